"""What the operators write is seen by autograd, as what torch's in-place operations write."""
import importlib

import pytest
import torch

import gpu_helpers as H

pytestmark = pytest.mark.gpu

NS = importlib.import_module(H.PKG)


def _dev():
    assert torch.cuda.is_available(), "GPU test run without a CUDA device"
    return torch.device("cuda:0")


def _writes():
    """(name, the tensors that a call writes, the call)"""
    x, out = torch.randn(3, 50, device=_dev()), torch.zeros(3, 50, device=_dev())
    status = [torch.zeros(1, dtype=torch.int32, device=_dev()) for _ in range(4)]
    pools = [torch.randn(6, 4, device=_dev()), torch.randn(6, 2, 3, device=_dev())]
    pool, ids = torch.zeros(6, 4, dtype=torch.int32, device=_dev()), torch.zeros(4, dtype=torch.int32, device=_dev())
    table, off = torch.zeros(1, dtype=torch.int32, device=_dev()), torch.tensor([0, 1], device=_dev())
    here = x.clone()
    tokens = torch.zeros(3, dtype=torch.int64, device=_dev())
    return [
        ("out", [out, status[0]], lambda: NS.process_logits(x, out=out, status=status[0])),
        ("in place", [here], lambda: NS.process_logits(here, out=here)),
        ("status alone", [status[1]], lambda: NS.process_logits(x, status=status[1])),
        ("log-probabilities", [status[2]], lambda: NS.token_logprobs(x, tokens, 1, status=status[2])),
        ("copies", pools, lambda: NS.copy_pages(pools, [0, 1], [2, 3])),
        ("gather", [ids, status[3]], lambda: NS.gather_paged_history(pool, table, off, off * 4, out=ids, status=status[3])),
    ]


def test_what_is_written_has_a_new_version():
    for name, written, call in _writes():
        before = [t._version for t in written]
        call()
        assert all(t._version > b for t, b in zip(written, before)), name
    x = torch.randn(3, 50, device=_dev())
    r = NS.process_logits(x)
    assert x._version == 0 and r._version == 0


def test_a_saved_tensor_that_was_overwritten_is_noticed():
    w = torch.randn(3, 50, device=_dev(), requires_grad=True)
    for kind in ("process", "copy"):
        t = torch.randn(3, 50, device=_dev())
        loss = (w * t).sum()
        if kind == "process":
            NS.process_logits(torch.randn(3, 50, device=_dev()), out=t)
        else:
            NS.copy_pages(t, [0], [1])
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()


def test_a_result_that_wants_a_gradient_is_refused():
    x = torch.randn(3, 50, device=_dev())
    leaf = torch.randn(3, 50, device=_dev(), requires_grad=True)
    was = leaf.detach().clone()
    for out in (leaf, leaf * 1):
        with pytest.raises(RuntimeError, match="no gradient"):
            NS.process_logits(x, out=out)
    assert torch.equal(leaf, was)
    with torch.no_grad():
        assert NS.process_logits(x, out=leaf) is leaf and torch.equal(leaf, x)


def test_tensors_made_in_inference_mode():
    """They have no version; calls in and out of the mode write them as before."""
    with torch.inference_mode():
        x, pool = torch.randn(2, 40, device=_dev()), torch.zeros(4, 8, device=_dev())
        pool[0] = 3.0
        NS.process_logits(x, out=x)
        NS.copy_pages(pool, [0], [1])
    with torch.no_grad():
        y = torch.empty_like(x)
        NS.process_logits(x, out=y)
        NS.process_logits(y, out=x)
        NS.copy_pages(pool, [0], [2])
    assert torch.equal(y, x) and pool[:, 0].tolist() == [3.0, 3.0, 3.0, 0.0]
    assert NS.token_logprobs(x, torch.zeros(2, dtype=torch.int64, device=_dev())).ranks.shape == (2,)
