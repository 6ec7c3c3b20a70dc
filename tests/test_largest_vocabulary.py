"""Vocabularies up to the largest that 32-bit ids can number: 2^31 - 1."""
import importlib

import numpy as np
import pytest

from conftest import PKG_NAME, pkg

cabi = pkg("_cabi")
LARGEST = 2**31 - 1


def _process(**kw):
    a = cabi.NsProcessArgs()
    base = dict(logits=4096, logits_dtype=0, vocab_size=LARGEST, num_logit_rows=1, logits_row_stride=LARGEST, num_rows=1,
                out_dtype=0, out=1 << 40, out_row_stride=LARGEST)
    for k, v in {**base, **kw}.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("vocab", [LARGEST, LARGEST - 12031, 2**30])
def test_sizes_are_checked_without_overflow(vocab):
    rows = 2**31 // (vocab // 12032)
    with pytest.raises(cabi.NsError, match="too large"):
        cabi.ns_process_logits(_process(vocab_size=vocab, logits_row_stride=vocab, out_row_stride=vocab, num_rows=rows,
                                        num_logit_rows=rows, out=1 << 58))


@pytest.mark.parametrize("stride", [1, 2**26 - 1])
def test_masks_that_are_too_short_are_refused(stride):
    with pytest.raises(cabi.NsError, match="mask_stride"):
        cabi.ns_process_logits(_process(allowed=64, mask_stride=stride, num_masks=1))


@pytest.mark.gpu
@pytest.mark.parametrize("inplace", [False, True])
@pytest.mark.parametrize("ids", [40, 6000])
def test_largest_vocabulary(inplace, ids):
    """One bf16 row of 2^31 - 1 ids (4.3 GB): the named ids change, all others are left."""
    import torch

    NS = importlib.import_module(PKG_NAME)
    dev = torch.device("cuda:0")
    rng = np.random.default_rng(ids)
    hist = np.concatenate([rng.integers(0, LARGEST, ids), LARGEST - 1 - rng.integers(0, 20000, ids), [0, LARGEST - 1, 5]])
    x = torch.full((1, LARGEST), 2.0, dtype=torch.bfloat16, device=dev)
    off = torch.tensor([0, hist.size], device=dev)
    bias_ids = np.unique(hist[:20])
    st = torch.zeros(1, dtype=torch.int32, device=dev)
    got = NS.process_logits(
        x, history_offsets=off, history_ids=torch.from_numpy(hist.astype(np.int32)).to(dev),
        presence_penalty=torch.ones(1, device=dev), bias_offsets=torch.tensor([0, bias_ids.size], device=dev),
        bias_ids=torch.from_numpy(bias_ids.astype(np.int32)).to(dev),
        bias_values=torch.full((bias_ids.size,), 8.0, device=dev), out=x if inplace else None, status=st)
    assert st.item() == 0 and (inplace or (x == 2.0).all())
    named, biased = torch.from_numpy(np.unique(hist)).to(dev), torch.from_numpy(bias_ids).to(dev)
    assert (got[0, biased] == 9.0).all()
    got[0, biased] = 1.0
    assert (got[0, named] == 1.0).all()
    got[0, named] = 2.0
    for part in got[0].split(1 << 28):
        assert (part == 2.0).all()
