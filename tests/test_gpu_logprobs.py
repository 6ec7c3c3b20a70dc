"""token_logprobs on the GPU against its plain 64-bit form."""
import importlib

import numpy as np
import pytest
import torch

import gpu_helpers as H
import operator_refs as R

pytestmark = pytest.mark.gpu

NS = importlib.import_module(H.PKG)
cabi = H.cabi


def _dev():
    assert torch.cuda.is_available(), "GPU test run without a CUDA device"
    return torch.device("cuda:0")


def _check(r, rows, tokens, n):
    lp, rk, ids, tl, err = R.logprob_rows(rows, tokens, n)
    got = r.logprobs.double().cpu().numpy()
    assert np.array_equal(r.ranks.cpu().numpy(), rk)
    assert np.array_equal(r.top_ids.cpu().numpy(), ids)
    assert np.array_equal(np.isnan(got), np.isnan(lp))
    for g, w, e in ((got[:, None], lp[:, None], err[:, :1]), (r.top_logprobs.double().cpu().numpy(), tl, err[:, 1:])):
        fin = np.isfinite(w)
        assert np.array_equal(g[~fin & ~np.isnan(w)], w[~fin & ~np.isnan(w)])
        bad = np.abs(g[fin] - w[fin]) > e[fin]
        assert not bad.any(), (g[fin][bad][:4], w[fin][bad][:4], e[fin][bad][:4])


def _rows(rng, S, V, dtype, kind="peaked"):
    if kind == "flat":
        x = rng.normal(0, 0.01, (S, V))
    elif kind == "ties":
        x = rng.integers(-3, 4, (S, V)).astype(np.float64)
    elif kind == "rising":
        x = np.broadcast_to(np.linspace(-20, 20, V), (S, V)).copy()
    elif kind == "falling":
        x = np.broadcast_to(np.linspace(20, -20, V), (S, V)).copy()
    elif kind == "constant":
        x = np.full((S, V), -1.5)
    elif kind == "wide":
        x = rng.normal(0, 1000, (S, V))
    else:
        x = rng.normal(0, 2, (S, V))
        for r in range(S):
            x[r, rng.integers(0, V, 20)] += 8
    return torch.from_numpy(x.astype(np.float32)).to(_dev()).to(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("S,V,n", [(1, 1, 1), (2, 2, 2), (3, 7, 0), (3, 31, 31), (2, 33, 32), (4, 1000, 5), (3, 4099, 20),
                                   (5, 32003, 1), (2, 50257, 32), (3, 128256, 20), (40, 8192, 7), (300, 2049, 3)])
def test_matches_the_plain_form(S, V, n, dtype):
    rng = np.random.default_rng(S + V + n)
    x = _rows(rng, S, V, dtype)
    t = rng.integers(0, V, S)
    t[0] = int(x[0].float().argmax())
    tok = torch.from_numpy(t).to(_dev())
    st = torch.zeros(1, dtype=torch.int32, device=_dev())
    r = NS.token_logprobs(x, tok, n, status=st)
    assert r.top_ids.dtype == torch.int64 and st.item() == 0
    _check(r, x.double().cpu().numpy(), t, n)
    r32 = NS.token_logprobs(x, tok.to(torch.int32), n)
    assert r32.top_ids.dtype == torch.int32
    assert torch.equal(r32.top_ids.long(), r.top_ids) and torch.equal(r32.logprobs, r.logprobs)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind", ["flat", "ties", "rising", "falling", "constant", "wide"])
@pytest.mark.parametrize("S,V", [(2, 20000), (160, 5001)])
def test_distributions(kind, S, V, dtype):
    """Ties (the lowest ids win), rows that rise or fall, flat and very wide rows."""
    rng = np.random.default_rng(5)
    x = _rows(rng, S, V, dtype, kind)
    t = rng.integers(0, V, S)
    for n in (1, 20, 32):
        _check(NS.token_logprobs(x, torch.from_numpy(t).to(_dev()), n), x.double().cpu().numpy(), t, n)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_masked_and_degenerate_rows(dtype):
    """Rows of -inf but for a few ids (fewer than n too), and the rows that the sampler's guard makes uniform."""
    rng = np.random.default_rng(6)
    S, V, n = 9, 6000, 8
    x = _rows(rng, S, V, torch.float32)
    x[0, 5:] = -np.inf                       # fewer than n allowed
    x[1, torch.from_numpy(rng.random(V) < 0.99).to(_dev())] = -np.inf
    x[2] = -np.inf                           # nothing allowed
    x[3, 4000] = np.nan
    x[4, 17] = np.inf
    x[5] = -np.inf
    x[5, V - 1] = 3.0                        # one token
    x[6, :] = torch.finfo(torch.bfloat16).min
    x[7, 0], x[7, 1], x[7, 2:] = 0.0, -0.0, -5.0  # equal
    x[8, : V // 2] = -np.inf
    x = x.to(dtype)
    for t in ([0] * S, [V - 1] * S, [1, 2, 3, 4000, 17, V - 1, 8, 1, 0]):
        _check(NS.token_logprobs(x, torch.tensor(t, device=_dev()), n), x.double().cpu().numpy(), t, n)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [1, 2, 5, 31, 33, 63, 64, 65, 100, 700, 20000])
def test_more_top_tokens_than_are_allowed(V, dtype):
    """Rows of few allowed tokens, anywhere in the row: the masked ones follow by id."""
    rng = np.random.default_rng(V)
    S, n = 24, min(V, 32)
    x = rng.normal(0, 3, (S, V)).astype(np.float32)
    for i in range(S):
        keep = rng.choice(V, min(V, int(rng.integers(0, 40))), replace=False) if i else np.arange(min(V, 31))
        mask = np.ones(V, dtype=bool)
        mask[keep] = False
        x[i, mask] = -np.inf
    x = torch.from_numpy(x).to(_dev()).to(dtype)
    t = rng.integers(0, V, S)
    _check(NS.token_logprobs(x, torch.from_numpy(t).to(_dev()), n), x.double().cpu().numpy(), t, n)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("S,V", [(700, 9001), (600, 1474), (1300, 203), (594, 40013)])
def test_many_short_rows(S, V, dtype):
    """More rows than the GPU takes at once, each of another kind, with masks that leave all, some or a few."""
    rng = np.random.default_rng(S)
    kinds = ["peaked", "flat", "ties", "rising", "falling", "constant", "wide"]
    x = _rows(rng, S, V, torch.float32)
    for i, kind in enumerate(kinds):
        x[i::len(kinds)] = _rows(rng, len(range(i, S, len(kinds))), V, torch.float32, kind)
    for i in range(0, S, 3):
        x[i, torch.from_numpy(rng.random(V) < rng.choice([0.5, 0.99, 1.0])).to(_dev())] = -np.inf
    x = x.to(dtype)
    t = rng.integers(0, V, S)
    for n in (0, 1, 12, 32):
        _check(NS.token_logprobs(x, torch.from_numpy(t).to(_dev()), n), x.double().cpu().numpy(), t, n)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("offset", [0, 1, 5])
def test_strided_rows_and_sample_indices(dtype, offset):
    rng = np.random.default_rng(offset)
    V, T, n = 5003, 12, 6
    buf = _rows(rng, T, V + 13, dtype)
    x = buf[:, offset:offset + V]
    idx = [11, 0, 3, 3, 9]
    t = rng.integers(0, V, 5)
    r = NS.token_logprobs(x, torch.from_numpy(t).to(_dev()), n, sample_indices=torch.tensor(idx, device=_dev()))
    _check(r, x.double().cpu().numpy()[idx], t, n)
    t = rng.integers(0, V, T)
    r = NS.token_logprobs(x.t().contiguous().t(), torch.from_numpy(t).to(_dev()), n)
    _check(r, x.double().cpu().numpy(), t, n)
    one = x[4:5].expand(T, V)
    r = NS.token_logprobs(one, torch.from_numpy(t).to(_dev()), n)
    _check(r, one.double().cpu().numpy(), t, n)


def test_bad_tokens_and_indices_are_reported():
    x = torch.randn(3, 50, device=_dev())
    st = torch.zeros(1, dtype=torch.int32, device=_dev())
    r = NS.token_logprobs(x, torch.tensor([1, 50, -1], device=_dev()), 2, status=st)
    assert st.item() == cabi.NS_STATUS_BAD_TOKEN_ID
    _check(r, x.double().cpu().numpy(), [1, 50, -1], 2)
    st.zero_()
    r = NS.token_logprobs(x, torch.tensor([4, 4], device=_dev()), 2, status=st,
                          sample_indices=torch.tensor([3, -2], device=_dev()))
    assert st.item() == cabi.NS_STATUS_BAD_SAMPLE_INDEX
    _check(r, x[[0, 0]].double().cpu().numpy(), [4, 4], 2)


def test_refusals_and_no_rows():
    x = torch.randn(3, 50, device=_dev())
    t = torch.zeros(3, dtype=torch.int64, device=_dev())
    with pytest.raises(ValueError, match="top_n"):
        NS.token_logprobs(x, t, 33)
    with pytest.raises(ValueError, match="top_n"):
        NS.token_logprobs(x[:, :4], t, 5)
    with pytest.raises(ValueError, match="top_n"):
        NS.token_logprobs(x, t, -1)
    with pytest.raises(RuntimeError, match="one element per row"):
        NS.token_logprobs(x, t[:2])
    with pytest.raises(RuntimeError, match="int64 or int32"):
        NS.token_logprobs(x, t.float())
    with pytest.raises(RuntimeError, match="float32 or bfloat16"):
        NS.token_logprobs(x.half(), t)
    with pytest.raises(RuntimeError, match="CUDA"):
        NS.token_logprobs(x, t.cpu())
    with pytest.raises(RuntimeError, match="no gradient"):
        NS.token_logprobs(x.clone().requires_grad_(), t)
    r = NS.token_logprobs(x[:0], t[:0], 4)
    assert r.logprobs.shape == (0,) and r.top_ids.shape == (0, 4)


def test_graph_replay_streams_and_repeats():
    """A captured call replays over new inputs, calls on several streams do not disturb one another, and the
    same inputs give the same bits."""
    rng = np.random.default_rng(8)
    S, V, n = 24, 32000, 20
    x = _rows(rng, S, V, torch.float32)
    tok = torch.from_numpy(rng.integers(0, V, S)).to(_dev())
    NS.token_logprobs(x, tok, n)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        r = NS.token_logprobs(x, tok, n)
    for seed in (1, 2):
        x.copy_(_rows(np.random.default_rng(seed), S, V, torch.float32))
        g.replay()
        torch.cuda.synchronize()
        _check(r, x.double().cpu().numpy(), tok.tolist(), n)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    many = []
    for s in streams:
        with torch.cuda.stream(s):
            many.append(NS.token_logprobs(x, tok, n))
    torch.cuda.synchronize()
    for m in many:
        assert all(torch.equal(a, b) for a, b in zip(m, r))


def test_rows_past_2_to_the_31_elements():
    V, T = 128256, 16800
    x = torch.zeros(T, V, dtype=torch.bfloat16, device=_dev())
    x[T - 1] = torch.randn(V, device=_dev()).to(torch.bfloat16)
    t = torch.full((T,), V - 1, device=_dev())
    r = NS.token_logprobs(x, t, 3)
    last = type(r)(*[v[T - 1:] for v in r])
    _check(last, x[T - 1:].double().cpu().numpy(), [V - 1], 3)
    assert (r.ranks[: T - 1] == 1).all() and (r.top_ids[: T - 1] == torch.arange(3, device=_dev())).all()
