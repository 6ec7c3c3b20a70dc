"""process_logits on the GPU against its plain 64-bit form."""
import importlib

import numpy as np
import pytest
import torch

import gpu_helpers as H
import operator_refs as R

pytestmark = pytest.mark.gpu

NS = importlib.import_module(H.PKG)
cabi = H.cabi
HALF_STEP = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8}


def _dev():
    assert torch.cuda.is_available(), "GPU test run without a CUDA device"
    return torch.device("cuda:0")


def _csr(lists, dtype=np.int32):
    off = np.zeros(len(lists) + 1, dtype=np.int64)
    off[1:] = np.cumsum([len(x) for x in lists])
    flat = np.array([v for x in lists for v in x], dtype=dtype)
    return torch.from_numpy(off).to(_dev()), torch.from_numpy(flat).to(_dev())


def _f32(a):
    return torch.from_numpy(np.asarray(a, dtype=np.float32)).to(_dev())


def _step(rng, S, V, hist=64, bias=8, mask=True):
    """Host inputs of one step: every row with penalties, biases and a mask (some rows without)."""
    common = rng.integers(0, V, size=max(1, min(V, 40)))  # repeated ids
    hists = []
    for i in range(S):
        n = int(rng.integers(0, hist + 1))
        h = np.where(rng.random(n) < 0.5, rng.choice(common, n), rng.integers(0, V, n))
        hists.append(h.tolist())
    d = dict(
        hists=hists,
        prompts=[int(rng.integers(0, len(h) + 2)) for h in hists],
        rep=rng.choice([1.0, 1.1, 1.3, 0.8], S), pres=rng.choice([0.0, 0.7, -0.4], S), freq=rng.choice([0.0, 0.3, 1.9], S),
        biases=[[(int(v), float(b)) for v, b in zip(rng.choice(V, min(bias, V), replace=False), rng.normal(0, 3, min(bias, V)))]
                for _ in range(S)],
        masks=[None if i % 3 == 2 else rng.random(V) < (0.1 if i % 3 else 0.9) for i in range(S)] if mask else None,
    )
    return d


def _device(d, V, words=None):
    """The keyword arguments of process_logits for a step."""
    ho, hi = _csr(d["hists"])
    kw = dict(history_offsets=ho, history_ids=hi, prompt_lens=torch.tensor(d["prompts"], dtype=torch.int32, device=_dev()),
              repetition_penalty=_f32(d["rep"]), presence_penalty=_f32(d["pres"]), frequency_penalty=_f32(d["freq"]))
    bo, bi = _csr([[v for v, _ in b] for b in d["biases"]])
    kw.update(bias_offsets=bo, bias_ids=bi, bias_values=_f32([x for b in d["biases"] for _, x in b]))
    if d["masks"] is not None:
        there = [m for m in d["masks"] if m is not None] or [np.ones(V, dtype=bool)]
        rows, k = [], 0
        for m in d["masks"]:
            rows.append(-1 if m is None else k)
            k += m is not None
        kw.update(allowed=torch.from_numpy(R.pack_masks(there, words)).to(_dev()),
                  allowed_rows=torch.tensor(rows, dtype=torch.int32, device=_dev()))
    return kw


def _check(got, rows, d, dtype):
    want, err = R.process_rows(rows, d["hists"], d["prompts"], d["rep"], d["pres"], d["freq"], d["biases"], d["masks"])
    R.assert_processed(got.double().cpu().numpy(), want, err, HALF_STEP[dtype])


TYPES = [(torch.float32, torch.float32), (torch.bfloat16, torch.float32), (torch.bfloat16, torch.bfloat16)]


@pytest.mark.parametrize("types", TYPES, ids=["f32", "bf16-f32", "bf16"])
@pytest.mark.parametrize("S,V", [(1, 1), (2, 2), (3, 31), (1, 33), (5, 50), (4, 1000), (3, 8191), (2, 8192), (3, 8193),
                                 (7, 32003), (3, 50257), (2, 128256)])
def test_matches_the_plain_form(S, V, types):
    rng = np.random.default_rng(S * 1000 + V)
    d = _step(rng, S, V)
    x = torch.from_numpy(rng.normal(0, 3, (S, V)).astype(np.float32)).to(_dev()).to(types[0])
    before = x.clone()
    status = torch.zeros(1, dtype=torch.int32, device=_dev())
    got = NS.process_logits(x, out_dtype=types[1], status=status, **_device(d, V))
    assert got.dtype == types[1]
    _check(got, x.double().cpu().numpy(), d, types[1])
    assert torch.equal(x, before)
    assert status.item() == 0


@pytest.mark.parametrize("mask", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("S,V", [(1, 5), (6, 1001), (3, 16384), (2, 128256)])
def test_in_place_equals_out_of_place(S, V, dtype, mask):
    rng = np.random.default_rng(V)
    d = _step(rng, S, V, mask=mask)
    x = torch.from_numpy(rng.normal(0, 3, (S, V)).astype(np.float32)).to(_dev()).to(dtype)
    kw = _device(d, V)
    want = NS.process_logits(x, **kw)
    rows = x.double().cpu().numpy()
    got = NS.process_logits(x, out=x, **kw)
    assert got is x and torch.equal(got, want)
    _check(got, rows, d, dtype)


def test_each_part_alone():
    """What is not given is not applied; a call with nothing is a copy."""
    rng = np.random.default_rng(3)
    S, V = 4, 9000
    x = torch.from_numpy(rng.normal(0, 3, (S, V)).astype(np.float32)).to(_dev())
    rows = x.double().cpu().numpy()
    assert torch.equal(NS.process_logits(x), x)
    d = _step(rng, S, V)
    kw = _device(d, V)
    none = dict(d, prompts=None, rep=None, pres=None, freq=None, biases=None, masks=None)
    hist = {k: kw[k] for k in ("history_offsets", "history_ids")}
    for name, key in (("repetition_penalty", "rep"), ("presence_penalty", "pres"), ("frequency_penalty", "freq")):
        want, err = R.process_rows(rows, d["hists"], **{key: d[key]})
        R.assert_processed(NS.process_logits(x, **hist, **{name: kw[name]}).double().cpu().numpy(), want, err, 2.0**-24)
    _check(NS.process_logits(x, **{k: kw[k] for k in ("bias_offsets", "bias_ids", "bias_values")}), rows,
           dict(none, biases=d["biases"]), torch.float32)
    _check(NS.process_logits(x, allowed=kw["allowed"], allowed_rows=kw["allowed_rows"]), rows, dict(none, masks=d["masks"]),
           torch.float32)
    # without allowed_rows row i has mask i
    masks = [rng.random(V) < 0.5 for _ in range(S)]
    _check(NS.process_logits(x, allowed=torch.from_numpy(R.pack_masks(masks)).to(_dev())), rows, dict(none, masks=masks),
           torch.float32)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("offset", [0, 1, 3])
def test_strided_and_unaligned_rows(dtype, offset):
    """Rows inside wider buffers, at any element offset, read through sample_indices (one of them twice)."""
    rng = np.random.default_rng(offset)
    S, V, T = 5, 8200, 9
    d = _step(rng, S, V)
    buf = torch.from_numpy(rng.normal(0, 3, (T, V + 17)).astype(np.float32)).to(_dev()).to(dtype)
    x = buf[:, offset:offset + V]
    idx = np.array([8, 0, 3, 3, 7])
    out_buf = torch.full((S, V + 9), 7.0, dtype=dtype, device=_dev())
    out = out_buf[:, offset + 1:offset + 1 + V]
    kw = _device(d, V, words=(V + 31) // 32 + 2)
    NS.process_logits(x, sample_indices=torch.from_numpy(idx).to(_dev()), out=out, **kw)
    _check(out, x.double().cpu().numpy()[idx], d, dtype)
    assert (out_buf[:, :offset + 1] == 7).all() and (out_buf[:, offset + 1 + V:] == 7).all()
    # in place on such rows
    mine = out_buf[:, 2:2 + V]
    rows = mine.double().cpu().numpy()
    left, right = out_buf[:, :2].clone(), out_buf[:, 2 + V:].clone()
    NS.process_logits(mine, out=mine, **kw)
    _check(mine, rows, d, dtype)
    assert torch.equal(out_buf[:, :2], left) and torch.equal(out_buf[:, 2 + V:], right)
    # one row read by all (stride 0), and columns that are not contiguous
    one = buf[2:3, offset:offset + V].expand(S, V)
    _check(NS.process_logits(one, **kw), one.double().cpu().numpy(), d, dtype)
    _check(NS.process_logits(x[:S].t().contiguous().t(), **kw), x[:S].double().cpu().numpy(), d, dtype)


@pytest.mark.parametrize("mask", [False, True])
@pytest.mark.parametrize("types", TYPES + [(torch.float32, None), (torch.bfloat16, None)],
                         ids=["f32", "bf16-f32", "bf16", "f32-in-place", "bf16-in-place"])
def test_long_repetitive_histories(types, mask):
    """Counts of many thousands, neighbouring ids of which one has many, histories longer than the vocabulary, and
    more different ids than a block lists."""
    rng = np.random.default_rng(9)
    S, V = 4, 40000
    hists = [[17] * 30000 + [39999] * 5 + [16, 18], rng.integers(0, V, 131072).tolist(), (np.arange(60000) * 32 % V).tolist(),
             [20000] * 6990 + [20001] * 7100 + rng.integers(0, 9000, 5000).tolist()]
    d = dict(hists=hists, prompts=[10, 70000, 0, 4], rep=[1.2, 1.1, 1.0, 1.3], pres=[0.1, 0.2, 0.3, 0.4],
             freq=[0.01, 0.5, 0.25, 0.125], biases=[[(16, 2.0)], [(5, 1.0)], [], [(20001, -1.0), (20001, 4.0), (30000, 1.0)]],
             masks=[rng.random(V) < 0.5 for _ in range(S)] if mask else None)
    x = torch.from_numpy(rng.normal(0, 3, (S, V)).astype(np.float32)).to(_dev()).to(types[0])
    rows = x.double().cpu().numpy()
    got = NS.process_logits(x, out=x if types[1] is None else None, out_dtype=types[1], **_device(d, V))
    _check(got, rows, d, types[1] or types[0])


@pytest.mark.parametrize("mask", [False, True])
@pytest.mark.parametrize("types", TYPES + [(torch.float32, None), (torch.bfloat16, None)],
                         ids=["f32", "bf16-f32", "bf16", "f32-in-place", "bf16-in-place"])
@pytest.mark.parametrize("S,V", [(600, 77), (500, 4003), (450, 4100), (450, 8191), (200, 9001)])
def test_many_short_rows(S, V, types, mask):
    """More rows than are worked on at once, picked in another order, with a few long histories among them."""
    rng = np.random.default_rng(S + V)
    d = _step(rng, S, V, hist=30, bias=3, mask=mask)
    d["hists"][7] = [3] * 9000 + [4] * 7100 + rng.integers(0, V, 900).tolist()
    d["hists"][S - 1] = rng.integers(0, V, 6000).tolist()
    d["biases"][9] = [(int(v), 0.5) for v in rng.integers(0, V, 700)]
    x = torch.from_numpy(rng.normal(0, 3, (S + 1, V)).astype(np.float32)).to(_dev()).to(types[0])
    kw = _device(d, V)
    if types[1] is None:
        x = x[1:]
        rows = x.double().cpu().numpy()
        got = NS.process_logits(x, out=x, **kw)
    else:
        idx = np.arange(S)[::-1] + 1
        rows = x.double().cpu().numpy()[idx]
        got = NS.process_logits(x, sample_indices=torch.from_numpy(idx.copy()).to(_dev()), out_dtype=types[1], **kw)
    _check(got, rows, d, types[1] or types[0])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_in_place_with_a_few_long_rows_among_many(dtype):
    """Rows whose ids fit the block's table, and rows that other blocks share, in one call of over 1024 rows."""
    rng = np.random.default_rng(10)
    S, V = 1100, 33000
    long = {3: 5000, 600: 9001, 601: 4097, 1099: 20000}
    hists = [rng.integers(0, V, long.get(i, int(rng.integers(0, 5)))).tolist() for i in range(S)]
    hists[5] = rng.integers(0, V, 4096).tolist()
    hists[6] = (np.arange(4000) * 4096 % V).tolist() + [7] * 90
    d = dict(hists=hists, prompts=[int(rng.integers(0, len(h) + 1)) for h in hists], rep=[1.25] * S, pres=[0.5] * S,
             freq=[0.25] * S, biases=[[(int(v), 1.5) for v in rng.choice(V, 3, replace=False)] for _ in range(S)], masks=None)
    d["biases"][600] = [(int(v), -2.0) for v in rng.choice(V, 6000, replace=False)] + [(hists[600][0], 3.0)]
    x = torch.from_numpy(rng.normal(0, 3, (S, V)).astype(np.float32)).to(_dev()).to(dtype)
    kw = _device(d, V)
    want = NS.process_logits(x, **kw)
    pick = [0, 3, 5, 6, 600, 601, 1098, 1099]
    rows = x[pick].double().cpu().numpy()
    NS.process_logits(x, out=x, **kw)
    assert torch.equal(x, want)
    sub = {k: None if v is None else [v[i] for i in pick] for k, v in d.items()}
    _check(x[pick], rows, sub, dtype)


def test_a_bias_given_twice_counts_once_the_last():
    rng = np.random.default_rng(11)
    S, V = 3, 20000
    biases = [[(5, 1.0), (9000, 2.0), (5, 3.0), (19999, -1.0), (5, -7.5)],
              [(int(v), float(i)) for i, v in enumerate(rng.integers(0, 50, 4000))],
              [(7, 1.0)] * 3000 + [(7, 2.5)]]
    d = dict(hists=[[5, 5], [3], []], prompts=[0, 0, 0], rep=[1.5, 1.5, 1.0], pres=[1.0, 1.0, 0.0], freq=[0.5, 0.5, 0.0],
             biases=biases, masks=None)
    x = torch.from_numpy(rng.normal(0, 3, (S, V)).astype(np.float32)).to(_dev())
    kw = _device(d, V)
    first = NS.process_logits(x, **kw)
    _check(first, x.double().cpu().numpy(), d, torch.float32)
    for _ in range(5):
        assert torch.equal(NS.process_logits(x, **kw), first)


def test_special_values():
    """-inf, +inf and NaN logits, masked and not; infinite biases; rows whose mask allows nothing."""
    V = 300
    x = torch.zeros(4, V, device=_dev())
    x[:, 0], x[:, 1], x[:, 2], x[:, 3] = -np.inf, np.inf, np.nan, torch.finfo(torch.float32).min
    x[:, 4], x[:, 5] = -0.0, 1e-45
    x[:, 6] = torch.finfo(torch.float32).max
    masks = [None, np.arange(V) >= 8, np.zeros(V, dtype=bool), np.ones(V, dtype=bool)]
    d = dict(hists=[list(range(8))] * 4, prompts=[0] * 4, rep=[1.5] * 4, pres=[0.5] * 4, freq=[0.25] * 4,
             biases=[[(0, 1.0), (1, -np.inf), (20, -np.inf), (21, np.inf), (2, 1.0)]] * 4, masks=masks)
    want, err = R.process_rows(x.double().cpu().numpy(), d["hists"], d["prompts"], d["rep"], d["pres"], d["freq"],
                               d["biases"], masks)
    with np.errstate(all="ignore"):
        want = np.where(np.abs(want) > 3.4028235677973366e38, np.sign(want) * np.inf, want)  # fp32 overflows
    for inp in (x, x.clone()):
        got = NS.process_logits(inp, out=None if inp is x else inp, **_device(d, V))
        R.assert_processed(got.double().cpu().numpy(), want, err, 2.0**-24)
    assert (got[2] == -np.inf).all()


def test_empty_histories_and_no_rows():
    x = torch.randn(3, 100, device=_dev())
    z = torch.zeros(4, dtype=torch.int64, device=_dev())
    none = torch.empty(0, dtype=torch.int32, device=_dev())
    assert torch.equal(NS.process_logits(x, history_offsets=z, history_ids=none, repetition_penalty=_f32([2, 2, 2]),
                                         bias_offsets=z, bias_ids=none, bias_values=_f32([])), x)
    assert NS.process_logits(x[:0]).shape == (0, 100)
    assert NS.process_logits(x, sample_indices=torch.empty(0, dtype=torch.int64, device=_dev())).shape == (0, 100)


def test_bad_device_data_is_reported_and_not_followed():
    S, V = 4, 100
    x = torch.randn(S, V, device=_dev())
    st = torch.zeros(1, dtype=torch.int32, device=_dev())
    rp = _f32([2.0] * S)
    off = torch.tensor([0, 2, 4, 4, 4], device=_dev())

    def run(**kw):
        st.zero_()
        r = NS.process_logits(x, status=st, **kw)
        return r, st.item()

    ids = torch.tensor([3, 100, -1, 7], dtype=torch.int32, device=_dev())
    got, s = run(history_offsets=off, history_ids=ids, repetition_penalty=rp)
    assert s == cabi.NS_STATUS_BAD_HISTORY_ID
    want, err = R.process_rows(x.double().cpu().numpy(), [[3], [7], [], []], rep=[2.0] * S)
    R.assert_processed(got.double().cpu().numpy(), want, err, 2.0**-24)
    got, s = run(bias_offsets=off, bias_ids=ids, bias_values=_f32([1, 2, 3, 4]))
    assert s == cabi.NS_STATUS_BAD_TOKEN_ID
    assert got[0, 3].item() == pytest.approx(x[0, 3].item() + 1) and torch.equal(got[2:], x[2:])
    for bad in ([0, 5, 4, 4, 4], [-1, 2, 4, 4, 4], [0, 2, 1, 4, 4]):
        got, s = run(history_offsets=torch.tensor(bad, device=_dev()), history_ids=ids.clamp(0, 50), repetition_penalty=rp)
        assert s & cabi.NS_STATUS_BAD_ROW_RANGE
    got, s = run(allowed=torch.zeros(2, 4, dtype=torch.int32, device=_dev()),
                 allowed_rows=torch.tensor([0, 1, 2, -5], dtype=torch.int32, device=_dev()))
    assert s == cabi.NS_STATUS_BAD_MASK_ROW
    assert (got[:2] == -np.inf).all() and torch.equal(got[2:], x[2:])
    got, s = run(sample_indices=torch.tensor([1, 4, -1], device=_dev()))
    assert s == cabi.NS_STATUS_BAD_SAMPLE_INDEX and torch.equal(got, x[[1, 0, 0]])


def test_refusals():
    x = torch.randn(4, 64, device=_dev())
    i32 = dict(dtype=torch.int32, device=_dev())
    with pytest.raises(RuntimeError, match="overlap"):
        NS.process_logits(x[:3], out=x[1:])
    with pytest.raises(RuntimeError, match="overlap"):
        NS.process_logits(x, sample_indices=torch.arange(4, device=_dev()), out=x)
    with pytest.raises(RuntimeError, match="overlap"):
        b = x.to(torch.bfloat16)
        NS.process_logits(b[:2], out=b.view(-1).view(torch.float32)[:128].view(2, 64))
    with pytest.raises(RuntimeError, match="columns"):
        NS.process_logits(x, out=torch.empty(4, 63, device=_dev()))
    with pytest.raises(RuntimeError, match="one row per row"):
        NS.process_logits(x, out=torch.empty(3, 64, device=_dev()))
    with pytest.raises(RuntimeError, match="float32 or bfloat16"):
        NS.process_logits(x.half())
    with pytest.raises(RuntimeError, match="go together"):
        NS.process_logits(x, history_offsets=torch.zeros(5, dtype=torch.int64, device=_dev()))
    with pytest.raises(RuntimeError, match="repetition_penalty must have 4"):
        NS.process_logits(x, repetition_penalty=_f32([1.0]))
    with pytest.raises(RuntimeError, match="dtype"):
        NS.process_logits(x, presence_penalty=torch.zeros(4, dtype=torch.float64, device=_dev()))
    with pytest.raises(RuntimeError, match="words"):
        NS.process_logits(x, allowed=torch.zeros(4, 1, **i32))
    with pytest.raises(RuntimeError, match="one row per row"):
        NS.process_logits(x, allowed=torch.zeros(3, 2, **i32))
    with pytest.raises(RuntimeError, match="without allowed"):
        NS.process_logits(x, allowed_rows=torch.zeros(4, **i32))
    with pytest.raises(RuntimeError, match="must be on|CUDA"):
        NS.process_logits(x, prompt_lens=torch.zeros(4, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="no gradient"):
        NS.process_logits(x.clone().requires_grad_())
    with pytest.raises(ValueError, match="out_dtype"):
        NS.process_logits(x, out_dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="rows must be contiguous"):
        y = torch.randn(64, 4, device=_dev()).t()
        NS.process_logits(y, out=y)
    with pytest.raises(RuntimeError, match="stride"):
        NS.process_logits(x, out=torch.empty(64, device=_dev()).expand(4, 64))


def test_graph_replay_and_streams():
    """A captured call replays over new inputs; a call on another stream runs there."""
    rng = np.random.default_rng(4)
    S, V = 8, 32000
    d = _step(rng, S, V)
    kw = _device(d, V)
    x = torch.randn(S, V, device=_dev())
    out = torch.empty_like(x)
    NS.process_logits(x, out=out, **kw)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        NS.process_logits(x, out=out, **kw)
    for seed in (1, 2):
        x.copy_(torch.randn(S, V, generator=torch.Generator(device="cuda").manual_seed(seed), device=_dev()))
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        _check(out, x.double().cpu().numpy(), d, torch.float32)
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    torch.cuda.synchronize()
    for s in streams:
        with torch.cuda.stream(s):
            outs.append(NS.process_logits(x, **kw))
    torch.cuda.synchronize()
    for o in outs:
        assert torch.equal(o, out)


def test_rows_past_2_to_the_31_elements():
    V, T = 128256, 16800  # T * V > 2^31
    x = torch.zeros(T, V, dtype=torch.bfloat16, device=_dev())
    x[T - 1] = torch.randn(V, device=_dev()).to(torch.bfloat16)
    rows = x[T - 1:].double().cpu().numpy()
    d = _step(np.random.default_rng(2), 1, V)
    idx = torch.tensor([T - 1], device=_dev())
    _check(NS.process_logits(x, sample_indices=idx, **_device(d, V)), rows, d, torch.bfloat16)
    # and the output's last row, in place
    off = torch.zeros(T + 1, dtype=torch.int64, device=_dev())
    off[T:] = 2
    ids = torch.tensor([1, V - 1], dtype=torch.int32, device=_dev())
    NS.process_logits(x, bias_offsets=off, bias_ids=ids, bias_values=_f32([4.0, -4.0]), out=x)
    want = rows[0].copy()
    want[1] += 4
    want[V - 1] -= 4
    R.assert_processed(x[T - 1:].double().cpu().numpy(), want[None], np.full((1, V), 1e-6), 2.0**-8)
    assert not x[: T - 1].any()
