"""Page copies, paged history gathers and the paged history store on the GPU."""
import importlib

import numpy as np
import pytest
import torch

import gpu_helpers as H

pytestmark = pytest.mark.gpu

NS = importlib.import_module(H.PKG)
W = importlib.import_module(H.PKG + ".workloads")
SP = NS.SamplingParams
cabi = H.cabi


def _dev():
    assert torch.cuda.is_available(), "GPU test run without a CUDA device"
    return torch.device("cuda:0")


def _bits(shape, dtype, seed):
    """A tensor of random bytes."""
    size = torch.empty(0, dtype=dtype).element_size()
    g = torch.Generator(device="cuda").manual_seed(seed)
    b = torch.randint(0, 256, (int(np.prod(shape)) * size,), generator=g, dtype=torch.uint8, device=_dev())
    return b.view(dtype).view(shape)


def _same(a, b):
    return torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


def _copied(pools, src, dst):
    want = [p.clone() for p in pools]
    s, d = torch.as_tensor(src, device=_dev()), torch.as_tensor(dst, device=_dev())
    for w in want:
        w[d] = w[s]
    return want


@pytest.mark.parametrize("shape,dtype", [
    ((40, 16), torch.int32), ((40, 1), torch.uint8), ((40, 3), torch.uint8), ((33, 7, 5), torch.bfloat16),
    ((64, 16, 8, 128), torch.bfloat16), ((20, 5), torch.int64), ((30,), torch.float32), ((24, 1, 4099), torch.float32),
    ((17, 2, 16384), torch.float16), ((14, 100003), torch.uint8)])
@pytest.mark.parametrize("count", [1, 7])
def test_copies_pages_of_any_size(shape, dtype, count):
    pools = [_bits(shape, dtype, k) for k in range(3)]
    order = np.random.default_rng(count).permutation(shape[0])
    src, dst = order[:count], order[-count:]
    want = _copied(pools, src, dst)
    NS.copy_pages(pools, src, dst)
    for p, w in zip(pools, want):
        assert _same(p, w)


def test_copies_strided_unaligned_and_mixed_pools():
    """Halves of one buffer, pools at odd byte addresses, pools of different types in one call."""
    n = 50
    kv = _bits((n, 2, 16, 64), torch.bfloat16, 1)
    raw = _bits((n * 77 + 1,), torch.uint8, 2)
    odd = raw[1:].view(n, 77)
    wide = _bits((n, 100), torch.int32, 3)
    pools = [kv[:, 0], kv[:, 1], odd, wide[:, 3:50], _bits((n, 16), torch.int32, 4)]
    src, dst = [3, 3, 49, 0], [10, 11, 1, 48]
    before = [b.clone() for b in (kv, raw, wide)]
    want = _copied(pools, src, dst)
    NS.copy_pages(pools, src, dst)
    for p, w in zip(pools, want):
        assert _same(p, w)
    for now, was, cols in ((wide, before[2], [0, 1, 2] + list(range(50, 100))),):
        assert torch.equal(now[:, cols], was[:, cols])
    assert raw[0] == before[1][0]


@pytest.mark.parametrize("pools,pages,moves", [(130, 20, 9), (1, 20000, 9000), (3, 8000, 3501), (2, 7000, 3500)])
def test_many_pools_and_pages(pools, pages, moves):
    ps = [_bits((pages, 16), torch.int32, k) for k in range(pools)]
    order = np.random.default_rng(1).permutation(pages)
    src, dst = order[:moves], order[moves:2 * moves]
    want = _copied(ps, src, dst)
    NS.copy_pages(ps, torch.from_numpy(src), dst.tolist())
    for p, w in zip(ps, want):
        assert _same(p, w)


def test_pools_past_2_to_the_31_bytes():
    n = 70000
    p = torch.zeros(n, 32768, dtype=torch.uint8, device=_dev())  # 2.3 GB
    p[n - 1], p[5] = 7, 9
    NS.copy_pages(p, [n - 1, 5], [n - 2, 6])
    assert (p[n - 2] == 7).all() and (p[6] == 9).all() and not p[7].any() and not p[n - 3].any()


def test_listed_copies():
    """Page numbers in device memory: one launch, pages outside the pool skipped and reported."""
    p = _bits((9000, 16), torch.int32, 3)
    order = np.random.default_rng(2).permutation(9000)
    src, dst = order[:4400], order[4400:8800]
    want = _copied([p], src, dst)[0]
    bad = [(9000, int(order[8900])), (-1, int(order[8901])), (int(order[8902]), 9000), (int(order[8903]), -7)]
    s = torch.tensor([*src.tolist(), *[a for a, _ in bad]], dtype=torch.int32, device=_dev())
    d = torch.tensor([*dst.tolist(), *[b for _, b in bad]], dtype=torch.int32, device=_dev())
    st = torch.zeros(1, dtype=torch.int32, device=_dev())
    pool = [(p.data_ptr(), 64, 64)]
    stream = torch.cuda.current_stream().cuda_stream
    cabi.ns_pages_copy_listed(pool, 9000, s.data_ptr(), d.data_ptr(), 4400, st.data_ptr(), stream)
    assert st.item() == 0 and torch.equal(p, want)
    cabi.ns_pages_copy_listed(pool, 9000, s.data_ptr(), d.data_ptr(), 4404, st.data_ptr(), stream)
    assert st.item() == cabi.NS_STATUS_BAD_POOL_RANGE and torch.equal(p, want)


def test_long_lists_in_a_graph():
    """More pages than a launch takes, captured: the page numbers become part of the graph."""
    p = _bits((20000, 16), torch.int32, 3)
    order = torch.randperm(20000)
    src, dst = order[:8000].clone(), order[8000:16000].clone()
    NS.copy_pages(p, [0], [1])
    g = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(g, stream=side):
        NS.copy_pages(p, src, dst)
    p.copy_(_bits((20000, 16), torch.int32, 4))
    want = _copied([p], src, dst)[0]
    src.zero_(), dst.zero_()
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(p, want)


def test_copy_refusals_leave_the_pools():
    p = _bits((8, 16), torch.int32, 1)
    was = p.clone()
    for src, dst, match in (([0, 1], [2, 2], "twice"), ([0, 1], [1, 2], "both"), ([3], [3], "both"), ([8], [1], "outside"),
                            ([0], [-1], "outside"), ([0, 1], [2], "destination"), ([0.5], [1], "whole"),
                            ([True], [False], "whole")):
        with pytest.raises(ValueError, match=match):
            NS.copy_pages([p], src, dst)
    with pytest.raises(RuntimeError, match="host"):
        NS.copy_pages([p], torch.tensor([0], device=_dev()), [1])
    with pytest.raises(RuntimeError, match="same number of pages"):
        NS.copy_pages([p, p[:4].clone()], [0], [1])
    with pytest.raises(RuntimeError, match="contiguous"):
        NS.copy_pages([_bits((8, 4, 6), torch.int32, 2).transpose(1, 2)], [0], [1])
    with pytest.raises(RuntimeError, match="overlap"):
        NS.copy_pages([p[0].expand(8, 16)], [0], [1])
    with pytest.raises(RuntimeError, match="CUDA"):
        NS.copy_pages([p.cpu()], [0], [1])
    NS.copy_pages([p], [], [])
    NS.copy_pages([], [], [])
    NS.copy_pages([p[:, :0]], [0], [1])
    assert torch.equal(p, was)


def test_copy_graph_replay_and_streams():
    p = [_bits((64, 16, 8, 128), torch.bfloat16, k) for k in range(2)]
    src, dst = list(range(0, 20)), list(range(30, 50))
    NS.copy_pages(p, [60], [61])
    g = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(g, stream=side):
        NS.copy_pages(p, src, dst)
    for seed in (5, 6):
        for k, x in enumerate(p):
            x.copy_(_bits(tuple(x.shape), x.dtype, seed + 10 * k))
        want = _copied(p, src, dst)
        g.replay()
        torch.cuda.synchronize()
        assert all(_same(a, b) for a, b in zip(p, want))


@pytest.mark.parametrize("page", [1, 3, 16, 100, 256])
@pytest.mark.parametrize("rows,hi", [(1, 1), (7, 40), (300, 900), (3, 50000), (9000, 900)])
def test_gather_equals_indexing(page, rows, hi):
    rng = np.random.default_rng(page + rows)
    lens = rng.integers(0, hi + 1, rows)
    lens[0] = hi
    need = -(-lens // page)
    n = int(need.sum()) + 5
    pool = rng.integers(0, 1 << 30, (n, page)).astype(np.int32)
    table = rng.permutation(n)[: int(need.sum())].astype(np.int32)
    po, ho = np.concatenate([[0], np.cumsum(need)]), np.concatenate([[0], np.cumsum(lens)])
    want = np.concatenate([pool[table[po[r]:po[r + 1]]].reshape(-1)[: lens[r]] for r in range(rows)])
    d = lambda a: torch.from_numpy(a).to(_dev())  # noqa: E731
    out = torch.full((want.size + 9,), -7, dtype=torch.int32, device=_dev())
    st = torch.zeros(1, dtype=torch.int32, device=_dev())
    got = NS.gather_paged_history(d(pool), d(table), d(po), d(ho), out=out, status=st)
    assert got is out and st.item() == 0
    assert np.array_equal(out[: want.size].cpu().numpy(), want)
    assert (out[want.size:] == -7).all()


@pytest.mark.parametrize("rows,p_empty", [(300, 0.9), (70000, 0.999), (5000, 0.0)])
def test_gather_with_empty_and_one_id_rows(rows, p_empty):
    """Long runs of empty rows, rows of one id, and a long row among them."""
    rng = np.random.default_rng(rows)
    lens = np.where(rng.random(rows) < p_empty, 0, 1)
    lens[rows // 2] = 3000
    need = -(-lens // 4)
    table = rng.permutation(int(need.sum())).astype(np.int32)
    pool = rng.integers(0, 1 << 30, (table.size, 4)).astype(np.int32)
    po, ho = np.concatenate([[0], np.cumsum(need)]), np.concatenate([[0], np.cumsum(lens)])
    row = np.repeat(np.arange(rows), lens)
    j = np.arange(row.size) - ho[row]
    want = pool[table[po[row] + j // 4], j % 4]
    d = lambda a: torch.from_numpy(a).to(_dev())  # noqa: E731
    out = torch.full((want.size + 700,), -7, dtype=torch.int32, device=_dev())
    st = torch.zeros(1, dtype=torch.int32, device=_dev())
    NS.gather_paged_history(d(pool), d(table), d(po), d(ho), out=out, status=st)
    assert st.item() == 0 and np.array_equal(out[: want.size].cpu().numpy(), want) and (out[want.size:] == -7).all()


@pytest.mark.parametrize("page", [1, 5, 16])
@pytest.mark.parametrize("rows,hi", [(1, 1), (33, 3), (513, 7), (20000, 7), (20000, 1), (6000, 15)])
def test_gather_of_many_short_rows(page, rows, hi):
    """Rows of a few ids each, some runs of them empty, into an array that is just long enough."""
    rng = np.random.default_rng(rows + page)
    lens = rng.integers(0, hi + 1, rows)
    lens[rows // 4: rows // 2] = 0
    lens[-1] = hi
    need = -(-lens // page)
    table = rng.permutation(int(need.sum())).astype(np.int32)
    pool = rng.integers(0, 1 << 30, (table.size, page)).astype(np.int32)
    po, ho = np.concatenate([[0], np.cumsum(need)]), np.concatenate([[0], np.cumsum(lens)])
    row = np.repeat(np.arange(rows), lens)
    j = np.arange(row.size) - ho[row]
    want = pool[table[po[row] + j // page], j % page]
    d = lambda a: torch.from_numpy(a).to(_dev())  # noqa: E731
    out = torch.full((want.size,), -7, dtype=torch.int32, device=_dev())
    st = torch.zeros(1, dtype=torch.int32, device=_dev())
    NS.gather_paged_history(d(pool), d(table), d(po), d(ho), out=out, status=st)
    assert st.item() == 0 and np.array_equal(out.cpu().numpy(), want)


def test_gather_reports_bad_tables():
    pool = torch.arange(40, dtype=torch.int32, device=_dev()).view(10, 4)
    i64 = dict(dtype=torch.int64, device=_dev())
    st = torch.zeros(1, dtype=torch.int32, device=_dev())

    def run(pages, po, ho, n):
        st.zero_()
        out = torch.full((n,), -7, dtype=torch.int32, device=_dev())
        NS.gather_paged_history(pool, torch.tensor(pages, dtype=torch.int32, device=_dev()), torch.tensor(po, **i64),
                                torch.tensor(ho, **i64), out=out, status=st)
        return out.tolist(), st.item()

    bad = cabi.NS_STATUS_BAD_POOL_RANGE
    assert run([2, 10], [0, 2], [0, 6], 6) == ([8, 9, 10, 11, -1, -1], bad)     # page past the pool
    assert run([2, -1], [0, 2], [0, 5], 5) == ([8, 9, 10, 11, -1], bad)         # negative page
    assert run([2, 3], [0, 1], [0, 6], 6) == ([8, 9, 10, 11, -1, -1], bad)      # the row's table is too short
    assert run([2], [0, 5], [0, 6], 6) == ([8, 9, 10, 11, -1, -1], bad)         # the tables end before
    assert run([2, 3], [-1, 1], [0, 5], 5) == ([-1, -1, -1, -1, 8], bad)        # a negative offset
    assert run([2, 3], [0, 2], [0, 6], 4) == ([8, 9, 10, 11], bad)              # out is too short
    out, flag = run([2, 3], [0, 1, 2], [0, 3, 2], 3)                             # falling offsets: reported, in bounds
    assert flag == bad and all(g in (w, -1, -7) for g, w in zip(out, [8, 9, 10]))
    out, flag = run([2, 3], [0, 1, 2], [0, -9, 4], 4)
    assert flag == bad and set(out) <= {-7, -1, *range(40)}
    assert run([2, 3], [0, 1, 2], [0, 4, 8], 8) == ([8, 9, 10, 11, 12, 13, 14, 15], 0)


def test_gather_refusals():
    pool = torch.zeros(4, 4, dtype=torch.int32, device=_dev())
    t = torch.zeros(1, dtype=torch.int32, device=_dev())
    o = torch.zeros(2, dtype=torch.int64, device=_dev())
    with pytest.raises(RuntimeError, match="page_offsets must have"):
        NS.gather_paged_history(pool, t, o[:1], o, out=t)
    with pytest.raises(RuntimeError, match="page_size"):
        NS.gather_paged_history(pool.view(-1), t, o, o, out=t)
    with pytest.raises(RuntimeError, match="dtype"):
        NS.gather_paged_history(pool, t.long(), o, o, out=t)
    with pytest.raises(RuntimeError, match="contiguous"):
        NS.gather_paged_history(pool[:, :2], t, o, o, out=t)
    with pytest.raises(RuntimeError, match="CUDA"):
        NS.gather_paged_history(pool.cpu(), t, o, o, out=t)


# -- the store --------------------------------------------------------------------------------------------------
def _store(pages=400, page_size=8, vocab=1000, caches=0):
    cs = [_bits((pages, page_size, 4), torch.float32, k) for k in range(caches)]
    return NS.PagedHistoryStore(_dev(), pages, vocab, page_size, caches=cs)


@pytest.mark.parametrize("page_size", [1, 4, 16])
def test_store_random_life(page_size):
    """Adds, forks, appends, truncations, releases and compactions in random order: every request's ids are what a
    list of Python lists has, a cache that moves along holds the same, and no page is lost."""
    rng = np.random.default_rng(page_size)
    pages = 600
    cache = torch.zeros(pages, page_size, dtype=torch.int32, device=_dev())
    st = NS.PagedHistoryStore(_dev(), pages, 1 << 20, page_size, caches=[cache])
    live = {}

    def note(h):  # the cache row of each token is the token itself, written where the page table says
        for i, p in enumerate(st.pages(h)[: -(-len(live[h]) // page_size)]):
            part = live[h][i * page_size:(i + 1) * page_size]
            cache[p, : len(part)] = torch.tensor(part, dtype=torch.int32, device=_dev())

    for step in range(120):
        what = rng.integers(0, 7)
        handles = list(live)
        if what == 0 or not handles:
            ids = rng.integers(0, 1 << 20, rng.integers(0, 40)).tolist()
            h = st.add(ids, int(rng.integers(0, 3)))
            live[h] = ids
            note(h)
        elif what == 1:
            h = handles[rng.integers(len(handles))]
            for f in st.fork(h, int(rng.integers(0, 4))):
                live[f] = list(live[h])
        elif what in (2, 3):
            some = [h for h in handles if rng.random() < 0.7]
            if some:
                tok = rng.integers(0, 1 << 20, len(some))
                st.append(some, torch.from_numpy(tok).to(_dev()))
                for h, t in zip(some, tok.tolist()):
                    live[h].append(t)
                    note(h)
        elif what == 4:
            h = handles[rng.integers(len(handles))]
            n = int(rng.integers(0, len(live[h]) + 1))
            st.truncate(h, n)
            live[h] = live[h][:n]
        elif what == 5 and len(handles) > 4:
            h = handles[rng.integers(len(handles))]
            st.release(h)
            del live[h]
        else:
            st.compact()
            used = {p for h in live for p in st.pages(h)}
            assert used == set(range(len(used))) and st.free_pages() == pages - len(used)
        if step % 10 == 9:
            for h, ids in live.items():
                assert st.length(h) == len(ids) and st.tokens(h) == ids
                at = st.pages(h)[: -(-len(ids) // page_size)]
                assert cache[at].reshape(-1)[: len(ids)].tolist() == ids
    for h in live:
        st.release(h)
    assert st.free_pages() == pages and st.status.item() == 0


def test_store_refusals_change_nothing():
    st = _store(pages=6, page_size=4, vocab=100)
    a = st.add(list(range(10)))  # three pages
    b, = st.fork(a)              # shares two, owns one
    assert st.free_pages() == 2
    with pytest.raises(MemoryError):
        st.add(list(range(20)))
    with pytest.raises(MemoryError):
        st.fork(a, 3)
    with pytest.raises(IndexError):
        st.add([100])
    with pytest.raises(ValueError):
        st.truncate(a, 11)
    with pytest.raises(ValueError, match="twice"):
        st.append([a, a], torch.tensor([1, 2], device=_dev()))
    with pytest.raises(MemoryError):
        st.reserve(a, 50)
    with pytest.raises(KeyError):
        st.release(99)
    assert st.free_pages() == 2 and st.tokens(a) == st.tokens(b) == list(range(10))
    # a truncation into a shared page takes a page of its own
    st.truncate(b, 6)
    st.append([b], torch.tensor([77], device=_dev()))
    assert st.tokens(a) == list(range(10)) and st.tokens(b) == [0, 1, 2, 3, 4, 5, 77]
    st.append([a, b], torch.tensor([55, 66], dtype=torch.int32, device=_dev()))
    assert st.tokens(a) == [*range(10), 55] and st.tokens(b) == [0, 1, 2, 3, 4, 5, 77, 66]


def test_store_refuses_caches_it_cannot_copy():
    ok = torch.zeros(8, 2, 3, device=_dev())
    for bad in (torch.zeros(7, 2, device=_dev()), torch.zeros(8, 2), torch.zeros(8, 3, 2, device=_dev()).transpose(1, 2),
                torch.zeros((), device=_dev())):
        with pytest.raises((ValueError, RuntimeError)):
            NS.PagedHistoryStore(_dev(), 8, 10, 4, caches=[ok, bad])
    NS.PagedHistoryStore(_dev(), 8, 10, 4, caches=[ok])


def test_a_full_pool_is_found_out_before_sampling():
    st = _store(pages=3, page_size=2, vocab=50)
    a, b = st.add([1, 2]), st.add([3, 4])
    s = NS.Sampler(_dev())
    lg = torch.randn(2, 50, device=_dev())
    with pytest.raises(MemoryError):
        st.sample(s, lg, [SP(), SP()], [a, b])
    with pytest.raises(ValueError, match="twice"):
        st.sample(s, lg, [SP(), SP()], [a, a])
    assert st.free_pages() == 1 and st.tokens(a) == [1, 2] and s._step == 0
    out = st.sample(s, lg[:1], [SP()], [a])
    assert st.tokens(a) == [1, 2, int(out)] and st.free_pages() == 0


def test_paged_pack_equals_host_packing():
    rng = np.random.default_rng(12)
    V = 128256
    params = W.mixed_params(40) + [SP(temperature=0.8, repetition_penalty=1.25)] * 5
    hists = W.histories(rng, len(params), 0, 700, V)
    hists[3] = []
    st = NS.PagedHistoryStore(_dev(), 4000, V, 16)
    handles = [st.add(h) for h in hists]
    rp, off, ids, order = st.pack(params, handles, sms=148)
    ref = H.packing.pack(params, hists, V, sms=148)
    assert rp.cpu().numpy().tobytes() == ref.row_params.tobytes()
    assert np.array_equal(off.cpu().numpy(), ref.offsets) and np.array_equal(ids.cpu().numpy(), ref.ids)
    assert np.array_equal(order.cpu().numpy(), ref.order)


@pytest.mark.parametrize("extended", [False, True])
@pytest.mark.parametrize("kind", ["regions", "pages"])
def test_decode_steps_through_the_stores_match_lists(kind, extended):
    """Three steps, forked requests among them: the tokens and log-probabilities through a store equal those over
    Python lists; the histories grow by the sampled ids."""
    rng = np.random.default_rng(31)
    S, V = 20, 32000
    params = W.mixed_params(S)
    if extended:
        params = [NS.ExtendedSamplingParams(
            temperature=p.temperature, top_k=p.top_k, top_p=p.top_p, repetition_penalty=p.repetition_penalty,
            presence_penalty=0.6 if i % 2 else 0.0, frequency_penalty=0.3 if i % 3 else 0.0,
            logit_bias={5: 2.0, 100 + i: -np.inf} if i % 4 == 1 else None) for i, p in enumerate(params)]
    hists = W.histories(rng, S, 0, 60, V)
    prompts = [len(h) for h in hists]
    if kind == "pages":
        st = NS.PagedHistoryStore(_dev(), 400, V, 8)
        handles = [st.add(h) for h in hists[:S // 2]]
        handles += [st.fork(h)[0] for h in handles]
        hists = [list(h) for h in hists[:S // 2] + hists[:S // 2]]
        prompts = [len(h) for h in hists]
    else:
        st = NS.HistoryStore(_dev(), 10000, V)
        handles = [st.add(h, 8) for h in hists]
    a, b = NS.Sampler(_dev()), NS.Sampler(_dev())
    for step in range(3):
        lg = torch.from_numpy(W.peaked_logits(rng, S, V)).to(_dev())
        for r in range(S):
            if hists[r]:
                lg[r, hists[r][-1]] += 9.0
        kw = dict(prompt_lens=prompts) if extended else {}
        (ta, la) = a.sample(lg, params, hists, seed=5, logprobs=3, **kw)
        (tb, lb) = st.sample(b, lg, params, handles, seed=5, logprobs=3)
        assert ta.tolist() == tb.tolist(), step
        assert all(torch.equal(x, y) for x, y in zip(la, lb))
        if kind == "pages" and step == 1:
            st.compact()
        for h, t in zip(hists, ta.tolist()):
            h.append(t)
    for h, handle in zip(hists, handles):
        assert st.tokens(handle) == h
    assert st.status.item() == 0
