"""Host side of the operators around sampling: the C ABI's checks, the page allocator, packing (no GPU needed)."""
import ctypes
import random
import subprocess

import numpy as np
import pytest

from conftest import REPO, pkg

cabi = pkg("_cabi")
packing = pkg("packing")
pages = pkg("pages")
NS = pkg()
HEADER = REPO / "include" / "nanoserve_sampler.h"


def test_struct_layouts_match_the_header(tmp_path):
    structs = (cabi.NsProcessArgs, cabi.NsLogprobArgs, cabi.NsPagePool)
    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{HEADER}"', "int main(void){"]
    for st in structs:
        lines.append(f'printf("{st.__name__} %zu\\n", sizeof({st.__name__}));')
        lines += [f'printf("{st.__name__}.{n} %zu\\n", offsetof({st.__name__}, {n}));' for n, _ in st._fields_]
    (tmp_path / "l.c").write_text("\n".join(lines + ["return 0;}"]))
    subprocess.run(["gcc", str(tmp_path / "l.c"), "-o", str(tmp_path / "l")], check=True)
    got = dict(l.split() for l in subprocess.run([str(tmp_path / "l")], capture_output=True, text=True).stdout.splitlines())
    for st in structs:
        assert int(got[st.__name__]) == ctypes.sizeof(st)
        for n, _ in st._fields_:
            assert int(got[f"{st.__name__}.{n}"]) == getattr(st, n).offset, (st.__name__, n)


def _process(**kw):
    a = cabi.NsProcessArgs()
    base = dict(logits=4096, logits_dtype=0, vocab_size=100, num_logit_rows=2, logits_row_stride=100, num_rows=2, out_dtype=0,
                out=1 << 20, out_row_stride=100)
    for k, v in {**base, **kw}.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,match", [
    (dict(num_rows=-1), "num_rows"), (dict(logits=None), "required"), (dict(out=None), "required"),
    (dict(logits_dtype=5), "logits_dtype"), (dict(out_dtype=1), "out_dtype"), (dict(vocab_size=0), "vocab_size"),
    (dict(logits_row_stride=-1), "stride"), (dict(out_row_stride=99), "out_row_stride"), (dict(num_logit_rows=0), "num_logit_rows"),
    (dict(num_logit_rows=1), "fewer logits rows"), (dict(history_offsets=64, num_history_ids=3), "history_ids"),
    (dict(num_history_ids=-1), "< 0"), (dict(bias_offsets=64, num_biases=2, bias_ids=64), "bias_values"),
    (dict(allowed=64, mask_stride=3, num_masks=2), "mask_stride"), (dict(allowed=64, mask_stride=4, num_masks=1), "fewer masks"),
    (dict(reserved=1), "reserved"), (dict(logits=4098), "aligned"), (dict(out=4096 + 400), "overlaps"),
    (dict(out=4096, sample_indices=64), "overlaps"), (dict(out=4096, out_row_stride=101), "overlaps"),
    (dict(num_rows=1 << 30, num_logit_rows=1 << 30, out=1 << 50, vocab_size=1 << 20, logits_row_stride=1 << 20,
          out_row_stride=1 << 20), "too large"),
])
def test_process_is_checked_on_the_host(kw, match):
    with pytest.raises(cabi.NsError, match=match):
        cabi.ns_process_logits(_process(**kw))


@pytest.mark.parametrize("kw,match", [
    (dict(num_rows=-1), "num_rows"), (dict(token_ids=None), "required"), (dict(logits_dtype=2), "logits_dtype"),
    (dict(ids_dtype=2), "ids_dtype"), (dict(vocab_size=-3), "vocab_size"), (dict(logits_row_stride=-1), "stride"),
    (dict(num_logit_rows=1), "fewer logits rows"), (dict(top_n=33), "top_n"), (dict(top_n=-1), "top_n"),
    (dict(top_n=5, vocab_size=4), "top_n"), (dict(top_n=2), "out_top_ids"), (dict(reserved=1), "reserved"),
    (dict(logits=4097), "aligned"),
])
def test_logprobs_are_checked_on_the_host(kw, match):
    a = cabi.NsLogprobArgs()
    base = dict(logits=4096, vocab_size=100, num_logit_rows=2, logits_row_stride=100, num_rows=2, token_ids=64, out_logprobs=64,
                out_ranks=64)
    for k, v in {**base, **kw}.items():
        setattr(a, k, v)
    with pytest.raises(cabi.NsError, match=match):
        cabi.ns_token_logprobs(a)


@pytest.mark.parametrize("pool,pages_n,src,dst,match", [
    ((64, 16, 16), -1, [0], [1], "< 0"), ((0, 16, 16), 4, [0], [1], "no base"), ((64, 8, 16), 4, [0], [1], "overlap"),
    ((64, 16, 0), 4, [0], [1], "no bytes"), ((64, 16, 16), 4, [4], [1], "outside"), ((64, 16, 16), 4, [0], [-1], "outside"),
    ((64, 16, 16), 4, [0, 1], [2, 2], "twice"), ((64, 16, 16), 4, [0, 2], [2, 3], "both"), ((64, 16, 16), 4, [1], [1], "both"),
    ((64, 16, 16), 1 << 32, [0], [1], "2\\^31"),
])
def test_page_copies_are_checked_on_the_host(pool, pages_n, src, dst, match):
    with pytest.raises(cabi.NsError, match=match):
        cabi.ns_pages_copy([pool], pages_n, src, dst)


def test_page_checks_on_long_lists():
    """Random plans with one thing wrong somewhere, among sound ones; a refusal leaves nothing behind."""
    rng = random.Random(4)
    for n, pages_n in ((1, 2), (5, 40), (300, 1000), (4000, 9000), (500, 100000)):
        for _ in range(6):
            order = rng.sample(range(pages_n), 2 * n)
            src, dst = order[:n], order[n:]
            cabi.ns_pages_check(pages_n, src, dst)
            cabi.ns_pages_check(pages_n, [src[0]] * n, dst)
            low, high = sorted(order)[:n], sorted(order)[n:]
            cabi.ns_pages_check(pages_n, high, low)  # as a compaction's
            cabi.ns_pages_check(pages_n, low, high)
            i, j = rng.randrange(n), rng.randrange(n)
            for bad, match in ((-1, "outside"), (pages_n, "outside"), (1 << 62, "outside"), (src[j], "both")):
                with pytest.raises(cabi.NsError, match=match):
                    cabi.ns_pages_check(pages_n, src, dst[:i] + [bad] + dst[i + 1:])
            for bad, match in ((-5, "outside"), (pages_n, "outside"), (dst[j], "both")):
                with pytest.raises(cabi.NsError, match=match):
                    cabi.ns_pages_check(pages_n, src[:i] + [bad] + src[i + 1:], dst)
            if n > 1 and i != j:
                with pytest.raises(cabi.NsError, match="twice"):
                    cabi.ns_pages_check(pages_n, src, dst[:i] + [dst[j]] + dst[i + 1:])
                with pytest.raises(cabi.NsError, match="twice"):
                    cabi.ns_pages_check(pages_n, high, [low[max(k, 1) - 1] if k == max(i, 1) else x for k, x in enumerate(low)])
                with pytest.raises(cabi.NsError, match="outside"):
                    cabi.ns_pages_check(pages_n, high[:-1] + [pages_n + 3], low)
    with pytest.raises(cabi.NsError, match="null"):
        cabi._call("ns_pages_check", 5, None, None, 2)
    with pytest.raises(cabi.NsError, match="< 0"):
        cabi.ns_pages_check(-1, [0], [1])


def test_listed_copies_are_checked_on_the_host():
    for args, match in ((([(64, 16, 16)], 4, 0, 16, 1), "null"), (([(64, 8, 16)], 4, 16, 16, 1), "overlap"),
                        (([(64, 16, 16)], 4, 16, 16, -1), "< 0"), (([(64, 16, 16)], 1 << 31, 16, 16, 1), "2\\^31")):
        with pytest.raises(cabi.NsError, match=match):
            cabi.ns_pages_copy_listed(*args)
    cabi.ns_pages_copy_listed([], 0, 0, 0, 0)


def test_gather_is_checked_on_the_host():
    for args, match in (((16, 4, 0, 16, 4, 16, 16, 1, 16, 4), "page_size"), ((16, -1, 4, 16, 4, 16, 16, 1, 16, 4), "< 0"),
                        ((16, 4, 4, 16, 4, 0, 16, 1, 16, 4), "null"), ((0, 4, 4, 16, 4, 16, 16, 1, 16, 4), "null"),
                        ((16, 4, 4, 0, 4, 16, 16, 1, 16, 4), "null")):
        with pytest.raises(cabi.NsError, match=match):
            cabi.ns_paged_history_gather(*args)


def test_more_rows_than_row_numbers_hold_are_refused():
    with pytest.raises(cabi.NsError, match="2\\^30 rows"):
        cabi.ns_paged_history_gather(16, 4, 4, 16, 4, 16, 16, (1 << 30) + 1, 16, 4)
    for out in (1 << 45, 4096):  # another array, and in place
        a = cabi.NsProcessArgs()
        for k, v in dict(logits=4096, out=out, vocab_size=1, num_logit_rows=0x7fffffff, logits_row_stride=1, out_row_stride=1,
                         num_rows=0x7fffffff - 40).items():
            setattr(a, k, v)
        with pytest.raises(cabi.NsError, match="too large"):
            cabi.ns_process_logits(a)


def test_nothing_to_do_needs_no_gpu():
    cabi.ns_process_logits(cabi.NsProcessArgs())
    cabi.ns_token_logprobs(cabi.NsLogprobArgs())
    cabi.ns_pages_copy([], 0, [], [])
    cabi.ns_pages_copy([(64, 16, 16)], 4, [], [])
    cabi.ns_paged_history_gather(0, 0, 1, 0, 0, 0, 0, 0, 0, 0)


def test_there_is_no_cpu_path():
    import torch

    x = torch.zeros(2, 10)
    with pytest.raises(RuntimeError, match="CUDA"):
        NS.process_logits(x)
    with pytest.raises(RuntimeError, match="CUDA"):
        NS.token_logprobs(x, torch.zeros(2, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="CUDA"):
        NS.copy_pages(x, [0], [1])
    with pytest.raises(RuntimeError, match="CUDA"):
        NS.gather_paged_history(x.int(), x, x, x, out=x)
    with pytest.raises(RuntimeError, match="CUDA"):
        NS.PagedHistoryStore("cpu", 4, 10)


def test_ops_register():
    import torch

    NS.load_ops()
    for name in ("process_logits", "token_logprobs", "copy_pages", "paged_history_gather"):
        assert "!" in str(getattr(torch.ops.nanoserve_b200, name).default._schema)  # each says what it writes


def test_allocator_takes_the_lowest_page_and_counts_users():
    a = pages.PageAllocator(6)
    p = a.alloc(4)
    assert p == [0, 1, 2, 3] and a.live_total() == 4
    a.share([1, 3])
    a.free([0, 1])
    assert a.users(1) == 1 and a.users(0) == 0 and a.free_total() == 3
    with pytest.raises(MemoryError):
        a.alloc(4)
    assert a.free_total() == 3
    for bad in ([0], [1, 1], [-1], [6]):
        with pytest.raises(ValueError):
            a.free(bad)
    for bad in ([4], [-2], [6], [1, 0]):
        with pytest.raises(ValueError):
            a.share(bad)
    assert a.users(1) == 1 and a.alloc(1) == [0]
    with pytest.raises(ValueError):
        a.alloc(-1)
    with pytest.raises(ValueError):
        pages.PageAllocator(-1)
    assert pages.PageAllocator(0).alloc(0) == []


def test_allocator_random_life_and_compaction():
    rng = random.Random(3)
    a = pages.PageAllocator(300)
    users = {}
    for step in range(2000):
        r = rng.random()
        if r < 0.45:
            n = rng.randrange(6)
            if n <= a.free_total():
                for p in a.alloc(n):
                    assert p not in users
                    users[p] = 1
        elif r < 0.6 and users:
            p = rng.choice(list(users))
            a.share([p])
            users[p] += 1
        elif r < 0.97 and users:
            p = rng.choice(list(users))
            a.free([p])
            users[p] -= 1
            if not users[p]:
                del users[p]
        else:
            src, dst = a.plan_compact()
            assert len(set(dst.tolist())) == dst.size and not set(src.tolist()) & set(dst.tolist())
            a.move(src, dst)
            for s, d in zip(src.tolist(), dst.tolist()):
                users[d] = users.pop(s)
            assert sorted(users) == list(range(len(users)))
            assert all(p.size == 0 for p in a.plan_compact())
        assert a.live_total() == len(users) and all(a.users(p) == n for p, n in users.items())


def test_processing_is_packed_only_where_it_is_asked_for():
    SP, EP = NS.SamplingParams, NS.ExtendedSamplingParams
    assert not packing.wants_processing([SP(), SP(repetition_penalty=1.2)])
    assert not packing.wants_processing([EP(), EP(logit_bias={})]) and not packing.wants_processing([])
    for kw in (dict(presence_penalty=0.1), dict(frequency_penalty=-1.0), dict(logit_bias={3: 0.0})):
        assert packing.wants_processing([SP(), EP(**kw)])
    params = [SP(repetition_penalty=1.1), EP(frequency_penalty=0.5, logit_bias={7: 1.5, 2: -np.inf}), SP(), EP(presence_penalty=1.0)]
    pr = packing.pack_processing(params, [3, 4, 5, 0], [1, 2, 3, 0], 10)
    assert pr.lens.tolist() == [3, 4, 0, 0] and pr.offsets.tolist() == [0, 3, 7, 7, 7]
    assert pr.bias_offsets.tolist() == [0, 0, 2, 2, 2] and pr.bias_ids.tolist() == [7, 2]
    assert pr.bias_values.tolist() == [1.5, -np.inf] and pr.prompt_lens.tolist() == [1, 2, 3, 0]
    ids = packing.flatten_histories([[1, 2, 3], [4, 5, 6, 7], [99], []], pr.lens, 10)
    assert ids.tolist() == [1, 2, 3, 4, 5, 6, 7]
    for bad in ({10: 1.0}, {-1: 1.0}):
        with pytest.raises(IndexError):
            packing.pack_processing([EP(logit_bias=bad)], [0], None, 10)
    with pytest.raises(IndexError):
        packing.flatten_histories([[1, 10]], np.array([2]), 10)
    with pytest.raises(ValueError):
        packing.pack_processing([SP()], [0], [1, 2], 10)
