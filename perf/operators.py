"""Timed cases of the operators around sampling: logits processing, token log-probabilities, page copies and
paged history gathers.

Every case runs in two ways on the same inputs: in elementary torch operations (``own`` false), and as the
calls that a user makes of this package (``own`` true).  ``listed`` gives the named cases, ``draw`` one more of
the same ranges, ``prepare`` the inputs of a case, ``run`` one pass, ``work`` the bytes and operations that a pass
cannot do without, and ``exact`` the results in 64 bits.
"""
import importlib
import math

import numpy as np
import torch

own = False

PKG = "nanoserve---custom-llm-inference-engine_b200"
VOCAB = 128256
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
PAGE = 16                      # tokens of a cache page
KV_SHAPE = (PAGE, 8, 128)      # one page of keys (or values) of one layer: 32 KiB in bf16
LARGEST = 1 << 30              # bytes of logits that a drawn case reads at most


def listed():
    return [
        # -- penalties, biases and grammar masks on logits --------------------------------------------------
        # a few interactive users: the eight sampled rows of a step, penalties only; latency counts
        {"name": "process 8 rows", "op": "process", "rows": 8, "from_rows": 16, "vocab": VOCAB, "dtype": "f32",
         "out": "f32", "hist_lo": 32, "hist_hi": 256, "bias": 0, "mask": False, "inplace": False},
        # a decode step of a full batch, every request with penalties and a logit_bias of 32 ids
        {"name": "process 256 rows", "op": "process", "rows": 256, "from_rows": 0, "vocab": VOCAB, "dtype": "f32",
         "out": "f32", "hist_lo": 128, "hist_hi": 2048, "bias": 32, "mask": False, "inplace": False},
        # the same step on a buffer of logits that nobody reads again
        {"name": "process 256 in place", "op": "process", "rows": 256, "from_rows": 0, "vocab": VOCAB, "dtype": "f32",
         "out": "f32", "hist_lo": 128, "hist_hi": 2048, "bias": 32, "mask": False, "inplace": True},
        # chunked prefill: 64 rows of 4096 are sampled, two thirds of them under a grammar, long prompts
        {"name": "process 64 of 4096 grammar", "op": "process", "rows": 64, "from_rows": 4096, "vocab": VOCAB,
         "dtype": "bf16", "out": "f32", "hist_lo": 512, "hist_hi": 4096, "bias": 0, "mask": True, "inplace": False},
        # offline generation: many rows of an odd vocabulary (rows off the 16-byte grid), everything at once
        {"name": "process 2048 odd vocab", "op": "process", "rows": 2048, "from_rows": 0, "vocab": 50257,
         "dtype": "f32", "out": "f32", "hist_lo": 0, "hist_hi": 1024, "bias": 300, "mask": True, "inplace": False},
        # -- log-probabilities of given tokens, their ranks, and the best n ---------------------------------
        # the sampled tokens of a small step, five alternatives each
        {"name": "logprobs 8 rows top 5", "op": "logprobs", "rows": 8, "vocab": VOCAB, "dtype": "f32", "top": 5,
         "masked": False},
        # a decode step where every request asks for twenty alternatives, half of the rows under a grammar
        {"name": "logprobs 256 rows top 20", "op": "logprobs", "rows": 256, "vocab": VOCAB, "dtype": "f32", "top": 20,
         "masked": True},
        # scoring a prompt of 4096 tokens
        {"name": "logprobs 4096 rows top 1", "op": "logprobs", "rows": 4096, "vocab": VOCAB, "dtype": "bf16", "top": 1,
         "masked": False},
        # -- copies of cache pages --------------------------------------------------------------------------
        # forking 32 requests: the last page of each, keys and values of eight layers
        {"name": "copy 32 pages of 16", "op": "copy", "pools": 16, "pages": 512, "moves": 32, "kind": "kv"},
        # compacting a cache: 300 pages of each pool move into the holes at its front
        {"name": "copy 300 pages of 16", "op": "copy", "pools": 16, "pages": 1024, "moves": 300, "kind": "kv"},
        # -- token histories out of a paged cache -----------------------------------------------------------
        # the histories of a decode step
        {"name": "gather 256 rows", "op": "gather", "rows": 256, "page": PAGE, "lo": 128, "hi": 2048},
        # the histories of a large offline batch
        {"name": "gather 16384 rows", "op": "gather", "rows": 16384, "page": PAGE, "lo": 128, "hi": 1024},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["process", "process", "logprobs", "logprobs", "copy", "gather"])
    if op == "process":
        vocab, dtype = _log_int(rng, 1000, 160000), rng.choice(["f32", "bf16"])
        rows = _log_int(rng, 1, max(1, min(4096, LARGEST // 8 // (4 * vocab))))
        inplace = rng.random() < 0.25
        hi = _log_int(rng, 1, 8192 if rows <= 256 else 1024)
        return {"op": op, "rows": rows, "from_rows": 0 if inplace or rng.random() < 0.5 else rows + rng.randrange(64),
                "vocab": vocab, "dtype": dtype, "out": dtype if inplace or dtype == "f32" else rng.choice(["f32", "bf16"]),
                "hist_lo": rng.randrange(hi + 1), "hist_hi": hi, "bias": min(vocab // 4, rng.choice([0, _log_int(rng, 1, 300)])),
                "mask": rng.random() < 0.5, "inplace": inplace}
    if op == "logprobs":
        vocab, dtype = _log_int(rng, 1000, 160000), rng.choice(["f32", "bf16"])
        return {"op": op, "rows": _log_int(rng, 1, max(1, min(4096, LARGEST // 2 // (4 * vocab)))), "vocab": vocab,
                "dtype": dtype, "top": rng.randrange(21), "masked": rng.random() < 0.3}
    if op == "copy":
        if rng.random() < 0.5:
            pages = _log_int(rng, 64, 1024)
            return {"op": op, "pools": rng.randrange(1, 17), "pages": pages, "moves": _log_int(rng, 1, pages // 3), "kind": "kv"}
        pages = _log_int(rng, 64, 1 << 18)
        return {"op": op, "pools": 1, "pages": pages, "moves": _log_int(rng, 1, pages // 3), "kind": "ids"}
    hi = _log_int(rng, 1, 4096)
    return {"op": op, "rows": _log_int(rng, 1, min(16384, (10 << 20) // hi)), "page": rng.choice([1, 5, 16, 32, 64, 256]),
            "lo": rng.randrange(hi + 1), "hi": hi}


# -- inputs -----------------------------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _peaked(g, rows, vocab, dtype):
    """Logits as a language model's head gives them: a Gaussian bulk and about twenty likely ids a row."""
    x = torch.empty(rows, vocab, dtype=dtype, device="cuda").normal_(0.0, 2.0, generator=g)
    n = min(20, vocab)
    at = torch.randint(vocab, (rows, n), generator=g, device="cuda")
    return x.scatter_add_(1, at, torch.full((rows, n), 8.0, dtype=dtype, device="cuda"))


def _lengths(g, rows, lo, hi):
    """Lengths spread evenly over [lo, hi], in an order of the seed's (their sum is the same for every seed)."""
    i = torch.randperm(rows, generator=g, device="cuda")
    lens = lo + (2 * i + 1) * (hi - lo + 1) // (2 * rows)
    offsets = torch.zeros(rows + 1, dtype=torch.int64, device="cuda")
    offsets[1:] = lens.cumsum(0)
    return lens, offsets


def _tokens(g, n, vocab):
    """Token ids of text: a few ids are very common, most are rare."""
    u = torch.rand(n, generator=g, device="cuda", dtype=torch.float64)
    return (u**4 * vocab).long().clamp_(max=vocab - 1).to(torch.int32)


def _uniform(g, n, lo, hi):
    return torch.rand(n, generator=g, device="cuda") * (hi - lo) + lo


def prepare(case, seed):
    g = _gen(seed)
    s = {"case": dict(case)}
    if own:
        s["ns"] = importlib.import_module(PKG)
    op = case["op"]
    if op == "process":
        rows, vocab = case["rows"], case["vocab"]
        s["logits"] = _peaked(g, case["from_rows"] or rows, vocab, DTYPES[case["dtype"]])
        s["sample_indices"] = None
        if case["from_rows"]:
            s["sample_indices"] = torch.randperm(case["from_rows"], generator=g, device="cuda")[:rows].contiguous()
        lens, s["history_offsets"] = _lengths(g, rows, case["hist_lo"], case["hist_hi"])
        s["history_ids"] = _tokens(g, int(s["history_offsets"][-1]), vocab)
        s["prompt_lens"] = (lens * torch.rand(rows, generator=g, device="cuda")).to(torch.int32)
        s["repetition_penalty"] = _uniform(g, rows, 1.0, 1.3)
        s["presence_penalty"] = _uniform(g, rows, -0.5, 1.0)
        s["frequency_penalty"] = _uniform(g, rows, 0.0, 0.5)
        s["bias_offsets"] = s["bias_ids"] = s["bias_values"] = None
        if case["bias"]:
            # a request's logit_bias is a dict: an id appears once in a row
            n = case["bias"]
            s["bias_offsets"] = torch.arange(rows + 1, device="cuda") * n
            first = torch.randint(vocab, (rows, 1), generator=g, device="cuda")
            step = torch.randint(1, vocab // n + 1, (rows, 1), generator=g, device="cuda")
            s["bias_ids"] = ((first + step * torch.arange(n, device="cuda")) % vocab).reshape(-1).to(torch.int32)
            v = torch.randn(rows * n, generator=g, device="cuda") * 2.0
            v[torch.rand(rows * n, generator=g, device="cuda") < 0.1] = -100.0
            v[torch.rand(rows * n, generator=g, device="cuda") < 0.02] = -math.inf  # banned ids
            s["bias_values"] = v
        s["allowed"] = s["allowed_rows"] = None
        if case["mask"]:
            # a third of the rows allow about 1/16 of the vocabulary (inside a structure), a third 15/16 (inside a
            # string), a third is free
            shape = (max(2, 2 * ((rows + 2) // 3)), (vocab + 31) // 32)
            words = [torch.randint(-(2**31), 2**31, shape, generator=g, device="cuda", dtype=torch.int32) for _ in range(4)]
            tight = words[0] & words[1] & words[2] & words[3]
            loose = words[0] | words[1] | words[2] | words[3]
            odd = (torch.arange(shape[0], device="cuda") % 2 == 1)[:, None]
            s["allowed"] = torch.where(odd, loose, tight).contiguous()
            i = torch.arange(rows, device="cuda")
            s["allowed_rows"] = torch.where(i % 3 == 2, -1, 2 * (i // 3) + i % 3).to(torch.int32)
    elif op == "logprobs":
        rows, vocab = case["rows"], case["vocab"]
        x = _peaked(g, rows, vocab, DTYPES[case["dtype"]])
        if case["masked"]:  # every other row keeps about a tenth of its ids
            for r in range(0, rows, 2):
                x[r, torch.rand(vocab, generator=g, device="cuda") < 0.9] = -math.inf
            x[:, 0] = 0.0
        s["logits"] = x
        # the tokens that a sampler took: likely ones
        noise = torch.rand(rows, min(vocab, 64), generator=g, device="cuda")
        at = torch.randint(vocab, noise.shape, generator=g, device="cuda")
        score = x.gather(1, at).float() - torch.log(-torch.log(noise.clamp(1e-6, 1 - 1e-6)))
        s["token_ids"] = at.gather(1, score.argmax(1, keepdim=True))[:, 0].contiguous()
    elif op == "copy":
        pages, moves = case["pages"], case["moves"]
        if case["kind"] == "kv":
            s["pools"] = [torch.empty(pages, *KV_SHAPE, dtype=torch.bfloat16, device="cuda").normal_(generator=g)
                          for _ in range(case["pools"])]
        else:
            s["pools"] = [_tokens(g, pages * PAGE, VOCAB).reshape(pages, PAGE) for _ in range(case["pools"])]
        # the plan of a host allocator: sources and destinations are different pages
        order = torch.randperm(pages, generator=torch.Generator().manual_seed(int(seed)))
        s["src"], s["dst"] = order[:moves].clone(), order[moves : 2 * moves].clone()
    else:
        rows, page = case["rows"], case["page"]
        lens, s["history_offsets"] = _lengths(g, rows, case["lo"], case["hi"])
        s["total"] = int(s["history_offsets"][-1])
        counts = (lens + page - 1) // page
        s["page_offsets"] = torch.zeros(rows + 1, dtype=torch.int64, device="cuda")
        s["page_offsets"][1:] = counts.cumsum(0)
        live = int(s["page_offsets"][-1])
        num_pages = live + live // 4 + 1
        s["pages"] = torch.randperm(num_pages, generator=g, device="cuda")[:live].to(torch.int32)
        s["pool"] = _tokens(g, num_pages * page, VOCAB).reshape(num_pages, page)
        s["out"] = torch.empty(s["total"], dtype=torch.int32, device="cuda")
    return s


# -- one pass ---------------------------------------------------------------------------------------------------
def run(s):
    return {"process": _process, "logprobs": _logprobs, "copy": _copy, "gather": _gather}[s["case"]["op"]](s)


def _process(s):
    c, logits = s["case"], s["logits"]
    out_dtype = DTYPES[c["out"]]
    if own:
        return s["ns"].process_logits(
            logits, sample_indices=s["sample_indices"], history_offsets=s["history_offsets"], history_ids=s["history_ids"],
            prompt_lens=s["prompt_lens"], repetition_penalty=s["repetition_penalty"],
            presence_penalty=s["presence_penalty"], frequency_penalty=s["frequency_penalty"],
            bias_offsets=s["bias_offsets"], bias_ids=s["bias_ids"], bias_values=s["bias_values"], allowed=s["allowed"],
            allowed_rows=s["allowed_rows"], out=logits if c["inplace"] else None, out_dtype=out_dtype)
    rows, vocab = c["rows"], c["vocab"]
    x = (logits if s["sample_indices"] is None else logits[s["sample_indices"]]).float()
    # where each history id stands, and whether it was generated
    at = torch.arange(s["history_ids"].numel(), device=x.device)
    row = torch.searchsorted(s["history_offsets"], at, right=True) - 1
    flat = row * vocab + s["history_ids"]
    generated = at - s["history_offsets"][row] >= s["prompt_lens"][row]
    seen = torch.zeros(rows * vocab, dtype=torch.bool, device=x.device)
    seen[flat] = True
    count = torch.zeros(rows * vocab, dtype=torch.float32, device=x.device).index_add_(0, flat, generated.float())
    seen, count = seen.view(rows, vocab), count.view(rows, vocab)
    rp = s["repetition_penalty"][:, None]
    x = torch.where(seen, torch.where(x < 0, x * rp, x / rp), x)
    x = x - s["frequency_penalty"][:, None] * count
    x = torch.where(count > 0, x - s["presence_penalty"][:, None], x)
    if s["bias_ids"] is not None:
        at = torch.arange(s["bias_ids"].numel(), device=x.device)
        flat = (torch.searchsorted(s["bias_offsets"], at, right=True) - 1) * vocab + s["bias_ids"]
        x.view(-1)[flat] = x.view(-1)[flat] + s["bias_values"]
    if s["allowed"] is not None:
        v = torch.arange(vocab, device=x.device)
        bits = (s["allowed"][s["allowed_rows"].clamp(min=0)][:, v // 32] >> (v % 32)) & 1
        x = torch.where((bits == 0) & (s["allowed_rows"] >= 0)[:, None], -math.inf, x)
    return logits.copy_(x) if c["inplace"] else x.to(out_dtype)


def _logprobs(s):
    n = s["case"]["top"]
    if own:
        r = s["ns"].token_logprobs(s["logits"], s["token_ids"], n)
        return [r.logprobs, r.ranks, r.top_ids, r.top_logprobs]
    x = s["logits"].float()
    top = x.amax(1, keepdim=True)
    lse = top + torch.log(torch.exp(x - top).sum(1, keepdim=True))
    mine = x.gather(1, s["token_ids"][:, None])
    ranks = 1 + (x > mine).sum(1)
    logprobs = (mine - lse)[:, 0]
    if n == 0:
        empty = torch.empty(x.shape[0], 0, device=x.device)
        return [logprobs, ranks.to(torch.int32), empty.long(), empty]
    # one sortable whole number for each (logit, id): larger logits first, then lower ids
    bits = (x + 0.0).view(torch.int32)  # -0 counts as 0
    key = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long() * 2**32 + (x.shape[1] - 1 - torch.arange(x.shape[1], device=x.device))
    best = x.shape[1] - 1 - (key.topk(n, 1).values & 0xFFFFFFFF)
    return [logprobs, ranks.to(torch.int32), best, x.gather(1, best) - lse]


def _copy(s):
    if own:
        s["ns"].copy_pages(s["pools"], s["src"], s["dst"])
        return s["pools"]
    src, dst = s["src"].cuda(non_blocking=True), s["dst"].cuda(non_blocking=True)
    for p in s["pools"]:
        p[dst] = p[src]
    return s["pools"]


def _gather(s):
    if own:
        return s["ns"].gather_paged_history(s["pool"], s["pages"], s["page_offsets"], s["history_offsets"], out=s["out"])
    page = s["case"]["page"]
    at = torch.arange(s["total"], device="cuda")
    row = torch.searchsorted(s["history_offsets"], at, right=True) - 1
    j = at - s["history_offsets"][row]
    held = s["pages"][s["page_offsets"][row] + j // page].long()
    s["out"].copy_(s["pool"][held, j % page])
    return s["out"]


# -- what a pass cannot do without ------------------------------------------------------------------------------
def work(case):
    op = case["op"]
    size = {"f32": 4, "bf16": 2}
    if op == "process":
        rows, vocab = case["rows"], case["vocab"]
        n = rows * (case["hist_lo"] + case["hist_hi"]) / 2
        small = 4 * n + 8 * rows * case["bias"] + rows * (8 + 4 * 4)
        if case["mask"]:
            small += 2 / 3 * rows * vocab / 8
        if case["inplace"]:
            # the ids that a penalty or a bias names are read and written, the masked ones written
            touched = 2 * size[case["dtype"]] * (n + rows * case["bias"])
            masked = rows * vocab * size[case["dtype"]] / 3 if case["mask"] else 0
            return {"bytes": small + touched + masked, "flops": 6 * n}
        return {"bytes": small + rows * vocab * (size[case["dtype"]] + size[case["out"]]), "flops": 6 * n}
    if op == "logprobs":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * size[case["dtype"]] + case["rows"] * (16 + 12 * case["top"]), "flops": 4 * n}
    if op == "copy":
        page = 2 * math.prod(KV_SHAPE) if case["kind"] == "kv" else 4 * PAGE
        return {"bytes": 2 * case["pools"] * case["moves"] * page + 16 * case["moves"], "flops": 0}
    n = case["rows"] * (case["lo"] + case["hi"]) / 2
    return {"bytes": 8 * n + 4 * n / case["page"] + 24 * case["rows"], "flops": 0}


# -- the results in 64 bits -------------------------------------------------------------------------------------
def exact(case, seed):
    if case["op"] in ("copy", "gather"):
        return None  # values are moved, not computed
    s = prepare(case, seed)
    if case["op"] == "logprobs":
        return _exact_logprobs(s)
    rows, vocab = case["rows"], case["vocab"]
    if rows * vocab > 1.2e8:
        return None
    host = {k: v.cpu().numpy() for k, v in s.items() if isinstance(v, torch.Tensor) and k != "logits"}
    picked = s["logits"] if s["sample_indices"] is None else s["logits"].index_select(0, s["sample_indices"])
    result = picked.double().cpu().numpy()
    for r in range(rows):
        y = result[r]
        ids = host["history_ids"][host["history_offsets"][r] : host["history_offsets"][r + 1]]
        known = np.unique(ids)
        rp = float(host["repetition_penalty"][r])
        y[known] = np.where(y[known] < 0, y[known] * rp, y[known] / rp)
        said, times = np.unique(ids[host["prompt_lens"][r] :], return_counts=True)
        y[said] -= float(host["frequency_penalty"][r]) * times + float(host["presence_penalty"][r])
        if "bias_ids" in host:
            b = slice(host["bias_offsets"][r], host["bias_offsets"][r + 1])
            y[host["bias_ids"][b]] += host["bias_values"][b]
        if "allowed" in host and host["allowed_rows"][r] >= 0:
            bits = np.unpackbits(host["allowed"][host["allowed_rows"][r]].view(np.uint8), bitorder="little")[:vocab]
            y[bits == 0] = -np.inf
    return result


def _exact_logprobs(s):
    n, parts = s["case"]["top"], []
    for x, t in zip(s["logits"].split(128), s["token_ids"].split(128)):
        x = x.double()
        lse = torch.logsumexp(x, 1)
        mine = x[torch.arange(x.shape[0], device=x.device), t]
        value, index = torch.sort(x, dim=1, descending=True, stable=True)
        parts.append([mine - lse, (value > mine[:, None]).sum(1).to(torch.int32) + 1, index[:, :n], value[:, :n] - lse[:, None]])
    return [torch.cat(p) for p in zip(*parts)]
