"""Plain 64-bit forms of the operators around sampling, with the error that
fp32 kernels may make (test infrastructure)."""
from __future__ import annotations

import numpy as np

HALF = 2.0**-24  # half a step of fp32, relative


def process_rows(rows, hists, prompts=None, rep=None, pres=None, freq=None, biases=None, masks=None):
    """(result, error bound) of logits processing, float64 [S, V].

    ``rows`` float64 [S, V]; ``hists`` lists of ids; ``biases`` lists of (id, value);
    ``masks`` a list of boolean [V] arrays or None.  The bound adds half a step of
    fp32 for every operation whose result fp32 rounds: the repetition penalty,
    freq * c, its subtraction, the presence penalty's, and the bias's; the
    factor covers their products."""
    S, V = rows.shape
    out, err = rows.astype(np.float64).copy(), np.zeros((S, V))
    f32 = lambda a, i, d: d if a is None else float(np.float32(a[i]))  # noqa: E731
    with np.errstate(all="ignore"):
        for i in range(S):
            y, e = out[i], err[i]
            r, p, f = f32(rep, i, 1.0), f32(pres, i, 0.0), f32(freq, i, 0.0)
            h = np.asarray(hists[i], dtype=np.int64) if hists is not None else np.zeros(0, np.int64)
            h_gen = h[max(0, int(prompts[i])) if prompts is not None else 0:]
            seen = np.unique(h[(h >= 0) & (h < V)])
            if r != 1.0:
                y[seen] = np.where(y[seen] < 0, y[seen] * r, y[seen] / r)
                e[seen] += HALF * np.abs(y[seen])
            ids, c = np.unique(h_gen[(h_gen >= 0) & (h_gen < V)], return_counts=True)
            if f or p:
                y[ids] = y[ids] - f * c
                e[ids] += HALF * np.abs(f * c) + HALF * np.abs(y[ids])
                y[ids] = y[ids] - p
                e[ids] += HALF * np.abs(y[ids])
            if biases is not None:
                for v, b in dict(biases[i]).items():  # the last entry for an id counts
                    if 0 <= v < V:
                        y[v] += float(np.float32(b))
                        e[v] += HALF * abs(y[v])
            if masks is not None and masks[i] is not None:
                y[~masks[i]] = -np.inf
                e[~masks[i]] = 0.0
    err[~np.isfinite(err)] = 0.0
    return out, err * (1 + 2.0**-20) + 2.0**-148


def assert_processed(got, want, err, half_step):
    """``got`` (the kernel's, as float64) is ``want`` within ``err`` and half a step of its type."""
    assert got.shape == want.shape
    assert np.array_equal(np.isnan(got), np.isnan(want))
    fin = np.isfinite(want)
    assert np.array_equal(got[~fin & ~np.isnan(want)], want[~fin & ~np.isnan(want)])
    d = np.abs(got[fin] - want[fin])
    tol = err[fin] + half_step * (np.abs(want[fin]) + err[fin])
    bad = d > tol
    assert not bad.any(), (np.argwhere(fin)[bad][:4], got[fin][bad][:4], want[fin][bad][:4], d[bad].max())


def pack_masks(masks, words=None):
    """Boolean masks as int32 words, bit v % 32 of word v // 32; the bits behind V are 0."""
    V = masks[0].shape[0]
    words = words or (V + 31) // 32
    out = np.zeros((len(masks), words * 4), dtype=np.uint8)
    for i, m in enumerate(masks):
        b = np.packbits(m.astype(np.uint8), bitorder="little")
        out[i, : b.size] = b
    return out.view(np.int32)


def logprob_rows(rows, tokens, n):
    """(logprobs, ranks, top ids, top logprobs, error bound) in float64, rows float64 [S, V].

    The bound: the kernel's sum of exponentials has, per term, the rounding of
    the shifted argument and of its product with log2(e), that constant's
    own (3 half steps of |d|, d = x - max), and the hardware exponential's
    2^-22; weighted by the terms, |d| is on average at most log V.  Sums run
    over at most ADDS terms in fp32 before they continue in more
    bits.  A relative error of the sum is an absolute one of its logarithm;
    x - max, the logarithm (one step) and their difference round too."""
    S, V = rows.shape
    lp, rk = np.zeros(S), np.zeros(S, dtype=np.int64)
    ids, tl, err = np.zeros((S, n), dtype=np.int64), np.zeros((S, n)), np.zeros((S, n + 1))
    sum_err = (3 * np.log(max(V, 2)) + 4 + ADDS) * HALF
    for i in range(S):
        x, t = rows[i], int(tokens[i])
        ok = 0 <= t < V
        if np.isnan(x).any() or np.isposinf(x).any() or not (x > -np.inf).any():
            lp[i], rk[i] = (-np.log(V), 1) if ok else (np.nan, 0)
            ids[i], tl[i] = np.arange(n), -np.log(V)
            err[i] = 2 * HALF * np.log(V)
            continue
        m = x.max()
        logsum = np.log(np.exp(x - m).sum())
        order = np.argsort(-x, kind="stable")[:n]
        ids[i], tl[i] = order, x[order] - m - logsum
        lp[i], rk[i] = (x[t] - m - logsum, 1 + int((x > x[t]).sum())) if ok else (np.nan, 0)
        vals = np.concatenate([[x[t] if ok else 0.0], x[order]])
        e = sum_err + HALF * (np.abs(vals - m) + 2 * abs(logsum) + np.abs(vals - m - logsum))
        err[i] = np.where(np.isfinite(e), e, 0.0)
    return lp, rk, ids, tl, err * (1 + 2.0**-20)


ADDS = 256
