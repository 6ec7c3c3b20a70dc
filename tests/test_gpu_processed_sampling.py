"""Requests with penalties, biases, grammars and log-probabilities through Sampler.sample."""
import importlib

import numpy as np
import pytest
import torch

import gpu_helpers as H
import operator_refs as R
from oracle import sampler_oracle as O

pytestmark = pytest.mark.gpu

NS = importlib.import_module(H.PKG)
W = importlib.import_module(H.PKG + ".workloads")
EP = NS.ExtendedSamplingParams


def _dev():
    assert torch.cuda.is_available(), "GPU test run without a CUDA device"
    return torch.device("cuda:0")


def test_samples_from_the_processed_logits():
    """The whole chain of a request: processing, then the sampler's own oracle on the processed rows, then the
    log-probabilities of what was drawn."""
    rng = np.random.default_rng(1)
    S, V = 40, 32000
    base = W.mixed_params(S)
    params = [EP(temperature=p.temperature, top_k=p.top_k, top_p=p.top_p, repetition_penalty=p.repetition_penalty,
                 presence_penalty=float(i % 3) / 2, frequency_penalty=0.25 * (i % 2),
                 logit_bias={int(v): float(b) for v, b in zip(rng.integers(0, V, 5), rng.normal(0, 4, 5))} if i % 5 else None)
              for i, p in enumerate(base)]
    x = W.peaked_logits(rng, S, V)
    hists = W.histories(rng, S, 0, 80, V)
    for r in range(S):
        for t in hists[r][:10]:
            x[r, t] += 7.0
    prompts = [len(h) // 2 for h in hists]
    masks = [None if i % 3 else rng.random(V) < 0.3 for i in range(S)]
    there = [m for m in masks if m is not None]
    rows = np.cumsum([m is not None for m in masks]) - 1
    kw = dict(allowed=torch.from_numpy(R.pack_masks(there)).to(_dev()),
              allowed_rows=torch.from_numpy(np.where([m is not None for m in masks], rows, -1).astype(np.int32)).to(_dev()))
    uni = torch.from_numpy(rng.random(S).astype(np.float32)).to(_dev())
    lg = torch.from_numpy(x).to(_dev())
    s = NS.Sampler(_dev())
    (out, dbg), lp = s.sample(lg, params, hists, uniforms=uni, prompt_lens=prompts, return_debug=True, logprobs=4, **kw)
    assert torch.equal(lg.cpu(), torch.from_numpy(x))
    want, err = R.process_rows(x.astype(np.float64), hists, prompts, [p.repetition_penalty for p in params],
                               [p.presence_penalty for p in params], [p.frequency_penalty for p in params],
                               [list((p.logit_bias or {}).items()) for p in params], masks)
    got = dbg["penalized"].cpu().numpy()
    R.assert_processed(got.astype(np.float64), want, err, 2.0**-24)
    plain = [NS.SamplingParams(temperature=p.temperature, top_k=p.top_k, top_p=p.top_p) for p in params]
    rep = H.compare(dict(tokens=out.cpu().numpy(), filtered=dbg["filtered"].cpu().numpy(), probs=dbg["probs"].cpu().numpy()),
                    got, plain, [[]] * S, uni.cpu().numpy())
    assert not rep.failures, "\n".join(rep.failures)
    l, rk, ids, tl, e = R.logprob_rows(got.astype(np.float64), out.tolist(), 4)
    assert np.array_equal(lp.ranks.cpu().numpy(), rk) and np.array_equal(lp.top_ids.cpu().numpy(), ids)
    assert (np.abs(lp.logprobs.cpu().numpy() - l) <= e[:, 0]).all()


def test_a_masked_token_is_never_drawn():
    S, V = 64, 5000
    lg = torch.randn(S, V, device=_dev())
    mask = np.zeros(V, dtype=bool)
    mask[[7, 4999]] = True
    allowed = torch.from_numpy(R.pack_masks([mask])).to(_dev())
    s = NS.Sampler(_dev())
    for _ in range(5):
        out = s.sample(lg, [NS.SamplingParams()] * S, [[]] * S, allowed=allowed,
                       allowed_rows=torch.zeros(S, dtype=torch.int32, device=_dev()))
        assert set(out.tolist()) <= {7, 4999}


def test_repetition_penalty_is_the_same_on_both_paths():
    """A row's repetition penalty is applied bit for bit as the sampler does, whether its batch is processed or not."""
    rng = np.random.default_rng(2)
    S, V = 12, 32000
    x = torch.from_numpy(W.peaked_logits(rng, S, V)).to(_dev())
    hists = W.histories(rng, S, 1, 300, V)
    plain = [NS.SamplingParams(temperature=0.8, repetition_penalty=1.3, seed=i) for i in range(S)]
    ext = [EP(temperature=0.8, repetition_penalty=1.3, seed=i, logit_bias={0: 0.0}) for i in range(S)]
    s = NS.Sampler(_dev())
    a, da = s.sample(x, plain, hists, return_debug=True)
    b, db = s.sample(x, ext, hists, return_debug=True)
    assert torch.equal(da["penalized"], db["penalized"]) and a.tolist() == b.tolist()


def test_gathered_bf16_rows():
    w = W.make(3, rows=8, seed=5)
    lg = H.to_bf16_tensor(w.logits, _dev())
    idx = torch.from_numpy(w.sample_indices).to(_dev())
    ext = [EP(temperature=0.0, repetition_penalty=1.2, frequency_penalty=0.1) for _ in w.params]
    out, lp = NS.Sampler(_dev()).sample(lg, ext, w.histories, sample_indices=idx, logprobs=0)
    want, _ = R.process_rows(w.gathered().astype(np.float64), w.histories, rep=[1.2] * 8, freq=[0.1] * 8)
    assert out.tolist() == want.argmax(1).tolist() and (lp.ranks == 1).all() and lp.top_ids.shape == (8, 0)


def test_refusals():
    lg = torch.randn(2, 100, device=_dev())
    s = NS.Sampler(_dev())
    p = [EP(presence_penalty=1.0)] * 2
    with pytest.raises(IndexError):
        s.sample(lg, [EP(logit_bias={100: 1.0})] * 2, [[], []])
    with pytest.raises(IndexError):
        s.sample(lg, p, [[100], []])
    with pytest.raises(ValueError, match="prompt lengths"):
        s.sample(lg, p, [[1], []], prompt_lens=[1])
    with pytest.raises(ValueError, match="without allowed"):
        s.sample(lg, p, [[1], []], allowed_rows=torch.zeros(2, dtype=torch.int32, device=_dev()))
    with pytest.raises(ValueError, match="ids only"):
        s.sample_async(lg, p, [[1], []], logprobs=1)
    assert s.sample_async(lg, [EP(temperature=0.0, logit_bias={5: 100.0})] * 2, [[], []]).wait() == [5, 5]
