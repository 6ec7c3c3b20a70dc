"""Steps of requests with penalties, masks and log-probabilities: what they score, report and draw."""
import importlib

import numpy as np
import pytest
import torch

import gpu_helpers as H
import operator_refs as R

pytestmark = pytest.mark.gpu

NS = importlib.import_module(H.PKG)
W = importlib.import_module(H.PKG + ".workloads")
cabi = H.cabi
SP, EP = NS.SamplingParams, NS.ExtendedSamplingParams


def _dev():
    assert torch.cuda.is_available(), "GPU test run without a CUDA device"
    return torch.device("cuda:0")


def _scores(lp, tokens, penalized):
    """``lp`` is what the penalised logits give for ``tokens``."""
    n = lp.top_ids.shape[1]
    l, rk, ids, tl, err = R.logprob_rows(penalized.double().cpu().numpy(), tokens.tolist(), n)
    assert np.array_equal(lp.ranks.cpu().numpy(), rk) and np.array_equal(lp.top_ids.cpu().numpy(), ids)
    assert (np.abs(lp.logprobs.double().cpu().numpy() - l) <= err[:, 0]).all()
    assert (np.abs(lp.top_logprobs.double().cpu().numpy() - tl) <= err[:, 1:]).all()


def _step(S, V, dtype, seed=3):
    """Logits whose likely ids are in the histories, so that a repetition penalty moves ranks."""
    rng = np.random.default_rng(seed)
    x = W.peaked_logits(rng, S, V)
    hists = W.histories(rng, S, 1, 200, V)
    for r in range(S):
        hists[r] += [int(t) for t in np.argsort(-x[r])[:6:2]]
    uni = torch.from_numpy(rng.random(S).astype(np.float32)).to(_dev())
    return torch.from_numpy(x).to(_dev()).to(dtype), hists, uni


# -- log-probabilities ------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind", [SP, EP])
@pytest.mark.parametrize("S", [1, 5, 40])
def test_logprobs_are_those_of_the_penalised_logits(S, kind, dtype):
    """Requests with a repetition penalty and nothing else: scored on what they are drawn from, and drawn as
    without log-probabilities."""
    x, hists, uni = _step(S, 32000, dtype)
    params = [kind(temperature=0.8, repetition_penalty=1.0 if i % 4 == 3 else 1.3 + 0.1 * (i % 3)) for i in range(S)]
    s = NS.Sampler(_dev())
    (out, dbg), lp = s.sample(x, params, hists, uniforms=uni, return_debug=True, logprobs=5)
    _scores(lp, out, dbg["penalized"])
    assert torch.equal(s.sample(x, params, hists, uniforms=uni), out)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_logprobs_do_not_depend_on_the_other_requests(dtype):
    x, hists, uni = _step(3, 32000, dtype)
    params = [SP(temperature=0.8, repetition_penalty=1.4), SP(), SP()]
    s = NS.Sampler(_dev())
    a_out, a = s.sample(x, params, hists, uniforms=uni, logprobs=5)
    b_out, b = s.sample(x, params[:2] + [EP(logit_bias={7: 1.0})], hists, uniforms=uni, logprobs=5)
    assert a_out.tolist()[:2] == b_out.tolist()[:2]
    for p, q in zip(a, b):
        assert torch.equal(p[:2], q[:2])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_logprobs_of_gathered_rows(dtype):
    """The same through sample_indices, histories empty for some rows and for all."""
    x, hists, uni = _step(6, 5001, dtype)
    idx = torch.tensor([4, 1, 1, 5], device=_dev())
    params = [SP(temperature=0.9, repetition_penalty=1.5)] * 4
    s = NS.Sampler(_dev())
    for h in ([hists[i] for i in idx.tolist()], [[], hists[1], [], []], [[]] * 4):
        (out, dbg), lp = s.sample(x, params, h, sample_indices=idx, uniforms=uni[:4], return_debug=True, logprobs=3)
        _scores(lp, out, dbg["penalized"])


@pytest.mark.parametrize("kind", ["regions", "pages"])
def test_logprobs_through_the_stores(kind):
    S, V = 6, 32000
    x, hists, uni = _step(S, V, torch.float32)
    params = [SP(temperature=0.8, repetition_penalty=1.3)] * S
    st = NS.HistoryStore(_dev(), 4000, V) if kind == "regions" else NS.PagedHistoryStore(_dev(), 400, V, 16)
    handles = [st.add(h, 4) for h in hists]
    (out, dbg), lp = st.sample(NS.Sampler(_dev()), x, params, handles, uniforms=uni, return_debug=True, logprobs=4)
    _scores(lp, out, dbg["penalized"])
    assert [st.tokens(h)[-1] for h in handles] == out.tolist()
