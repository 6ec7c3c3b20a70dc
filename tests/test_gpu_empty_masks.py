"""What a step draws where a mask leaves nothing that can be drawn."""
import importlib

import numpy as np
import pytest
import torch

import gpu_helpers as H
import operator_refs as R

pytestmark = pytest.mark.gpu

NS = importlib.import_module(H.PKG)
SP, EP = NS.SamplingParams, NS.ExtendedSamplingParams


def _dev():
    assert torch.cuda.is_available(), "GPU test run without a CUDA device"
    return torch.device("cuda:0")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_whose_mask_leaves_nothing_are_drawn_from_the_whole_vocabulary(dtype):
    """An empty mask, and one whose only tokens are banned by a bias, by their logits or by a NaN among them: the
    sampler's guard makes the row uniform; log-probabilities of -log(V) tell."""
    S, V = 5, 900
    x = torch.randn(S, V, device=_dev()).to(dtype)
    x[2, :2] = -np.inf
    x[3, 0] = np.nan
    few = np.zeros(V, dtype=bool)
    few[:2] = True
    allowed = torch.from_numpy(R.pack_masks([np.zeros(V, dtype=bool), few, few, few, few])).to(_dev())
    params = [SP(), EP(logit_bias={0: -np.inf, 1: -np.inf}), SP(), SP(), SP()]
    uni = torch.full((S,), 0.9, device=_dev())
    (out, dbg), lp = NS.Sampler(_dev()).sample(x, params, [[]] * S, allowed=allowed, uniforms=uni, return_debug=True, logprobs=2)
    # one division of fp32, and the sum of what fp32 holds: two half steps
    assert (dbg["probs"][:4].double() * V - 1).abs().max().item() <= 2 * 2.0**-24 * (1 + 2.0**-20)
    assert (out[:4] > V // 2).all() and out[4] < 2
    # log V rounded, and the logarithm's own step
    assert (lp.logprobs[:4].double() + np.log(V)).abs().max().item() <= 3 * 2.0**-24 * np.log(V)
    assert lp.top_ids[:4].tolist() == [[0, 1]] * 4 and lp.ranks[:4].tolist() == [1] * 4
    assert set(lp.top_ids[4].tolist()) == {0, 1}
    greedy = [EP(temperature=0.0, logit_bias=getattr(p, "logit_bias", None)) for p in params]
    x[3, 1], x[4, 0], x[4, 1] = np.nan, -1.0, np.inf
    x[3, 0] = 2.0
    out = NS.Sampler(_dev()).sample(x, greedy, [[]] * S, allowed=allowed)
    assert out.tolist() == [0, 0, 0, 1, 1]
