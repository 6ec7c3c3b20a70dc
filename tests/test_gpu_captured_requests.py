"""Extended requests in a captured step: process_logits, then sample_packed of what is left of the requests."""
import importlib

import numpy as np
import pytest
import torch

import gpu_helpers as H

pytestmark = pytest.mark.gpu

NS = importlib.import_module(H.PKG)
W = importlib.import_module(H.PKG + ".workloads")
SP, EP = NS.SamplingParams, NS.ExtendedSamplingParams
upload_packed = importlib.import_module(H.PKG + ".sampler").upload_packed


def _dev():
    assert torch.cuda.is_available(), "GPU test run without a CUDA device"
    return torch.device("cuda:0")


@pytest.mark.parametrize("S", [6, 48])
def test_a_captured_step_draws_what_sample_draws(S):
    rng = np.random.default_rng(S)
    V = 32000
    params = [EP(temperature=p.temperature, top_k=p.top_k, top_p=p.top_p, repetition_penalty=p.repetition_penalty,
                 presence_penalty=0.5, logit_bias={7: 3.0, i: -np.inf}) for i, p in enumerate(W.mixed_params(S))]
    hists = W.histories(rng, S, 0, 60, V)
    uni = torch.from_numpy(rng.random(S).astype(np.float32)).to(_dev())
    lg = torch.zeros(S, V, device=_dev())
    pr = H.packing.pack_processing(params, [len(h) for h in hists], None, V)
    ids = H.packing.flatten_histories(hists, pr.lens, V)
    d = lambda a: torch.from_numpy(a).to(_dev())  # noqa: E731
    given = dict(history_offsets=d(pr.offsets), history_ids=d(ids), repetition_penalty=d(pr.repetition),
                 presence_penalty=d(pr.presence), frequency_penalty=d(pr.frequency), bias_offsets=d(pr.bias_offsets),
                 bias_ids=d(pr.bias_ids), bias_values=d(pr.bias_values))
    # what is left of the requests when process_logits has applied its part
    left = [SP(temperature=p.temperature, top_k=p.top_k, top_p=p.top_p) for p in params]
    rp, off, hid, order = upload_packed(H.packing.pack(left, [[]] * S, V, sms=148), _dev())
    s = NS.Sampler(_dev())

    def step():
        return s.sample_packed(NS.process_logits(lg, **given), rp, off, hid, uniforms=uni, row_order=order)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        out = step()
    for _ in range(2):
        lg.copy_(torch.from_numpy(W.peaked_logits(rng, S, V)))
        g.replay()
        torch.cuda.synchronize()
        assert out.tolist() == NS.Sampler(_dev()).sample(lg, params, hists, uniforms=uni).tolist()
