"""What a step that processes its logits reports."""
import importlib

import pytest
import torch

import gpu_helpers as H

pytestmark = pytest.mark.gpu

NS = importlib.import_module(H.PKG)
cabi = H.cabi
SP, EP = NS.SamplingParams, NS.ExtendedSamplingParams


def _dev():
    assert torch.cuda.is_available(), "GPU test run without a CUDA device"
    return torch.device("cuda:0")


def _status(params, idx, **kw):
    x = torch.randn(4, 1000, device=_dev(), generator=torch.Generator(device="cuda").manual_seed(1))
    out, dbg = NS.Sampler(_dev()).sample(x, params, [[1, 2], [3]], sample_indices=torch.tensor(idx, device=_dev()),
                                         return_debug=True, **kw)
    assert dbg["status"].shape == (1,) and dbg["status"].dtype == torch.int32
    return dbg["status"].item()


def test_a_processed_step_reports_what_a_plain_one_reports():
    plain, extended = [SP(repetition_penalty=1.2)] * 2, [EP(repetition_penalty=1.2, presence_penalty=0.1)] * 2
    for params in (plain, extended):
        assert _status(params, [0, 3]) == 0
        for bad in ([0, 4], [-1, 3]):
            assert _status(params, bad) == cabi.NS_STATUS_BAD_SAMPLE_INDEX
    masks = torch.full((2, 32), -1, dtype=torch.int32, device=_dev())
    rows = lambda *a: torch.tensor(a, dtype=torch.int32, device=_dev())  # noqa: E731
    assert _status(plain, [0, 3], allowed=masks, allowed_rows=rows(1, -1)) == 0
    assert _status(plain, [0, 3], allowed=masks, allowed_rows=rows(0, 2)) == cabi.NS_STATUS_BAD_MASK_ROW


@pytest.mark.parametrize("extended", [False, True])
def test_a_bad_page_of_a_history_is_reported(extended):
    """The gather gives -1 for the ids of a page that does not exist, and the step reports them."""
    st = NS.PagedHistoryStore(_dev(), 8, 100, 4)
    h = st.add(list(range(10)))
    st._requests[h].pages[1] = 8
    p = EP(repetition_penalty=1.2, frequency_penalty=0.1 if extended else 0.0)
    lg = torch.randn(1, 100, device=_dev())
    out, dbg = st.sample(NS.Sampler(_dev()), lg, [p], [h], append=False, return_debug=True)
    assert dbg["status"].item() == cabi.NS_STATUS_BAD_HISTORY_ID
    assert st.status.item() == cabi.NS_STATUS_BAD_POOL_RANGE
