"""process_logits with rows of very many biases."""
import importlib

import numpy as np
import pytest
import torch

import gpu_helpers as H
import operator_refs as R

pytestmark = pytest.mark.gpu

NS = importlib.import_module(H.PKG)
cabi = H.cabi
MOST = 1 << 18


def _dev():
    assert torch.cuda.is_available(), "GPU test run without a CUDA device"
    return torch.device("cuda:0")


@pytest.mark.parametrize("inplace", [False, True])
@pytest.mark.parametrize("V", [200, 20000])
def test_longer_lists_than_a_row_may_have_are_left_out(V, inplace):
    """The longest list is applied (the last entry of an id counts); one entry more, and the row has no biases."""
    rng = np.random.default_rng(V)
    ids = rng.integers(0, V, 2 * MOST + 1).astype(np.int32)
    values = rng.normal(0, 3, ids.size).astype(np.float32)
    x = torch.from_numpy(rng.normal(0, 3, (3, V)).astype(np.float32)).to(_dev())
    rows = x.double().cpu().numpy()
    off = np.array([0, MOST, 2 * MOST + 1, 2 * MOST + 1])
    st = torch.zeros(1, dtype=torch.int32, device=_dev())
    got = NS.process_logits(x, bias_offsets=torch.from_numpy(off).to(_dev()), bias_ids=torch.from_numpy(ids).to(_dev()),
                            bias_values=torch.from_numpy(values).to(_dev()), out=x if inplace else None, status=st)
    biases = [list(zip(ids[:MOST].tolist(), values[:MOST].tolist())), [], []]
    want, err = R.process_rows(rows, None, biases=biases)
    R.assert_processed(got.double().cpu().numpy(), want, err, 2.0**-24)
    assert st.item() == cabi.NS_STATUS_BAD_ROW_RANGE
