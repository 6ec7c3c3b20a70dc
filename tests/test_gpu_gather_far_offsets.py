"""gather_paged_history with page offsets far outside the tables, near the ends of 64 bits."""
import importlib

import pytest
import torch

import gpu_helpers as H

pytestmark = pytest.mark.gpu

NS = importlib.import_module(H.PKG)
cabi = H.cabi
LAST = 2**63 - 1


def _dev():
    assert torch.cuda.is_available(), "GPU test run without a CUDA device"
    return torch.device("cuda:0")


@pytest.mark.parametrize("page", [1, 2, 3, 4, 16])
@pytest.mark.parametrize("length", [1, 40, 3000])
@pytest.mark.parametrize("first,end", [
    (5, -LAST - 1), (0, -LAST - 1), (5, -LAST), (-LAST - 1, 2), (-LAST - 1, -LAST - 1), (-LAST, LAST), (-LAST - 1, LAST),
    (LAST, -LAST - 1), (LAST, LAST), (-2**31, 8), (-2**40, 8), (8, 8), (2**40, 2**41), (LAST - 1, LAST)])
def test_ids_of_a_table_that_is_not_there_are_reported(first, end, page, length):
    """No page of the row lies in the table: every id is -1, and the rows around it keep theirs."""
    pool = torch.arange(8 * page, dtype=torch.int32, device=_dev()).view(8, page)
    table = torch.arange(8, dtype=torch.int32, device=_dev())
    i64 = dict(dtype=torch.int64, device=_dev())
    st = torch.zeros(1, dtype=torch.int32, device=_dev())
    # the row alone, and as one of two, whose other row's table begins where this one's ends
    for po, ho in (([first, end], [0, length]), ([first, end, 8], [0, length, length])):
        out = torch.full((length + 3,), -7, dtype=torch.int32, device=_dev())
        st.zero_()
        NS.gather_paged_history(pool, table, torch.tensor(po, **i64), torch.tensor(ho, **i64), out=out, status=st)
        assert out.tolist() == [-1] * length + [-7] * 3
        assert st.item() == cabi.NS_STATUS_BAD_POOL_RANGE


@pytest.mark.parametrize("page", [1, 3, 4])
def test_history_offsets_far_away(page):
    """History offsets that leave the array on either side: reported, and nothing written outside."""
    pool = torch.arange(8 * page, dtype=torch.int32, device=_dev()).view(8, page)
    table = torch.arange(8, dtype=torch.int32, device=_dev())
    i64 = dict(dtype=torch.int64, device=_dev())
    st = torch.zeros(1, dtype=torch.int32, device=_dev())
    for ho in ([0, LAST], [-LAST - 1, 4], [-LAST - 1, LAST], [4, -LAST - 1], [LAST, 4], [LAST, LAST], [-5, 4]):
        out = torch.full((9,), -7, dtype=torch.int32, device=_dev())
        st.zero_()
        NS.gather_paged_history(pool, table, torch.tensor([0, 8], **i64), torch.tensor(ho, **i64), out=out[:6], status=st)
        assert st.item() == cabi.NS_STATUS_BAD_POOL_RANGE and out[6:].tolist() == [-7] * 3
        assert set(out[:6].tolist()) <= {-7, -1, *range(8 * page)}


@pytest.mark.parametrize("page", [256, 300])
def test_a_table_that_begins_before_a_long_array(page):
    """The row's first page lies before the array, and the array is longer than 2^32 ids have pages."""
    pool = torch.arange(2 * page, dtype=torch.int32, device=_dev()).view(2, page)
    n = 2**32 // page + 9
    st = torch.zeros(1, dtype=torch.int32, device=_dev())
    out = torch.full((page + 50,), -7, dtype=torch.int32, device=_dev())
    NS.gather_paged_history(pool, torch.ones(n, dtype=torch.int32, device=_dev()), torch.tensor([-1, n], device=_dev()),
                            torch.tensor([0, page + 40], device=_dev()), out=out, status=st)
    assert out.tolist() == [-1] * page + list(range(page, page + 40)) + [-7] * 10
    assert st.item() == cabi.NS_STATUS_BAD_POOL_RANGE
