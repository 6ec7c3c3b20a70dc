"""The most that a list of page copies may move (checked on the host)."""
import pytest

from conftest import pkg

cabi = pkg("_cabi")


@pytest.mark.parametrize("page_bytes,count", [(2**31 - 1, 2**31 - 1), (2**30, 2**11 + 1), (2**31 - 1, 2**10 + 1)])
def test_lists_of_more_bytes_than_a_launch_has_blocks_for_are_refused(page_bytes, count):
    """The blocks of a launch are counted in 31 bits; a larger count would be cut off, and with it the copies."""
    with pytest.raises(cabi.NsError, match="2\\^41 bytes"):
        cabi.ns_pages_copy_listed([(64, 16, 16), (64, page_bytes, page_bytes)], 1 << 20, 64, 64, count)


@pytest.mark.gpu
def test_a_pool_that_is_named_twice():
    import torch

    p = torch.randn(64, 32768, device="cuda:0")
    want = p.clone()
    want[32:] = want[:32]
    pkg().copy_pages([p, p], list(range(32)), list(range(32, 64)))
    assert torch.equal(p, want)
