"""A copy that fails leaves a PagedHistoryStore as it was."""
import importlib

import pytest
import torch

import gpu_helpers as H

pytestmark = pytest.mark.gpu

NS = importlib.import_module(H.PKG)
pages = importlib.import_module(H.PKG + ".pages")


def _dev():
    assert torch.cuda.is_available(), "GPU test run without a CUDA device"
    return torch.device("cuda:0")


def _fails(*args):
    raise RuntimeError("no copy")


def test_pages_are_given_back_where_a_copy_fails(monkeypatch):
    st = NS.PagedHistoryStore(_dev(), 12, 100, 4)
    a = st.add(list(range(10)))  # three pages
    b, = st.fork(a)              # shares two, owns one
    own = st.pages(b)
    with monkeypatch.context() as m:
        m.setattr(pages, "copy_pages", _fails)
        with pytest.raises(RuntimeError, match="no copy"):
            st.fork(a, 3)
        assert st.free_pages() == 8
        with pytest.raises(RuntimeError, match="no copy"):
            st.truncate(b, 6)  # into a shared page; the page behind it would become the copy
        assert st.free_pages() == 8 and st.pages(b) == own and st.length(b) == 10
        st.truncate(b, 8)
        with pytest.raises(RuntimeError, match="no copy"):
            st.truncate(b, 6)  # a free page would
        assert st.free_pages() == 9 and st.pages(b) == own[:2] and st.length(b) == 8
    with monkeypatch.context() as m:
        m.setattr(pages.torch, "from_numpy", _fails)
        with pytest.raises(RuntimeError, match="no copy"):
            st.add(list(range(9)), 7)
    assert st.free_pages() == 9 and st.tokens(a) == list(range(10)) and st.tokens(b) == list(range(8))
    c = st.add(list(range(36)))
    assert st.free_pages() == 0 and st.tokens(c) == list(range(36))
    for h in (a, b, c):
        st.release(h)
    assert st.free_pages() == 12
