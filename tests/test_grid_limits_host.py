"""Calls whose launch would hold 2^32 threads or more are refused on the host."""

import pytest

from test_more_operators_host import select
from turbopolar_amd import _lib


@pytest.mark.parametrize("pages", [2 ** 28, 2 ** 29, 2 ** 30 - 1])
def test_pages_of_a_selection(pages):
    st, text = select(n=pages, cap=pages, count=5, wsb=2 ** 40)
    assert st == _lib.TP_ERR_INVALID and "n_pages" in text, (st, text)
