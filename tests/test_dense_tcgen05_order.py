"""The ordering rules of tests/test_tcgen05_order.py on the sources of the dense attention's tcgen05 kernels."""
import pytest

from tests import test_tcgen05_order as order

SOURCES = ["dense_tc.cu", "dense_bwd_tc.cu"]


@pytest.mark.parametrize("name", SOURCES)
def test_every_tcgen05_access_behind_a_wait_is_fenced(name):
    assert order._unfenced(order._source(name)) == []


@pytest.mark.parametrize("name", SOURCES)
def test_a_reported_code_names_one_barrier(name):
    codes = order._codes_of_waits(order._source(name))
    assert len(codes) > 15
    assert {c: b for c, b in codes.items() if len(b) > 1} == {}
