"""Arguments of the paged K/V cache's C functions at the ends of their ranges, refused before any launch."""

from __future__ import annotations

import pytest

from turbo_roformer_amd import _hip

from .test_paged_host import _attend, _p


@pytest.fixture(scope="module")
def lib():
    return _hip.open_library()


@pytest.mark.parametrize("max_length", (-1, 0, 257, 2**31 - 1))
def test_a_plan_is_no_longer_than_its_table(lib, max_length):
    assert lib.trf_page_plan_limited(_p(256), _p(), 4, 8, _p(), 16, 64, _p(), 4, max_length, _p(4096), _p(), _p(), _p(), None) == 1
    assert b"max_length must be 1..256" in lib.trf_last_error()


@pytest.mark.parametrize("at,stride", [((1 << 16) + 16, 512), ((1 << 16) - 8 * 512 * 2 + 16, 512), (1 << 16, 520), ((1 << 16) + 1024, 1024)])
def test_attention_refuses_an_output_across_its_queries(lib, at, stride):
    """Eight rows of 512 elements at 2^16: another workgroup's rows of O would be read as q."""
    assert _attend(lib, q=_p(1 << 16), qs=stride, O=_p(at)) == 1
    assert b"O must not overlap q" in lib.trf_last_error()
