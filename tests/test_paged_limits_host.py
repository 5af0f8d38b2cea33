"""Arguments of the paged K/V cache's C functions at the ends of their ranges, refused before any launch."""

from __future__ import annotations

import pytest

from turbo_roformer_amd import _hip

from .test_paged_host import _append, _attend, _p


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


@pytest.mark.parametrize("kw", [dict(rows=(1 << 24) - 1, heads=8, kv=8, qs=1024, ks=1024, vs=1024, q=_p(1 << 16), q_out=_p(1 << 45)),
                                dict(rows=(1 << 27) - 1, q=None, kv=2, ks=256, vs=256), dict(rows=(1 << 28) - 1, q=None, kv=1, ks=128, vs=128)])
def test_append_refuses_more_workgroups_than_a_launch_numbers(lib, kw):
    """256 threads for each 16 rows and head, all of them in 32 bits."""
    assert _append(lib, dim=128, **kw) == 1
    assert b"n_rows" in lib.trf_last_error()
