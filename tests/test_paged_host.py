"""The C ABI of the paged K/V cache refuses what it cannot run before touching the device."""

from __future__ import annotations

import ctypes

import pytest
import torch

from oracle import paged
from turbo_roformer_amd import _hip

BIG = 1 << 20


@pytest.fixture(scope="module")
def lib():
    return _hip.open_library()


def _p(at: int = 256):
    return ctypes.c_void_p(at)


def _plan(lib, **kw):
    a = dict(state=_p(256), n_new=_p(), R=4, rows=8, pool=_p(), pages=16, page=64, table=_p(), max_pages=4, out=_p(4096),
             starts=_p(), slots=_p(), positions=_p())
    a.update(kw)
    return lib.trf_page_plan(*a.values(), None)


def _release(lib, **kw):
    a = dict(state=_p(256), done=_p(), R=4, pool=_p(), pages=16, page=64, table=_p(), max_pages=4, out=_p(4096))
    a.update(kw)
    return lib.trf_page_release(*a.values(), None)


def _append(lib, **kw):
    a = dict(q=_p(1 << 16), qs=512, heads=8, k=_p(), ks=512, v=_p(), vs=512, dtype=1, rows=8, slots=_p(), positions=_p(),
             rope=_p(), P=100, K=_p(), V=_p(), pages=16, page=64, kv=8, dim=64, q_out=_p(1 << 18))
    a.update(kw)
    return lib.trf_paged_append(*a.values(), None)


def _attend(lib, **kw):
    a = dict(q=_p(), qs=512, heads=8, K=_p(), V=_p(), dtype=1, pages=16, page=64, kv=8, dim=64, table=_p(), max_pages=4,
             starts=_p(), lens=_p(), R=4, rows=8, max_new=2, max_len=256, scale=0.125, causal=1, window=0, gate=None, O=_p(),
             ws=None, ws_bytes=0)
    a.update(kw)
    return lib.trf_paged_attention(*a.values(), None)


@pytest.mark.parametrize("kw,word", [
    (dict(page=48), b"page_size"), (dict(page=512), b"page_size"), (dict(page=8), b"page_size"),
    (dict(pages=0), b"n_pages"), (dict(pages=1 << 25), b"n_pages"), (dict(R=0), b"n_requests"),
    (dict(R=8193), b"n_requests"), (dict(R=8192, max_pages=1 << 18), b"n_requests"), (dict(max_pages=0), b"max_pages"),
    (dict(max_pages=(1 << 24) + 1, R=1), b"max_pages"), (dict(out=_p(256)), b"overlap"), (dict(out=_p(256 + 20)), b"overlap"),
    (dict(state=_p(257)), b"aligned"), (dict(state=None), b"state"), (dict(pool=None), b"pool"), (dict(table=None), b"table"),
])
def test_plan_and_release_refuse(lib, kw, word):
    for call in (_plan, _release):
        assert call(lib, **kw) == 1, call
        assert word in lib.trf_last_error()


@pytest.mark.parametrize("call,kw,word", [
    (_plan, dict(rows=-1), b"n_rows"), (_plan, dict(rows=1 << 30), b"n_rows"), (_plan, dict(n_new=None), b"n_new"),
    (_plan, dict(starts=None), b"starts"), (_plan, dict(slots=None), b"slots"), (_plan, dict(positions=_p(2)), b"positions"),
    (_release, dict(done=None), b"done"),
    (_append, dict(dtype=0), b"dtype"), (_append, dict(dim=96), b"head_dim"), (_append, dict(kv=0), b"kv_heads"),
    (_append, dict(heads=0), b"heads"), (_append, dict(rows=-1), b"n_rows"), (_append, dict(rows=1 << 24), b"n_rows"),
    (_append, dict(k=None), b"k must"), (_append, dict(ks=516), b"multiple of 8"), (_append, dict(vs=504), b"fewer than"),
    (_append, dict(ks=0), b"fewer than"), (_append, dict(qs=256), b"fewer than"), (_append, dict(v=_p(8)), b"aligned"),
    (_append, dict(slots=None), b"slots"), (_append, dict(positions=None), b"positions"), (_append, dict(P=0), b"rope_len"),
    (_append, dict(q_out=None), b"q_out"), (_append, dict(q_out=_p((1 << 16) + 1024)), b"overlap"),
    (_append, dict(q_out=_p(1 << 16), qs=1536), b"overlap"), (_append, dict(K=_p(264)), b"K must"),
    (_append, dict(page=24), b"page_size"),
    (_attend, dict(dtype=3), b"dtype"), (_attend, dict(heads=12), b"multiple of kv_heads"), (_attend, dict(heads=0), b"heads"),
    (_attend, dict(dim=32), b"head_dim"), (_attend, dict(scale=0.0), b"scale"), (_attend, dict(scale=-1.0), b"scale"),
    (_attend, dict(scale=float("nan")), b"scale"), (_attend, dict(scale=float("inf")), b"scale"),
    (_attend, dict(window=-1), b"window"), (_attend, dict(causal=2), b"causal"), (_attend, dict(max_new=-1), b"max_new"),
    (_attend, dict(max_len=-1), b"max_len"), (_attend, dict(rows=1 << 28), b"n_rows"), (_attend, dict(q=None), b"q must"),
    (_attend, dict(qs=500), b"multiple of 8"), (_attend, dict(O=_p(8)), b"O must"), (_attend, dict(table=None), b"table"),
    (_attend, dict(lens=_p(2)), b"lens"), (_attend, dict(R=1 << 21), b"too many"), (_attend, dict(gate=_p(2)), b"gate"),
])
def test_refusals(lib, call, kw, word):
    assert call(lib, **kw) == 1
    assert word in lib.trf_last_error()


def test_nothing_to_do(lib):
    assert _append(lib, rows=0, k=None, v=None, slots=None) == 0
    assert _attend(lib, rows=0, q=None, O=None) == 0
    assert _attend(lib, max_new=0, q=None, O=None) == 0


def test_a_cache_is_refused_before_it_is_made():
    for kw, word in ((dict(page_size=20), "page_size"), (dict(head_dim=80), "head_dim"), (dict(dtype=torch.float32), "dtype")):
        with pytest.raises(ValueError, match=word):
            _hip.paged_cache(**{**dict(pages=4, page_size=16, kv_heads=1, head_dim=64, device="cpu"), **kw})
    K, V = _hip.paged_cache(3, 32, 2, 128, torch.float16, "cpu")
    assert K.shape == (3, 2, 2, 16, 16, 8) and V.shape == (3, 2, 4, 128, 8)
    assert _hip._cache(K, V) == (2, 3, 32, 2, 128)
    for bad in ((K, V[:2]), (K.float(), V), (K, V.to(torch.bfloat16)), (K.transpose(0, 1), V)):
        with pytest.raises(ValueError):
            _hip._cache(*bad)


def test_the_module_refuses_before_any_launch(lib):
    """Arguments that are no tensors, not on the device, of the wrong number; an address that is none."""
    native = _hip.bind_native(lib)
    with pytest.raises(ValueError, match="address"):
        native.bind(1, 2, 0, 4)
    with pytest.raises(TypeError, match="4 functions"):
        native.bind(1)
    ints = torch.zeros(8, dtype=torch.int32)
    table = ints.view(2, 4)
    for args, error, word in (
        ((0, 0, ints, ints, ints, table, 16, ints), TypeError, "expected 11 arguments, got 8"),
        ((0, 0, 5, ints, ints, table, 16, ints, ints, ints, ints), TypeError, "state must be a tensor, got int"),
        ((0, 0, None, ints, ints, table, 16, ints, ints, ints, ints), TypeError, "state must be a tensor, got NoneType"),
        ((0, 0, ints, ints, ints, table, 16, ints, ints, ints, ints), ValueError, "state is on cpu"),
        (("x", 0, ints, ints, ints, table, 16, ints, ints, ints, ints), TypeError, "int"),
    ):
        with pytest.raises(error, match=word):
            native.page_plan(*args)


def test_oracle_layouts_and_softmax():
    """The oracle's row views invert the layouts of the header, and its attention is torch's on one request."""
    K, V = _hip.paged_cache(3, 32, 2, 64, torch.float16, "cpu")
    g = torch.Generator().manual_seed(0)
    K.copy_(torch.randn(K.shape, generator=g))
    V.copy_(torch.randn(V.shape, generator=g))
    slot, h, d = 2 * 32 + 21, 1, 43
    assert paged.k_rows(K)[slot, h, d] == K[2, h, 21 // 16, d // 8, 21 % 16, d % 8]
    assert paged.v_rows(V)[slot, h, d] == V[2, h, 21 // 8, d, 21 % 8]
    table = torch.tensor([[2, 0]], dtype=torch.int32)
    q = torch.randn(5, 4, 64, generator=g)
    O, _, size = paged.attention(q, K, V, table, torch.tensor([0, 5]), torch.tensor([40]))
    at = torch.cat((torch.arange(64, 96), torch.arange(0, 8)))
    k, v = (rows(x)[at].double().repeat_interleave(2, 1) for rows, x in ((paged.k_rows, K), (paged.v_rows, V)))
    s = torch.einsum("nhd,khd->hnk", q.double(), k) / 8
    s[:, torch.arange(40)[None, :] > torch.arange(35, 40)[:, None]] = -float("inf")
    torch.testing.assert_close(O, torch.einsum("hnk,khd->nhd", s.softmax(-1), v))
    assert size[:, 0, 0].tolist() == [36, 37, 38, 39, 40]
