"""Attention over the paged K/V cache where its kernels for many columns differ from each other, and with its keys cut
into as many parts as there are, against the plain form; tolerances as in test_gpu_paged.py.

At head dim 64 a request of more than 1024 columns (rows times heads of a K/V head), not causal or with more than 2048
keys times that group, has two column tiles a wave, whose steps take turns."""

from __future__ import annotations

import itertools

import pytest
import torch

from oracle import paged
from turbo_roformer_amd import _hip

from .test_gpu_paged import BF, DEV, HF, _attn_case, _attn_close, _run_attn, _say
from .test_gpu_paged_nan import _set_rows, _slot

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", (BF, HF))
@pytest.mark.parametrize("causal,window", [(True, 0), (True, 700), (True, 899), (False, 0), (False, 3), (False, 650)])
def test_two_column_tiles_masks(hip, dtype, causal, window):
    for page, lens, new in ((16, [900], [600]), (64, [613, 900, 30], [600, 260, 30])):
        c = _attn_case(lens, new, 4, 1, 64, page, dtype, window + 5, padding=3)
        gate = torch.rand(c["q"].shape[0], 4, generator=torch.Generator().manual_seed(2))
        _say("two column tiles", dtype, causal, window, page)
        _attn_close(_run_attn(c, gate=gate, causal=causal, window=window, max_new=max(new), max_len=max(lens)), c, gate=gate,
                    causal=causal, window=window)


@pytest.mark.parametrize("dtype", (BF, HF))
def test_two_column_tiles_scores_that_rise_late(hip, dtype):
    """Keys tens and hundreds above all earlier ones, for all columns and for those of one tile of a wave only: one tile's
    maximum is raised while the other's P is still to be applied."""
    for only in (None, 0, 1):
        c = _attn_case([900], [600], 4, 1, 64, 64, dtype, 22)
        k = paged.k_rows(c["K"]).clone()
        for i, at in enumerate((100, 267, 301, 431, 690, 820)):
            k[_slot(c, 0, at)] = 0.0
            k[_slot(c, 0, at), 0, 0] = 20.0 * (i + 1)
        _set_rows(c, k)
        c["q"][..., 0] = 3.0
        if only is not None:  # columns are 4 row + head: rows of 8 are a tile of 32
            c["q"][torch.arange(600) // 8 % 2 == 1 - only, :, 0] = -1.0
        _say("late rise", dtype, only)
        for causal in (True, False):
            _attn_close(_run_attn(c, scale=1.0, causal=causal), c, scale=1.0, causal=causal)


@pytest.mark.parametrize("dtype", (BF, HF))
@pytest.mark.parametrize("causal,window", [(True, 0), (True, 700), (False, 0)])
def test_two_column_tiles_skip_table_entries_that_are_no_pages(hip, dtype, causal, window):
    c = _attn_case([900], [600], 4, 1, 64, 16, dtype, 8)
    for at, entry in ((0, -1), (3, 2**31 - 1), (18, -7), (30, c["K"].shape[0]), (55, -(2**31))):
        c["table"][0, at] = entry
    _attn_close(_run_attn(c, causal=causal, window=window), c, causal=causal, window=window)
    c["table"][:] = -1
    assert bool((_run_attn(c, causal=causal, window=window) == 0).all())


@pytest.mark.parametrize("dtype", (BF, HF))
@pytest.mark.parametrize("causal,window", [(True, 0), (True, 700), (False, 650)])
def test_two_column_tiles_unseen_infinities_and_nan_change_nothing(hip, dtype, causal, window):
    """NaN and infinities wherever no row looks, and in V at positions that some columns of a tile see and others do not."""
    c = _attn_case([900], [600], 4, 1, 64, 32, dtype, 12)
    key = torch.arange(900)
    held = torch.zeros(c["K"].shape[0] * 32, dtype=torch.bool)
    held[c["table"][0, key // 32].long() * 32 + key % 32] = True
    k, v = paged.k_rows(c["K"]).clone(), paged.v_rows(c["V"]).clone()
    k[~held], v[~held] = float("nan"), float("inf")
    v[~held, :, 1::2] = float("nan")
    for at, value in ((133, float("nan")), (310, float("inf")), (583, float("-inf")), (890, float("nan"))):
        v[_slot(c, 0, at), 0, at % 64] = value
    _set_rows(c, k, v)
    got = _run_attn(c, causal=causal, window=window)
    _attn_close(got, c, causal=causal, window=window)
    assert bool(got.isfinite().any(-1).all())


@pytest.mark.parametrize("dtype,D", itertools.product((BF, HF), (64, 128)))
@pytest.mark.parametrize("lens,new,heads,page", [([20_001], [1], 2, 16), ([9_000, 40_000], [1, 1], 1, 256), ([17_011], [20], 2, 64),
                                                 ([8_300], [70], 1, 32)])
def test_thirty_two_parts(hip, dtype, D, lens, new, heads, page):
    """Keys cut into as many parts as there are at most."""
    c = _attn_case(lens, new, heads, 1, D, page, dtype, 15)
    need = _hip.paged_attention_workspace_bytes(heads, c["K"], c["V"], *c["table"].shape, sum(new), max(new), max(lens))
    assert need == 32 * sum(new) * heads * (D + 2) * 4
    _say("32 parts", dtype, D, lens, new)
    _attn_close(_run_attn(c, max_new=max(new), max_len=max(lens)), c)



@pytest.mark.parametrize("D", (64, 128))
def test_entries_that_are_no_pages_in_some_of_the_parts(hip, D):
    """Each part of the keys looks at the table entries of its own keys: the first, one in the middle, the last."""
    for entries in ((0,), (300,), (518,), (0, 255, 256, 518)):
        c = _attn_case([8_300], [70], 1, 1, D, 16, BF, 16)
        c["table"][0, list(entries)] = -1
        _attn_close(_run_attn(c, max_new=70, max_len=8_300), c)


@pytest.mark.parametrize("D", (64, 128))
@pytest.mark.parametrize("lens,new,heads", [([90, 40], [3, 1], 4), ([3000], [1], 8), ([500, 90], [200, 90], 1), ([2000], [60], 1),
                                            ([700], [400], 4)])
def test_attention_in_place_of_its_queries(hip, D, lens, new, heads):
    c = _attn_case(lens, new, heads, 1, D, 16, BF, 18, padding=2)
    d = {k: v.to(DEV) for k, v in c.items()}
    n = c["q"].shape[0]
    want = torch.cat((_run_attn(c, max_new=max(new))[:-2], c["q"][-2:]))
    _hip.paged_attention(**d, O=d["q"].view(n, heads * D), max_new=max(new))
    torch.cuda.synchronize()
    assert torch.equal(d["q"].cpu(), want)
