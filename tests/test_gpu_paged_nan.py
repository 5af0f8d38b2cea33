"""NaN and infinities in one column of the paged attention's products (a row of a head) reach no other column."""

from __future__ import annotations

import itertools

import pytest
import torch

from oracle import paged

from .test_gpu_paged import BF, HF, _attn_case, _run_attn

pytestmark = pytest.mark.gpu


def _set_rows(c, k=None, v=None):
    """Rows [slot, heads, D] laid out as the cache."""
    P, kv, groups, chunks = c["K"].shape[:4]
    page, D = 16 * groups, 8 * chunks
    if k is not None:
        c["K"] = k.view(P, groups, 16, kv, chunks, 8).permute(0, 3, 1, 4, 2, 5).contiguous()
    if v is not None:
        c["V"] = v.view(P, page // 8, 8, kv, D).permute(0, 3, 1, 4, 2).contiguous()


def _slot(c, r, position):
    page = 16 * c["K"].shape[2]
    return int(c["table"][r, position // page]) * page + position % page


@pytest.mark.parametrize("dtype,D", itertools.product((BF, HF), (64, 128)))
@pytest.mark.parametrize("lens,new,heads", [([90], [1], 32), ([90], [32], 1), ([3000], [1], 32), ([90], [80], 1),
                                            ([1200], [1100], 1), ([2100], [1100], 1)])
def test_a_nan_in_one_column_stays_in_it(hip, dtype, D, lens, new, heads):
    """q of one column NaN, for every place that a column can have in its tile: its row and head, and no other."""
    c = _attn_case(lens, new, heads, 1, D, 16, dtype, 14)
    q = c["q"]
    clean = _run_attn(c, max_new=max(new), causal=False)
    for at in range(32) if new[0] * heads <= 32 else (0, 1, 15, 16, 17, 31, 32, 33, 47, 48, 63, 64):
        c["q"] = q.clone()
        c["q"].view(-1, D)[at, 5] = float("nan")
        got = _run_attn(c, max_new=max(new), causal=False).view(-1, D)
        assert bool(got[at].isnan().all()), at
        got[at] = clean.view(-1, D)[at]
        assert torch.equal(got, clean.view(-1, D)), at


@pytest.mark.parametrize("dtype,D", itertools.product((BF, HF), (64, 128)))
@pytest.mark.parametrize("lens,new", [([90], [32]), ([90], [80]), ([1200], [1100]), ([2100], [1100])])
@pytest.mark.parametrize("value", (float("nan"), float("inf")))
def test_rows_that_do_not_see_a_nan_or_infinite_key_keep_their_bits(hip, dtype, D, lens, new, value):
    c = _attn_case(lens, new, 1, 1, D, 16, dtype, 17)
    c["q"] = c["q"].abs() + 0.1
    clean = _run_attn(c, max_new=max(new))
    k = paged.k_rows(c["K"])
    for at in (lens[0] - new[0] + i for i in (1, 9, 17, 30, new[0] - 1)):
        bad = k.clone()
        bad[_slot(c, 0, at), 0, 3] = value
        x = dict(c)
        _set_rows(x, bad)
        got = _run_attn(x, max_new=max(new))
        sees = torch.arange(lens[0] - new[0], lens[0]) >= at
        assert bool(got[sees].isnan().all()) and torch.equal(got[~sees], clean[~sees]), at
