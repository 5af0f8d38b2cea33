"""HipPagedCache at the limits that its caller sets."""

from __future__ import annotations

import pytest
import torch

from oracle import paged
from turbo_roformer_amd import _hip
from turbo_roformer_amd.paged import HipPagedCache

from .test_gpu_paged import BF, _attn_close, _ints, _pages, _Plain, _rope, _same, _say

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("longest,page", [(70, 16), (70, 64), (64, 64), (1, 256)])
def test_a_request_ends_at_max_length(hip, longest, page):
    """A length between max_length and the end of its last page is refused, and a table of angles of max_length is enough:
    every row that the plan accepts is written."""
    R, heads, kv, D = 3, 2, 1, 64
    cache = HipPagedCache(R, longest, kv, D, page_size=page)
    cache.K.fill_(float("nan")), cache.V.fill_(float("nan"))
    plain, rope = _Plain(R), _rope(longest, D)
    g = torch.Generator().manual_seed(longest)
    lens = [0] * R
    for new in ([longest - 1, longest, longest + 1], [1, 1, longest], [0, 0, 1], [2, -1, 0]):
        want = [n + max(m, 0) if n + max(m, 0) <= longest else n for n, m in zip(lens, new)]
        rows = sum(max(m, 0) for m in new) + 1
        qkv = torch.randn(rows, heads + 2 * kv, D, generator=g).to(BF)
        dev = qkv.to(DEV)
        _say("max_length", longest, page, new)
        step = cache.plan(_ints(new).to(DEV), rows)
        q = cache.append(step, dev[:, :heads], dev[:, heads:heads + kv], dev[:, heads + kv:], rope.to(DEV))
        O = torch.full((rows, heads * D), 7.0, dtype=BF, device=DEV)
        cache.attend(step, q, out=O)
        torch.cuda.synchronize()
        assert cache.lengths.tolist() == want
        assert cache.refused == sum(m > 0 and n == w for n, m, w in zip(lens, new, want))
        K, V = paged.k_rows(cache.K.cpu()), paged.v_rows(cache.V.cpu())
        at, live = 0, torch.zeros(rows, dtype=torch.bool)
        for r, m in enumerate(new):
            m = max(m, 0)
            if want[r] == lens[r] + m:
                live[at:at + m] = True
                plain.k[r] += list(K[step.slots[at:at + m].long().cpu()])
                plain.v[r] += list(V[step.slots[at:at + m].long().cpu()])
                assert torch.equal(torch.stack(plain.v[r][-m:]) if m else qkv[:0, 0], qkv[at:at + m, heads + kv:] if m else qkv[:0, 0])
            at += m
        lens = want
        if bool(live.any()):
            starts = torch.tensor([0] + [int(live[:int(s)].sum()) for s in step.starts[1:]])
            c = dict(plain.dense(kv, D, BF), q=q.cpu()[live], starts=starts)
            assert bool(c["K"].isfinite().all())
            _attn_close(O.cpu().view(rows, heads, D)[live], c)


def test_a_table_of_angles_that_ends_before_max_length_is_refused(hip):
    cache = HipPagedCache(2, 70, 1, 64, page_size=16)
    step = cache.plan(_ints([3, 1]).to(DEV), 4)
    k = torch.zeros(4, 1, 64, dtype=BF, device=DEV)
    with pytest.raises(ValueError, match="69 positions.*70"):
        cache.append(step, None, k, k, _rope(69, 64).to(DEV))
    cache.append(step, None, k, k, _rope(70, 64).to(DEV))


@pytest.mark.parametrize("R,page,most", [(5, 16, 40), (62, 64, 700), (1025, 32, 33)])
def test_plan_within_a_length(hip, R, page, most):
    g = torch.Generator().manual_seed(R)
    lens = torch.randint(0, most + 1, (R,), generator=g).tolist()
    new = torch.randint(0, most // 2 + 1, (R,), generator=g)
    lens[1], new[1] = most + 3, 0  # longer than it may be, no more rows
    lens[2], new[2] = most + 3, 1
    table, pool, state = _pages(lens, page, -(-2 * most // page) + 1, 3 * R, R)
    n_rows = int(new.sum())
    for longest in (1, most - 1, most, table.shape[1] * page, None):
        dev = [t.to(DEV) for t in (state, new.int(), pool, table)]
        out = [torch.full((n,), -99, dtype=torch.int32, device=DEV) for n in (2 + R, R + 1, n_rows, n_rows)]
        _say("plan within", R, page, longest)
        _hip.page_plan(*dev, page, *out, max_length=longest)
        torch.cuda.synchronize()
        _same(dict(zip(("state_out", "starts", "slots", "positions"), (t.cpu() for t in out)), table=dev[3].cpu()),
              paged.plan(state, new, pool, table, page, n_rows, longest))
    for longest in (-1, table.shape[1] * page + 1):
        with pytest.raises(RuntimeError, match="max_length"):
            _hip.page_plan(*dev, page, *out, max_length=longest)


def test_refused_is_the_last_plans_after_a_release(hip):
    """A step reads it at its end, where it can wait for the device."""
    cache = HipPagedCache(3, 64, 1, 64, pages=3, page_size=16)
    assert cache.refused == 0
    cache.plan(_ints([16, 20, 5]).to(DEV), 41)
    cache.release(torch.tensor([True, False, False], device=DEV))
    assert cache.refused == 1 and cache.lengths.tolist() == [0, 20, 0] and cache.free_pages == 1
    cache.release(torch.tensor([False, True, False], device=DEV))
    assert cache.refused == 1 and cache.lengths.tolist() == [0, 0, 0] and cache.free_pages == 3
    cache.plan(_ints([0, 0, 5]).to(DEV), 5)
    assert cache.refused == 0
