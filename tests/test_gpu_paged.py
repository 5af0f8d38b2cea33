"""The paged K/V cache on the GPU against its plain form (oracle/paged.py): pages dealt and taken back, rows written,
attention of new rows over the pages, and runs of them together.

Tolerances.  Page numbers, slots, positions, lengths and V's bits are equal.  A rotated value has one rounding to its
type, half a step, after fp32 products and a sum (2^-22 of the pair's size covers three roundings of 2^-24).  Attention:
with weights w and u = half a step of the type, the output's rounding is u |O|; P = 2^(s - m) is rounded by u of itself,
which is u sum(w |v|); the fp32 scores, sums and exponentials add e = 2^-24 (keys + 4 D max(scale sum |q| |k|) + 64) of
sum(w |v|).  fp16 is subnormal below 2^-14: P is then off by up to 2^-25 of the largest P, in all by
2^-25 keys max|v|, the output by 2^-25."""

from __future__ import annotations

import itertools

import pytest
import torch

from oracle import paged
from turbo_roformer_amd import _hip
from turbo_roformer_amd.paged import HipPagedCache

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, HF = torch.bfloat16, torch.float16


def _ints(x) -> torch.Tensor:
    return torch.tensor(list(x), dtype=torch.int32)


def _say(*what) -> None:
    print(*what, flush=True)


# ---------------------------------------------------------------------------------------------- plan and release


def _pages(lens, page, max_pages, spare, seed):
    """Table, pool and state with these lengths, pages dealt at random, `spare` free."""
    g = torch.Generator().manual_seed(seed)
    have = [-(-n // page) for n in lens]
    perm = torch.randperm(sum(have) + spare, generator=g).int()
    table = torch.full((len(lens), max_pages), -1, dtype=torch.int32)
    at = 0
    for r, n in enumerate(have):
        table[r, :n] = perm[at:at + n]
        at += n
    pool = torch.full((len(perm),), -7, dtype=torch.int32)
    pool[:spare] = perm[at:]
    return table, pool, _ints([spare, 5, *lens])


def _run_plan(state, n_new, pool, table, page, n_rows):
    R = table.shape[0]
    d = {k: v.to(DEV) for k, v in dict(state=state, n_new=n_new, pool=pool, table=table).items()}
    out = {k: torch.full((n,), -99, dtype=torch.int32, device=DEV)
           for k, n in dict(state_out=2 + R, starts=R + 1, slots=n_rows, positions=n_rows).items()}
    _hip.page_plan(d["state"], d["n_new"], d["pool"], d["table"], page, out["state_out"], out["starts"], out["slots"],
                   out["positions"])
    torch.cuda.synchronize()
    assert torch.equal(d["state"].cpu(), state) and torch.equal(d["pool"].cpu(), pool)
    return dict({k: v.cpu() for k, v in out.items()}, table=d["table"].cpu())


def _same(got, want):
    for k in want:
        assert torch.equal(got[k], want[k]), k


@pytest.mark.parametrize("R,page,longest,most,padding,spare", [
    (1, 64, 0, 1, 0, 1), (1, 16, 100, 0, 3, 0), (62, 64, 1701, 1, 0, 62), (62, 16, 1701, 40, 7, 200), (3, 256, 1000, 700, 1, 9),
    (300, 32, 500, 50, 0, 500), (1024, 16, 40, 9, 5, 1200), (1025, 16, 40, 9, 0, 1200), (8192, 16, 60, 5, 11, 9000),
    (62, 64, 1701, 1701, 0, 1700),
    # pools that run out in the middle, at once, and just not
    (62, 16, 300, 40, 0, 40), (62, 16, 300, 40, 0, 0), (7, 16, 33, 20, 0, 7),
])
def test_plan(hip, R, page, longest, most, padding, spare):
    g = torch.Generator().manual_seed(R * 7 + page)
    lens = torch.randint(0, longest + 1, (R,), generator=g).tolist()
    new = torch.randint(0, most + 1, (R,), generator=g)
    table, pool, state = _pages(lens, page, -(-(longest + most) // page) + 1, spare, R)
    n_rows = int(new.sum()) + padding
    _say("plan", R, page, n_rows)
    _same(_run_plan(state, new.int(), pool, table, page, n_rows), paged.plan(state, new, pool, table, page, n_rows))


def test_plan_refusals_and_odd_counts(hip):
    """Requests past the row capacity, past the table and past the pool, negative counts, lengths and free counts
    that are no such thing, pool and table entries that are no pages."""
    page, max_pages = 16, 4
    table, pool, _ = _pages([20, 64, 0, 10, 33], page, max_pages, 6, 3)
    for state, new, n_rows in (
        ([6, 0, 20, 64, 0, 10, 33], [4, 1, 5, -3, 2], 30),  # request 1 is as long as its table row
        ([6, 0, 20, 64, 0, 10, 33], [4, 0, 45, 3, 2], 49),  # request 2's rows end at 49: 3 and 4 do not fit
        ([1, 0, 20, 64, 0, 10, 33], [13, 0, 5, 1, 2], 30),  # one page: request 2 wants the second
        ([99, 0, -5, 70, 0, 10, 33], [1, 1, 1, 1, 1], 5),
        ([-4, 0, 20, 64, 0, 10, 33], [1, 1, 1, 1, 1], 5),
        ([6, 0, 20, 64, 0, 10, 33], [2**31 - 1, 2**31 - 1, 2**31 - 1, 1, 2**31 - 1], 9),
        ([6, 0, 20, 64, 0, 10, 33], [0, 0, 0, 0, 0], 4),
        ([6, 0, 20, 64, 0, 10, 33], [0, 0, 0, 0, 0], 0),
    ):
        _say("plan", state, new, n_rows)
        _same(_run_plan(_ints(state), _ints(new), pool, table, page, n_rows),
              paged.plan(_ints(state), _ints(new), pool, table, page, n_rows))
    odd_pool, odd_table = pool.clone(), table.clone()
    odd_pool[4], odd_table[0, 1], odd_table[3, 0] = 10_000, -3, 2**31 - 1
    state, new = _ints([6, 0, 20, 64, 0, 10, 33]), _ints([4, 0, 20, 3, 2])
    _same(_run_plan(state, new, odd_pool, odd_table, page, 30), paged.plan(state, new, odd_pool, odd_table, page, 30))


@pytest.mark.parametrize("R,page,longest,share", [
    (1, 64, 1, 1.0), (62, 64, 1701, 0.5), (62, 16, 1701, 1.0), (5, 16, 8000, 0.6), (1024, 32, 90, 0.3), (8192, 16, 70, 0.9),
    (300, 16, 500, 0.0),
])
def test_release(hip, R, page, longest, share):
    g = torch.Generator().manual_seed(R + page)
    lens = torch.randint(0, longest + 1, (R,), generator=g).tolist()
    table, pool, state = _pages(lens, page, -(-longest // page) + 2, 3, R)
    done = torch.rand(R, generator=g) < share
    want = paged.release(state, done, pool, table, page)
    for flags in (done, done.to(torch.uint8) * 3):
        dev = [t.to(DEV) for t in (state, flags, pool, table)]
        out = torch.full_like(dev[0], -99)
        _say("release", R, page, flags.dtype)
        _hip.page_release(*dev, page, out)
        torch.cuda.synchronize()
        _same(dict(state_out=out.cpu(), pool=dev[2].cpu()), want)
        assert torch.equal(dev[3].cpu(), table)


def test_release_does_not_pass_the_pools_end(hip):
    """A state that claims more pages than there are: the pool is filled and no further."""
    table, pool, state = _pages([64, 64], 16, 4, 2, 0)
    state[0] = 7
    done = torch.tensor([True, True])
    dev = [t.to(DEV) for t in (state, done, pool, table)]
    out = torch.empty_like(dev[0])
    _hip.page_release(*dev, 16, out)
    torch.cuda.synchronize()
    _same(dict(state_out=out.cpu(), pool=dev[2].cpu()), paged.release(state, done, pool, table, 16))


# ---------------------------------------------------------------------------------------------- append


def _rope(P, D, seed=0):
    g = torch.Generator().manual_seed(seed)
    ang = torch.arange(P, dtype=torch.float64)[:, None] * torch.rand(D // 2, generator=g).double()
    return torch.stack((ang.cos(), ang.sin())).float()


def _half(dtype) -> float:
    return torch.finfo(dtype).eps / 2


def _rotated_close(got, x, rope, pos, what):
    want = paged.rotate(x, rope, pos)
    pair = x.double().reshape(*x.shape[:-1], -1, 2).abs().sum(-1).repeat_interleave(2, -1)
    tol = _half(x.dtype) * want.abs() + 2.0**-22 * pair + (2.0**-25 if x.dtype == HF else 0.0)
    assert bool(((got.double() - want).abs() <= tol).all()), what


# slots of the rows: runs that start anywhere in a page, single rows, rows without a place in between
def _slots(kind, n, page, pages, g):
    perm = torch.randperm(pages, generator=g)
    if kind == "single":  # each row in a page of its own, anywhere in it
        assert n <= pages
        return perm[:n] * page + torch.randint(0, page, (n,), generator=g)
    pos = torch.arange(n) + (5 if kind == "ragged" else 0)
    slots = perm[pos // page] * page + pos % page
    if kind == "ragged":
        slots[torch.rand(n, generator=g) < 0.1] = -1
        slots[n // 3] = pages * page  # no slot of the cache
    return slots


@pytest.mark.parametrize("dtype,D", itertools.product((BF, HF), (64, 128)))
@pytest.mark.parametrize("n,heads,kv,page,kind", [
    (1, 8, 8, 64, "single"), (62, 8, 8, 64, "single"), (37, 6, 3, 16, "ragged"), (8, 1, 1, 256, "run"), (7, 4, 1, 16, "run"),
    (1701, 8, 2, 64, "run"), (515, 5, 5, 32, "ragged"), (20001, 2, 1, 128, "ragged"),
])
def test_append(hip, dtype, D, n, heads, kv, page, kind):
    g = torch.Generator().manual_seed(n + D)
    pages = (n if kind == "single" else -(-(n + 5) // page)) + 1
    slots = _slots(kind, n, page, pages, g)
    P = 300
    pos = torch.randint(0, P, (n,), generator=g)
    if kind == "ragged":
        pos[n // 2], pos[n // 2 + 1] = -1, P  # no positions of the table
    qkv = torch.randn(n, heads + 2 * kv, D, generator=g).to(dtype)
    q, k, v = qkv[:, :heads], qkv[:, heads:heads + kv], qkv[:, heads + kv:]
    K0, V0 = _hip.paged_cache(pages, page, kv, D, dtype, "cpu")
    K0.copy_(torch.randn(K0.shape, generator=g))
    V0.copy_(torch.randn(V0.shape, generator=g))
    K, V = K0.to(DEV), V0.to(DEV)
    rope = _rope(P, D)
    dev = qkv.to(DEV)
    out = torch.full((n, heads, D), 7.0, dtype=dtype, device=DEV)
    _say("append", dtype, D, n, heads, kv, page, kind)
    _hip.paged_append(dev[:, heads:heads + kv], dev[:, heads + kv:], K, V, slots.int().to(DEV), pos.int().to(DEV),
                      rope.to(DEV), dev[:, :heads], out)
    torch.cuda.synchronize()
    live = (slots >= 0) & (slots < pages * page) & (pos >= 0) & (pos < P)
    at = slots[live]
    got_k, got_v = paged.k_rows(K.cpu()), paged.v_rows(V.cpu())
    _rotated_close(got_k[at], k[live], rope, pos[live], "K")
    _rotated_close(out.cpu()[live], q[live], rope, pos[live], "q")
    assert bool((out.cpu()[~live] == 7.0).all())
    want_v = paged.v_rows(V0).clone()
    want_v[at] = v[live]
    assert torch.equal(got_v.view(torch.int16), want_v.view(torch.int16))
    other = torch.ones(pages * page, dtype=torch.bool)
    other[at] = False
    assert torch.equal(got_k[other].view(torch.int16), paged.k_rows(K0)[other].view(torch.int16))


@pytest.mark.parametrize("dtype", (BF, HF))
def test_append_without_rotation_keeps_every_bit(hip, dtype):
    """rope None: k and q as they are, infinities, NaN and zeros' signs too; q in place."""
    n, kv, D, page, pages = 45, 3, 64, 32, 2
    g = torch.Generator().manual_seed(4)
    k, v, q = (torch.randint(-2**15, 2**15, (n, kv, D), generator=g, dtype=torch.int16).view(dtype) for _ in range(3))
    K, V = _hip.paged_cache(pages, page, kv, D, dtype, DEV)
    slots = torch.randperm(pages * page, generator=g)[:n]
    qd = q.to(DEV)
    _hip.paged_append(k.to(DEV), v.to(DEV), K, V, slots.int().to(DEV), q=qd, q_out=qd)
    torch.cuda.synchronize()
    for got, want in ((paged.k_rows(K.cpu())[slots], k), (paged.v_rows(V.cpu())[slots], v), (qd.cpu(), q)):
        assert torch.equal(got.view(torch.int16), want.view(torch.int16))


def test_append_rotates_q_in_place(hip):
    n, heads, kv, D = 33, 4, 2, 128
    g = torch.Generator().manual_seed(9)
    q, k, v = (torch.randn(n, h, D, generator=g).to(BF) for h in (heads, kv, kv))
    K, V = _hip.paged_cache(3, 16, kv, D, BF, DEV)
    rope, pos = _rope(50, D), torch.arange(10, 10 + n)
    qd = q.to(DEV)
    _hip.paged_append(k.to(DEV), v.to(DEV), K, V, torch.arange(n).int().to(DEV), pos.int().to(DEV), rope.to(DEV), qd, qd)
    torch.cuda.synchronize()
    _rotated_close(qd.cpu(), q, rope, pos, "q in place")
    _rotated_close(paged.k_rows(K.cpu())[:n], k, rope, pos, "K")


def test_append_of_rows_with_the_same_slot_keeps_one_of_them(hip):
    n, kv, D = 40, 2, 64
    g = torch.Generator().manual_seed(3)
    k, v = (torch.randn(n, kv, D, generator=g).to(BF) for _ in range(2))
    slots = torch.arange(n)
    slots[7], slots[30] = 20, 31  # 20 and 31 twice, 7 and 30 not at all
    K, V = _hip.paged_cache(4, 16, kv, D, BF, DEV)
    K.zero_(), V.zero_()
    _hip.paged_append(k.to(DEV), v.to(DEV), K, V, slots.int().to(DEV))
    torch.cuda.synchronize()
    for got, want in ((paged.k_rows(K.cpu()), k), (paged.v_rows(V.cpu()), v)):
        for s, a, b in ((20, 7, 20), (31, 30, 31)):
            assert bool(((got[s] == want[a]) | (got[s] == want[b])).all())
        once = [i for i in range(n) if i not in (7, 20, 30, 31)]
        assert torch.equal(got[once], want[once])
        assert bool((got[[7, 30]] == 0).all()) and bool((got[n:] == 0).all())


# ---------------------------------------------------------------------------------------------- attention


def _attn_case(lens, new, heads, kv, D, page, dtype, seed, sharp=1.0, padding=0):
    """A cache with every page random and requests of these lengths, the last new[r] rows of each in q."""
    g = torch.Generator().manual_seed(seed)
    max_pages = max(1, max(-(-n // page) for n in lens)) + 1
    table, pool, _ = _pages(lens, page, max_pages, 2, seed)
    K, V = _hip.paged_cache(len(pool), page, kv, D, dtype, "cpu")
    K.copy_(torch.randn(K.shape, generator=g))
    V.copy_(torch.randn(V.shape, generator=g) + 0.3)
    n = sum(new) + padding
    q = (sharp * torch.randn(n, heads, D, generator=g)).to(dtype)
    starts = torch.cat((torch.zeros(1, dtype=torch.int64), torch.tensor(new).cumsum(0))).int()
    return dict(q=q, K=K, V=V, table=table, starts=starts, lens=_ints(lens))


def _run_attn(c, O=None, **kw):
    d = {k: v.to(DEV) for k, v in c.items()}
    n, heads, D = c["q"].shape
    O = torch.full((n, heads * D), 7.0, dtype=c["q"].dtype, device=DEV) if O is None else O
    if kw.get("gate") is not None:
        kw["gate"] = kw["gate"].to(DEV)
    _hip.paged_attention(d["q"], d["K"], d["V"], d["table"], d["starts"], d["lens"], O, **kw)
    torch.cuda.synchronize()
    return O.cpu().view(n, heads, D)


def _attn_close(got, c, gate=None, **kw):
    n, heads, D = c["q"].shape
    want, mag, size = paged.attention(**c, gate=gate, **kw)
    rows = ~want[:, 0, 0].isnan() | (size[:, 0, 0] > 0)
    u = _half(got.dtype)
    e = 2.0**-24 * (size[..., :1] + 4 * D * size[..., 1:] + 64)
    tol = u * want.abs() + (u + e) * mag
    if got.dtype == HF:
        f = 1.0 if gate is None else gate.double().abs()[..., None].clamp(min=1.0)
        big = torch.nan_to_num(c["V"].double().abs(), posinf=0.0).max()
        tol = tol + 2.0**-25 * (1 + f * size[..., :1] * big)
    bad = ~((got.double() - want).abs() <= tol)
    bad &= ~(got.double().isnan() & want.isnan()) & ~(got.double() == want)
    assert not bool(bad[rows].any()), (int(bad[rows].sum()), float(((got.double() - want).abs() / (tol + 1e-30))[rows].max()))
    assert bool((got[~rows] == 7.0).all())


ATTN = [  # lens, new, heads, kv, page
    ([1], [1], 8, 8, 64), ([17], [1], 8, 8, 16), ([33, 64, 65, 128], [1, 1, 1, 1], 4, 4, 16), ([500, 3, 1701], [1, 1, 1], 8, 2, 64),
    ([40, 100], [7, 12], 4, 4, 32), ([300, 31], [33, 31], 2, 1, 16), ([90, 70, 200], [5, 0, 65], 8, 1, 128),
    ([257], [200], 3, 3, 256), ([700, 129], [129, 129], 6, 3, 32), ([2050], [3], 16, 1, 64), ([5, 1000], [5, 300], 4, 2, 64),
    # keys split over workgroups: single rows, some rows, many; requests far shorter than the longest
    ([3001], [1], 2, 2, 16), ([4000, 1, 0, 260], [1, 1, 0, 1], 8, 1, 64), ([2500, 31], [40, 31], 2, 1, 32), ([1500], [300], 2, 2, 128),
    # column tiles of more than 64 requests, and of requests of one length
    ([(37 * i) % 90 + 1 for i in range(70)], [min((37 * i) % 90 + 1, (13 * i) % 43) for i in range(70)], 4, 1, 16),
    ([200] * 5, [60, 3, 0, 45, 70], 4, 1, 32),
    # more than 1024 columns of a request
    ([300, 40], [290, 3], 4, 1, 16), ([1100], [259], 8, 2, 64), ([600, 40], [290, 3], 4, 1, 32), ([1090, 1030], [1090, 3], 1, 1, 64),
]


@pytest.mark.parametrize("dtype,D", itertools.product((BF, HF), (64, 128)))
@pytest.mark.parametrize("lens,new,heads,kv,page", ATTN)
def test_attention(hip, dtype, D, lens, new, heads, kv, page):
    c = _attn_case(lens, new, heads, kv, D, page, dtype, sum(lens) + D)
    _say("attention", dtype, D, lens, new, heads, kv, page)
    _attn_close(_run_attn(c, max_new=max(new), max_len=max(lens)), c)


@pytest.mark.parametrize("causal,window", [(True, 1), (True, 16), (True, 50), (True, 900), (True, 10_000), (False, 0), (False, 7), (False, 33)])
@pytest.mark.parametrize("lens,new,page", [([200, 77], [1, 1], 16), ([150, 90], [40, 90], 32), ([333], [130], 64),
                                           ([2100, 90], [1, 1], 16), ([1300], [45], 64), ([310], [270], 32)])
def test_attention_masks(hip, causal, window, lens, new, page):
    for dtype, D, heads, kv in ((BF, 64, 4, 1), (HF, 128, 2, 2)):
        c = _attn_case(lens, new, heads, kv, D, page, dtype, window + 3, padding=2)
        gate = torch.rand(c["q"].shape[0], heads, generator=torch.Generator().manual_seed(1))
        _say("attention", causal, window, lens, new, page, dtype)
        _attn_close(_run_attn(c, gate=gate, causal=causal, window=window, max_new=max(new)), c, gate=gate, causal=causal,
                    window=window)


@pytest.mark.parametrize("D", (64, 128))
def test_attention_rows_that_see_nothing_and_odd_lengths(hip, D):
    """Requests of length 0 and with fewer positions than rows, no rows, lengths past the table, negative ones, starts
    that go past the rows: zeros where no key is seen, no row beyond."""
    c = _attn_case([40, 40, 40, 40, 40], [2, 5, 0, 3, 2], 2, 1, D, 16, BF, 5, padding=3)
    c["lens"] = _ints([0, 3, 40, 1000, -5])
    c["table"][3] = torch.tensor([0, 1, 2, 3])
    got = _run_attn(c)
    _attn_close(got, c)
    assert bool((got[:4] == 0).all())  # request 0, and the first two rows of request 1
    _attn_close(_run_attn(c, causal=False), c, causal=False)
    c["starts"] = _ints([0, 4, 4, 9, 400, 500])
    _attn_close(_run_attn(c), c)
    c["starts"] = _ints([-3, 4, 2, 9, 12, 12])
    _run_attn(c)  # not ascending: nothing out of bounds


def test_attention_skips_table_entries_that_are_no_pages(hip):
    for lens, new in (([200], [1]), ([200, 100], [40, 60])):
        c = _attn_case(lens, new, 2, 1, 64, 16, HF, 8)
        c["table"][0, 0], c["table"][0, 3], c["table"][0, 11] = -1, 2**31 - 1, c["K"].shape[0]
        _attn_close(_run_attn(c), c)
        c["table"][:] = -1
        assert bool((_run_attn(c) == 0).all())


@pytest.mark.parametrize("dtype", (BF, HF))
@pytest.mark.parametrize("lens,new,page", [([50, 70], [1, 1], 64), ([100, 70, 33], [20, 40, 33], 16), ([300], [200], 32),
                                           ([1400], [3], 16), ([600], [550], 64)])
def test_unseen_infinities_and_nan_change_nothing(hip, dtype, lens, new, page):
    """K and V are NaN and infinite wherever no row may look (behind the lengths, in free pages), and V at a position that
    some rows of a tile see and others do not: only those that see it are touched, causal, windowed or both."""
    heads, kv, D = 2, 1, 64
    for causal, window in ((True, 0), (True, 9), (False, 9)):
        c = _attn_case(lens, new, heads, kv, D, page, dtype, 11)
        held = torch.zeros(c["K"].shape[0] * page, dtype=torch.bool)
        for r, n in enumerate(lens):
            key = torch.arange(n)
            held[c["table"][r, key // page].long() * page + key % page] = True
        k, v = paged.k_rows(c["K"]).clone(), paged.v_rows(c["V"]).clone()
        k[~held], v[~held] = float("nan"), float("inf")
        v[~held, :, 1::2] = float("nan")
        at = lens[0] - 1 - new[0] // 2
        spot = int(c["table"][0, at // page]) * page + at % page
        v[spot, 0, 3], v[spot, 0, 40], v[spot, 0, 63] = float("inf"), float("-inf"), float("nan")
        P = c["K"].shape[0]
        c["K"] = k.view(P, page // 16, 16, kv, D // 8, 8).permute(0, 3, 1, 4, 2, 5).contiguous()
        c["V"] = v.view(P, page // 8, 8, kv, D).permute(0, 3, 1, 4, 2).contiguous()
        got = _run_attn(c, causal=causal, window=window)
        _attn_close(got, c, causal=causal, window=window)
        assert bool(got.isfinite().any())


@pytest.mark.parametrize("lens,new", [([90], [1]), ([90], [60]), ([2000], [1])])
def test_seen_nan_and_infinities_come_out(hip, lens, new):
    """A NaN in q, in a key's K or an infinite score make NaN of the rows that have them, and of no other."""
    c = _attn_case(lens, new, 2, 2, 64, 16, BF, 13)
    c["q"][0, 0, 5] = float("nan")
    got = _run_attn(c, max_new=max(new))
    assert bool(got[0, 0].isnan().all()) and not bool(got[0, 1].isnan().any()) and not bool(got[1:].isnan().any())
    for value in (float("nan"), float("inf")):
        c = _attn_case(lens, new, 2, 2, 64, 16, BF, 13)
        c["q"][:] = c["q"].abs() + 0.1
        k = paged.k_rows(c["K"]).clone()
        at = lens[0] - 1 - new[0] // 2
        k[int(c["table"][0, at // 16]) * 16 + at % 16, 1, 7] = value
        P = c["K"].shape[0]
        c["K"] = k.view(P, 1, 16, 2, 8, 8).permute(0, 3, 1, 4, 2, 5).contiguous()
        got = _run_attn(c, max_new=max(new))
        sees = torch.arange(lens[0] - new[0], lens[0]) >= at
        assert bool(got[sees, 1].isnan().all()) and bool(got[~sees, 1].isfinite().all()) and bool(got[:, 0].isfinite().all())


@pytest.mark.parametrize("D,dtype", [(64, BF), (128, HF)])
def test_attention_scores_that_rise_late(hip, D, dtype):
    """Keys whose scores stand tens and hundreds above all earlier ones, late in a long sequence and one after the other."""
    for lens, new in (([900], [1]), ([900], [70])):
        c = _attn_case(lens, new, 2, 1, D, 64, dtype, 21)
        k = paged.k_rows(c["K"]).clone()
        for i, at in enumerate((100, 431, 690, 820)):
            slot = int(c["table"][0, at // 64]) * 64 + at % 64
            k[slot] = 0.0
            k[slot, 0, 0] = 20.0 * (i + 1)
        c["q"][..., 0] = 1.0 + 0.25 * D**0.5
        P = c["K"].shape[0]
        c["K"] = k.view(P, 4, 16, 1, D // 8, 8).permute(0, 3, 1, 4, 2, 5).contiguous()
        _attn_close(_run_attn(c, scale=1.0), c, scale=1.0)


def test_attention_row_strides_and_scale(hip):
    c = _attn_case([70, 40], [30, 9], 3, 1, 64, 32, BF, 31)
    n = c["q"].shape[0]
    wide = torch.full((n, 5, 64), float("nan"), dtype=BF, device=DEV)
    wide[:, 1:4] = c["q"].to(DEV)
    d = {k: v.to(DEV) for k, v in c.items()}
    O = torch.empty(n, 192, dtype=BF, device=DEV)
    _hip.paged_attention(wide[:, 1:4], d["K"], d["V"], d["table"], d["starts"], d["lens"], O, scale=0.3)
    torch.cuda.synchronize()
    _attn_close(O.cpu().view(n, 3, 64), c, scale=0.3)


@pytest.mark.parametrize("new", (1, 60))
def test_attention_workspace(hip, new):
    """A caller's workspace: of any content, exactly as large as asked for, and refused if smaller."""
    c = _attn_case([3000], [new], 4, 2, 64, 64, BF, 43)
    need = _hip.paged_attention_workspace_bytes(4, c["K"], c["V"], 1, c["table"].shape[1], new, new, 3000)
    assert need > 0
    ws = torch.full((need + 64,), 255, dtype=torch.uint8, device=DEV)  # NaN in any type
    kw = dict(max_new=new, max_len=3000)
    got = _run_attn(c, ws=ws[:need], **kw)
    assert bool((ws[need:] == 255).all())
    _attn_close(got, c)
    assert torch.equal(got, _run_attn(c, **kw))
    with pytest.raises(RuntimeError, match="workspace"):
        _run_attn(c, ws=ws[:need - 16], **kw)


def test_attention_bounds_that_are_not_tight(hip):
    """max_len far from the lengths, both ways, and max_new above the rows: other launches, the same result."""
    c = _attn_case([1900, 40], [5, 2], 4, 2, 64, 64, BF, 44)
    for kw in (dict(), dict(max_len=1), dict(max_len=1900, max_new=5), dict(max_new=7, max_len=100_000), dict(max_new=1 << 30)):
        _attn_close(_run_attn(c, **kw), c)


def test_attention_of_thousands_of_requests(hip):
    """Column tiles found among 5000 requests: of no rows, of a few, of several tiles; of no positions."""
    lens = [(37 * i) % 60 for i in range(5000)]
    lens[0], lens[4100], lens[-1] = 300, 250, 140
    new = [min(n, (13 * i) % 4) for i, n in enumerate(lens)]
    new[0], new[4100], new[-1] = 200, 170, 140
    c = _attn_case(lens, new, 2, 1, 64, 16, BF, 45, padding=3)
    _say("attention of 5000 requests")
    _attn_close(_run_attn(c, max_new=200, max_len=300), c)


@pytest.mark.parametrize("R,max_new", [(5, 1), (5, 200), (64, 200), (65, 200)])
def test_attention_of_starts_out_of_order_stays_in_its_rows(hip, R, max_new):
    """starts that descend, are negative or pass the rows: what the rows get means nothing, and only rows are written."""
    n, heads, D = 150, 2, 64
    c = _attn_case([40 + i for i in range(R)], [0] * R, heads, 1, D, 16, BF, 46, padding=n)
    c["starts"] = torch.randint(-100, 400, (R + 1,), generator=torch.Generator().manual_seed(R)).int()
    c["starts"][:2] = _ints([-(1 << 31), (1 << 31) - 1])
    room = torch.full((n + 64, heads * D), 7.0, dtype=BF, device=DEV)
    _say("attention, starts out of order", R, max_new)
    _run_attn(c, O=room[32:32 + n], max_new=max_new, max_len=100)
    assert bool((room[:32] == 7.0).all()) and bool((room[32 + n:] == 7.0).all())


def test_attention_is_the_same_bits_again_and_at_another_place_in_the_batch(hip):
    c = _attn_case([1500, 90, 700], [1, 1, 1], 4, 2, 64, 16, BF, 41)
    a = _run_attn(c, max_new=1)
    assert torch.equal(a, _run_attn(c, max_new=1))
    swapped = dict(c, q=c["q"].flip(0), table=c["table"].flip(0), lens=c["lens"].flip(0))
    assert torch.equal(a.flip(0), _run_attn(swapped, max_new=1))


def test_attention_of_a_cache_past_32_bits(hip):
    """K and V of 4.5 GB each: pages whose elements start past 2^31 and whose bytes start past 2^32."""
    page, kv, D = 256, 8, 128
    pages = 9000  # x 256 x 8 x 128 x 2 bytes
    K, V = _hip.paged_cache(pages, page, kv, D, BF, DEV)
    use = torch.tensor([8999, 4200, 8100, 17, 8192], dtype=torch.int32)
    small = _attn_case([1200], [3], 8, kv, D, page, BF, 51)
    small["table"] = torch.arange(5, dtype=torch.int32)[None]
    K[use.long().to(DEV)], V[use.long().to(DEV)] = small["K"][:5].to(DEV), small["V"][:5].to(DEV)
    k, v = (torch.randn(3, kv, D, generator=torch.Generator().manual_seed(i)).to(BF) for i in (1, 2))
    slots = (8192 * page + torch.arange(1200 - 3, 1200) % page).int()
    _say("append and attention past 32 bits")
    _hip.paged_append(k.to(DEV), v.to(DEV), K, V, slots.to(DEV))
    O = torch.empty(3, 8 * D, dtype=BF, device=DEV)
    _hip.paged_attention(small["q"].to(DEV), K, V, use[None].to(DEV), small["starts"].to(DEV), small["lens"].to(DEV), O)
    torch.cuda.synchronize()
    small["K"], small["V"] = K[use.long().to(DEV)].cpu(), V[use.long().to(DEV)].cpu()
    assert torch.equal(paged.k_rows(small["K"])[4 * page + slots.long() % page], k)
    assert torch.equal(paged.v_rows(small["V"])[4 * page + slots.long() % page], v)
    _attn_close(O.cpu().view(3, 8, D), small)


# ---------------------------------------------------------------------------------------------- together


class _Plain:
    """What HipPagedCache keeps, in plain form: every request's rotated K rows and V rows in lists."""

    def __init__(self, R):
        self.k, self.v = [[] for _ in range(R)], [[] for _ in range(R)]

    def dense(self, kv, D, dtype):
        """The rows as a cache with one page per request."""
        longest = max(1, max(len(x) for x in self.k))
        page = -(-longest // 16) * 16
        K, V = (torch.zeros(len(self.k), page, kv, D, dtype=dtype) for _ in range(2))
        for r, (k, v) in enumerate(zip(self.k, self.v)):
            if k:
                K[r, :len(k)], V[r, :len(v)] = torch.stack(k), torch.stack(v)
        R = len(self.k)
        K = K.view(R, page // 16, 16, kv, D // 8, 8).permute(0, 3, 1, 4, 2, 5).contiguous()
        V = V.view(R, page // 8, 8, kv, D).permute(0, 3, 1, 4, 2).contiguous()
        return dict(K=K, V=V, table=torch.arange(R, dtype=torch.int32)[:, None], lens=_ints(len(x) for x in self.k))


@pytest.mark.parametrize("dtype,D,heads,kv,page", [(BF, 64, 8, 8, 64), (HF, 128, 4, 2, 16)])
def test_a_run_of_steps(hip, dtype, D, heads, kv, page):
    """Ragged pieces, single rows, padding, requests that end and their pages dealt again."""
    R = 5
    g = torch.Generator().manual_seed(D)
    cache = HipPagedCache(R, 400, kv, D, pages=R * 400 // page, page_size=page, dtype=dtype)
    plain = _Plain(R)
    rope = _rope(400, D)
    for step, new in enumerate(([70, 0, 33, 1, 100], [1, 1, 1, 1, 1], [0, 40, 17, 64, 3], [5, 90, 0, 1, 130], [1, 1, 1, 1, 1])):
        n = sum(new)
        rows = n + (step % 3)
        qkv = torch.randn(rows, heads + 2 * kv, D, generator=g).to(dtype)
        dev = qkv.to(DEV)
        gate = torch.rand(rows, heads, generator=g)
        _say("step", step, new)
        plan = cache.plan(_ints(new).to(DEV), rows, max(new))
        q = cache.append(plan, dev[:, :heads], dev[:, heads:heads + kv], dev[:, heads + kv:], rope.to(DEV))
        O = torch.full((rows, heads * D), 7.0, dtype=dtype, device=DEV)
        cache.attend(plan, q, gate=gate.to(DEV), out=O)
        torch.cuda.synchronize()
        assert cache.refused == 0
        at = 0
        K = paged.k_rows(cache.K.cpu())
        for r, m in enumerate(new):
            for i in range(m):
                pos = torch.tensor([len(plain.k[r])])
                _rotated_close(K[int(plan.slots[at])][None], qkv[at:at + 1, heads:heads + kv], rope, pos, "K")
                _rotated_close(q[at:at + 1].cpu(), qkv[at:at + 1, :heads], rope, pos, "q")
                plain.k[r].append(K[int(plan.slots[at])])
                plain.v[r].append(qkv[at, heads + kv:])
                at += 1
        assert cache.lengths.tolist() == [len(x) for x in plain.k]
        c = dict(plain.dense(kv, D, dtype), q=q.cpu(), starts=plan.starts.cpu())
        _attn_close(O.cpu().view(rows, heads, D), c, gate=gate)
        if step == 2:
            done = torch.tensor([True, False, False, True, False])
            cache.release(done.to(DEV))
            for r in (0, 3):
                plain.k[r], plain.v[r] = [], []
            assert cache.lengths.tolist() == [len(x) for x in plain.k]
    held = sum(-(-len(x) // page) for x in plain.k)
    assert cache.free_pages == cache.pages - held
    live = torch.cat([cache.table[r, :-(-len(x) // page)] for r, x in enumerate(plain.k)])
    assert sorted(live.tolist() + cache.pool[:cache.free_pages].tolist()) == list(range(cache.pages))


def test_a_refused_request_says_so_and_keeps_its_length(hip):
    cache = HipPagedCache(3, 64, 1, 64, pages=3, page_size=16)
    cache.plan(_ints([16, 20, 5]).to(DEV), 41)
    assert cache.refused == 1 and cache.lengths.tolist() == [16, 20, 0] and cache.free_pages == 0
    cache.release(torch.tensor([True, False, False], device=DEV))
    cache.plan(_ints([0, 0, 5]).to(DEV), 5)
    assert cache.refused == 0 and cache.lengths.tolist() == [0, 20, 5]


def test_captured_step_replays_with_growing_lengths(hip):
    """plan, append and attend of one row per request captured once and replayed, each replay against an eager cache
    that takes the same rows, with eager work of the program's own in between."""
    R, heads, kv, D = 6, 4, 2, 64
    rope = _rope(500, D).to(DEV)
    a, b = (HipPagedCache(R, 500, kv, D, page_size=16) for _ in range(2))
    g = torch.Generator().manual_seed(2)
    lens = [0, 15, 16, 100, 300, 31]
    first = torch.randn(sum(lens), heads + 2 * kv, D, generator=g).to(BF).to(DEV)
    n_new, ones = _ints(lens).to(DEV), torch.ones(R, dtype=torch.int32, device=DEV)
    rows = torch.zeros(R, heads + 2 * kv, D, dtype=BF, device=DEV)

    def step(cache, x, new, most):
        plan = cache.plan(new, x.shape[0], most)
        q = cache.append(plan, x[:, :heads], x[:, heads:heads + kv], x[:, heads + kv:], rope)
        return cache.attend(plan, q)

    for cache in (a, b):
        cache.K.zero_(), cache.V.zero_()
        step(cache, first, n_new, max(lens))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        O = step(a, rows, ones, 1)
    torch.cuda.synchronize()
    for i in range(4):
        x = torch.randn(R, heads + 2 * kv, D, generator=g).to(BF).to(DEV)
        rows.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        want = step(b, x, ones, 1)
        torch.cuda.synchronize()
        assert torch.equal(O, want), i
        assert torch.equal(a.state, b.state) and torch.equal(a.table, b.table)


def test_two_streams_at_once(hip):
    """Two caches stepped on two streams with nothing between them."""
    c = [_attn_case([800, 90], [1, 1], 4, 2, 64, 16, BF, s) for s in (61, 62)]
    want = [_run_attn(x) for x in c]
    dev = [{k: v.to(DEV) for k, v in x.items()} for x in c]
    out = [torch.empty(2, 256, dtype=BF, device=DEV) for _ in c]
    streams = [torch.cuda.Stream() for _ in c]
    torch.cuda.synchronize()
    for _ in range(5):
        for d, o, s in zip(dev, out, streams):
            with torch.cuda.stream(s):
                _hip.paged_attention(d["q"], d["K"], d["V"], d["table"], d["starts"], d["lens"], o)
    torch.cuda.synchronize()
    for o, w in zip(out, want):
        assert torch.equal(o.cpu().view(w.shape), w)


def test_wrappers_refuse(hip):
    c = {k: v.to(DEV) for k, v in _attn_case([40, 20], [3, 1], 4, 2, 64, 16, BF, 71).items()}
    n = c["q"].shape[0]
    O = torch.empty(n, 256, dtype=BF, device=DEV)

    def attend(**kw):
        a = dict(c, O=O)
        a.update(kw)
        _hip.paged_attention(**a)

    for kw in (dict(q=c["q"].to(HF)), dict(q=c["q"][:, :3]), dict(q=c["q"].cpu()), dict(O=O[:, :128]), dict(O=O.float()),
               dict(table=c["table"].long()), dict(starts=c["starts"][:2]), dict(lens=c["lens"].cpu()),
               dict(gate=torch.ones(n, 3, device=DEV)), dict(q=c["q"].transpose(1, 2)), dict(q=c["q"].flatten(1)),
               dict(V=c["V"][:-1])):
        with pytest.raises(ValueError):
            attend(**kw)
    for kw in (dict(scale=0.0), dict(window=-1), dict(max_new=-1)):
        with pytest.raises(RuntimeError):
            attend(**kw)
    kv = torch.zeros(3, 2, 64, dtype=BF, device=DEV)
    slots = torch.zeros(3, dtype=torch.int32, device=DEV)
    for kw in (dict(k=kv[:2]), dict(k=kv.float()), dict(slots=slots.long()), dict(rope=torch.zeros(2, 9, 32, device=DEV)),
               dict(q=kv), dict(v=kv.expand(3, 2, 64)[:, :1]), dict(slots=slots.cpu())):
        a = dict(k=kv, v=kv, K=c["K"], V=c["V"], slots=slots)
        a.update(kw)
        with pytest.raises(ValueError):
            _hip.paged_append(**a)
    with pytest.raises(RuntimeError, match="fewer than"):
        _hip.paged_append(kv[:1].expand(3, 2, 64), kv, c["K"], c["V"], slots)
    with pytest.raises(ValueError, match="requests"):
        HipPagedCache(0, 10)
