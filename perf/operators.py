"""The operators of streaming attention over a paged K/V cache, as ``perf/cases.py`` has the ones of whole chunks: cases,
inputs, the calls, their plain forms and what they compute in 64 bits.

A server of live streams and songs keeps the K and V rows of the frames so far in pages of ``page`` positions, a row of
page numbers per request (one request is one band's frame sequence: a stereo stream of the 62-band model has 62). A
step takes ``new`` frames per request: ``page_plan`` deals pages and says where the new rows go, ``paged_append`` rotates q
and k and writes k and v there, ``paged_attention`` attends the new rows over their requests' positions, and
``page_release`` takes the pages of finished requests back. The forms:

    K cache [pages][kv heads][page / 16][D / 8][16 positions][8 features]
    V cache [pages][kv heads][page / 8][D features][8 positions]
    state   [free pages, refused requests, length of each request]

Lengths of a case are spread evenly over their range, so that a case alone fixes its work; the seed orders them, places
the pages and fills the tensors.
"""

from __future__ import annotations

import math
import random
import sys
from pathlib import Path

import numpy as np
import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ------------------------------------------------------------------------------------------------ the cases


def listed() -> list[dict]:
    return [
        # One live stream takes one frame: 62 bands, a row each.
        dict(name="plan_live", kind="plan", requests=62, lo=600, hi=1701, new_lo=1, new_hi=1, page=64, max_pages=32),
        # 66 songs are fed in ragged pieces, about 105,000 rows, onto small pages.
        dict(name="plan_songs", kind="plan", requests=4092, lo=0, hi=1701, new_lo=0, new_hi=51, page=16, max_pages=112),
        # Half of two live streams' bands end.
        dict(name="release_live", kind="release", requests=124, lo=600, hi=1701, done=0.5, page=64, max_pages=32),
        # A third of 66 long recordings ends at once.
        dict(name="release_songs", kind="release", requests=4092, lo=1, hi=8191, done=0.33, page=16, max_pages=512),
        # One frame of a live stream enters the cache: latency.
        dict(name="append_live", kind="append", requests=62, lo=600, hi=1701, new_lo=1, new_hi=1, heads=8, kv=8, dim=64,
             page=64, dtype="bf16"),
        # Odd pieces of several recordings, grouped heads of 128 in fp16 on small pages.
        dict(name="append_pieces", kind="append", requests=29, lo=0, hi=5003, new_lo=1, new_hi=601, heads=32, kv=8,
             dim=128, page=16, dtype="fp16"),
        # A 17 s chunk's 1701 frames of 62 bands enter at once.
        dict(name="append_17s", kind="append", requests=62, lo=0, hi=0, new_lo=1701, new_hi=1701, heads=8, kv=8, dim=64,
             page=64, dtype="bf16"),
        # The first frames of one sequence: the smallest call.
        dict(name="attn_first", kind="attn", requests=1, lo=17, hi=17, new_lo=1, new_hi=1, heads=8, kv=8, dim=64, page=64,
             dtype="bf16", causal=True, window=0, gated=True),
        # One frame of a live stream over up to 17 s of its past, 62 bands with gates.
        dict(name="attn_live", kind="attn", requests=62, lo=600, hi=1701, new_lo=1, new_hi=1, heads=8, kv=8, dim=64, page=64,
             dtype="bf16", causal=True, window=0, gated=True),
        # Single rows over about 20 minutes of frames each, grouped heads of 128: few rows, long caches.
        dict(name="attn_long", kind="attn", requests=5, lo=99_991, hi=131_071, new_lo=1, new_hi=1, heads=32, kv=8, dim=128,
             page=16, dtype="fp16", causal=True, window=0, gated=False),
        # Pieces of 3 to 7 s over a past of 20 to 60 s, causal in a window of 40 s, grouped heads of 128.
        dict(name="attn_pieces", kind="attn", requests=9, lo=2001, hi=6007, new_lo=301, new_hi=701, heads=32, kv=8, dim=128,
             page=32, dtype="fp16", causal=True, window=4001, gated=False),
        # A 17 s chunk at once, every frame over every frame as the model's time attention has it.
        dict(name="attn_17s", kind="attn", requests=62, lo=1701, hi=1701, new_lo=1701, new_hi=1701, heads=8, kv=8, dim=64,
             page=64, dtype="bf16", causal=False, window=0, gated=True),
    ]


def _log(rng: random.Random, lo: int, hi: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _range(rng: random.Random, hi: int) -> tuple[int, int]:
    return (hi, hi) if rng.random() < 0.25 else (rng.randint(0, hi), hi)


def draw(rng: random.Random) -> dict:
    kind = rng.choice(("plan", "release", "append", "append", "attn", "attn", "attn", "attn"))
    page = rng.choice((16, 32, 64, 128))
    if kind in ("plan", "release"):
        R = _log(rng, 1, 4092)
        lo, hi = _range(rng, _log(rng, 1, min(8191, 512 * page - 64)))
        if kind == "release":
            return dict(kind=kind, requests=R, lo=lo, hi=hi, done=round(rng.uniform(0.1, 1.0), 3), page=page,
                        max_pages=-(-hi // page) + rng.randint(0, 3))
        new_hi = _log(rng, 1, max(1, min(1701, 100_000 // R)))
        return dict(kind=kind, requests=R, lo=lo, hi=hi, new_lo=rng.randint(0, new_hi), new_hi=new_hi, page=page,
                    max_pages=-(-(hi + new_hi) // page) + rng.randint(0, 3))
    kv, group, dim = rng.choice((1, 2, 4, 8)), rng.choice((1, 1, 2, 4, 8)), rng.choice((64, 64, 128))
    dtype = rng.choice(("bf16", "bf16", "fp16"))
    heads = kv * group
    if kind == "append":
        most = 105_462 * 24 * 64 // ((heads + 2 * kv) * dim)
        R = _log(rng, 1, min(4092, most))
        new_hi = _log(rng, 1, max(1, min(4096, most // R)))
        lo, hi = _range(rng, _log(rng, 1, 8191))
        return dict(kind=kind, requests=R, lo=lo, hi=hi, new_lo=rng.randint(0 if R > 1 else 1, new_hi), new_hi=new_hi,
                    heads=heads, kv=kv, dim=dim, page=page, dtype=dtype)
    if rng.random() < 0.5:  # single rows
        hi = _log(rng, 2, 131_071)
        R = _log(rng, 1, max(1, min(512, 260_000_000 // (hi * kv * dim))))
        new_lo = new_hi = 1
    else:
        new_hi = _log(rng, 2, 2048)
        hi = new_hi + _log(rng, 1, 16_384)
        R = _log(rng, 1, max(1, min(512, 200_000_000 // (hi * kv * dim), 1_000_000_000 // (hi * new_hi * heads))))
        new_lo = rng.randint(1, new_hi)
    lo = rng.randint(new_hi, hi)
    return dict(kind="attn", requests=R, lo=lo, hi=hi, new_lo=new_lo, new_hi=new_hi, heads=heads, kv=kv, dim=dim, page=page,
                dtype=dtype, causal=rng.random() < 0.75, window=0 if rng.random() < 0.7 else _log(rng, 1, hi),
                gated=rng.random() < 0.5)


def _spread(lo: int, hi: int, n: int, step: float) -> list[int]:
    """n whole numbers that cover lo..hi evenly, in an order of no pattern: multiples of an irrational step."""
    return [lo + int((hi - lo + 1) * (((i + 1) * step) % 1.0)) for i in range(n)]


def _lengths(case: dict) -> list[tuple[int, int]]:
    """(length, new rows) of each request; the length counts the new rows where K and V already hold them (attn)."""
    R = case["requests"]
    lens = _spread(case["lo"], case["hi"], R, 0.6180339887498949)
    new = _spread(case["new_lo"], case["new_hi"], R, 0.7548776662466927) if "new_lo" in case else [0] * R
    return list(zip(lens, new))


# ------------------------------------------------------------------------------------------------ prepare


def _gen(seed: int, stream: int) -> torch.Generator:
    return torch.Generator(device=DEV).manual_seed(seed * 64 + stream)


def _normal(seed: int, stream: int, shape: tuple, dtype: torch.dtype, heads: int) -> torch.Tensor:
    """Normal rows [n, heads, D] of a spread and a mean that differ from head to head, as projections have them."""
    g = _gen(seed, stream)
    s = 0.6 + 0.8 * torch.rand(heads, 1, generator=g, device=DEV)
    m = 0.2 * torch.randn(heads, shape[-1], generator=g, device=DEV)
    return (torch.randn(shape, generator=g, device=DEV) * s + m).to(dtype)


def _pages(case: dict, seed: int, lens: list[int], pages_more: int) -> dict:
    """Pages dealt at random to requests of these lengths, `pages_more` left free: table, pool and state."""
    page, R = case["page"], len(lens)
    have = [-(-n // page) for n in lens]
    held = sum(have)
    n_pages = held + pages_more
    perm = np.random.RandomState(seed % (1 << 32)).permutation(n_pages).astype(np.int32)
    max_pages = case.get("max_pages", max(1, max(have)))
    table = np.full((R, max_pages), -1, dtype=np.int32)
    table[np.arange(max_pages)[None, :] < np.array(have)[:, None]] = perm[:held]
    pool = np.full(n_pages, -1, dtype=np.int32)
    pool[:pages_more] = perm[held:]
    dev = {k: torch.from_numpy(v).to(DEV) for k, v in dict(table=table, pool=pool).items()}
    dev["state"] = torch.tensor([pages_more, 0, *lens], dtype=torch.int32, device=DEV)
    return dict(dev, n_pages=n_pages)


def _rows(s: dict, lens: list[int], new: list[int]) -> None:
    """starts, and position and slot of every new row; lens count the new rows."""
    n, ln = np.array(new, dtype=np.int64), np.array(lens, dtype=np.int64)
    starts = np.concatenate([[0], np.cumsum(n)])
    r = np.repeat(np.arange(len(new)), n)
    pos = np.arange(starts[-1]) - starts[r] + (ln - n)[r]
    s["starts"] = torch.from_numpy(starts.astype(np.int32)).to(DEV)
    s["lens"] = torch.from_numpy(ln.astype(np.int32)).to(DEV)
    p = torch.from_numpy(pos).to(DEV)
    pages = s["table"][torch.from_numpy(r).to(DEV), p // s["page"]].long()
    s["positions"], s["slots"] = p.int(), (pages * s["page"] + p % s["page"]).int()


def prepare(case: dict, seed: int) -> dict:
    kind, page = case["kind"], case["page"]
    s = dict(case)
    order = np.random.RandomState((seed + 1) % (1 << 32)).permutation(case["requests"])
    pairs = [_lengths(case)[i] for i in order]
    lens, new = [p[0] for p in pairs], [p[1] for p in pairs]
    R = len(lens)
    if kind == "plan":
        wanted = sum(-(-(a + b) // page) + (-a // page) for a, b in pairs)
        s.update(_pages(case, seed, lens, wanted + 7))
        s["n_new"] = torch.tensor(new, dtype=torch.int32, device=DEV)
        n = max(1, sum(new))
        for name, size in (("state_out", 2 + R), ("starts", R + 1), ("slots", n), ("positions", n)):
            s[name] = torch.empty(size, dtype=torch.int32, device=DEV)
        return s
    if kind == "release":
        s.update(_pages(case, seed, lens, 7))
        ended = np.random.RandomState((seed + 2) % (1 << 32)).permutation(R) < max(1, round(case["done"] * R))
        s["done"] = torch.from_numpy(ended).to(DEV)
        s["state_out"] = torch.empty(2 + R, dtype=torch.int32, device=DEV)
        return s
    if kind == "append":
        lens = [a + b for a, b in pairs]
    s.update(_pages(case, seed, lens, 1))
    _rows(s, lens, new)
    n, dt, D, Hq, Hkv = sum(new), DTYPES[case["dtype"]], case["dim"], case["heads"], case["kv"]
    P = s["n_pages"]
    # what the pages hold: rows of the same distribution (of other requests and times where these lengths do not reach)
    s["K"] = _normal(seed, 1, (P, page, Hkv, D), dt, Hkv).view(P, page // 16, 16, Hkv, D // 8, 8)
    s["K"] = s["K"].permute(0, 3, 1, 4, 2, 5).contiguous()
    s["V"] = _normal(seed, 2, (P, page, Hkv, D), dt, Hkv).view(P, page // 8, 8, Hkv, D).permute(0, 3, 1, 4, 2).contiguous()
    if kind == "append":  # q, k and v are slices of one projection's rows
        qkv = _normal(seed, 3, (n, Hq + 2 * Hkv, D), dt, Hq + 2 * Hkv)
        s["q"], s["k"], s["v"] = qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:]
        freqs = 10000.0 ** (-torch.arange(0, D, 2, dtype=torch.float64, device=DEV) / D)
        ang = torch.arange(max(lens), dtype=torch.float64, device=DEV)[:, None] * freqs
        s["rope"] = torch.stack((ang.cos(), ang.sin())).float()
        s["q_out"] = torch.empty(n, Hq, D, dtype=dt, device=DEV)
        return s
    s["q"] = _normal(seed, 3, (n, Hq, D), dt, Hq)
    s["gate"] = torch.rand(n, Hq, generator=_gen(seed, 4), device=DEV) if case["gated"] else None
    s["O"] = torch.empty(n, Hq * D, dtype=dt, device=DEV)
    s["max_new"], s["max_len"] = max(new), max(lens)
    return s


# ------------------------------------------------------------------------------------------------ run


def run(s: dict):
    kind = s["kind"]
    if own:
        root = str(Path(__file__).resolve().parents[1] / "turbo-roformer_amd")
        if root not in sys.path:
            sys.path.insert(0, root)
        from turbo_roformer_amd import _hip

        if kind == "plan":
            _hip.page_plan(s["state"], s["n_new"], s["pool"], s["table"], s["page"], s["state_out"], s["starts"], s["slots"],
                           s["positions"])
            return {k: s[k] for k in ("state_out", "starts", "slots", "positions", "table")}
        if kind == "release":
            _hip.page_release(s["state"], s["done"], s["pool"], s["table"], s["page"], s["state_out"])
            return {k: s[k] for k in ("state_out", "pool")}
        if kind == "append":
            _hip.paged_append(s["k"], s["v"], s["K"], s["V"], s["slots"], s["positions"], s["rope"], s["q"], s["q_out"])
            return {k: s[k] for k in ("q_out", "K", "V")}
        _hip.paged_attention(s["q"], s["K"], s["V"], s["table"], s["starts"], s["lens"], s["O"], causal=s["causal"],
                             window=s["window"], gate=s["gate"], max_new=s["max_new"], max_len=s["max_len"])
        return s["O"]
    return dict(plan=_plan, release=_release, append=_append, attn=_attention)[kind](s)


def _plan(s: dict) -> dict:
    state, page, table = s["state"].long(), s["page"], s["table"]
    R, max_pages = table.shape
    n = s["slots"].numel()
    free, length, new = state[0], state[2:].clamp(0, max_pages * page), s["n_new"].long().clamp(min=0)
    end = new.cumsum(0)
    begin = end - new
    have = (length + page - 1) // page
    want = (length + new + page - 1) // page - have
    fits = (end <= n) & (length + new <= max_pages * page)
    upto = (want * fits).cumsum(0)
    ok = fits & ((want == 0) | (upto <= free))
    given = want * ok
    j = torch.arange(max_pages, device=DEV) - have[:, None]
    at = (free - 1 - (upto - want)[:, None] - j).clamp(0, s["pool"].numel() - 1)
    table.copy_(torch.where((j >= 0) & (j < given[:, None]), s["pool"][at], table))
    row = torch.arange(n, device=DEV)
    r = torch.searchsorted(end, row, right=True)
    live = r < R
    r = r.clamp(max=R - 1)
    pos = torch.where(live & ok[r], length[r] + row - begin[r], -1)
    slot = torch.where(pos >= 0, table[r, pos.clamp(min=0) // page] * page + pos % page, -1)
    s["state_out"].copy_(torch.cat(((free - given.sum())[None], (~ok & (new > 0)).sum()[None], length + new * ok)))
    s["starts"].copy_(torch.cat((torch.zeros_like(end[:1]), end)).clamp(max=n))
    s["slots"].copy_(slot)
    s["positions"].copy_(pos)
    return {k: s[k] for k in ("state_out", "starts", "slots", "positions", "table")}


def _release(s: dict) -> dict:
    state, page, table, pool = s["state"].long(), s["page"], s["table"], s["pool"]
    max_pages, n_pages = table.shape[1], pool.numel()
    free, length = state[0], state[2:].clamp(0, max_pages * page)
    gone = (length + page - 1) // page * s["done"]
    upto = gone.cumsum(0)
    j = torch.arange(max_pages, device=DEV)
    to = torch.where(j < gone[:, None], free + (upto - gone)[:, None] + j, n_pages).clamp(max=n_pages)
    pool.copy_(torch.cat((pool, pool[:1])).scatter(0, to.reshape(-1), table.reshape(-1))[:n_pages])
    s["state_out"].copy_(torch.cat(((free + upto[-1]).clamp(max=n_pages)[None], state[1:2] * 0, length * ~s["done"])))
    return {k: s[k] for k in ("state_out", "pool")}


def _turned(x: torch.Tensor, rope: torch.Tensor, pos: torch.Tensor) -> torch.Tensor:
    """Feature pairs (2i, 2i + 1) of x [n, heads, D] turned by the table's angles at pos, in 32 bits."""
    c, sn = (t[pos.long()][:, None] for t in rope)
    a, b = x[..., 0::2].float(), x[..., 1::2].float()
    return torch.stack((a * c - b * sn, a * sn + b * c), -1).flatten(-2).to(x.dtype)


def _append(s: dict) -> dict:
    slot, page = s["slots"].long(), s["page"]
    n, kv, D = s["k"].shape
    pg, at = slot // page, slot % page
    k = _turned(s["k"], s["rope"], s["positions"])
    s["K"][pg, :, at // 16, :, at % 16] = k.reshape(n, kv, D // 8, 8)
    s["V"][pg, :, at // 8, :, at % 8] = s["v"]
    s["q_out"].copy_(_turned(s["q"], s["rope"], s["positions"]))
    return {k: s[k] for k in ("q_out", "K", "V")}


def _attention(s: dict) -> torch.Tensor:
    page, (R, P) = s["page"], s["table"].shape
    n, Hq, D = s["q"].shape
    kv, L, new = s["kv"], P * page, s["max_new"]
    group = Hq // kv
    table = s["table"].long().clamp(min=0)
    # every request's rows side by side, padded to the longest
    k = s["K"][table].float().permute(0, 2, 1, 3, 5, 4, 6).reshape(R, kv, L, D)  # [R][P][kv][g][D/8][16][8]
    v = s["V"][table].float().permute(0, 2, 1, 3, 5, 4).reshape(R, kv, L, D)  # [R][P][kv][page/8][D][8]
    starts, lens = s["starts"].long(), s["lens"].long()
    i = torch.arange(new, device=DEV)
    q = s["q"].float()[(starts[:-1, None] + i).clamp(max=n - 1)].view(R, new, kv, group, D).permute(0, 2, 1, 3, 4)
    w = torch.matmul(q.reshape(R, kv, new * group, D), k.transpose(2, 3).contiguous()).mul_(D**-0.5)
    p = (lens - (starts[1:] - starts[:-1]))[:, None, None] + i[:, None]  # [R][new][1]
    key = torch.arange(L, device=DEV)
    seen = key < lens[:, None, None]
    if s["causal"]:
        seen = seen & (key <= p)
    if s["window"]:
        seen = seen & (key > p - s["window"])
    w = w.view(R, kv, new, group, L).masked_fill_(~seen[:, None, :, None, :], -math.inf)
    w = w.sub_(w.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)).exp_()
    total = w.sum(-1, keepdim=True)
    o = torch.matmul(w.view(R, kv, new * group, L), v).view(R, kv, new, group, D)
    o = torch.where(total > 0, o / total, 0.0).permute(0, 2, 1, 3, 4).reshape(R, new, Hq, D)
    row = torch.arange(n, device=DEV)
    r = torch.searchsorted(starts[1:], row, right=True)
    o = o[r, row - starts[r]]
    if s["gate"] is not None:
        o = o * s["gate"][:, :, None]
    s["O"].copy_(o.reshape(n, Hq * D))
    return s["O"]


# ------------------------------------------------------------------------------------------------ work


def _seen(case: dict) -> tuple[int, int]:
    """(keys that some row of a request sees, pairs of a row and a key that it sees), over all requests."""
    keys = pairs = 0
    for length, new in _lengths(case):
        p = np.arange(length - new, length, dtype=np.int64)
        hi = p + 1 if case["causal"] else np.full_like(p, length)
        lo = np.maximum(0, p - case["window"] + 1) if case["window"] else np.zeros_like(p)
        if new:
            keys += int(hi.max() - lo.min())
            pairs += int(np.maximum(hi - lo, 0).sum())
    return keys, pairs


def work(case: dict) -> dict:
    R, kind = case["requests"], case["kind"]
    pairs = _lengths(case)
    rows = sum(p[1] for p in pairs)
    page = case["page"]
    if kind == "plan":
        deals = sum(-(-(a + b) // page) + (-a // page) for a, b in pairs)
        # state and counts in, state and starts out; a row's slot and position; a page read from the pool, into the table
        return dict(bytes=16 * R + 8 * rows + 8 * deals, flops=0)
    if kind == "release":
        each = sum(-(-a // page) for a, _ in pairs) / R
        return dict(bytes=9 * R + 8 * each * max(1, round(case["done"] * R)), flops=0)
    D, Hq, Hkv = case["dim"], case["heads"], case["kv"]
    if kind == "append":
        turned = rows * (Hq + Hkv) * D
        angles = 8 * (D // 2) * min(rows, max(a + b for a, b in pairs))  # each table row that is used, once
        return dict(bytes=2 * 2 * (turned + rows * Hkv * D) + 8 * rows + angles, flops=3 * turned)
    keys, seen = _seen(case)
    bytes_ = 2 * 2 * keys * Hkv * D + 2 * 2 * rows * Hq * D + 4 * keys / page + (4 * rows * Hq if case["gated"] else 0) + 8 * R
    return dict(bytes=bytes_, flops=4.0 * D * Hq * seen)


# ------------------------------------------------------------------------------------------------ 64 bits


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    kind, page = case["kind"], case["page"]
    if kind == "plan":
        return _plan64(s)
    if kind == "release":
        return _release64(s)
    if kind == "append":
        D = case["dim"]
        slot, pos = s["slots"].cpu().numpy().astype(np.int64), s["positions"].long()
        # row-major copies of the cache [slot, kv, D], written there and laid out again
        K = s["K"].double().permute(0, 2, 4, 1, 3, 5).reshape(-1, case["kv"], D)
        V = s["V"].double().permute(0, 2, 4, 1, 3).reshape(-1, case["kv"], D)
        at = torch.from_numpy(slot).to(DEV)

        def turn(x):
            z = torch.view_as_complex(x.double().reshape(*x.shape[:2], D // 2, 2).contiguous())
            unit = torch.complex(s["rope"][0].double(), s["rope"][1].double())[pos]
            return torch.view_as_real(z * unit[:, None, :]).reshape(x.shape)

        K[at], V[at] = turn(s["k"]), s["v"].double()
        P = s["n_pages"]
        return dict(q_out=turn(s["q"]), K=K.view(P, page // 16, 16, case["kv"], D // 8, 8).permute(0, 3, 1, 4, 2, 5).contiguous(),
                    V=V.view(P, page // 8, 8, case["kv"], D).permute(0, 3, 1, 4, 2).contiguous())
    if work(case)["flops"] > 5e11:
        return None
    return _attention64(s)


def _plan64(s: dict) -> dict:
    """The same deal, request by request on the host."""
    state, new, table = s["state"].tolist(), s["n_new"].tolist(), s["table"].cpu().numpy().copy()
    pool, page = s["pool"].tolist(), s["page"]
    R, max_pages = table.shape
    n = s["slots"].numel()
    free, refused, lens, starts, slots, positions = state[0], 0, [], [0], [-1] * n, [-1] * n
    row = owed = 0
    for r in range(R):
        length, more = min(max(state[2 + r], 0), max_pages * page), max(new[r], 0)
        have, need = -(-length // page), -(-(length + more) // page)
        room = row + more <= n and length + more <= max_pages * page
        owed += need - have if room else 0
        if room and (need == have or owed <= state[0]):
            for j in range(have, need):
                free -= 1
                table[r, j] = pool[free]
            for i in range(more):
                positions[row + i] = length + i
                slots[row + i] = int(table[r, (length + i) // page]) * page + (length + i) % page
            length += more
        else:
            refused += more > 0
        lens.append(length)
        row += more
        starts.append(min(row, n))
    whole = dict(state_out=[free, refused, *lens], starts=starts, slots=slots, positions=positions)
    return dict({k: np.array(v, dtype=np.int64) for k, v in whole.items()}, table=table.astype(np.int64))


def _release64(s: dict) -> dict:
    state, done, table, pool, page = s["state"].tolist(), s["done"].tolist(), s["table"].tolist(), s["pool"].tolist(), s["page"]
    free, lens = state[0], list(state[2:])
    for r, d in enumerate(done):
        if d:
            for p in table[r][:-(-lens[r] // page)]:
                pool[free] = p
                free += 1
            lens[r] = 0
    return dict(state_out=np.array([free, 0, *lens], dtype=np.int64), pool=np.array(pool, dtype=np.int64))


def _attention64(s: dict) -> torch.Tensor:
    """Request by request and head by head: softmax by its definition in 64 bits."""
    page, D, Hq, kv = s["page"], s["dim"], s["heads"], s["kv"]
    K = s["K"].permute(0, 2, 4, 1, 3, 5).reshape(-1, kv, D)  # [slot, kv, D]
    V = s["V"].permute(0, 2, 4, 1, 3).reshape(-1, kv, D)
    starts, lens, table = s["starts"].tolist(), s["lens"].tolist(), s["table"].long()
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    for r, length in enumerate(lens):
        a, b = starts[r], starts[r + 1]
        key = torch.arange(length, device=DEV)
        at = table[r, key // page] * page + key % page
        pos = torch.arange(length - (b - a), length, device=DEV)[:, None]
        hidden = torch.zeros(b - a, length, dtype=torch.bool, device=DEV)
        if s["causal"]:
            hidden |= key > pos
        if s["window"]:
            hidden |= pos - key >= s["window"]
        for g in range(kv):
            k, v = K[at, g].double(), V[at, g].double()
            for h in range(g * (Hq // kv), (g + 1) * (Hq // kv)):
                score = (s["q"][a:b, h].double() @ k.T.contiguous()) / math.sqrt(D)
                score[hidden] = -math.inf
                out[a:b, h] = torch.softmax(score, -1).nan_to_num(0.0) @ v
    if s["gate"] is not None:
        out *= s["gate"].double()[:, :, None]
    return out.reshape(out.shape[0], -1)
