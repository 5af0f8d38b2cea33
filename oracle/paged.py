"""The paged K/V cache in plain form: pages dealt request by request, rows written one by one, softmax by its
definition in 64 bits.  For tests only; everything is on the CPU."""

from __future__ import annotations

import math

import torch

Tensor = torch.Tensor


def plan(state, n_new, pool, table, page: int, n_rows: int, max_length: int | None = None) -> dict[str, Tensor]:
    """The deal of ``trf_page_plan_limited``: state_out, starts, slots, positions and table (a copy)."""
    R, max_pages = table.shape
    longest = max_pages * page if max_length is None else max_length
    n_pages = pool.numel()
    table = table.clone()
    free = min(max(int(state[0]), 0), n_pages)
    left, refused, owed, row = free, 0, 0, 0
    starts, lens = [0], []
    slots, positions = torch.full((n_rows,), -1, dtype=torch.int32), torch.full((n_rows,), -1, dtype=torch.int32)
    for r in range(R):
        n, length = max(int(n_new[r]), 0), min(max(int(state[2 + r]), 0), max_pages * page)
        have, need = -(-length // page), -(-(length + n) // page)
        fits = row + n <= n_rows and length + n <= longest
        owed += need - have if fits else 0
        if fits and (need == have or owed <= free):
            for j in range(have, need):
                left -= 1
                table[r, j] = pool[left]
            for i in range(n):
                p = length + i
                positions[row + i] = p
                pg = int(table[r, p // page])
                if 0 <= pg < n_pages:
                    slots[row + i] = pg * page + p % page
            length += n
        else:
            refused += n > 0
        row += n
        starts.append(min(row, n_rows))
        lens.append(length)
    ints = dict(dtype=torch.int32)
    return dict(state_out=torch.tensor([left, refused, *lens], **ints), starts=torch.tensor(starts, **ints), slots=slots,
                positions=positions, table=table)


def release(state, done, pool, table, page: int) -> dict[str, Tensor]:
    """``trf_page_release``: state_out and pool (a copy)."""
    max_pages = table.shape[1]
    pool = pool.clone()
    free = min(max(int(state[0]), 0), pool.numel())
    lens = [min(max(int(n), 0), max_pages * page) for n in state[2:]]
    for r, d in enumerate(done.tolist()):
        if d:
            for j in range(-(-lens[r] // page)):
                if free < pool.numel():
                    pool[free] = table[r, j]
                    free += 1
            lens[r] = 0
    return dict(state_out=torch.tensor([free, 0, *lens], dtype=torch.int32), pool=pool)


def rotate(x: Tensor, rope: Tensor, positions: Tensor) -> Tensor:
    """Pairs (2i, 2i + 1) of x [n, heads, D] turned by the table's angles, in 64 bits."""
    c, s = (rope[i].double()[positions.long()][:, None] for i in (0, 1))
    a, b = x[..., 0::2].double(), x[..., 1::2].double()
    return torch.stack((a * c - b * s, a * s + b * c), -1).flatten(-2)


def k_rows(K: Tensor) -> Tensor:
    """K [pages, heads, page / 16, D / 8, 16, 8] as rows [slot, heads, D]."""
    pages, heads, groups, chunks = K.shape[:4]
    return K.permute(0, 2, 4, 1, 3, 5).reshape(pages * groups * 16, heads, chunks * 8)


def v_rows(V: Tensor) -> Tensor:
    """V [pages, heads, page / 8, D, 8] as rows [slot, heads, D]."""
    pages, heads, octets, dim = V.shape[:4]
    return V.permute(0, 2, 4, 1, 3).reshape(pages * octets * 8, heads, dim)


def attention(q, K, V, table, starts, lens, scale: float | None = None, causal: bool = True, window: int = 0,
              gate: Tensor | None = None) -> tuple[Tensor, Tensor, Tensor]:
    """(O [n, heads, D], the same with |V|, the number of keys of each row [n, heads] and of its largest
    scale * sum |q| |k|), in 64 bits: what ``trf_paged_attention`` gives, and what bounds its rounding.  Rows of no
    request are NaN."""
    page = K.shape[2] * 16
    n, heads, D = q.shape
    kv = K.shape[1]
    scale = D**-0.5 if scale is None else scale
    kr, vr = k_rows(K), v_rows(V)
    out = torch.full((n, heads, D), math.nan, dtype=torch.float64)
    mag, size = torch.zeros_like(out), torch.zeros(n, heads, 2, dtype=torch.float64)
    n_pages, cap = K.shape[0], table.shape[1] * page
    for r in range(table.shape[0]):
        a = min(max(int(starts[r]), 0), n)
        b = min(max(int(starts[r + 1]), a), n)
        length = min(max(int(lens[r]), 0), cap)
        key = torch.arange(length)
        pg = table[r, key // page].long()
        real = (pg >= 0) & (pg < n_pages)
        at = torch.where(real, pg, 0) * page + key % page
        for i in range(b - a):
            p = length - (b - a) + i
            seen = real.clone()
            if causal:
                seen &= key <= p
            if window:
                seen &= key > p - window
            for h in range(heads):
                g = h // (heads // kv)
                k, v = kr[at[seen], g].double(), vr[at[seen], g].double()
                qi = q[a + i, h].double()
                w = torch.softmax(scale * (k @ qi), 0)
                f = 1.0 if gate is None else float(gate[a + i, h])
                out[a + i, h] = f * (w @ v)
                finite = torch.nan_to_num(v.abs(), posinf=0.0)
                mag[a + i, h] = abs(f) * (w @ finite)
                size[a + i, h, 0] = seen.sum()
                if seen.any():
                    size[a + i, h, 1] = scale * (k.abs() @ qi.abs()).max()
    return out, mag, size
