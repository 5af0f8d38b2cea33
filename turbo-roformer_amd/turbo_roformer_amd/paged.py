"""A paged K/V cache for attention over frames that arrive piece by piece, on the gfx950 kernels.

``HipPagedCache`` owns what a program that serves such sequences keeps between steps: the K and V pages, the page
table, the pool of free pages and the requests' lengths, all on the device.  The stack's time attention has a sequence
per band, so a live stereo stream of a 62-band model is 62 requests.  A step of new rows is

    step = cache.plan(n_new, rows)                    # pages, row starts, slots and positions
    q = cache.append(step, q, k, v, rope)             # rotate, write K and V, rotated q
    O = cache.attend(step, q, gate=G)                 # the rows over their requests' positions
    ...
    cache.release(done)                               # finished requests give their pages back

Lengths stay on the device: nothing here waits for it, and a step can be captured in a graph and replayed.  Work runs
on the current stream of the cache's device, which has to be the current device; one step at a time per cache.  There
is no CPU fallback: construction raises ``HipUnavailable`` without the HIP library or a gfx950 GPU.
"""

from __future__ import annotations

from dataclasses import dataclass

import torch

from . import _hip

Tensor = torch.Tensor


def rope_table(freqs: Tensor, positions: int) -> Tensor:
    """[2, positions, head dim / 2] fp32 (cos, sin) of angle p * freq_i, formed in 64 bits.  ``stack.rope_table`` forms the
    angles in 32, as the reference does for its chunks: past 65,536 positions it is off by up to 0.004, half a step of
    bf16's."""
    ang = torch.arange(positions, dtype=torch.float64)[:, None] * freqs.detach().double().cpu()[None, :]
    return torch.stack((ang.cos(), ang.sin())).float()


@dataclass
class PageStep:
    """Where the rows of one step go: ``starts`` [requests + 1] (first row of each request), and for each row its ``slots``
    and ``positions`` (-1: no place), with ``max_new``, the caller's bound on a request's rows."""

    starts: Tensor
    slots: Tensor
    positions: Tensor
    max_new: int


class HipPagedCache:
    """K/V pages of ``requests`` sequences of at most ``max_length`` positions; ``pages``: how many there are in all (None:
    enough for every request at its longest)."""

    def __init__(self, requests: int, max_length: int, kv_heads: int = _hip.HEADS, head_dim: int = _hip.HEAD_DIM,
                 pages: int | None = None, page_size: int = 64, dtype: torch.dtype = torch.bfloat16,
                 device: str | torch.device = "cuda"):
        if requests < 1 or max_length < 1:
            raise ValueError(f"requests and max_length must be >= 1, got {requests} and {max_length}")
        _hip.load_native()
        self.device = torch.device(device)
        self.page_size = page_size
        self.max_length = max_length
        self.max_pages = -(-max_length // page_size) if page_size > 0 else 0
        self.pages = requests * self.max_pages if pages is None else pages
        self.K, self.V = _hip.paged_cache(self.pages, page_size, kv_heads, head_dim, dtype, self.device)
        self.table = torch.full((requests, self.max_pages), -1, dtype=torch.int32, device=self.device)
        self.pool = torch.arange(self.pages, dtype=torch.int32, device=self.device)
        self.state = torch.zeros(2 + requests, dtype=torch.int32, device=self.device)
        self.state[:1] = self.pages
        self._planned, self._released = torch.zeros_like(self.state), torch.zeros_like(self.state)

    @property
    def lengths(self) -> Tensor:
        """Positions that each request holds [requests], on the device."""
        return self.state[2:]

    @property
    def free_pages(self) -> int:
        """Pages in the pool (waits for the device)."""
        return int(self.state[0])

    @property
    def refused(self) -> int:
        """Requests that the last ``plan`` refused, for want of pages, of rows or of length (waits for the device); a
        ``release`` since then does not change it."""
        return int(self._planned[1])

    def plan(self, n_new: Tensor, rows: int, max_new: int | None = None) -> PageStep:
        """Deal pages for ``n_new`` [requests] int32 more rows of each request, ``rows`` of them in all or more (the rest is
        padding); ``max_new``: a bound on a request's rows (None: ``rows``), past which ``attend`` may leave rows out."""
        ints = dict(dtype=torch.int32, device=self.device)
        step = PageStep(torch.empty(self.table.shape[0] + 1, **ints), torch.empty(rows, **ints), torch.empty(rows, **ints),
                        rows if max_new is None else max_new)
        _hip.page_plan(self.state, n_new, self.pool, self.table, self.page_size, self._planned, step.starts, step.slots,
                       step.positions, self.max_length)
        self.state.copy_(self._planned)
        return step

    def append(self, step: PageStep, q: Tensor | None, k: Tensor, v: Tensor, rope: Tensor | None = None) -> Tensor | None:
        """Write the step's rows k and v [rows, kv heads, head dim] to the cache, k rotated by ``rope`` [2, P, head dim / 2]
        with P at least ``max_length``; returns q [rows, heads, head dim] rotated (rows without a place are not written)."""
        if rope is not None and rope.dim() == 3 and rope.shape[1] < self.max_length:
            raise ValueError(f"rope has {rope.shape[1]} positions, the cache's requests have up to {self.max_length}")
        out = None if q is None else torch.empty(q.shape, dtype=q.dtype, device=q.device)
        _hip.paged_append(k, v, self.K, self.V, step.slots, step.positions, rope, q, out)
        return out

    def attend(self, step: PageStep, q: Tensor, scale: float | None = None, causal: bool = True, window: int = 0,
               gate: Tensor | None = None, out: Tensor | None = None, max_length: int | None = None) -> Tensor:
        """The step's rows q (rotated) over their requests' positions -> [rows, heads * head dim]; see
        ``_hip.paged_attention``.  Padding rows of a new ``out`` are not written.  ``max_length``: a bound on the requests'
        lengths (None: the cache's)."""
        O = out if out is not None else torch.empty(q.shape[0], q.shape[1] * q.shape[2], dtype=q.dtype, device=q.device)
        _hip.paged_attention(q, self.K, self.V, self.table, step.starts, self.lengths, O, scale, causal, window, gate,
                             step.max_new, max_length)
        return O

    def release(self, done: Tensor) -> None:
        """Take the pages of the requests with ``done`` [requests] (bool) back; their lengths become 0."""
        _hip.page_release(self.state, done, self.pool, self.table, self.page_size, self._released)
        self.state.copy_(self._released)
