"""The paged K/V cache beside the model's own time attention: the same sequences, whole chunk and piece by piece."""

from __future__ import annotations

import math

import pytest
import torch

from oracle import paged
from turbo_roformer_amd import _hip
from turbo_roformer_amd.paged import HipPagedCache

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("T", (70, 700))
def test_pieces_of_a_chunk_attend_as_the_models_time_attention(hip, T):
    """Both against the definition in 64 bits: bf16's half step of the output, and of P for each."""
    F, H, D = 3, 8, 64
    g = torch.Generator().manual_seed(T)
    q, k, v = (torch.randn(F, T, H, D, generator=g).to(torch.bfloat16) for _ in range(3))
    gate = torch.rand(F, T, H, generator=g)
    # the model's buffers: q.k is a power of two's exponent there, so its scale is ln 2
    Q, K, Vt, G = _hip.seq_buffers(0, 1, T, F, DEV)
    O = torch.empty(T * F, H * D, dtype=torch.bfloat16, device=DEV)
    for buf, x in ((Q, q), (K, k)):
        buf.zero_()
        buf[:, :, :, :T] = x.permute(0, 2, 3, 1).reshape(F, H, 8, 8, T).permute(0, 1, 2, 4, 3).to(DEV)
    Vt.zero_()
    Vt[..., :T] = v.permute(0, 2, 3, 1).to(DEV)
    G.copy_(gate.permute(1, 0, 2).reshape(G.shape))
    _hip.attention(Q, K, Vt, G, O, 0, 1, T, F)
    whole = O.view(T, F, H, D).permute(1, 0, 2, 3).cpu()

    # K and V come in two pieces, and all rows attend at once
    cache = HipPagedCache(F, T + 5, H, D, page_size=16)
    cut = T // 3
    for a, b in ((0, cut), (cut, T)):
        step = cache.plan(torch.full((F,), b - a, dtype=torch.int32, device=DEV), F * (b - a), b - a)
        cache.append(step, None, *(x[:, a:b].reshape(-1, H, D).to(DEV) for x in (k, v)))
    starts = torch.arange(F + 1, dtype=torch.int32, device=DEV) * T
    out = torch.empty(F * T, H * D, dtype=torch.bfloat16, device=DEV)
    _hip.paged_attention(q.reshape(-1, H, D).to(DEV), cache.K, cache.V, cache.table, starts, cache.lengths, out, math.log(2.0),
                         causal=False, gate=gate.reshape(-1, H).to(DEV), max_new=T, max_len=T)
    torch.cuda.synchronize()
    pieces = out.view(F, T, H, D).cpu()

    page = -(-T // 16) * 16
    rows = [torch.zeros(F, page, H, D, dtype=torch.bfloat16) for _ in range(2)]
    rows[0][:, :T], rows[1][:, :T] = k, v
    want = paged.attention(q[:, :8].reshape(-1, H, D), rows[0].view(F, page // 16, 16, H, 8, 8).permute(0, 3, 1, 4, 2, 5),
                           rows[1].view(F, page // 8, 8, H, D).permute(0, 3, 1, 4, 2), torch.arange(F)[:, None],
                           torch.arange(F + 1) * 8, torch.full((F,), T), math.log(2.0), False, 0, gate[:, :8].reshape(-1, H))
    o, mag, size = (x.view(F, 8, H, -1) for x in want)
    u = torch.finfo(torch.bfloat16).eps / 2
    tol = u * o.abs() + (u + 2.0**-24 * (T + 4 * D * size[..., 1:] + 64)) * mag
    assert bool(((pieces[:, :8].double() - o).abs() <= tol).all())
    assert bool(((whole[:, :8].double() - o).abs() <= tol).all())
    # every row: each side by its half steps of |O| and of sum(w |v|), which the gate and the largest |v| bound, and fp32's
    # 2^-24 (T + 4 D 60 + 64), below 2^-10 for scores whose sum |q| |k| ln 2 is 60 at most
    most = 2 * (u * whole.double().abs() * (1 + 2 * u) + (u + 2.0**-10) * gate[..., None] * v.double().abs().max())
    assert bool(((pieces.double() - whole.double()).abs() <= most).all())
