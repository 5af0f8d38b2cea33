"""The paged attention's weights in fp16: what the type's range holds of a long tail, and of the largest scores."""

from __future__ import annotations

import math

import pytest
import torch

from turbo_roformer_amd import _hip

from .test_gpu_paged import BF, HF

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _shared_pages(k, v, R, rows, heads, q, dtype, page=256):
    """R requests of `rows` rows each over the same n positions k, v [n, D], with q for all rows and heads; one K/V head.
    Enough requests that no keys are split."""
    n, D = k.shape
    pages = -(-n // page)
    K, V = _hip.paged_cache(pages, page, 1, D, dtype, DEV)
    kk, vv = (torch.zeros(pages * page, D, dtype=dtype) for _ in range(2))
    kk[:n], vv[:n] = k, v
    K.copy_(kk.view(pages, page // 16, 16, 1, D // 8, 8).permute(0, 3, 1, 4, 2, 5))
    V.copy_(vv.view(pages, page // 8, 8, 1, D).permute(0, 3, 1, 4, 2))
    table = torch.arange(pages, dtype=torch.int32, device=DEV).repeat(R, 1)
    starts = torch.arange(R + 1, dtype=torch.int32, device=DEV) * rows
    O = torch.empty(R * rows, heads * D, dtype=dtype, device=DEV)
    qq = q.to(dtype).expand(R * rows, heads, D).contiguous().to(DEV)
    assert _hip.paged_attention_workspace_bytes(heads, K, V, R, pages, R * rows, rows, n) == 0
    _hip.paged_attention(qq, K, V, table, starts, torch.full((R,), n, dtype=torch.int32, device=DEV), O, scale=1.0, causal=False,
                         max_new=rows, max_len=n)
    torch.cuda.synchronize()
    return O.cpu().view(R * rows * heads, D)


@pytest.mark.parametrize("D", (64, 128))
@pytest.mark.parametrize("rows,heads", [(1, 1), (40, 1), (300, 4)])
def test_a_tail_of_small_weights_is_kept(hip, D, rows, heads):
    """One key in front and 131,071 behind it with 2^-26 of its weight each: 2^-9 of the sum.  P is 2^(s - m + 7) in fp16,
    off by up to 2^-25 where it is subnormal, which is 2^-32 of the key in front: 2^-32 keys of the output in all.  The rest
    as in test_gpu_paged.py: half a step of the output, half a step of the P that are normal, fp32's
    e = 2^-24 (keys + 4 D score + 64) of sum(w |v|)."""
    n, score = 131_072, 18.03125  # exp(-score) is 2^-26.01
    k, v, q = torch.zeros(n, D, dtype=HF), torch.ones(n, D, dtype=HF), torch.zeros(D, dtype=HF)
    k[0, 0], q[0], v[0] = 1.0, score, 0.0
    got = _shared_pages(k, v, 172 if rows < 300 else 31, rows, heads, q, HF).double()
    w = math.exp(-score)
    want = (n - 1) * w / (1 + (n - 1) * w)
    u = torch.finfo(HF).eps / 2
    tol = 2 * u * want + 2.0**-25 + 2.0**-32 * n + 2.0**-24 * (n + 4 * D * score + 64) * want
    assert float((got - want).abs().max()) <= tol, (float(got.min()), float(got.max()), want, tol)


@pytest.mark.parametrize("D", (64, 128))
@pytest.mark.parametrize("rows,heads", [(1, 1), (40, 1), (300, 4)])
def test_the_weights_of_a_tail_add_to_one(hip, D, rows, heads):
    """The sum that divides is that of the rounded weights that are applied, subnormal ones too: ones come out as ones (P.V
    and the sum differ by 2^-24 of each of a few thousand additions, and one's half step is 2^-12 below it)."""
    n = 131_072
    k, q = torch.zeros(n, D, dtype=HF), torch.zeros(D, dtype=HF)
    k[0, 0], q[0] = 1.0, 18.03125
    got = _shared_pages(k, torch.ones(n, D, dtype=HF), 172 if rows < 300 else 31, rows, heads, q, HF)
    assert bool((got == 1).all()), (float(got.min()), float(got.max()))


@pytest.mark.parametrize("dtype", (BF, HF))
@pytest.mark.parametrize("rows,heads", [(1, 1), (40, 1), (300, 4)])
def test_scores_of_millions(hip, dtype, rows, heads):
    """Scores of 2^15 .. 2^23 in steps of 2^15, rising, falling and mixed: the row is the one key's values, to the last bit
    (P v / P is v but for a few 2^-24, which no rounding to 16 bits shows)."""
    n, D = 256, 64
    g = torch.Generator().manual_seed(rows)
    q, v = torch.zeros(D, dtype=dtype), torch.randn(n, D, generator=g).to(dtype)
    q[0] = 2048.0
    for order in (torch.arange(n), torch.arange(n - 1, -1, -1), torch.randperm(n, generator=g)):
        k = torch.zeros(n, D, dtype=dtype)
        k[:, 0] = (16.0 * (order + 1)).to(dtype)
        got = _shared_pages(k, v, 172 if rows < 300 else 31, rows, heads, q, dtype)
        assert bool((got == v[int(order.argmax())]).all())
