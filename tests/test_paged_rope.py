"""The paged cache's table of angles at far positions."""

from __future__ import annotations

import math

import pytest
import torch

from turbo_roformer_amd import paged, stack


@pytest.mark.parametrize("dim", (64, 128))
def test_angles_of_far_positions(dim):
    """Every value within half a step of fp32 (2^-25 below one), and 2^-40 for the 64-bit angle and function."""
    freqs = (10000.0 ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim)).float()
    n = 131_072
    table = paged.rope_table(freqs, n)
    assert table.shape == (2, n, dim // 2) and table.dtype is torch.float32
    for p in (0, 1, 1701, 65_537, 100_003, n - 1):
        for i in (0, 1, dim // 4, dim // 2 - 1):
            a = p * float(freqs[i])
            assert abs(float(table[0, p, i]) - math.cos(a)) <= 2.0**-25 + 2.0**-40
            assert abs(float(table[1, p, i]) - math.sin(a)) <= 2.0**-25 + 2.0**-40


def test_it_is_the_stacks_table_at_a_chunks_positions():
    """p * freq rounded to 24 bits is off by half a step, 2^-24 of the angle, which is below 1701; each value by 2^-24 more."""
    freqs = (10000.0 ** (-torch.arange(0, 64, 2, dtype=torch.float64) / 64)).float()
    diff = (paged.rope_table(freqs, 1701).double() - stack.rope_table(freqs, 1701).double()).abs()
    assert float(diff.max()) <= 2.0**-24 * 1701 + 2.0**-23
