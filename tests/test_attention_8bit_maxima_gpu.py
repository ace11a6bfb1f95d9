"""Attention over a cache in 8 bits where rows' maxima lie around the lag of the running ones: weights up to the most that
f16 is meant to hold, and references that have to move."""
from __future__ import annotations

import math

import pytest
import torch

from test_attention_8bit_gpu import BF, DEV, E4M3, E8M0, F32, check, exact, i32, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("gap", [7.5, 8.0, 8.0625, 8.5, 8.9375, 9.0, 9.5, 16.5])
@pytest.mark.parametrize("T,dtype,d,raised", [(1, BF, 128, 0), (1, BF, 64, 5), (3, BF, 128, 60), (1, F32, 128, 0), (2, F32, 64, 7), (2, BF, 96, 3)])
def test_later_keys_score_higher_by_about_the_lag(T, dtype, d, raised, gap):
    """The first 128 keys score 0, half of the later ones `gap` in powers of two; `raised`: by how many powers the later
    blocks of v are larger."""
    B, H, Hkv, page, block, n = 2, 8, 4, 32, 16, 700
    M = -(-n // page)
    g = torch.Generator(device=DEV).manual_seed(11)
    k = torch.zeros(B * M, Hkv, page, d, device=DEV)
    later = k.view(B, M, Hkv, page, d)[:, 4:]
    later[..., ::2, 0] = 1.0
    v = torch.randint(-448, 449, k.shape, generator=g, device=DEV).float()
    ks, vs = (torch.full((B * M, Hkv, page // block), 120, dtype=torch.uint8, device=DEV) for _ in range(2))
    vs.view(B, M, Hkv, -1)[:, 4:] += raised
    q = torch.zeros(B, T, H, d, device=DEV, dtype=dtype)
    q[..., 0] = gap * 128  # exact; k's powers are 2^-7
    new = torch.zeros(B, T, Hkv, d, device=DEV, dtype=dtype)
    x = (q, new, new, k.to(E4M3), v.to(E4M3), torch.arange(B * M, device=DEV).view(B, M).int(), i32([n, n - 333]), ks.view(E8M0), vs.view(E8M0))
    check(run(x, None, math.log(2)), *exact(x, None, math.log(2)), dtype)
