"""New rows behind rows whose block has a scale that a caller chose."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from _cache8 import scale_for, to8, values
from flour_amd import ops

pytestmark = pytest.mark.gpu

E, I = torch.float8_e4m3fn, torch.int8


def i32(x, device):
    return torch.tensor(x, dtype=torch.int32, device=device)


@pytest.mark.parametrize("D", [64, 20])
@pytest.mark.parametrize("pool", [E, I])
def test_write_behind_rows_of_any_scale(device, pool, D):
    """One row behind five of a block: its scale becomes the stored one's next power of two or what the new
    row needs; -0 is 0, subnormal scales become 2^-126."""
    bs, kept = 16, 5
    olds = [0.0, -0.0, 1.0, 1.5, 0.75, 3e-39, 2.0 ** -126, 2.0 ** 126, 1.5 * 2.0 ** 126, 2.0 ** 127]
    G, n = 1, len(olds)
    gen = torch.Generator().manual_seed(41)
    b = torch.randint(0, 256, (2, G, n * bs, D), generator=gen).to(torch.uint8)
    b[(b & 127) == 127] = 9
    b[b == 128] = 7
    for new_mag in (1e-3, 100.0, 1e38):
        kv = b.clone().view(pool).to(device)
        s = torch.tensor(olds, dtype=torch.float64).float().view(1, 1, n).repeat(2, G, 1).to(device)
        x = (new_mag * (torch.rand((n, G, D), generator=gen) + 0.5)).to(device)
        before = values(kv).reshape(2, n, bs, D)
        ops.kv_write_q8(x, x, kv[0], kv[1], s[0], s[1], i32(list(range(n + 1)), device),
                        i32([kept + 1] * n, device), i32([[i] for i in range(n)], device), bs)
        got_s, got = s.cpu().double().numpy(), values(kv).reshape(2, n, bs, D)
        for i, old in enumerate(olds):
            old = float(np.float32(old))
            row = x[i, 0].cpu().double().numpy()
            mine = max(2.0 ** math.ceil(math.log2(old)), 2.0 ** -126) if old > 0 else 0.0
            S = max(mine, scale_for(float(np.abs(row).max()), pool))
            assert (got_s[:, 0, i] == S).all(), (old, new_mag)
            for z in range(2):
                assert np.array_equal(got[z, i, :kept], to8(before[z, i, :kept] * (old / S), pool))
                assert np.array_equal(got[z, i, kept], to8(row / S, pool)), (old, new_mag)
                assert np.array_equal(got[z, i, kept + 1:], before[z, i, kept + 1:])
