"""Sums of attention weights where scores are no numbers."""
from __future__ import annotations

import pytest
import torch

from flour_amd import ops

pytestmark = pytest.mark.gpu

I = torch.int8
BF, HF, F = torch.bfloat16, torch.float16, torch.float32


def i32(x, device):
    return torch.tensor(x, dtype=torch.int32, device=device)


@pytest.mark.parametrize("pool", [BF, HF, F, I])
@pytest.mark.parametrize("D,bs", [(128, 16), (64, 16), (96, 16), (20, 5)])
def test_a_nan_score_makes_its_heads_sums_nan_and_no_others(device, pool, D, bs):
    """One K row of NaN (in 8 bits a block) in kv head 0 of sequence 0: its positions' sums are NaN and stay
    so, those of the other head, of the other sequence and behind the end are as without it. The eviction
    takes such sums as the lowest: the first positions and the latest stay."""
    G, H, lens = 2, 4, [40, 33]
    gen = torch.Generator().manual_seed(31)
    nb = [(n + bs - 1) // bs for n in lens]
    blocks = sum(nb)
    tab = [list(range(nb[0])), list(range(nb[0], blocks)) + [-1] * (nb[0] - nb[1])]
    q = torch.randn((2, H, D), generator=gen).to(pool if pool != I else BF).to(device)
    if pool == I:
        k, v = (torch.randint(-100, 100, (G, blocks * bs, D), generator=gen).to(I).to(device) for _ in "kv")
        s = torch.full((G, blocks), 2.0 ** -6, device=device)
        bad = s.clone()
        bad[0, 1] = float("nan")
    else:
        k, v = (torch.randn((G, blocks * bs, D), generator=gen).to(pool).to(device) for _ in "kv")
        bad = k.clone()
        bad[0, bs + 2, 3] = float("nan")
    args = (i32(tab, device), i32(lens, device), 0.1, max(lens))

    def step(x, w):
        if pool == I:
            ops.paged_decode_q8(q, k, v, x, s, *args, bs, weights=w)
        else:
            ops.paged_decode_weights(q, x, v, *args, w, bs)

    start = torch.rand((2, G, 45), generator=gen).to(device)
    clean, w = start.clone(), start.clone()
    step(s if pool == I else k, clean)
    assert torch.isfinite(clean).all()
    step(bad, w)
    assert torch.isnan(w[0, 0, :40]).all()
    w[0, 0, :40] = clean[0, 0, :40]
    assert torch.equal(w, clean)
    w[0, 0, :40] = float("nan")
    step(s if pool == I else k, w)
    assert torch.isnan(w[0, 0, :40]).all() and not torch.isnan(w[:, 1]).any()
    new = i32([[0, 1, 2, 3, 4, 5, 6, 7]] * 2, device) + blocks  # (ids outside the pool: positions only)
    kept = ops.kv_evict(k, v, w, *args[:2], i32([9, 9], device), new, 40, 9, 4, bs,
                        **(dict(k_scale=s, v_scale=s) if pool == I else {}))
    assert kept[0, 0].tolist() == [0, 1, 2, 3, 4, 36, 37, 38, 39]
