"""Eviction where K and V hold NaN or blocks of scale NaN: what the kept rows and their neighbours are, bit
for bit."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from _cache8 import quantised, scale_for, values
from flour_amd import ops

pytestmark = pytest.mark.gpu

E, I = torch.float8_e4m3fn, torch.int8
BF, HF, F = torch.bfloat16, torch.float16, torch.float32


def i32(x, device):
    return torch.tensor(x, dtype=torch.int32, device=device)


def case(G, bs, L, keep, seed):
    """A source and a destination table, and weights in whose order every position is listed, most of them
    (of one head other ones) kept."""
    gen = torch.Generator().manual_seed(seed)
    nb, nd = (L + bs - 1) // bs, (keep + bs - 1) // bs
    perm = torch.randperm(nb + nd + 2, generator=gen).tolist()
    w = torch.rand((1, G, L), generator=gen) + 0.1
    w[0, 0, ::4] = 0.01  # positions that head 0 gives up
    return gen, nb + nd + 2, perm[:nb], perm[nb:nb + nd], w


@pytest.mark.parametrize("dtype", [BF, HF, F])
@pytest.mark.parametrize("bs,D", [(16, 64), (16, 128), (5, 20)])
def test_a_nan_stays_in_its_row(device, bs, D, dtype):
    """A NaN in a kept row of K and one in a row that is given up: the destination holds exactly the kept
    rows' bits."""
    G, L, keep = 2, 90, 60
    gen, blocks, src, dst, w = case(G, bs, L, keep, 3)
    kp = torch.randn((G, blocks * bs, D), generator=gen).to(dtype).to(device)
    vp = torch.randn((G, blocks * bs, D), generator=gen).to(dtype).to(device)

    def slot(p):
        return src[p // bs] * bs + p % bs

    w[0, :, 37] = 5.0  # kept by both heads
    w[0, :, 40] = 0.0  # by none
    kp[1, slot(37), 3] = float("nan")
    kp[0, slot(40), 1] = float("nan")
    vp[0, slot(37)] = float("inf")
    before = [x.clone() for x in (kp, vp)]
    kept = ops.kv_evict(kp, vp, w.to(device), i32([src], device), i32([L], device), i32([keep], device),
                        i32([dst], device), L, keep, 0, bs)
    bits = {2: torch.int16, 4: torch.int32}[dtype.itemsize]
    for x, old in zip((kp, vp), before):
        want = old.clone()
        for g in range(G):
            pos = kept[0, g].tolist()
            assert 37 in pos and 40 not in pos
            for i, p in enumerate(pos):
                want[g, dst[i // bs] * bs + i % bs] = old[g, slot(p)]
        assert torch.equal(x.view(bits), want.view(bits))


@pytest.mark.parametrize("bs,D", [(16, 64), (16, 40), (80, 64)])
@pytest.mark.parametrize("pool", [E, I])
def test_a_poisoned_block_poisons_its_rows_blocks_alone(device, pool, bs, D):
    """One source block of scale NaN in K, another in V: the destination blocks that take a row of it have
    the scale NaN, all others the scale and the bits that their rows come to."""
    G, L, keep = 2, 4 * bs, 3 * bs
    gen, blocks, src, dst, w = case(G, bs, L, keep, 4)
    b = torch.randint(0, 256, (2, G, blocks * bs, D), generator=gen).to(torch.uint8)
    b[(b & 127) == 127] = 6
    b[b == 128] = 2
    kv = b.view(pool).to(device)
    s = torch.exp2(torch.randint(-4, 5, (2, G, blocks), generator=gen).float()).to(device)
    s[0, 0, src[1]] = float("nan")
    s[1, 1, src[3]] = float("nan")
    old_s, old_q = s.cpu().double().numpy().copy(), values(kv)
    kept = ops.kv_evict(kv[0], kv[1], w.to(device), i32([src], device), i32([L], device),
                        i32([keep], device), i32([dst], device), L, keep, 0, bs, k_scale=s[0],
                        v_scale=s[1])
    got_s, got_q = s.cpu().double().numpy(), values(kv)
    poisoned = 0
    for x in range(2):
        for g in range(G):
            pos = kept[0, g].tolist()
            for lb in range(keep // bs):
                p = np.array(pos[lb * bs:(lb + 1) * bs])
                from_blocks = np.array(src)[p // bs]
                sc = old_s[x, g, from_blocks]
                if np.isnan(sc).any():
                    assert np.isnan(got_s[x, g, dst[lb]])
                    poisoned += 1
                    continue
                rows = old_q[x, g, from_blocks * bs + p % bs] * sc[:, None]
                S = scale_for(float(np.abs(rows).max()), pool)
                assert got_s[x, g, dst[lb]] == S
                to = got_q[x, g, dst[lb] * bs:(dst[lb] + 1) * bs]
                assert np.array_equal(to, quantised(rows, S, pool))
    assert 2 <= poisoned < 2 * G * (keep // bs)
