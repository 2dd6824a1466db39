"""The 8-bit cache on the GPU: the quantising write and the way back bit for bit, decode, prefill and
the sums of attention weights within the bounds of fp32 arithmetic, against tests/_cache8.py."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from _cache8 import Cache, attend, close, values
from flour_amd import ops
from flour_amd._lib import ERR_INVALID_ARGUMENT, ERR_UNSUPPORTED, FlourError, lib

pytestmark = pytest.mark.gpu

E, I = torch.float8_e4m3fn, torch.int8
BF, HF, F = torch.bfloat16, torch.float16, torch.float32


def i32(x, device):
    return torch.tensor(x, dtype=torch.int32, device=device)


def tables(lens, bs, blocks, gen, extra=0):
    """Disjoint random tables of sequences of `lens` positions, padded with ids outside the pool."""
    perm = torch.randperm(blocks, generator=gen).tolist()
    width = max((n + bs - 1) // bs for n in lens) + extra
    rows, at = [], 0
    for n in lens:
        nb = (n + bs - 1) // bs
        rows.append(perm[at:at + nb] + [2 ** 31 - 1, -1][:width - nb] + [-7] * (width - nb - 2))
        at += nb
    assert at <= blocks
    return rows


def random_pool(G, blocks, bs, D, dtype, gen, device, scales="pow2"):
    """An 8-bit pool of every byte but e4m3's NaN, and its scales."""
    b = torch.randint(0, 256, (G, blocks * bs, D), generator=gen).to(torch.uint8)
    if dtype == E:
        b[(b & 127) == 127] = 5
        b &= 0xBF  # |values| < 2: mixed magnitudes without a few that decide everything
    else:
        b[b == 128] = 1
    e = torch.randint(-7, -4, (G, blocks), generator=gen).float() + (5 if dtype == E else 0)
    s = torch.exp2(e)
    if scales == "any":
        s *= 1 + torch.rand((G, blocks), generator=gen)
        s[:, ::7] = 0.0
    return b.view(dtype).to(device), s.to(device)


def packed(x):
    cu = [0]
    for n in x:
        cu.append(cu[-1] + n)
    return cu


# ------------------------------------------------------------------ write
WRITES = [  # (G, D, bs, [(rows, kv)])
    (2, 128, 16, [(1, 1), (1, 16), (1, 17), (1, 40), (33, 33), (20, 30), (0, 9), (0, 0)]),
    (3, 64, 16, [(48, 48), (16, 32), (5, 100)]),
    (1, 128, 32, [(1, 31), (1, 33), (64, 70)]),
    (2, 20, 16, [(7, 9), (1, 3), (30, 31)]),
    (2, 72, 5, [(1, 6), (11, 13), (1, 5)]),
    (2, 256, 16, [(17, 35)]),
    (1, 8, 1, [(3, 5), (1, 1)]),
]


@pytest.mark.parametrize("shape", range(len(WRITES)))
@pytest.mark.parametrize("dtype", [BF, HF, F])
@pytest.mark.parametrize("pool", [E, I])
def test_write_bits(device, pool, dtype, shape):
    G, D, bs, seqs = WRITES[shape]
    gen = torch.Generator().manual_seed(shape)
    rows, lens = [n for n, _ in seqs], [kv for _, kv in seqs]
    blocks = sum((n + bs - 1) // bs for n in lens) + 3
    tab = tables(lens, bs, blocks, gen)
    kp, ks = random_pool(G, blocks, bs, D, pool, gen, device)
    vp, vs = random_pool(G, blocks, bs, D, pool, gen, device)
    T = sum(rows)
    # magnitudes from far below the blocks' present scales to far above
    mag = torch.exp2(torch.randint(-12, 6, (T, G, 1), generator=gen).float())
    k = (torch.randn((T, G, D), generator=gen) * mag).to(dtype).to(device)
    v = (torch.randn((T, G, D), generator=gen) * mag).to(dtype).to(device)
    v[: T // 2] = 0  # blocks of zeros
    want = [Cache(kp, ks, bs), Cache(vp, vs, bs)]
    cu = packed(rows)
    for w, x in zip(want, (k, v)):
        for s, (n, kv) in enumerate(seqs):
            w.write(x[cu[s]:cu[s + 1]].cpu().double().numpy(), tab[s], kv)
    before = [kp.clone(), vp.clone()]
    if shape == 0:  # the reference's head-major rows
        k = k.transpose(0, 1).contiguous().transpose(0, 1)
        v = v.transpose(0, 1).contiguous().transpose(0, 1)
    ops.kv_write_q8(k, v, kp, vp, ks, vs, i32(cu, device), i32(lens, device), i32(tab, device), bs)
    torch.cuda.synchronize()
    for w, p, s, old in zip(want, (kp, vp), (ks, vs), before):
        assert np.array_equal(s.cpu().double().numpy(), w.s)
        assert np.array_equal(values(p).reshape(w.q.shape), w.q)
    # blocks that no sequence writes keep their bytes, and so do the rows behind a sequence's last
    touched = torch.zeros(blocks * bs, dtype=torch.bool)
    for s, (n, kv) in enumerate(seqs):
        for j in range((kv - n) // bs * bs if n else kv, kv):
            touched[tab[s][j // bs] * bs + j % bs] = True
    for p, old in zip((kp, vp), before):
        a, b = p.view(torch.uint8).cpu()[:, ~touched], old.view(torch.uint8).cpu()[:, ~touched]
        assert torch.equal(a, b)


@pytest.mark.parametrize("pool", [E, I])
def test_write_non_finite_and_extremes(device, pool):
    G, D, bs = 1, 64, 16
    kp = torch.zeros((G, 4 * bs, D), dtype=torch.int8, device=device).view(pool)
    vp, ks = kp.clone(), torch.ones((G, 4), device=device)
    vs = ks.clone()
    x = torch.ones((3 * bs, G, D), device=device)
    x[3, 0, 5] = float("nan")
    x[bs + 1, 0, 0] = float("-inf")
    x[2 * bs:] = 3.4e38
    y = torch.full((3 * bs, G, D), 1e-45, device=device)
    y[bs:] = 0.0
    tab, cu, kv = i32([[2, 0, 3]], device), i32([0, 3 * bs], device), i32([3 * bs], device)
    ops.kv_write_q8(x, y, kp, vp, ks, vs, cu, kv, tab)
    s = ks[0].cpu()
    assert torch.isnan(s[2]) and torch.isnan(s[0]) and s[1] == 1.0
    # 127 * 2^121 = 3.376e38 and 448 * 2^119 = 2.977e38 are below 3.4e38
    assert s[3] == (2.0 ** 122 if pool == I else 2.0 ** 120)
    assert vs[0].cpu().tolist() == [0.0, 1.0, 2.0 ** -126, 0.0]
    # one more row into a poisoned block keeps it so; a fresh start clears it
    one = torch.ones((1, G, D), device=device)
    ops.kv_write_q8(one, one, kp, vp, ks, vs, i32([0, 1], device), i32([5], device), tab)
    assert torch.isnan(ks[0, 2])
    ops.kv_write_q8(one, one, kp, vp, ks, vs, i32([0, 1], device), i32([1], device), tab)
    assert ks[0, 2] == (2.0 ** -6 if pool == I else 2.0 ** -8)


def test_write_skips_what_it_must_not_touch(device):
    """kv < q_len, ids outside the pool, positions past the table, rows past total_q's sequences."""
    G, D, bs = 2, 64, 16
    kp = torch.full((G, 4 * bs, D), 3, dtype=torch.int8, device=device)
    vp, ks = kp.clone(), torch.ones((G, 4), device=device)
    vs = ks.clone()
    x = torch.randn((40, G, D), device=device)
    tab = i32([[0, 1], [-1, 4], [2, 3]], device)
    # sequence 0: kv < rows; 1: bad ids; 2: rows end past its table of two blocks
    ops.kv_write_q8(x, x, kp, vp, ks, vs, i32([0, 10, 20, 40], device), i32([9, 20, 50], device),
                    tab)
    assert (kp[:, :2 * bs] == 3).all() and (ks[:, :3] == 1).all() and (kp[:, 2 * bs:3 * bs] == 3).all()
    assert (ks[:, 3] == 1).all()  # its new rows start at position 30: block 3's rows 14 and 15
    assert not (kp[:, 3 * bs + 14:] == 3).all() and (kp[:, 3 * bs:3 * bs + 14] == 3).all()


# ------------------------------------------------------------------ read back
@pytest.mark.parametrize("dtype", [BF, HF, F])
@pytest.mark.parametrize("pool", [E, I])
@pytest.mark.parametrize("D,bs", [(128, 16), (20, 16), (64, 5)])
def test_dequant(device, D, bs, pool, dtype):
    gen = torch.Generator().manual_seed(D)
    G, lens = 2, [1, 0, 33, 16]
    blocks = sum((n + bs - 1) // bs for n in lens) + 1
    kp, ks = random_pool(G, blocks, bs, D, pool, gen, device, "any")
    vp, vs = random_pool(G, blocks, bs, D, pool, gen, device)
    tab, out_tab = tables(lens, bs, blocks, gen), tables(lens, bs, blocks + 2, gen)
    ko = torch.full((G, (blocks + 2) * bs, D), 7.0, dtype=dtype, device=device)
    vo = ko.clone()
    ops.kv_dequant(kp, vp, ks, vs, i32(tab, device), i32(lens, device), ko, vo,
                   i32(out_tab, device), max(lens), bs)
    for p, s, o in ((kp, ks, ko), (vp, vs, vo)):
        c, want = Cache(p, s, bs), np.full(o.shape, 7.0)
        for t, ot, n in zip(tab, out_tab, lens):
            for j, row in enumerate(c.rows(t, n)):
                want[:, ot[j // bs] * bs + j % bs] = row
        w = torch.from_numpy(want).float().to(dtype)  # products of two fp32 rounded to fp32 first
        assert torch.equal(o.cpu(), w)


def test_dequant_every_byte_and_f16_saturates(device):
    G, D, bs = 1, 256, 1
    for pool in (E, I):
        b = torch.arange(256, dtype=torch.int32).to(torch.uint8).view(1, 1, 256)
        kp = b.view(pool).to(device)
        s = torch.full((1, 1), 2.0 ** 10, device=device)
        one = i32([[0]], device)
        ko = torch.zeros((1, 1, 256), dtype=HF, device=device)
        vo = torch.zeros_like(ko)
        ops.kv_dequant(kp, kp, s, s, one, i32([1], device), ko, vo, one, 1, bs)
        want = np.clip(values(b.view(pool)) * 1024.0, -65504, 65504)
        assert np.array_equal(ko.cpu().double().numpy(), want, equal_nan=True)


# ------------------------------------------------------------------ decode
DECODES = [  # (H, G, D, bs, context lengths)
    (8, 2, 128, 16, [1, 0, 15, 16, 17, 64, 33]),
    (14, 2, 64, 16, [100, 31, 1]),
    (4, 4, 64, 16, [5, 700]),
    (32, 8, 128, 16, [1030]),
    (28, 4, 128, 16, [65, 2, 129]),
    (16, 1, 128, 32, [40, 90]),
    (17, 1, 64, 16, [37]),
    (6, 3, 128, 48, [100, 47]),
    (4, 2, 96, 16, [50, 3]),
    (2, 1, 20, 5, [23, 4]),
    (4, 2, 256, 16, [33]),
    (2, 2, 64, 8, [19, 70]),
]


def decode_case(shape, pool, dtype, device, scales="pow2"):
    H, G, D, bs, lens = DECODES[shape]
    gen = torch.Generator().manual_seed(100 + shape)
    blocks = sum((n + bs - 1) // bs for n in lens) + 2
    tab = tables(lens, bs, blocks, gen, extra=1)
    kp, ks = random_pool(G, blocks, bs, D, pool, gen, device, scales)
    vp, vs = random_pool(G, blocks, bs, D, pool, gen, device, scales)
    q = torch.randn((len(lens), H, D), generator=gen).to(dtype).to(device)
    # positions behind a sequence's end hold NaN bytes (e4m3) and whatever else
    if pool == E:
        flat = kp.view(torch.uint8), vp.view(torch.uint8)
        for t, n in zip(tab, lens):
            if n % bs:
                lo = t[n // bs] * bs + n % bs
                for f in flat:
                    f[:, lo:lo + bs - n % bs] = 127
    return q, kp, vp, ks, vs, tab, lens, bs


def want_decode(q, kp, vp, ks, vs, tab, lens, bs, scale):
    """(output, bound, weights (b, G, L), their bound) in 64 bits."""
    ck, cv, G = Cache(kp, ks, bs), Cache(vp, vs, bs), kp.shape[0]
    B, H, D = q.shape
    out, bound = np.zeros((B, H, D)), np.zeros((B, H, D))
    w, wb = np.zeros((B, G, max(lens))), np.zeros((B, G, max(lens)))
    for b, n in enumerate(lens):
        if n == 0:
            continue
        k, v = ck.rows(tab[b], n), cv.rows(tab[b], n)
        o, p, err = attend(q[b:b + 1].cpu().double().numpy(), k, v, scale)
        out[b], p = o[0], p[0]
        big = np.abs(v).max()
        bound[b] = 2 * err[0][:, None] * big
        w[b, :, :n] = p.reshape(G, H // G, n).sum(1)
        wb[b, :, :n] = (p * 2 * err[0][:, None]).reshape(G, H // G, n).sum(1) + 2.0 ** -40
    return out, bound, w, wb


@pytest.mark.parametrize("shape", range(len(DECODES)))
@pytest.mark.parametrize("dtype", [BF, HF, F])
@pytest.mark.parametrize("pool", [E, I])
def test_decode(device, pool, dtype, shape):
    q, kp, vp, ks, vs, tab, lens, bs = decode_case(shape, pool, dtype, device,
                                                   "any" if shape % 2 else "pow2")
    scale = q.shape[2] ** -0.5
    want, bound, w, wb = want_decode(q, kp, vp, ks, vs, tab, lens, bs, scale)
    args = (q, kp, vp, ks, vs, i32(tab, device), i32(lens, device), scale, max(lens), bs)
    ws = ops.Workspace(device)
    for out_dtype in {F, dtype}:
        close(ops.paged_decode_q8(*args, out_dtype=out_dtype, workspace=ws), want, bound)
    # the same with the weights added to sums, twice
    sums = torch.rand((len(lens) + 1, kp.shape[0], max(lens) + 3), device=device)
    before = sums.cpu().double().numpy()
    for _ in range(2):
        out = ops.paged_decode_q8(*args, out_dtype=F, workspace=ws, weights=sums)
    close(out, want, bound)
    after = before.copy()
    after[:len(lens), :, :max(lens)] += 2 * w
    wbound = np.zeros_like(before)
    wbound[:len(lens), :, :max(lens)] = 2 * wb + 2.0 ** -23 * after[:len(lens), :, :max(lens)]
    close(sums, after, wbound)
    for b, n in enumerate(lens):  # nothing behind a sequence's end, nothing in the spare row
        assert np.array_equal(sums[b, :, n:].cpu().double().numpy(), before[b, :, n:])
    assert np.array_equal(sums[len(lens)].cpu().double().numpy(), before[len(lens)])


@pytest.mark.parametrize("shape", [0, 1, 3, 5, 6, 8, 9])
@pytest.mark.parametrize("dtype", [BF, HF, F])
def test_decode_weights_over_plain_pools(device, dtype, shape):
    H, G, D, bs, lens = DECODES[shape]
    gen = torch.Generator().manual_seed(200 + shape)
    blocks = sum((n + bs - 1) // bs for n in lens) + 2
    tab = tables(lens, bs, blocks, gen, extra=1)
    kp = torch.randn((G, blocks * bs, D), generator=gen).to(dtype).to(device)
    vp = torch.randn((G, blocks * bs, D), generator=gen).to(dtype).to(device)
    q = torch.randn((len(lens), H, D), generator=gen).to(dtype).to(device)
    scale = D ** -0.5
    rows = list(range(len(lens), 0, -1))
    rows[0] = len(lens) + 5  # no such row
    if len(rows) > 2:
        rows[2] = -1
    sums = torch.rand((len(lens) + 1, G, max(lens)), device=device)
    before = sums.cpu().double().numpy()
    out = ops.paged_decode_weights(q, kp, vp, i32(tab, device), i32(lens, device), scale, max(lens),
                                   sums, bs, out_dtype=F, weight_rows=i32(rows, device))
    after, wbound = before.copy(), np.zeros_like(before)
    for b, n in enumerate(lens):
        o, bound = np.zeros((1, H, D)), np.zeros((1, H, D))
        if n:
            j = np.arange(n)
            at = np.array(tab[b])[j // bs] * bs + j % bs
            k, v = (p.cpu().double().numpy()[:, at].transpose(1, 0, 2) for p in (kp, vp))
            o, p, err = attend(q[b:b + 1].cpu().double().numpy(), k, v, scale)
            bound[0] = 2 * err[0][:, None] * np.abs(v).max()
            if 0 <= rows[b] <= len(lens):
                add = p[0].reshape(G, H // G, n)
                after[rows[b], :, :n] += add.sum(1)
                wbound[rows[b], :, :n] = (add * 2 * err[0].reshape(G, -1, 1)).sum(1) + 2.0 ** -22
        close(out[b:b + 1], o, bound)
    close(sums, after, wbound)


@pytest.mark.parametrize("shape", [0, 8])
def test_decode_poisoned_block_reaches_only_those_that_attend_to_it(device, shape):
    q, kp, vp, ks, vs, tab, lens, bs = decode_case(shape, I, BF, device)
    b = len(lens) - 1 if lens[-1] > 1 else 0
    args = (kp, vp, ks, vs, i32(tab, device), i32(lens, device), 0.1, max(lens), bs)
    clean = ops.paged_decode_q8(q, *args)
    for s in (ks, vs):
        keep = s.clone()
        s[0, tab[b][0]] = float("nan")
        # blocks that no sequence holds
        used = {x for t, n in zip(tab, lens) for x in t[:(n + bs - 1) // bs]}
        for x in set(range(s.shape[1])) - used:
            s[:, x] = float("nan")
        got = ops.paged_decode_q8(q, *args)
        rep = q.shape[1] // kp.shape[0]
        assert torch.isnan(got[b, :rep]).all()
        got[b, :rep] = clean[b, :rep]
        assert torch.equal(got, clean)
        s.copy_(keep)


@pytest.mark.parametrize("dtype", [BF, F])
def test_decode_range_of_scales(device, dtype):
    """Blocks whose V scales lie 2^60 apart, the heaviest position in the smallest, one block of
    zeros: each weight still counts."""
    H, G, D, bs, n = 4, 2, 64, 16, 64
    gen = torch.Generator().manual_seed(3)
    kp, ks = random_pool(G, 4, bs, D, I, gen, device)
    vp, vs = random_pool(G, 4, bs, D, I, gen, device)
    vs[:] = torch.tensor([2.0 ** -50, 0.0, 2.0 ** 10, 1.0], device=device)
    vp[:, bs:2 * bs] = 0
    q = (3 * torch.randn((1, H, D), generator=gen)).to(dtype).to(device)
    tab = [[0, 1, 2, 3]]
    want, bound, _, _ = want_decode(q, kp, vp, ks, vs, tab, [n], bs, 1.0)
    got = ops.paged_decode_q8(q, kp, vp, ks, vs, i32(tab, device), i32([n], device), 1.0, n, bs,
                              out_dtype=F)
    close(got, want, bound)


def test_decode_queries_beyond_f16(device):
    """bf16 and fp32 queries whose elements f16 could not hold."""
    H, G, D, bs, n = 4, 2, 128, 16, 40
    gen = torch.Generator().manual_seed(4)
    kp, ks = random_pool(G, 3, bs, D, E, gen, device)
    vp, vs = random_pool(G, 3, bs, D, E, gen, device)
    for dtype in (BF, F):
        for mag in (1e20, 1e-20):
            q = (mag * torch.randn((1, H, D), generator=gen)).to(dtype).to(device)
            scale = 0.1 / mag
            want, bound, _, _ = want_decode(q, kp, vp, ks, vs, [[0, 1, 2]], [n], bs, scale)
            got = ops.paged_decode_q8(q, kp, vp, ks, vs, i32([[0, 1, 2]], device),
                                      i32([n], device), scale, n, bs, out_dtype=F)
            close(got, want, bound)
    q = torch.zeros((1, H, D), dtype=BF, device=device)  # all scores alike
    want, bound, _, _ = want_decode(q, kp, vp, ks, vs, [[0, 1, 2]], [n], bs, 1.0)
    close(ops.paged_decode_q8(q, kp, vp, ks, vs, i32([[0, 1, 2]], device), i32([n], device), 1.0,
                              n, bs, out_dtype=F), want, bound)
    q[0, 1, 3] = float("nan")
    got = ops.paged_decode_q8(q, kp, vp, ks, vs, i32([[0, 1, 2]], device), i32([n], device), 1.0, n)
    assert torch.isnan(got[0, 1]).all() and not torch.isnan(got[0, [0, 2, 3]]).any()


def test_decode_context_clamped_and_offsets_past_32_bits(device):
    """max_context_len bounds the contexts; a pool of more than 2^32 elements a pool."""
    H, G, D, bs = 2, 2, 128, 16
    blocks = (1 << 32) // (G * bs * D) + 64
    kp = torch.zeros((G, blocks * bs, D), dtype=torch.int8, device=device)
    vp = torch.zeros_like(kp)
    ks = torch.ones((G, blocks), device=device)
    gen = torch.Generator().manual_seed(5)
    tab = [[blocks - 1, 3, blocks // 2 + 7]]
    small_k, _ = random_pool(G, 3, bs, D, I, gen, device)
    small_v, _ = random_pool(G, 3, bs, D, I, gen, device)
    for i, b in enumerate(tab[0]):
        kp[:, b * bs:(b + 1) * bs] = small_k[:, i * bs:(i + 1) * bs]
        vp[:, b * bs:(b + 1) * bs] = small_v[:, i * bs:(i + 1) * bs]
    s3 = torch.ones((G, 3), device=device)
    q = torch.randn((1, H, D), generator=gen).to(BF).to(device)
    want, bound, _, _ = want_decode(q, small_k, small_v, s3, s3, [[0, 1, 2]], [40], bs, 0.001)
    got = ops.paged_decode_q8(q, kp, vp, ks, ks, i32(tab, device), i32([47], device), 0.001, 40)
    close(got, want, bound)
    x = torch.randn((4, G, D), generator=gen).to(BF).to(device)
    c = Cache(small_k, s3, bs)
    c.write(x.cpu().double().numpy(), [0, 1, 2], 47)
    ops.kv_write_q8(x, x, kp, vp, ks, torch.ones_like(ks), i32([0, 4], device), i32([47], device),
                    i32(tab, device))
    b = tab[0][2]
    assert np.array_equal(values(kp[:, b * bs:(b + 1) * bs]), c.q[:, 2])
    del kp, vp


# ------------------------------------------------------------------ prefill
PREFILLS = [  # (H, G, D, bs, [(rows, kv)])
    (8, 2, 128, 16, [(1, 1), (5, 40), (0, 12), (17, 17), (3, 2), (2, 100)]),
    (14, 2, 64, 16, [(4, 33), (7, 130)]),
    (28, 4, 128, 16, [(130, 200), (1, 64)]),
    (4, 2, 128, 16, [(300, 300)]),
    (4, 4, 64, 32, [(40, 70), (8, 8)]),
    (6, 2, 96, 16, [(9, 20)]),
    (2, 1, 20, 5, [(6, 13), (2, 2)]),
    (17, 1, 128, 16, [(3, 50)]),
    (16, 2, 128, 16, [(8, 600), (2, 900)]),
]


@pytest.fixture
def prefill_mode():
    """Sets the path of 8-bit prefill (0 by the rule, 1 streamed, 2 staged, 3 the kernel for every
    shape); back to the rule afterwards."""
    yield lib().flour_hip_set_prefill_q8
    lib().flour_hip_set_prefill_q8(0)


@pytest.mark.parametrize("shape", range(len(PREFILLS)))
@pytest.mark.parametrize("dtype", [BF, HF, F])
@pytest.mark.parametrize("pool", [E, I])
@pytest.mark.parametrize("mode", [0, 1, 2])
def test_prefill(device, prefill_mode, mode, pool, dtype, shape):
    prefill_mode(mode)
    H, G, D, bs, seqs = PREFILLS[shape]
    gen = torch.Generator().manual_seed(300 + shape)
    rows, lens = [n for n, _ in seqs], [kv for _, kv in seqs]
    blocks = sum((n + bs - 1) // bs for n in lens) + 2
    tab = tables(lens, bs, blocks, gen, extra=1)
    kp, ks = random_pool(G, blocks, bs, D, pool, gen, device)
    vp, vs = random_pool(G, blocks, bs, D, pool, gen, device)
    q = torch.randn((sum(rows), H, D), generator=gen).to(dtype).to(device)
    if shape % 2:  # head-major
        q = q.transpose(0, 1).contiguous().transpose(0, 1)
    scale, cu = D ** -0.5, packed(rows)
    ck, cv = Cache(kp, ks, bs), Cache(vp, vs, bs)
    want, bound = np.zeros((sum(rows), H, D)), np.zeros((sum(rows), H, D))
    for s, (n, kv) in enumerate(seqs):
        if n and kv >= n:
            k, v = ck.rows(tab[s], kv), cv.rows(tab[s], kv)
            o, _, err = attend(q[cu[s]:cu[s + 1]].cpu().double().numpy(), k, v, scale)
            want[cu[s]:cu[s + 1]] = o
            # longer calls over 16-bit queries round each probability to f16 once (2^-11)
            p_eps = 2.0 ** -11 if dtype != F else 0.0
            bound[cu[s]:cu[s + 1]] = (2 * err[:, :, None] + p_eps) * np.abs(v).max()
    for out_dtype in {F, dtype}:
        out = torch.full((sum(rows) + 2, H, D), 9.0, dtype=out_dtype, device=device)
        ws = ops.Workspace(device)  # whose bytes are NaN in every type
        ws.get(ops.prefill_q8_workspace_bytes(len(seqs), max(rows), sum(rows), max(lens), H, G, D,
                                              bs, dtype)).fill_(255)
        ops.varlen_prefill_q8(q, kp, vp, ks, vs, i32(cu, device), i32(lens, device),
                              i32(tab, device), max(rows), max(lens), scale, bs,
                              out=out[:sum(rows)], workspace=ws)
        close(out[:sum(rows)], want, bound)
        assert (out[sum(rows):] == 9.0).all()


@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("mode", [1, 2, 3])
@pytest.mark.parametrize("D,bs", [(128, 16), (64, 32)])
def test_prefill_poisoned_block_reaches_only_the_rows_that_see_it(device, prefill_mode, D, bs, mode,
                                                                  dtype):
    H, G, rows, kv = 6, 2, 90, 150
    gen = torch.Generator().manual_seed(11)
    nb = (kv + bs - 1) // bs
    kp, ks = random_pool(G, nb + 1, bs, D, E, gen, device)
    vp, vs = random_pool(G, nb + 1, bs, D, E, gen, device)
    q = torch.randn((rows, H, D), generator=gen).to(dtype).to(device)
    tab = torch.randperm(nb, generator=gen).tolist()
    args = (i32([0, rows], device), i32([kv], device), i32([tab], device), rows, kv, 0.1, bs)
    prefill_mode(mode)
    clean = ops.varlen_prefill_q8(q, kp, vp, ks, vs, *args)
    assert not torch.isnan(clean).any()
    for s in (ks, vs):
        for lb in (0, nb // 2 + 1, nb - 1):
            keep = s.clone()
            s[1, tab[lb]] = float("nan")
            got = ops.varlen_prefill_q8(q, kp, vp, ks, vs, *args)
            sees = torch.arange(kv - rows, kv, device=device) >= lb * bs
            assert torch.isnan(got[sees, H // G:]).all()
            got[sees, H // G:] = clean[sees, H // G:]
            s.copy_(keep)
            if mode != 2:
                assert torch.equal(got, clean)
                continue
            # the prefill kernel recomputes an item with an output that is not finite, with each
            # probability in two parts instead of once rounded to f16 (off by at most 2^-11 of the
            # largest |v|, as the weights sum to 1); both results are rounded to the type once
            big = float(np.abs(Cache(vp, vs, bs).rows(tab, kv)).max())
            off = (got.double() - clean.double()).abs()
            assert (off <= 1.01 * 2.0 ** -11 * big + torch.finfo(dtype).eps * clean.double().abs()).all()


@pytest.mark.parametrize("mode", [1, 2])
def test_prefill_and_decode_of_many_sequences(device, prefill_mode, mode):
    """More sequences than a wave has lanes, some empty, some without rows."""
    H, G, D, bs, B = 4, 2, 64, 16, 83
    gen = torch.Generator().manual_seed(12)
    lens = torch.randint(0, 60, (B,), generator=gen).tolist()
    rows = [min(n, int(r)) for n, r in zip(lens, torch.randint(0, 9, (B,), generator=gen))]
    blocks = sum((n + bs - 1) // bs for n in lens) + 1
    tab = tables(lens, bs, blocks, gen)
    kp, ks = random_pool(G, blocks, bs, D, I, gen, device)
    vp, vs = random_pool(G, blocks, bs, D, I, gen, device)
    q = torch.randn((sum(rows), H, D), generator=gen).to(HF).to(device)
    cu, ck, cv = packed(rows), Cache(kp, ks, bs), Cache(vp, vs, bs)
    want, bound = np.zeros(q.shape), np.zeros(q.shape)
    for s, (n, kv) in enumerate(zip(rows, lens)):
        if n:
            k, v = ck.rows(tab[s], kv), cv.rows(tab[s], kv)
            o, _, err = attend(q[cu[s]:cu[s + 1]].cpu().double().numpy(), k, v, 0.125)
            want[cu[s]:cu[s + 1]] = o
            bound[cu[s]:cu[s + 1]] = (2 * err[:, :, None] + 2.0 ** -11) * np.abs(v).max()
    prefill_mode(mode)
    got = ops.varlen_prefill_q8(q, kp, vp, ks, vs, i32(cu, device), i32(lens, device),
                                i32(tab, device), max(rows), max(lens), 0.125, bs)
    close(got, want, bound)
    q = torch.randn((B, H, D), generator=gen).to(HF).to(device)
    sums = torch.zeros((B, G, max(lens)), device=device)
    want, bound, w, wb = want_decode(q, kp, vp, ks, vs, tab, lens, bs, 0.125)
    got = ops.paged_decode_q8(q, kp, vp, ks, vs, i32(tab, device), i32(lens, device), 0.125,
                              max(lens), bs, weights=sums)
    close(got, want, bound)
    close(sums, w, wb)


def test_staged_prefill_in_slices(device, prefill_mode):
    """Six sequences whose bound of 2^20 positions allows four in a staged copy: two slices."""
    H, G, D, bs, B, most = 4, 1, 64, 16, 6, 1 << 20
    gen = torch.Generator().manual_seed(13)
    lens, rows = [40, 33, 500, 7, 64, 130], [40, 2, 70, 7, 0, 129]
    blocks = sum((n + bs - 1) // bs for n in lens)
    tab = tables(lens, bs, blocks, gen)
    wide = torch.full((B, most // bs), -1, dtype=torch.int32)
    for s, t in enumerate(tab):
        wide[s, :len(t)] = torch.tensor(t)
    kp, ks = random_pool(G, blocks, bs, D, E, gen, device)
    vp, vs = random_pool(G, blocks, bs, D, E, gen, device)
    q = torch.randn((sum(rows), H, D), generator=gen).to(BF).to(device)
    nbytes = ops.prefill_q8_workspace_bytes(B, max(rows), sum(rows), most, H, G, D, bs, BF)
    assert nbytes < (1 << 30) + (1 << 25)
    outs = []
    for mode, bound in ((2, max(lens)), (2, most)):
        prefill_mode(mode)
        outs.append(ops.varlen_prefill_q8(q, kp, vp, ks, vs, i32(packed(rows), device),
                                          i32(lens, device), wide.to(device), max(rows), bound, 0.1,
                                          bs))
    assert torch.equal(*outs)


@pytest.mark.parametrize("shape", [0, 1, 2, 4, 5, 7])
@pytest.mark.parametrize("dtype", [BF, F])
def test_decode_by_chunks_of_64(device, dtype, shape):
    """A bound far above the contexts picks the kernel for long ones: the same output and sums."""
    q, kp, vp, ks, vs, tab, lens, bs = decode_case(shape, E, dtype, device, "any")
    want, bound, w, wb = want_decode(q, kp, vp, ks, vs, tab, lens, bs, 0.1)
    wide = torch.zeros((len(lens), 4096 // bs + 1), dtype=torch.int32)
    for s, t in enumerate(tab):
        wide[s, :len(t)] = torch.tensor(t)
    sums = torch.zeros((len(lens), kp.shape[0], 4096), device=device)
    got = ops.paged_decode_q8(q, kp, vp, ks, vs, wide.to(device), i32(lens, device), 0.1, 4096, bs,
                              out_dtype=F, weights=sums)
    close(got, want, bound)
    close(sums[:, :, :max(lens)], w, wb)
    assert (sums[:, :, max(lens):] == 0).all()
    plain = ops.paged_decode_q8(q, kp, vp, ks, vs, wide.to(device), i32(lens, device), 0.1, 4096, bs,
                                out_dtype=F)
    close(plain, want, bound)  # (a kernel of its own: the same within the bound, not bit for bit)


def test_rows_beyond_their_bound_stay_in_bounds(device, prefill_mode):
    """More rows than max_seqlen_q says: nothing is written outside the call's own rows."""
    H, G, D, bs = 4, 2, 64, 16
    gen = torch.Generator().manual_seed(14)
    kp, ks = random_pool(G, 4, bs, D, I, gen, device)
    q = torch.randn((20, H, D), generator=gen).to(BF).to(device)
    prefill_mode(1)
    n = ops.prefill_q8_workspace_bytes(1, 2, 20, 60, H, G, D, bs, BF)
    ws = ops.Workspace(device)
    buf = ws.get(n + 4096)
    buf.fill_(77)
    out = torch.full((22, H, D), 9.0, dtype=BF, device=device)
    ops.varlen_prefill_q8(q, kp, kp, ks, ks, i32([0, 20], device), i32([60], device),
                          i32([[0, 1, 2, 3]], device), 2, 60, 0.1, bs, out=out[:20], workspace=ws)
    torch.cuda.synchronize()
    assert (out[20:] == 9.0).all() and (buf[n:] == 77).all()


@pytest.mark.parametrize("D,bs", [(128, 16), (64, 32), (20, 5)])
@pytest.mark.parametrize("mode", [0, 1, 2, 3])
def test_padded_batch(device, prefill_mode, mode, D, bs):
    """Rows behind the last sequence and empty sequences at the end: the rows are neither written nor
    stored, their blocks and results stay as they were."""
    H, G, T = 4, 2, 64
    gen = torch.Generator().manual_seed(15)
    prefill_mode(mode)
    kp, ks = random_pool(G, 12, bs, D, I, gen, device)
    vp, vs = random_pool(G, 12, bs, D, I, gen, device)
    rows, lens = [3, 6, 0, 0], [bs + 3, 6, 0, 0]
    tab = [[3, 7, -1, -1], [5, 8, -1, -1], [-1] * 4, [-1] * 4]
    cu, n = packed(rows), sum(rows)
    k = torch.randn((T, G, D), generator=gen).to(BF).to(device)
    k[n:] = float("nan")
    q = torch.randn((T, H, D), generator=gen).to(BF).to(device)
    q[n:] = float("nan")
    before = kp.clone()
    ops.kv_write_q8(k, k, kp, vp, ks, vs, i32(cu, device), i32(lens, device), i32(tab, device), bs)
    others = [b for b in range(12) if b not in (3, 7, 5, 8)]
    assert torch.equal(kp.view(G, 12, bs, D)[:, others], before.view(G, 12, bs, D)[:, others])
    assert torch.isfinite(ks).all() and torch.isfinite(vs).all()
    out = torch.full((T, H, D), 9.0, dtype=F, device=device)
    ops.varlen_prefill_q8(q, kp, vp, ks, vs, i32(cu, device), i32(lens, device), i32(tab, device), 8,
                          2 * bs, 0.1, bs, out=out)
    ck, cv = Cache(kp, ks, bs), Cache(vp, vs, bs)
    for s in range(2):
        v = cv.rows(tab[s], lens[s])
        o, _, err = attend(q[cu[s]:cu[s + 1]].cpu().double().numpy(), ck.rows(tab[s], lens[s]), v, 0.1)
        close(out[cu[s]:cu[s + 1]], o, (2 * err[:, :, None] + 2.0 ** -11) * np.abs(v).max())
    assert (out[n:] == 9.0).all()


@pytest.mark.parametrize("D", [128, 64, 20])
@pytest.mark.parametrize("mode", [0, 1, 2, 3])
def test_prefill_strides(device, prefill_mode, mode, D):
    """Queries that are one row for every head (stride 0), and outputs inside larger rows, head by head:
    the bits of the contiguous call, nothing beside them written."""
    H, G, bs, T = 4, 2, 16, 9
    gen = torch.Generator().manual_seed(16)
    prefill_mode(mode)
    kp, ks = random_pool(G, 6, bs, D, E, gen, device)
    row = torch.randn((T, 1, D), generator=gen).to(BF).to(device)
    args = (kp, kp, ks, ks, i32([0, 4, T], device), i32([30, 40], device),
            i32([[0, 3, -1], [5, 1, 2]], device), 5, 40, 0.1, bs)
    want = ops.varlen_prefill_q8(row.expand(T, H, D).contiguous(), *args)
    for shape, view in (((H, T, 2 * D), lambda x: x.transpose(0, 1)[:, :, :D]),
                        ((T, 2 * H, D), lambda x: x[:, H:])):
        buf = torch.full(shape, 9.0, dtype=BF, device=device)
        out = ops.varlen_prefill_q8(row.expand(T, H, D), *args, out=view(buf))
        assert torch.equal(out, want)
        view(buf).fill_(9.0)
        assert (buf == 9.0).all()


@pytest.mark.parametrize("D", [128, 64, 20])
def test_one_sequence_listed_twice(device, D):
    """A sequence's table in two entries of a decode step (two samples of one prompt): equal rows, and each
    entry's weights in its own row."""
    H, G, bs = 8, 2, 16
    gen = torch.Generator().manual_seed(17)
    kp, ks = random_pool(G, 70, bs, D, I, gen, device)
    q = torch.randn((1, H, D), generator=gen).to(BF).to(device).repeat(3, 1, 1)
    tab = torch.randperm(70, generator=gen)[:63].to(torch.int32).to(device).repeat(3, 1)
    w = torch.zeros((4, G, 1000), device=device)
    out = ops.paged_decode_q8(q, kp, kp, ks, ks, tab, i32([1000, 1000, 7], device), 0.1, 1000, bs,
                              out_dtype=F, weights=w, weight_rows=i32([3, 0, 7], device))
    # The scores are the same bits. Cut into other pieces, sums of up to 1,000 terms, 32 or more an instruction,
    # are rounded in another order (up to 32 additions and as many pieces: 64 * 2^-24 of the sum of
    # magnitudes), and weights relative to another reference (2^-20): twice that of |v| < 4; of the
    # denominator alone for the weights, at most H / G a position.
    err = 2 * (64 * 2.0 ** -24 + 2.0 ** -20)
    close(out[1], out[0].cpu().double().numpy(), 4 * err)
    close(w[3], w[0].cpu().double().numpy(), H // G * err)
    assert abs(float(w[0].double().sum()) - H) < H * err
    assert (w[1:3] == 0).all()


# ------------------------------------------------------------------ streams and graphs
def test_decode_captured_and_replayed(device):
    """Two captured steps that share a workspace, replayed among eager calls of their own and of a
    larger step that makes the workspace grow."""
    q, kp, vp, ks, vs, tab, lens, bs = decode_case(0, E, BF, device)
    big = decode_case(3, E, BF, device)
    ws = ops.Workspace(device)
    t, n = i32(tab, device), i32(lens, device)
    sums = torch.zeros((len(lens), kp.shape[0], max(lens)), device=device)
    cu = i32(packed([1] * len(lens)), device)

    def step(w):
        o = ops.paged_decode_q8(q, kp, vp, ks, vs, t, n, 0.09, max(lens), bs, workspace=ws,
                                weights=w)
        p = ops.varlen_prefill_q8(q, kp, vp, ks, vs, cu, n, t, 1, max(lens), 0.09, bs, workspace=ws)
        return o, p

    eager = torch.zeros_like(sums)
    want = step(eager)
    graphs = []
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step(sums)
    torch.cuda.synchronize()
    sums.zero_()
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got = step(sums)
        graphs.append((g, got))
    total = torch.zeros_like(sums)
    for i in range(6):
        g, got = graphs[i % 2]
        for x in got:
            x.fill_(5.0)
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        total += eager
        assert torch.allclose(sums, total, rtol=2.0 ** -20, atol=0)
        ops.paged_decode_q8(big[0], *big[1:5], i32(big[5], device), i32(big[6], device), 0.1,
                            max(big[6]), big[7], workspace=ws,
                            weights=torch.zeros((1, 8, max(big[6])), device=device))
        torch.cuda.synchronize()


def test_two_streams_without_a_workspace(device):
    """Calls without a workspace share no scratch: two streams at once."""
    a, b = decode_case(3, I, HF, device), decode_case(0, E, HF, device)

    def call(c):
        q, kp, vp, ks, vs, tab, lens, bs = c
        w = torch.zeros((len(lens), kp.shape[0], max(lens)), device=device)
        return ops.paged_decode_q8(q, kp, vp, ks, vs, i32(tab, device), i32(lens, device), 0.1,
                                   max(lens), bs, weights=w), w

    want = [call(a), call(b)]
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    got = []
    for _ in range(4):
        with torch.cuda.stream(s1):
            x = call(a)
        with torch.cuda.stream(s2):
            y = call(b)
        got.append((x, y))
    torch.cuda.synchronize()
    for pair in got:
        for g, w in zip(pair, want):
            assert torch.equal(g[0], w[0]) and torch.equal(g[1], w[1])


# ------------------------------------------------------------------ refusals (nothing is launched)
def test_tensor_refusals(device):
    G, D, bs = 2, 64, 16
    kp = torch.zeros((G, 4 * bs, D), dtype=torch.int8, device=device)
    s = torch.ones((G, 4), device=device)
    t, n, cu = i32([[0, 1]], device), i32([20], device), i32([0, 1], device)
    q = torch.zeros((1, 4, D), dtype=BF, device=device)
    x = torch.zeros((1, G, D), dtype=BF, device=device)
    plain = torch.zeros((G, 4 * bs, D), dtype=BF, device=device)
    w = torch.zeros((1, G, 32), device=device)
    bad = [
        lambda: ops.paged_decode_q8(q, plain, plain, s, s, t, n, 1.0, 32),
        lambda: ops.paged_decode_q8(q, kp, kp, s[:, :3], s, t, n, 1.0, 32),
        lambda: ops.paged_decode_q8(q, kp, kp, s.double(), s, t, n, 1.0, 32),
        lambda: ops.paged_decode_q8(q, kp, kp, s, s.cpu(), t, n, 1.0, 32),
        lambda: ops.paged_decode_q8(q[:, :3], kp, kp, s, s, t, n, 1.0, 32),
        lambda: ops.paged_decode_q8(q, kp, kp, s, s, t, n, 1.0, 33),  # beyond the table
        lambda: ops.paged_decode_q8(q, kp, kp, s, s, t.long(), n, 1.0, 32),
        lambda: ops.paged_decode_q8(q, kp, kp, s, s, t, i32([20, 3], device), 1.0, 32),
        lambda: ops.paged_decode_q8(q, kp, kp, s, s, t, n, 1.0, 32, block_size=24),
        lambda: ops.paged_decode_q8(q, kp, kp, s, s, t, n, 1.0, 32, weights=w[:, :, :31]),
        lambda: ops.paged_decode_q8(q, kp, kp, s, s, t, n, 1.0, 32, weights=w[:0]),
        lambda: ops.paged_decode_q8(q, kp, kp, s, s, t, n, 1.0, 32, weight_rows=n),
        lambda: ops.paged_decode_q8(q.to(torch.float64), kp, kp, s, s, t, n, 1.0, 32),
        lambda: ops.paged_decode_weights(q, plain, plain, t, n, 1.0, 32, None),
        lambda: ops.paged_decode_weights(q.half(), plain, plain, t, n, 1.0, 32, w),
        lambda: ops.paged_decode_weights(q, kp, kp, t, n, 1.0, 32, w),
        lambda: ops.kv_write_q8(x, x[:, :1], kp, kp, s, s, cu, n, t),
        lambda: ops.kv_write_q8(x, x.half(), kp, kp, s, s, cu, n, t),
        lambda: ops.kv_write_q8(x, x, kp, kp, s, s, cu, i32([1, 2], device), t),
        lambda: ops.kv_write_q8(x, x, plain, plain, s, s, cu, n, t),
        lambda: ops.kv_dequant(kp, kp, s, s, t, n, plain, plain, t, 40),
        lambda: ops.kv_dequant(kp, kp, s, s, t, n, plain[:1], plain[:1], t, 32),
        lambda: ops.kv_dequant(kp, kp, s, s, t, n, kp, kp, t, 32),
        lambda: ops.varlen_prefill_q8(q, kp, kp, s, s, cu, n, t, 1, 33, 1.0),
        lambda: ops.varlen_prefill_q8(q[..., ::2], kp, kp, s, s, cu, n, t, 1, 32, 1.0),
        lambda: ops.kv_evict(kp, kp, w, t, n, n, t, 32, 32),  # no scales
        lambda: ops.kv_evict(plain, plain, w, t, n, n, t, 32, 32, k_scale=s, v_scale=s),
        lambda: ops.kv_evict(plain, plain, w, t, n, n, t, 32, 33),
        lambda: ops.kv_evict(plain, plain, w, t, n, n, t, 32, 32, recent=-1),
        lambda: ops.kv_evict(plain, plain, w, t, n, n, t, 32, 32, weights_out=w.half()),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(FlourError) as e:
            f()
        assert e.value.code in (ERR_INVALID_ARGUMENT, ERR_UNSUPPORTED), i
