"""Eviction by accumulated attention weight on the GPU: which positions stay, where their rows and
sums go, over plain and 8-bit pools, and a run of all operators of the small cache together."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from _cache8 import Cache, attend, close, evicted, quantised, scale_for, values
from flour_amd import ops

pytestmark = pytest.mark.gpu

E, I = torch.float8_e4m3fn, torch.int8
BF, HF, F = torch.bfloat16, torch.float16, torch.float32


def i32(x, device):
    return torch.tensor(x, dtype=torch.int32, device=device)


def nblocks(n, bs):
    return (n + bs - 1) // bs


def make(lens, keeps, G, D, bs, pool, device, seed, weights="heavy"):
    gen = torch.Generator().manual_seed(seed)
    src, dst = sum(nblocks(n, bs) for n in lens), sum(nblocks(min(k, n), bs) for k, n in zip(keeps, lens))
    blocks = src + dst + 2
    perm = torch.randperm(blocks, generator=gen).tolist()

    def table(ns, at):
        width = max(1, max(nblocks(n, bs) for n in ns))
        rows = []
        for n in ns:
            nb = nblocks(n, bs)
            rows.append(perm[at:at + nb] + [-1] * (width - nb))
            at += nb
        return rows

    tab = table(lens, 0)
    out_tab = table([min(k, n) for k, n in zip(keeps, lens)], src)
    if pool in (E, I):
        b = torch.randint(0, 256, (2, G, blocks * bs, D), generator=gen).to(torch.uint8)
        b[(b & 127) == 127] = 3
        b[b == 128] = 2
        kv = b.view(pool).to(device)
        s = torch.exp2(torch.randint(-9, 3, (2, G, blocks), generator=gen).float()).to(device)
    else:
        kv, s = torch.randn((2, G, blocks * bs, D), generator=gen).to(pool).to(device), [None, None]
    n = max(lens)
    w = torch.exp(2 * torch.randn((len(lens), G, n), generator=gen))
    if weights == "ties":
        w = torch.randint(0, 3, (len(lens), G, n), generator=gen).float()
    elif weights == "odd":
        w = torch.randn((len(lens), G, n), generator=gen)
        r = torch.rand((len(lens), G, n), generator=gen)
        w[r < 0.4] = 0.0
        w[(r > 0.2) & (r < 0.4)] = -0.0
        w[(r > 0.4) & (r < 0.6)] = float("nan")
        w[(r > 0.6) & (r < 0.65)] = float("inf")
        w[(r > 0.65) & (r < 0.7)] = float("-inf")
        w[(r > 0.7) & (r < 0.75)] = 1e-45
    return kv[0], kv[1], s[0], s[1], w.to(device), tab, out_tab


def check(lens, keeps, recent, G, D, bs, pool, device, seed, weights="heavy", separate=False):
    kp, vp, ks, vs, w, tab, out_tab = make(lens, keeps, G, D, bs, pool, device, seed, weights)
    before, w0 = [kp.clone(), vp.clone()], w.cpu().numpy().copy()
    scales = [None if s is None else s.clone() for s in (ks, vs)]
    wo = torch.full_like(w, 8.0) if separate else w
    most = max(min(k, n) for k, n in zip(keeps, lens))
    kept = ops.kv_evict(kp, vp, w, i32(tab, device), i32(lens, device), i32(keeps, device),
                        i32(out_tab, device), max(lens), most, recent, bs, k_scale=ks, v_scale=vs,
                        weights_out=wo if separate else None)
    torch.cuda.synchronize()
    want_kept = np.full((len(lens), G, most), -1)
    want_w = np.full(w0.shape, 8.0, dtype=np.float32) if separate else w0.copy()
    pos = {}
    for b, (n, k) in enumerate(zip(lens, keeps)):
        for g in range(G):
            p = pos[b, g] = evicted(w0[b, g], n, k, recent)
            want_kept[b, g, :len(p)] = p
            want_w[b, g, :len(p)] = w0[b, g, p]
            want_w[b, g, len(p):n] = 0.0
    assert np.array_equal(kept.cpu().numpy(), want_kept)
    assert np.array_equal(wo.cpu().numpy(), want_w, equal_nan=True)
    if separate:
        assert np.array_equal(w.cpu().numpy(), w0, equal_nan=True)
    for p, old, s, s0 in zip((kp, vp), before, (ks, vs), scales):
        if s is None:
            want = old.clone()
            for (b, g), j in pos.items():
                src = torch.tensor([tab[b][x // bs] * bs + x % bs for x in j], dtype=torch.long)
                to = torch.tensor([out_tab[b][i // bs] * bs + i % bs for i in range(len(j))],
                                  dtype=torch.long)
                want[g, to.to(device)] = old[g, src.to(device)]
            assert torch.equal(p, want)
            continue
        c = Cache(old, s0, bs)
        want_q, want_s = c.q.copy(), c.s.copy()
        for (b, g), j in pos.items():
            rows = c.q[g, np.array(tab[b])[j // bs], j % bs] * \
                c.s[g, np.array(tab[b])[j // bs]][:, None]
            for i0 in range(0, len(j), bs):
                x, to = rows[i0:i0 + bs], out_tab[b][i0 // bs]
                sc = want_s[g, to] = scale_for(float(np.abs(x).max()), pool)
                want_q[g, to, :len(x)] = quantised(x, sc, pool)
        assert np.array_equal(s.cpu().double().numpy(), want_s)
        assert np.array_equal(values(p).reshape(want_q.shape), want_q)


SHAPES = [  # (lens, keeps, recent, G, D, bs)
    ([40, 17, 1, 0, 64], [20, 30, 1, 5, 16], 4, 2, 128, 16),
    ([33, 50], [0, 50], 10, 3, 64, 16),
    ([100], [33], 0, 1, 64, 16),
    ([70, 20], [13, 7], 100, 2, 20, 5),
    ([2500, 1025, 1024], [1100, 64, 1000], 30, 2, 64, 16),
    ([90], [48], 7, 1, 8, 32),
    ([30, 31], [9, 16], 3, 2, 3, 1),
    ([5000], [17], 5, 1, 256, 16),
    ([9000, 40], [8000, 39], 3, 1, 64, 16),
    ([40000, 300], [2000, 200], 100, 1, 16, 16),
    ([66000], [65000], 64900, 1, 8, 16),
    ([200, 90], [150, 90], 9, 2, 64, 80),
    ([100], [70], 9, 2, 33, 128),
]


@pytest.mark.parametrize("weights", ["heavy", "ties", "odd"])
@pytest.mark.parametrize("pool", [BF, F, E, I])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_evict(device, shape, pool, weights):
    check(*SHAPES[shape], pool, device, shape, weights, separate=weights == "heavy")


def test_evict_all_alike_and_one_heavy(device):
    for value in (0.0, 1.0, float("nan")):
        kp, vp, ks, vs, w, tab, out_tab = make([300], [50], 1, 64, 16, HF, device, 1)
        w.fill_(value)
        w[0, 0, 200] = 2.0
        kept = ops.kv_evict(kp, vp, w, i32(tab, device), i32([300], device), i32([50], device),
                            i32(out_tab, device), 300, 50, 10)
        assert kept[0, 0].tolist() == list(range(39)) + [200] + list(range(290, 300))


def test_evict_rows_bounds_and_bad_ids(device):
    """weight_rows out of range skip their sequence; lengths beyond their bounds are clamped; ids
    outside the pool are not written."""
    kp, vp, _, _, w, tab, out_tab = make([40, 40, 40], [20, 20, 20], 2, 64, 16, BF, device, 2)
    out_tab[2] = [-1, 1 << 30]
    old, w0 = kp.clone(), w.cpu().numpy().copy()
    kept = ops.kv_evict(kp, vp, w, i32(tab, device), i32([40, 40, 99], device),
                        i32([20, 20, 70], device), i32(out_tab, device), 40, 20, 4,
                        weight_rows=i32([7, 0, 2], device))
    k = kept.cpu().numpy()
    assert (k[0] == -1).all()
    for b, r in ((1, 0), (2, 2)):
        for g in range(2):
            assert np.array_equal(k[b, g], evicted(w0[r, g], 40, 20, 4))
    to = torch.tensor([out_tab[1][i // 16] * 16 + i % 16 for i in range(20)], device=device)
    rest = torch.ones(kp.shape[1], dtype=torch.bool, device=device)
    rest[to] = False
    assert torch.equal(kp[:, rest], old[:, rest])
    assert np.array_equal(w[1].cpu().numpy(), w0[1])


@pytest.mark.parametrize("pool", [E, I, BF])
def test_evict_nan_values_stay_where_they_are(device, pool):
    """A poisoned source block poisons the destination blocks that take a row of it, no other."""
    kp, vp, ks, vs, w, tab, out_tab = make([64], [48], 1, 64, 16, pool, device, 3)
    if pool == BF:
        kp[0, tab[0][1] * 16 + 3] = float("nan")
    else:
        ks[0, tab[0][1]] = float("nan")
    kept = ops.kv_evict(kp, vp, w, i32(tab, device), i32([64], device), i32([48], device),
                        i32(out_tab, device), 64, 48, 0, k_scale=ks, v_scale=vs)
    hit = {i // 16 for i, p in enumerate(kept[0, 0].tolist()) if p // 16 == 1}
    for lb in range(3):
        if pool == BF:
            continue
        assert bool(torch.isnan(ks[0, out_tab[0][lb]])) == (lb in hit)
        assert not torch.isnan(vs[0, out_tab[0][lb]])


@pytest.mark.parametrize("bs,D", [(16, 64), (16, 40), (128, 64)])
@pytest.mark.parametrize("pool", [E, I])
def test_evict_zero_rows_of_a_huge_scale(device, pool, bs, D):
    """Rows of zeros under a scale of 2^120 beside rows under 2^-100: zeros stay zeros, the others keep
    their bits where the scale that they need is theirs (their quotient of 2^220 is no fp32 number)."""
    b = torch.randint(0, 256, (2, 1, 3 * bs, D), generator=torch.Generator().manual_seed(3)).to(torch.uint8)
    b[(b & 127) == 127] = 3
    b[b == 128] = 2
    b[:, :, :bs] = 0
    b[:, :, bs:, 0] = 0x7e if pool is E else 0x7f  # the largest element: the scale is needed
    kv = b.view(pool).to(device)
    s = torch.tensor([[[2.0 ** 120, 2.0 ** -100, 1.0]]] * 2, device=device)
    w = torch.ones((1, 1, 2 * bs), device=device)
    w[0, 0, ::2] = 2.0  # every other row is kept
    kept = ops.kv_evict(kv[0], kv[1], w, i32([[0, 1]], device), i32([2 * bs], device), i32([bs], device),
                        i32([[2]], device), 2 * bs, bs, 0, bs, k_scale=s[0], v_scale=s[1])
    assert kept[0, 0].tolist() == list(range(0, 2 * bs, 2))
    assert torch.equal(s[:, 0, 2].cpu(), torch.full((2,), 2.0 ** -100))
    assert torch.equal(kv.view(torch.uint8).cpu()[:, 0, 2 * bs:], b[:, 0, 0:2 * bs:2])


def test_evict_captured(device):
    lens, keeps = [1500, 90], [400, 64]
    kp, vp, ks, vs, w, tab, out_tab = make(lens, keeps, 2, 128, 16, E, device, 4)
    args = (i32(tab, device), i32(lens, device), i32(keeps, device), i32(out_tab, device), 1500,
            400, 32)
    wo, kept = torch.zeros_like(w), torch.zeros((2, 2, 400), dtype=torch.int32, device=device)

    def call():
        ops.kv_evict(kp, vp, w, *args, k_scale=ks, v_scale=vs, weights_out=wo, kept=kept)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        call()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call()
    for seed in range(4):
        w.copy_(torch.rand(w.shape, generator=torch.Generator().manual_seed(seed)))
        g.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in (kept, wo, ks, vs)] + [kp.view(I).clone(), vp.view(I).clone()]
        call()
        torch.cuda.synchronize()
        for a, b in zip(got, (kept, wo, ks, vs, kp.view(I), vp.view(I))):
            assert torch.equal(a, b)


# ------------------------------------------------------------------ together
@pytest.mark.parametrize("pool", [E, I])
def test_a_cache_in_service(device, pool):
    """Two sequences' prompts written and attended to, decode steps that add up weights, an eviction
    into new blocks, further steps on what is left: every output against the same in 64 bits."""
    H, G, D, bs, scale = 8, 2, 128, 16, 128 ** -0.5
    gen = torch.Generator().manual_seed(9)
    blocks = 24
    kp = torch.zeros((G, blocks * bs, D), dtype=torch.int8, device=device).view(pool)
    vp = kp.clone()
    ks, vs = torch.zeros((G, blocks), device=device), torch.zeros((G, blocks), device=device)
    ck, cv = Cache(kp, ks, bs), Cache(vp, vs, bs)
    ws, sums = ops.Workspace(device), torch.zeros((2, G, 96), device=device)
    want_sums = np.zeros((2, G, 96))
    tab = [[3, 9, 1, 20, 7], [15, 4, 12, 2, 0]]
    lens = [0, 0]

    def rows(n):
        return torch.randn((n, G, D), generator=gen).to(BF).to(device)

    def host(t):
        return t.cpu().double().numpy()

    def write(k, v, new):
        for s, n in enumerate(new):
            lens[s] += n
        cu = [0, new[0], sum(new)]
        ops.kv_write_q8(k, v, kp, vp, ks, vs, i32(cu, device), i32(lens, device), i32(tab, device))
        for s in range(2):
            ck.write(host(k[cu[s]:cu[s + 1]]), tab[s], lens[s])
            cv.write(host(v[cu[s]:cu[s + 1]]), tab[s], lens[s])
        return cu

    def want(q, cu):
        out, bound = np.zeros(q.shape), np.zeros(q.shape)
        p = [None, None]
        for s in range(2):
            k, v = ck.rows(tab[s], lens[s]), cv.rows(tab[s], lens[s])
            o, w, err = attend(host(q[cu[s]:cu[s + 1]]), k, v, scale)
            out[cu[s]:cu[s + 1]] = o
            bound[cu[s]:cu[s + 1]] = (2 * err[:, :, None] + 2.0 ** -11) * np.abs(v).max()
            p[s] = w.sum(0).reshape(G, H // G, -1).sum(1)
        return out, bound, p

    new = [37, 50]
    cu = write(rows(87), rows(87), new)
    q = torch.randn((87, H, D), generator=gen).to(BF).to(device)
    out = ops.varlen_prefill_q8(q, kp, vp, ks, vs, i32(cu, device), i32(lens, device),
                                i32(tab, device), 50, max(lens), scale, workspace=ws)
    o, bound, _ = want(q, cu)
    close(out, o, bound)

    def steps(n):
        for _ in range(n):
            cu = write(rows(2), rows(2), [1, 1])
            q = torch.randn((2, H, D), generator=gen).to(BF).to(device)
            out = ops.paged_decode_q8(q, kp, vp, ks, vs, i32(tab, device), i32(lens, device), scale,
                                      max(lens), workspace=ws, weights=sums)
            o, bound, p = want(q, cu)
            close(out, o, bound)
            for s in range(2):
                want_sums[s, :, :lens[s]] += p[s]

    steps(20)
    close(sums, want_sums, 1e-5 * (want_sums + 2.0 ** -20))
    new_tab, keep = [[5, 6, 8], [10, 11, 13]], [30, 33]
    # the kernel's own sums say what stays: the 64-bit ones could order two of them otherwise
    mine = sums.cpu().numpy()
    kept = ops.kv_evict(kp, vp, sums, i32(tab, device), i32(lens, device), i32(keep, device),
                        i32(new_tab, device), max(lens), 33, recent=8, k_scale=ks, v_scale=vs)
    for s in range(2):
        for g in range(G):
            j = evicted(mine[s, g], lens[s], keep[s], 8)
            assert kept[s, g, :keep[s]].tolist() == j.tolist()
            for c in (ck, cv):
                x = c.rows(tab[s], lens[s])[j, g]
                for i0 in range(0, keep[s], bs):
                    b = new_tab[s][i0 // bs]
                    c.s[g, b] = scale_for(float(np.abs(x[i0:i0 + bs]).max()), pool)
                    c.q[g, b, :len(x[i0:i0 + bs])] = quantised(x[i0:i0 + bs], c.s[g, b], pool)
            want_sums[s, g, :lens[s]] = np.concatenate([want_sums[s, g, j],
                                                        np.zeros(lens[s] - keep[s])])
    close(sums, want_sums, 1e-5 * (want_sums + 2.0 ** -20))
    tab, lens = [t + [b] for t, b in zip(new_tab, (16, 17))], list(keep)
    steps(18)
    close(sums, want_sums, 1e-5 * (want_sums + 2.0 ** -20))
