"""8-bit prefill over the whole range of scales and elements, on each of its paths (what a cache gives does
not depend on which one the shape of the batch selects), and in slices."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from _cache8 import Cache, attend, close
from flour_amd import _lib, ops
from flour_amd._lib import lib

pytestmark = pytest.mark.gpu

E, I = torch.float8_e4m3fn, torch.int8
BF, HF, F = torch.bfloat16, torch.float16, torch.float32


def i32(x, device):
    return torch.tensor(x, dtype=torch.int32, device=device)


def full_pool(G, blocks, bs, D, dtype, gen, device):
    """An 8-bit pool of every byte but e4m3's NaN and int8's -128."""
    b = torch.randint(0, 256, (G, blocks * bs, D), generator=gen).to(torch.uint8)
    if dtype == E:
        b[(b & 127) == 127] = 126
    else:
        b[b == 128] = 127
    return b.view(dtype).to(device)


@pytest.fixture
def prefill_mode():
    """Sets the path of 8-bit prefill (1 streamed, 2 staged, 3 the kernel for every shape); back to the
    rule afterwards."""
    yield lib().flour_hip_set_prefill_q8
    lib().flour_hip_set_prefill_q8(0)


def u_of(dtype):
    return torch.finfo(dtype).eps / 2


def check(device, pool, dtype, D, ks, vs, scale, stage_u, seed, qmag=1.0, H=6, lens=(130, 70),
          rows=(40, 70), bs=16):
    """Prefill of two sequences against 64 bits, each kv head by its own largest |v|; ks and vs (G,
    blocks). stage_u: the half step to which a staged copy rounds K and V, 0 where it is exact."""
    G, B = ks.shape[0], len(lens)
    gen = torch.Generator().manual_seed(seed)
    nb = [(n + bs - 1) // bs for n in lens]
    perm = torch.randperm(sum(nb), generator=gen).tolist()
    tab = [perm[sum(nb[:s]):sum(nb[:s + 1])] for s in range(B)]
    kp, vp = (full_pool(G, sum(nb), bs, D, pool, gen, device) for _ in "kv")
    q = (qmag * torch.randn((sum(rows), H, D), generator=gen)).to(dtype).to(device)
    ks, vs = ks.to(device), vs.to(device)
    cu = [0] + np.cumsum(rows).tolist()
    wide = [t + [0] * (max(nb) - len(t)) for t in tab]
    got = ops.varlen_prefill_q8(q, kp, vp, ks, vs, i32(cu, device), i32(lens, device),
                                i32(wide, device), max(rows), max(lens), scale, bs, out_dtype=F)
    ck, cv = Cache(kp, ks, bs), Cache(vp, vs, bs)
    # longer calls over 16-bit queries round each probability to f16 once
    p_u = 2.0 ** -11 if dtype != F else 0.0
    for s in range(B):
        k, v = ck.rows(tab[s], lens[s]), cv.rows(tab[s], lens[s])
        qs = q[cu[s]:cu[s + 1]].cpu().double().numpy()
        want, _, err = attend(qs, k, v, scale)
        rep = H // G
        big = np.repeat(np.abs(v).max((0, 2)), rep)  # of the query head's kv head
        # K rounded by u: every score off by u sum |q k|, every weight by a factor within exp(2 that)
        dots = np.einsum("ihd,jhd->ihj", np.abs(qs), np.abs(np.repeat(k, rep, 1))).max(2) * scale
        bound = 2 * err + p_u + np.expm1(2 * stage_u * dots) + stage_u
        close(got[cu[s]:cu[s + 1]], want, (bound * big)[:, :, None])


def blocks_of(lens=(130, 70), bs=16):
    return sum((n + bs - 1) // bs for n in lens)


@pytest.mark.parametrize("mode", [1, 2, 3])
@pytest.mark.parametrize("dtype", [BF, HF, F])
@pytest.mark.parametrize("D", [128, 64])
@pytest.mark.parametrize("pool", [E, I])
def test_prefill_over_scales_that_f16_does_not_hold(device, prefill_mode, pool, D, dtype, mode):
    """K blocks of values up to 2^20 and V blocks down to 2^-30 in some heads and sequences; one K block of
    values around 2^-30 beside ordinary ones."""
    prefill_mode(mode)
    n = blocks_of()
    one = 2.0 ** -9 if pool == E else 2.0 ** -7  # a block of values of about 1
    for kf, vf, scale in ((2.0 ** 20, 1.0, 2.0 ** -26), (1.0, 2.0 ** -30, 0.05),
                          (2.0 ** 12, 2.0 ** 18, 2.0 ** -18), (2.0 ** -30, 2.0 ** -40, 0.1),
                          (2.0 ** 7, 2.0 ** -17, 2.0 ** -10)):
        for part in range(3):
            ks, vs = torch.full((2, n), one), torch.full((2, n), one)
            if part == 0:
                ks *= kf
                vs *= vf
            elif part == 1:  # one head
                ks[1] *= kf
                vs[1] *= vf
            else:  # one block
                ks[0, n // 2] *= kf
                vs[0, n // 2] *= vf
            check(device, pool, dtype, D, ks, vs, scale, 0.0, 40 + part)


@pytest.mark.parametrize("mode", [1, 2, 3])
@pytest.mark.parametrize("dtype", [BF, HF, F])
@pytest.mark.parametrize("pool", [E, I])
def test_prefill_over_every_element_and_any_scales(device, prefill_mode, pool, dtype, mode):
    """Elements up to the type's largest under powers of two (exact on every path) and under scales that
    are none (rounded once to the type of the queries on the staged one)."""
    prefill_mode(mode)
    n = blocks_of()
    gen = torch.Generator().manual_seed(7)
    for D in (128, 64):
        s = torch.exp2(torch.randint(-9, -6, (2, 2, n), generator=gen).float())
        check(device, pool, dtype, D, s[0], s[1], 0.02, 0.0, 50)
        s = s * (1 + torch.rand((2, 2, n), generator=gen))
        check(device, pool, dtype, D, s[0], s[1], 0.01, u_of(dtype) if mode == 2 else 0.0, 51)


def test_slices_choose_their_kernel_by_their_own_rows(device, prefill_mode):
    """Six prompts whose bound of 2^20 positions allows four in a staged copy: the bits of the same prompts
    in calls of four and of two, which run on the kernels for 6,000 and 3,000 rows (9,000 in one call
    would run on another)."""
    H, G, D, bs, n, most = 4, 1, 64, 16, 1500, 1 << 20
    gen = torch.Generator().manual_seed(13)
    nb = (n + bs - 1) // bs
    kp, vp = (full_pool(G, 6 * nb, bs, D, E, gen, device) for _ in "kv")
    s = torch.full((G, 6 * nb), 2.0 ** -9, device=device)
    tab = torch.full((6, most // bs), -1, dtype=torch.int32)
    tab[:, :nb] = torch.randperm(6 * nb, generator=gen).to(torch.int32).view(6, nb)
    tab = tab.to(device)
    q = torch.randn((6 * n, H, D), generator=gen).to(HF).to(device)
    prefill_mode(2)

    def call(a, b):
        cu = i32([n * i for i in range(b - a + 1)], device)
        return ops.varlen_prefill_q8(q[n * a:n * b], kp, vp, s, s, cu, i32([n] * (b - a), device),
                                     tab[a:b], n, most, 0.05, bs, out_dtype=F)

    def call_with(nbytes):  # of workspace
        ws = torch.full((nbytes,), 255, dtype=torch.uint8, device=device)
        out = torch.empty((6 * n, H, D), dtype=F, device=device)
        cu, lens = i32([n * i for i in range(7)], device), i32([n] * 6, device)
        _lib.check(lib().flour_hip_varlen_prefill_q8(
            out.data_ptr(), _lib.F32, H * D, D, q.data_ptr(), H * D, D, _lib.F16, kp.data_ptr(),
            vp.data_ptr(), s.data_ptr(), s.data_ptr(), _lib.E4M3, cu.data_ptr(), lens.data_ptr(),
            tab.data_ptr(), most // bs, 6, n, 6 * n, H, G, D, bs, kp.shape[1], most, 0.05,
            ws.data_ptr(), nbytes, torch.cuda.current_stream().cuda_stream))
        return out

    assert torch.equal(call(0, 6), torch.cat([call(0, 4), call(4, 6)]))
    # a copy of one sequence takes 256 MiB and its table: parts of as many as the workspace holds
    one = (1 << 28) + (1 << 20)
    assert torch.equal(call_with(3 * one), torch.cat([call(0, 3), call(3, 6)]))
    assert torch.equal(call_with(one), torch.cat([call(i, i + 1) for i in range(6)]))


def test_few_rows_over_a_pool_of_2_31_bytes_a_head(device):
    """Such a pool is staged where its shape would be streamed: within the streamed kernel's workspace, one
    sequence of up to 65,536 positions (16 MiB of K, as much of V) at a time."""
    H, G, D, bs, most = 4, 1, 128, 16, 1 << 16
    blocks = (1 << 31) // (bs * D) + 40
    kp = torch.zeros((G, blocks * bs, D), dtype=I, device=device)
    s = torch.full((G, blocks), 2.0 ** -7, device=device)
    gen = torch.Generator().manual_seed(14)
    lens, rows = [600, 33, 100], [8, 3, 8]
    nb = [(n + bs - 1) // bs for n in lens]
    tab = torch.full((3, most // bs), -1, dtype=torch.int32)
    small = full_pool(G, sum(nb), bs, D, I, gen, device)
    where = [blocks - 1 - 7 * i for i in range(5)] + list(range(3, sum(nb) - 2))
    at = 0
    for x, n in enumerate(nb):
        tab[x, :n] = torch.tensor(where[at:at + n])
        at += n
    for i, b in enumerate(where):
        kp[:, b * bs:(b + 1) * bs] = small[:, i * bs:(i + 1) * bs]
    q = torch.randn((sum(rows), H, D), generator=gen).to(BF).to(device)
    cu = [0, 8, 11, 19]
    size = ops.prefill_q8_workspace_bytes(3, 8, 19, most, H, G, D, bs, BF)
    assert size < 3 * 2 * most * D * 2  # not all three at once
    ws = ops.Workspace(device)
    ws.get(size).fill_(255)
    got = ops.varlen_prefill_q8(q, kp, kp, s, s, i32(cu, device), i32(lens, device), tab.to(device), 8,
                                most, 0.03, bs, out_dtype=F, workspace=ws)
    c = Cache(small, torch.full((G, sum(nb)), 2.0 ** -7), bs)
    at = 0
    for x in range(3):
        v = c.rows(list(range(at, at + nb[x])), lens[x])
        at += nb[x]
        want, _, err = attend(q[cu[x]:cu[x + 1]].cpu().double().numpy(), v, v, 0.03)
        close(got[cu[x]:cu[x + 1]], want, (2 * err[:, :, None] + 2.0 ** -11) * np.abs(v).max())


def decode_against_64_bits(q, kp, vp, ks, vs, tab, lens, scale, bs, weights=False):
    """A decode step within the bounds of fp32 arithmetic relative to the sum of |weight v|, and its
    weights."""
    device = q.device
    B, H, D = q.shape
    G = kp.shape[0]
    w = torch.zeros((B, G, max(lens)), device=device) if weights else None
    got = ops.paged_decode_q8(q, kp, vp, ks, vs, i32(tab, device), i32(lens, device), scale, max(lens),
                              bs, out_dtype=F, weights=w)
    ck, cv = Cache(kp, ks, bs), Cache(vp, vs, bs)
    for b, n in enumerate(lens):
        k, v = ck.rows(tab[b], n), cv.rows(tab[b], n)
        want, p, err = attend(q[b:b + 1].cpu().double().numpy(), k, v, scale)
        av = np.abs(np.repeat(v, H // G, 1))  # (n, H, D)
        bound = 2 * err[0][:, None] * np.einsum("hj,jhd->hd", p[0], av)
        # probabilities as two f16 parts (2^-22) of the largest contribution to the head's row
        bound += 2.0 ** -21 * (p[0].T[:, :, None] * av).max((0, 2))[:, None]
        close(got[b:b + 1], want, bound[None])
        if weights:
            pg = p[0].reshape(G, H // G, n)
            close(w[b, :, :n], pg.sum(1), (2 * err[0].reshape(G, -1, 1) * pg).sum(1) + 2.0 ** -40)


@pytest.mark.parametrize("lens", [[48], [1500, 300]])
@pytest.mark.parametrize("dtype", [BF, HF, F])
@pytest.mark.parametrize("D", [128, 64])
@pytest.mark.parametrize("pool", [E, I])
def test_decode_over_v_scales_2_100_apart_that_all_count(device, pool, D, dtype, lens):
    """Blocks under V scales of 2^50, 1 and 2^-50, with weights that make up for them: each contributes
    about as much. One sequence is finished inside a wave's range, the others are merged from pieces."""
    H, G, bs = 4, 2, 16
    gen = torch.Generator().manual_seed(21)
    nb = [(n + bs - 1) // bs for n in lens]
    tab, at = [], 0
    for x in nb:
        tab.append(list(range(at, at + x)) + [0] * (max(nb) - x))
        at += x
    blocks = sum(nb)
    kind = torch.arange(blocks) % 3  # 0: 2^50, 1: 1, 2: 2^-50
    vs = torch.exp2(50.0 * (1 - kind)).repeat(G, 1).to(device)
    vp = full_pool(G, blocks, bs, D, pool, gen, device)
    # keys along one direction: the scores of the kinds are -50, 0 and 50 times ln 2 and some noise
    sign = torch.randint(0, 2, (G, 1, D), generator=gen) * 2 - 1
    noise = torch.randint(-2, 3, (G, blocks * bs, D), generator=gen)
    k = (sign * (32 * (kind - 1)).repeat_interleave(bs)[:, None] + noise).float()
    kp = k.to(E).to(device) if pool == E else k.to(I).to(device)
    ks = torch.full((G, blocks), 2.0 ** -5, device=device)
    q = sign.view(G, 1, D).repeat(1, H // G, 1).reshape(1, H, D).repeat(len(lens), 1, 1)
    q = q.to(dtype).to(device)
    decode_against_64_bits(q, kp, vp, ks, vs, tab, lens, 50 * np.log(2) / D, bs)


@pytest.mark.parametrize("dtype", [BF, HF, F])
@pytest.mark.parametrize("H,G,D", [(8, 2, 128), (4, 4, 64), (34, 2, 64), (4, 2, 96)])
@pytest.mark.parametrize("pool", [E, I])
def test_decode_over_every_element(device, pool, H, G, D, dtype):
    """Elements up to the type's largest, under powers of two and other scales, K's and V's of a block far
    apart; contexts in one piece and in several."""
    gen = torch.Generator().manual_seed(22)
    bs, lens = 16, [1, 17, 700, 64]
    nb = [(n + bs - 1) // bs for n in lens]
    tab, at = [], 0
    for x in nb:
        tab.append(list(range(at, at + x)) + [0] * (max(nb) - x))
        at += x
    kp, vp = (full_pool(G, sum(nb), bs, D, pool, gen, device) for _ in "kv")
    q = torch.randn((len(lens), H, D), generator=gen).to(dtype).to(device)
    for any_scale in (False, True):
        s = torch.exp2(torch.randint(-9, -6, (2, G, sum(nb)), generator=gen).float())
        s[1] *= 2.0 ** 12
        if any_scale:
            s *= 1 + torch.rand(s.shape, generator=gen)
        decode_against_64_bits(q, kp, vp, s[0].to(device), s[1].to(device), tab, lens, 0.02, bs,
                               weights=True)


@pytest.mark.parametrize("D,bs", [(64, 16), (20, 16)])
def test_bounds_of_2_31_positions(device, D, bs):
    """max_context_len and max_kv_len of 2^31 - 1 over a table that wide: decode and prefill as with the
    sequence's own length."""
    H, G, n, rows, most = 4, 2, 40, 5, (1 << 31) - 1
    gen = torch.Generator().manual_seed(23)
    kp, vp = (full_pool(G, 3, bs, D, I, gen, device) for _ in "kv")
    s = torch.full((G, 3), 2.0 ** -7, device=device)
    q = torch.randn((rows, H, D), generator=gen).to(BF).to(device)
    wide = torch.zeros((1, (most + bs - 1) // bs), dtype=torch.int32, device=device)
    wide[0, :3] = i32([2, 0, 1], device)
    lens, cu = i32([n], device), i32([0, rows], device)

    def calls(table, bound):
        return (ops.paged_decode_q8(q[:1], kp, vp, s, s, table, lens, 0.05, bound, bs, out_dtype=F),
                ops.varlen_prefill_q8(q, kp, vp, s, s, cu, lens, table, rows, bound, 0.05, bs,
                                      out_dtype=F))

    c, t = (Cache(x, s, bs) for x in (kp, vp)), [2, 0, 1]
    k, v = (x.rows(t, n) for x in c)
    got = calls(wide, most)
    for x, qs in zip(got, (q[:1], q)):
        want, _, err = attend(qs.cpu().double().numpy(), k, v, 0.05)
        close(x, want, 2 * err[:, :, None] * np.abs(v).max())


def test_staged_prefill_captured_and_replayed_over_changing_scales(device, prefill_mode):
    """A captured staged call with f16 queries looks at the scales in every replay: ordinary ones, a head
    beyond f16, ordinary ones again, each as the eager call, with eager work between them."""
    H, G, D, bs, rows, n = 4, 2, 128, 16, 70, 150
    gen = torch.Generator().manual_seed(24)
    nb = (n + bs - 1) // bs
    kp, vp = (full_pool(G, nb, bs, D, E, gen, device) for _ in "kv")
    q = torch.randn((rows, H, D), generator=gen).to(HF).to(device)
    ks, vs = (torch.full((G, nb), 2.0 ** -9, device=device) for _ in "kv")
    ws = ops.Workspace(device)
    args = (i32([0, rows], device), i32([n], device), i32([list(range(nb))], device), rows, n, 0.05, bs)
    prefill_mode(2)
    out = torch.empty((rows, H, D), dtype=F, device=device)

    def call(o):
        return ops.varlen_prefill_q8(q, kp, vp, ks, vs, *args, out=o, workspace=ws)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        call(out)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call(out)
    plain = None
    for v in (2.0 ** -9, 2.0 ** -40, 2.0 ** -9, 2.0 ** 30, 2.0 ** -9):
        vs[1] = v
        out.fill_(7.0)
        g.replay()
        torch.cuda.synchronize()
        got = out.clone()
        want = call(torch.empty_like(out))
        assert torch.equal(got, want)
        if v == 2.0 ** -9:
            plain = got if plain is None else plain
            assert torch.equal(got, plain)
        else:  # V under another power of two: the output times it, but for the probabilities' rounding
            assert torch.equal(got[:, :2], plain[:, :2])
            c = Cache(vp, torch.full((G, nb), v, device=device), bs)
            big = float(np.abs(c.rows(list(range(nb)), n)).max())
            off = (got[:, 2:].double() - plain[:, 2:].double() * (v * 2.0 ** 9)).abs().max()
            assert off <= 1.01 * 2.0 ** -11 * big
