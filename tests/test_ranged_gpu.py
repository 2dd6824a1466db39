"""Attention over a sliding window with sinks and over shared prefixes against the 64-bit forms."""
from __future__ import annotations

import math

import pytest
import torch

import _ranged as R
from flour_amd import _lib, ops

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def prefixes_on_their_own():
    """Small batches would not be cut at their prefixes: here they are, but for check_shared's other modes."""
    _lib.lib().flour_hip_set_shared_prefix(1)
    yield
    _lib.lib().flour_hip_set_shared_prefix(-1)


@pytest.fixture
def both_halves():
    """A function that runs another with a wave's columns its own, shared with a second one, and the latter
    behind prefixes only."""
    lib = _lib.lib()

    def each(f):
        for halves in (1, 2, 3):
            assert lib.flour_hip_set_tile_halves(halves) == 0
            f()

    yield each
    lib.flour_hip_set_tile_halves(0)


DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
# What a weight is rounded to on the way into a product: two bf16 or f16 parts in decode steps of up to 16
# query heads a kv head (half a step of 8 bits, twice: 2^-8 of 2^-8), one f16 number elsewhere (half a step,
# torch.finfo(torch.float16).eps / 2 = 2^-11).
DECODE_EPS = {"f32": 0.0, "bf16": 2.0 ** -16, "f16": 2.0 ** -16}
TILE_EPS = {"f32": 0.0, "bf16": 2.0 ** -11, "f16": 2.0 ** -11}


def decode_eps(dt, heads):
    return DECODE_EPS[dt] if heads[0] // heads[1] <= 16 else TILE_EPS[dt]


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def run(b, scale, window=None, sinks=0, decode=False, out_dtype=None, **more):
    """The call that the batch is for: with a window, or over its groups' prefixes."""
    args = [t.cuda() for t in (b.q, b.k_pool, b.v_pool)]
    kv, tables = i32(b.kv), b.tables.cuda()
    kw = dict(block_size=b.bs, out_dtype=out_dtype, **more)
    if window is not None:
        if decode:
            return ops.paged_decode_window(*args, tables, kv, scale, b.max_kv, window, sinks, **kw)
        return ops.varlen_prefill_window(*args, i32(b.cu), kv, tables, b.max_rows, b.max_kv, scale,
                                         window, sinks, **kw)
    groups = (i32(b.starts), i32(b.shared))
    most = max(b.shared + [0])
    if decode:
        return ops.paged_decode_shared(*args, tables, kv, *groups, scale, b.max_kv, most, **kw)
    return ops.varlen_prefill_shared(*args, i32(b.cu), kv, tables, *groups, b.max_rows, b.max_kv, most,
                                     scale, **kw)


def check(got, b, scale, eps, window=R.EVERY, sinks=0):
    want, mag, top, seen = R.expected(b, scale, window, sinks)
    v_max = float(b.v_pool[torch.isfinite(b.v_pool)].double().abs().max())
    R.close(got, want, R.bound(mag, top, seen, b.q.shape[2], eps, v_max))


def check_shared(b, scale, eps, **kw):
    """The prefixes once for their groups, without, and as the library chooses."""
    lib = _lib.lib()
    try:
        for mode in (1, 0, -1):
            assert lib.flour_hip_set_shared_prefix(mode) == 0
            check(run(b, scale, **kw), b, scale, eps)
    finally:
        lib.flour_hip_set_shared_prefix(1)


def check_steps(b, scale, eps, window, sinks):
    """Workgroups of a (sequence, kv head), ranges of chunks, and as the library chooses."""
    lib = _lib.lib()
    try:
        for mode in (1, 0, -1):
            assert lib.flour_hip_set_window_pairs(mode) == 0
            got = run(b, scale, window, sinks, decode=True)
            check(got, b, scale, eps, window, sinks)
    finally:
        lib.flour_hip_set_window_pairs(-1)
    return got


HEADS = [(8, 8, 64), (14, 2, 64), (32, 8, 128), (28, 4, 128)]


# ------------------------------------------------------------------ decode, window
@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("heads", HEADS + [(40, 2, 128), (6, 3, 96), (2, 1, 40), (3, 3, 256)], ids=str)
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (7, 3), (64, 4), (100, 33), (300, 0)])
def test_decode_window(dt, heads, window, sinks):
    kv = [0, 1, 2, window, window + 1, window + sinks, window + sinks + 1, 63, 64, 65, 500, 777]
    b = R.batch(DT[dt], *heads, 16, [1] * len(kv), kv, seed=window)
    scale = heads[2] ** -0.5
    got = check_steps(b, scale, decode_eps(dt, heads), window, sinks)
    assert got.dtype == DT[dt]
    assert not bool(got[0].any())


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("window,sinks", [(2 ** 31 - 1, 5), (3, 2 ** 31 - 1), (2 ** 31 - 1, 2 ** 31 - 1)])
def test_decode_window_over_everything(dt, window, sinks):
    b = R.batch(DT[dt], 8, 2, 64, 16, [1] * 4, [0, 1, 333, 2000], seed=24)
    check_steps(b, 0.125, DECODE_EPS[dt], window, sinks)


@pytest.mark.parametrize("bs", [1, 7, 8, 32, 48, 80])
@pytest.mark.parametrize("dt", DT)
def test_decode_window_other_pages(dt, bs):
    b = R.batch(DT[dt], 8, 2, 64, bs, [1] * 5, [3, 200, 1000, 333, 97], seed=bs)
    check_steps(b, 0.125, DECODE_EPS[dt], 90, 5)


@pytest.mark.parametrize("dt,odt", [("bf16", "f32"), ("f16", "bf16"), ("f32", "f16")])
def test_decode_window_output_types(dt, odt):
    b = R.batch(DT[dt], 32, 8, 128, 16, [1] * 4, [5, 200, 4000, 1333], seed=3)
    got = run(b, 0.1, 1000, 4, decode=True, out_dtype=DT[odt])
    assert got.dtype == DT[odt]
    check(got, b, 0.1, DECODE_EPS[dt], 1000, 4)


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("n", [1, 3, 70, 130])
def test_decode_window_batches(dt, n):
    kv = [(s * 7919) % 3000 for s in range(n)]
    b = R.batch(DT[dt], 8, 4, 128, 16, [1] * n, kv, seed=n)
    check_steps(b, 0.09, DECODE_EPS[dt], 600, 20)


# ------------------------------------------------------------------ prefill, window
@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("heads", HEADS + [(40, 2, 128), (6, 3, 96), (2, 1, 40)], ids=str)
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 2), (17, 5), (64, 0), (200, 70)])
def test_prefill_window(dt, heads, window, sinks, both_halves):
    rows = [1, 0, 33, 128, 5, 200, 2, 64]
    kv = [1, 9, 33, 300, 4, 200, 900, 65]  # (the fifth has fewer positions than rows: zeros)
    b = R.batch(DT[dt], *heads, 16, rows, kv, seed=window)
    scale = heads[2] ** -0.5

    def one():
        got = run(b, scale, window, sinks)
        check(got, b, scale, TILE_EPS[dt], window, sinks)
        assert not bool(got[b.cu[4]:b.cu[5]].any())

    both_halves(one)


@pytest.mark.parametrize("bs", [1, 7, 8, 32, 48, 80])
@pytest.mark.parametrize("dt", DT)
def test_prefill_window_other_pages(dt, bs, both_halves):
    b = R.batch(DT[dt], 8, 2, 64, bs, [150, 20, 1], [150, 400, 111], seed=bs)
    both_halves(lambda: check(run(b, 0.125, 60, 5), b, 0.125, TILE_EPS[dt], 60, 5))


@pytest.mark.parametrize("dt,odt", [("bf16", "f32"), ("f16", "bf16"), ("f32", "f16")])
def test_prefill_window_output_types(dt, odt):
    b = R.batch(DT[dt], 8, 2, 128, 16, [100, 30], [500, 30], seed=3)
    got = run(b, 0.1, 120, 4, out_dtype=DT[odt])
    assert got.dtype == DT[odt]
    check(got, b, 0.1, TILE_EPS[dt], 120, 4)


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("n", [70, 130])
def test_prefill_window_many_sequences(dt, n):
    kv = [1 + (s * 7919) % 300 for s in range(n)]
    rows = [min(L, (s * 31) % 40) for s, L in enumerate(kv)]
    b = R.batch(DT[dt], 14, 2, 64, 16, rows, kv, seed=n)
    check(run(b, 0.125, 50, 3), b, 0.125, TILE_EPS[dt], 50, 3)


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("heads", [(8, 2, 64), (7, 1, 128), (130, 1, 64)], ids=str)
@pytest.mark.parametrize("window,sinks", [(3000, 20), (2 ** 31 - 1, 0), (5, 2 ** 31 - 1)])
def test_prefill_window_few_rows_over_many_positions(dt, heads, window, sinks, both_halves):
    """Items cut along the positions, and (130 heads) rows that fill more than one item."""
    b = R.batch(DT[dt], *heads, 16, [5, 0, 1, 20], [5000, 9, 4100, 20], seed=21)
    both_halves(lambda: check(run(b, 0.1, window, sinks), b, 0.1, TILE_EPS[dt], min(window, R.EVERY), sinks))


def test_thousands_of_sequences():
    n, per = 4200, 60  # (more than the decode stream takes, and than two rounds of a wave's search)
    starts, shared = list(range(0, n + 1, per)), [16 * (g % 3) for g in range(n // per)]
    kv = [shared[s // per] + s % 5 for s in range(n)]
    for decode in (True, False):
        rows = [1] * n if decode else [min(L, s % 3) for s, L in enumerate(kv)]
        b = R.batch(torch.bfloat16, 2, 1, 64, 16, rows, kv, seed=22, starts=starts, shared=shared)
        check(run(b, 0.125, decode=decode), b, 0.125, TILE_EPS["bf16"])
        check(run(b, 0.125, 7, 2, decode=decode), b, 0.125, TILE_EPS["bf16"], 7, 2)


# ------------------------------------------------------------------ shared prefixes
GROUPS = [([0, 5], [160]), ([0, 2, 5], [32, 400]), ([1, 3, 3, 4], [100, 7, 0]), ([0, 1, 2, 3, 4, 5], [48] * 5),
          ([5, 5], [64]), ([0, 5], [1000])]


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("heads", HEADS + [(40, 2, 128), (6, 3, 96), (2, 1, 40)], ids=str)
@pytest.mark.parametrize("starts,shared", GROUPS, ids=str)
def test_decode_shared(dt, heads, starts, shared, both_halves):
    # (sequences longer and shorter than their prefixes, one of no position)
    kv = [450, 33, 0, 161, 1200]
    b = R.batch(DT[dt], *heads, 16, [1] * 5, kv, seed=len(starts), starts=starts, shared=shared)
    scale = heads[2] ** -0.5
    both_halves(lambda: check_shared(b, scale, TILE_EPS[dt], decode=True))


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("heads", HEADS + [(40, 2, 128), (6, 3, 96), (2, 1, 40)], ids=str)
@pytest.mark.parametrize("starts,shared", GROUPS, ids=str)
@pytest.mark.parametrize("rows", [[3, 8, 0, 5, 1], [150, 30, 9, 64, 200]], ids=["few", "many"])
def test_prefill_shared(dt, heads, starts, shared, rows, both_halves):
    kv = [450, 33, 5, 161, 1200]
    b = R.batch(DT[dt], *heads, 16, rows, kv, seed=len(starts), starts=starts, shared=shared)
    scale = heads[2] ** -0.5
    both_halves(lambda: check_shared(b, scale, TILE_EPS[dt]))


@pytest.mark.parametrize("bs", [1, 7, 32, 48])
@pytest.mark.parametrize("dt", DT)
def test_shared_other_pages(dt, bs):
    for decode in (True, False):
        rows = [1] * 4 if decode else [4, 1, 7, 2]
        b = R.batch(DT[dt], 8, 2, 64, bs, rows, [300, 250, 260, 500], seed=bs, starts=[0, 3, 4],
                    shared=[245, 77])
        check_shared(b, 0.125, TILE_EPS[dt], decode=decode)


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("n,groups", [(64, 1), (70, 5), (130, 100)])
def test_shared_large_batches(dt, n, groups):
    starts = sorted((g * n) // groups for g in range(groups)) + [n]
    shared = [16 * ((g * 7) % 12 + 1) for g in range(groups)]
    kv = []
    for g in range(groups):
        kv += [shared[g] + 1 + (s * 37) % 90 for s in range(starts[g], starts[g + 1])]
    for decode in (True, False):
        rows = [1] * n if decode else [1 + s % 4 for s in range(n)]
        kv = [max(L, r) for L, r in zip(kv, rows)]
        b = R.batch(DT[dt], 8, 2, 128, 16, rows, kv, seed=n, starts=starts, shared=shared)
        check_shared(b, 0.09, TILE_EPS[dt], decode=decode)


def test_no_groups_is_plain_attention():
    b = R.batch(torch.bfloat16, 8, 2, 128, 16, [1] * 3, [100, 7, 650], seed=1, starts=[0], shared=[])
    check_shared(b, 0.09, TILE_EPS["bf16"], decode=True)


# ------------------------------------------------------------------ values that are not numbers
def poison(b, window, sinks, value):
    """Everything that no row of the batch sees becomes `value`, the spare blocks and page ends too."""
    keep = torch.zeros(b.k_pool.shape[1], dtype=torch.bool)
    for s, L in enumerate(b.kv):
        n = b.cu[s + 1] - b.cu[s]
        j = torch.arange(L)
        lo = L - n - window + 1
        keep[b.slots(s, L)[(j >= lo) | (j < sinks)]] = True
    b.k_pool[:, ~keep], b.v_pool[:, ~keep] = value, value
    return b


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("heads", [(14, 2, 64), (32, 8, 128), (6, 3, 96)], ids=str)
def test_what_no_row_sees_does_not_matter(dt, heads, value):
    scale = heads[2] ** -0.5
    for window, sinks in ((5, 0), (40, 3), (100, 20)):
        kv = [1, 30, 39, 41, 120, 121, 700]
        b = R.batch(DT[dt], *heads, 16, [1] * 7, kv, seed=2)
        check_steps(poison(b, window, sinks, value), scale, DECODE_EPS[dt], window, sinks)
        b = R.batch(DT[dt], *heads, 16, [1, 30, 4, 1, 70, 1, 90], kv, seed=2)
        check(run(poison(b, window, sinks, value), scale, window, sinks), b, scale, TILE_EPS[dt],
              window, sinks)


@pytest.mark.parametrize("value", [math.nan, math.inf])
@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("heads", [(14, 2, 64), (32, 8, 128), (6, 3, 96)], ids=str)
@pytest.mark.parametrize("where", ["k", "v"])
def test_a_bad_row_spoils_those_who_see_it(dt, heads, value, where, both_halves):
    """Rows beside it in a tile, which do not see it, keep their numbers."""
    scale = heads[2] ** -0.5
    b = R.batch(DT[dt], *heads, 16, [200, 30], [260, 400], seed=4)
    pool = b.k_pool if where == "k" else b.v_pool
    for s, j in ((0, 150), (1, 377)):
        pool[0, b.slots(s, 400 if s else 260)[j], 3 if where == "v" else slice(None)] = value
    if where == "k" and value == math.inf:  # scores of +inf for some rows, -inf for others
        b.q[:, :, 0] = b.q[:, :, 0].abs() + 1
        b.q[:, :, 1:] = 0
    want, mag, top, seen = R.expected(b, scale, 40, 3)
    if where == "k":
        top = torch.nan_to_num(top, nan=0.0, posinf=0.0)
        rows = torch.isfinite(want).all(2).all(1)
        top[rows] = R.expected(_finite(b), scale, 40, 3)[2][rows]
    err = torch.nan_to_num(R.bound(mag, top, seen, heads[2], TILE_EPS[dt], 8.0), nan=0.0, posinf=0.0,
                           neginf=0.0)
    both_halves(lambda: R.close(run(b, scale, 40, 3), want, err))


def _finite(b):
    return R.Batch(b.q, torch.nan_to_num(b.k_pool, nan=0.0, posinf=0.0, neginf=0.0), b.v_pool, b.cu,
                   b.kv, b.tables, b.bs, b.starts, b.shared)


@pytest.mark.parametrize("dt", DT)
def test_scores_of_minus_infinity_weigh_nothing(dt):
    for heads in ((14, 2, 64), (8, 2, 128), (6, 3, 96)):
        b = R.batch(DT[dt], *heads, 16, [40, 20], [90, 20], seed=5, starts=[0, 2], shared=[0])
        b.q[:] = b.q.abs() + 0.1
        b.k_pool[:, b.slots(0, 90)[60:75]] = -math.inf  # some rows see nothing else
        b.k_pool[:, b.slots(0, 90)[0]] = -math.inf
        scale = heads[2] ** -0.5
        want, mag, top, seen = R.expected(b, scale, 10, 1)
        assert bool((want[b.cu[0]:b.cu[1]] == 0).all(2).any())
        top = R.expected(_finite(b), scale, 10, 1)[2]
        R.close(run(b, scale, 10, 1), want, R.bound(mag, top, seen, heads[2], TILE_EPS[dt], 8.0))


@pytest.mark.parametrize("size", [2.0 ** -20, 2.0 ** -40, 0.0, 2.0 ** 17, 2.0 ** 100])
@pytest.mark.parametrize("heads", [(14, 2, 64), (8, 2, 128)], ids=str)
def test_bf16_values_of_any_size(size, heads, both_halves):
    """Values beyond f16's numbers, above and below."""
    scale = heads[2] ** -0.5
    b = R.batch(torch.bfloat16, *heads, 16, [150, 3], [200, 300], seed=6, v_scale=size, starts=[0, 2],
                shared=[50])
    for kw in (dict(window=64, sinks=2), {}):
        want, mag, top, seen = R.expected(b, scale, kw.get("window", R.EVERY), kw.get("sinks", 0))
        err = R.bound(mag, top, seen, heads[2], 2.0 ** -11, 4.5 * size)
        # values below f16's numbers: off by what is small beside the block's root mean square
        err = err - 2.0 ** -25 + min(2.0 ** -25, 5e-4 * 4.5 * size)
        both_halves(lambda: R.close(run(b, scale, out_dtype=torch.float32, **kw), want, err))


# ------------------------------------------------------------------ layouts, tables, streams, graphs
def strided(t, pad):
    big = torch.full((t.shape[0], t.shape[1] + 1, t.shape[2] + pad), math.nan, dtype=t.dtype,
                     device="cuda")
    big[:, :t.shape[1], :t.shape[2]] = t.cuda()
    return big[:, :t.shape[1], :t.shape[2]]


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("pad", [8, 3])
def test_strided_queries_and_outputs(dt, pad):
    b = R.batch(DT[dt], 8, 2, 64, 16, [60, 4, 9], [60, 300, 200], seed=7, starts=[0, 3], shared=[32])
    args = (b.k_pool.cuda(), b.v_pool.cuda(), i32(b.cu), i32(b.kv), b.tables.cuda())
    for q in (strided(b.q, pad), b.q.transpose(0, 1).contiguous().cuda().transpose(0, 1)):
        out = strided(torch.zeros_like(b.q), pad)
        ops.varlen_prefill_window(q, *args, 60, 300, 0.125, 50, 2, out=out)
        check(out, b, 0.125, TILE_EPS[dt], 50, 2)
        out = strided(torch.zeros_like(b.q), pad)
        ops.varlen_prefill_shared(q, *args, i32(b.starts), i32(b.shared), 60, 300, 32, 0.125, out=out)
        check(out, b, 0.125, TILE_EPS[dt])


@pytest.mark.parametrize("dt", DT)
def test_unaligned_tensors(dt):
    b = R.batch(DT[dt], 8, 2, 64, 16, [20, 1], [60, 300], seed=8, starts=[0, 2], shared=[32])

    def shifted(t):
        flat = torch.zeros(t.numel() + 1, dtype=t.dtype, device="cuda")
        flat[1:] = t.flatten().cuda()
        return flat[1:].view(t.shape)

    args = (i32(b.cu), i32(b.kv), b.tables.cuda())
    for which in range(4):
        q, k, v = (shifted(t) if i == which else t.cuda()
                   for i, t in enumerate((b.q, b.k_pool, b.v_pool)))
        out = shifted(torch.zeros_like(b.q)) if which == 3 else None
        got = ops.varlen_prefill_window(q, k, v, *args, 20, 300, 0.125, 50, 2, out=out)
        check(got, b, 0.125, TILE_EPS[dt], 50, 2)
        got = ops.varlen_prefill_shared(q, k, v, *args, i32(b.starts), i32(b.shared), 20, 300, 32, 0.125,
                                        out=out)
        check(got, b, 0.125, TILE_EPS[dt])


@pytest.mark.parametrize("dt", DT)
def test_rows_behind_the_last_sequence_stay(dt):
    b = R.batch(DT[dt], 8, 2, 128, 16, [30, 2], [60, 300], seed=9, starts=[0, 2], shared=[48])
    q = torch.cat([b.q, torch.full((50, 8, 128), math.nan, dtype=DT[dt])]).cuda()
    args = (b.k_pool.cuda(), b.v_pool.cuda(), i32(b.cu), i32(b.kv), b.tables.cuda())
    for window in (True, False):
        out = torch.full(q.shape, 7.0, dtype=DT[dt], device="cuda")
        if window:
            ops.varlen_prefill_window(q, *args, 30, 300, 0.09, 33, 1, out=out)
        else:
            ops.varlen_prefill_shared(q, *args, i32(b.starts), i32(b.shared), 30, 300, 48, 0.09, out=out)
        check(out[:32], b, 0.09, TILE_EPS[dt], 33 if window else R.EVERY, 1 if window else 0)
        assert bool((out[32:] == 7.0).all())


@pytest.mark.parametrize("head_dim", [64, 80])  # the tile kernel, the one for every shape
@pytest.mark.parametrize("dt", DT)
def test_row_starts_behind_the_calls_rows_are_cut(dt, head_dim):
    """q's rows bound the sequences': the memory behind out is not theirs."""
    b = R.batch(DT[dt], 8, 2, head_dim, 16, [30, 2], [60, 300], seed=19, starts=[0, 2], shared=[48])
    args = (b.q.cuda(), b.k_pool.cuda(), b.v_pool.cuda(), i32([0, 30, 2 ** 31 - 1]), i32(b.kv), b.tables.cuda())
    for window in (True, False):
        memory = torch.full((64, 8, head_dim), 7.0, dtype=DT[dt], device="cuda")
        if window:
            ops.varlen_prefill_window(*args, 30, 300, 0.09, 33, 1, out=memory[:32])
        else:
            ops.varlen_prefill_shared(*args, i32(b.starts), i32(b.shared), 30, 300, 48, 0.09, out=memory[:32])
        check(memory[:32], b, 0.09, TILE_EPS[dt], 33 if window else R.EVERY, 1 if window else 0)
        assert bool((memory[32:] == 7.0).all())


@pytest.mark.parametrize("dt", DT)
def test_bounds_cut_longer_sequences_and_prefixes(dt):
    b = R.batch(DT[dt], 8, 2, 128, 16, [1, 1, 1], [600, 200, 90], seed=10, starts=[0, 3], shared=[80])
    cut = R.Batch(b.q, b.k_pool, b.v_pool, b.cu, [min(L, 150) for L in b.kv], b.tables, 16, b.starts,
                  b.shared)
    args = (b.q.cuda(), b.k_pool.cuda(), b.v_pool.cuda(), b.tables.cuda(), i32(b.kv))
    check(ops.paged_decode_window(*args, 0.09, 150, 70, 3), cut, 0.09, DECODE_EPS[dt], 70, 3)
    for most in (80, 48, 0):
        got = ops.paged_decode_shared(*args, i32(b.starts), i32(b.shared), 0.09, 150, most)
        check(got, cut, 0.09, TILE_EPS[dt])
    got = ops.paged_decode_shared(*args, i32(b.starts), i32([-5]), 0.09, 150, 80)
    check(got, cut, 0.09, TILE_EPS[dt])


@pytest.mark.parametrize("dt", DT)
def test_table_entries_that_are_not_visible_may_be_anything(dt):
    b = R.batch(DT[dt], 8, 2, 128, 16, [1, 1], [600, 900], seed=11)
    t = b.tables.clone()
    t[0, 1:30] = -1234567890  # sinks in block 0, the window from position 500 on
    t[1, 1:50] = 2000000000
    got = ops.paged_decode_window(b.q.cuda(), b.k_pool.cuda(), b.v_pool.cuda(), t.cuda(), i32(b.kv),
                                  0.09, 900, 100, 4)
    check(got, b, 0.09, DECODE_EPS[dt], 100, 4)
    got = ops.varlen_prefill_window(b.q.cuda(), b.k_pool.cuda(), b.v_pool.cuda(), i32(b.cu), i32(b.kv),
                                    t.cuda(), 1, 900, 0.09, 100, 4)
    check(got, b, 0.09, TILE_EPS[dt], 100, 4)


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("scale", [0.0, -0.1, 3.0])
def test_other_scales(dt, scale):
    b = R.batch(DT[dt], 8, 2, 64, 16, [40, 3], [100, 300], seed=12, starts=[0, 2], shared=[64])
    check(run(b, scale, 50, 2), b, scale, TILE_EPS[dt], 50, 2)
    check_shared(b, scale, TILE_EPS[dt])
    b = R.batch(DT[dt], 8, 2, 64, 16, [1, 1], [100, 300], seed=12, starts=[0, 2], shared=[64])
    check(run(b, scale, 50, 2, decode=True), b, scale, DECODE_EPS[dt], 50, 2)
    check_shared(b, scale, TILE_EPS[dt], decode=True)


def calls(b, d):
    """The four calls on the device tensors of a decode batch, as functions of (out, workspace)."""
    groups = (i32(b.starts), i32(b.shared))
    most = max(b.shared)
    cu = i32(b.cu)
    return [
        lambda o, w: ops.paged_decode_window(*d, 0.09, b.max_kv, 90, 4, out=o, workspace=w),
        lambda o, w: ops.varlen_prefill_window(*d[:3], cu, d[4], d[3], b.max_rows, b.max_kv, 0.09, 90, 4,
                                               out=o, workspace=w),
        lambda o, w: ops.paged_decode_shared(*d, *groups, 0.09, b.max_kv, most, out=o, workspace=w),
        lambda o, w: ops.varlen_prefill_shared(*d[:3], cu, d[4], d[3], *groups, b.max_rows, b.max_kv,
                                               most, 0.09, out=o, workspace=w)]


@pytest.mark.parametrize("dt", DT)
def test_equal_calls_give_equal_bits_also_captured_and_on_another_stream(dt):
    n = 9
    b = R.batch(DT[dt], 32, 8, 128, 16, [1] * n, [300 + 61 * s for s in range(n)], seed=13,
                starts=[0, 4, n], shared=[256, 320])
    d = [b.q.cuda(), b.k_pool.cuda(), b.v_pool.cuda(), b.tables.cuda(), i32(b.kv)]
    for i, f in enumerate(calls(b, d)):
        ws = ops.Workspace()
        want = f(None, ws)
        again, own = f(None, ws), f(None, None)
        assert torch.equal(want, again) and torch.equal(want, own)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            other = f(None, ops.Workspace())
        s.synchronize()
        assert torch.equal(want, other)
        out = torch.zeros_like(want)
        gws, graph = ops.Workspace(), torch.cuda.CUDAGraph()
        f(out, gws)
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            f(out, gws)
        for x in range(3):  # replays with new queries, eager work between them
            d[0].copy_(torch.randn(d[0].shape, generator=torch.Generator().manual_seed(x)).to(DT[dt]))
            out.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, f(None, ws)), i
        d[0].copy_(b.q)
        torch.cuda.synchronize()


def test_a_workspace_that_is_too_small_is_refused():
    b = R.batch(torch.bfloat16, 32, 8, 128, 16, [1] * 3, [300, 500, 400], starts=[0, 3], shared=[256])
    d = [b.q.cuda(), b.k_pool.cuda(), b.v_pool.cuda(), b.tables.cuda(), i32(b.kv)]
    lib = _lib.lib()
    for shared in (False, True):
        need = ops.shared_workspace_bytes(3, 1, 1, 3, 32, 8, 128, 500, 256, torch.bfloat16) if shared \
            else ops.window_workspace_bytes(3, 1, 3, 32, 8, 128, 500, 90, 4, torch.bfloat16)
        if need == 0:
            continue
        ws = torch.empty(need, dtype=torch.uint8, device="cuda")
        for p, n in ((ws.data_ptr(), need - 1), (None, need), (ws.data_ptr() + 128, need)):
            front = (d[0].data_ptr(), 1, d[0].data_ptr(), d[1].data_ptr(), d[2].data_ptr(),
                     d[3].data_ptr(), d[3].shape[1], d[4].data_ptr(), 3)
            if shared:
                g = (i32(b.starts), i32(b.shared))
                rc = lib.flour_hip_paged_decode_shared(*front, g[0].data_ptr(), g[1].data_ptr(), 1, 32, 8,
                                                       128, 16, d[1].shape[1], 500, 256, 0.09, 1, p, n,
                                                       None)
            else:
                rc = lib.flour_hip_paged_decode_window(*front, 32, 8, 128, 16, d[1].shape[1], 500, 90, 4,
                                                       0.09, 1, p, n, None)
            assert rc == _lib.ERR_WORKSPACE and "workspace" in _lib.last_error()


def test_arguments_that_do_not_fit_are_refused():
    b = R.batch(torch.bfloat16, 8, 2, 128, 16, [1] * 2, [30, 50], starts=[0, 2], shared=[16])
    q, k, v, t, kv = b.q.cuda(), b.k_pool.cuda(), b.v_pool.cuda(), b.tables.cuda(), i32(b.kv)
    cu, starts, shared = i32(b.cu), i32(b.starts), i32(b.shared)
    bad = [
        lambda: ops.paged_decode_window(q, k, v, t, kv, 0.1, 50, 0),
        lambda: ops.paged_decode_window(q, k, v, t, kv, 0.1, 50, 5, -1),
        lambda: ops.paged_decode_window(q.float(), k, v, t, kv, 0.1, 50, 5),
        lambda: ops.paged_decode_window(q, k, v, t, kv[:1], 0.1, 50, 5),
        lambda: ops.paged_decode_window(q, k, v, t.long(), kv, 0.1, 50, 5),
        lambda: ops.paged_decode_window(q, k, v, t, kv, 0.1, 50, 5, block_size=7),
        lambda: ops.paged_decode_window(q[:, :3], k, v, t, kv, 0.1, 50, 5),
        lambda: ops.paged_decode_window(q, k, v, t, kv, 0.1, 65, 5),
        lambda: ops.paged_decode_window(q, k, v, t, kv, 0.1, 50, 5, out=q[:1]),
        lambda: ops.varlen_prefill_window(q, k, v, cu, kv, t, 1, 50, 0.1, 0),
        lambda: ops.varlen_prefill_window(q[..., ::2], k, v, cu, kv, t, 1, 50, 0.1, 5),
        lambda: ops.varlen_prefill_window(q, k, v, cu[:2], kv, t, 1, 50, 0.1, 5),
        lambda: ops.varlen_prefill_window(q, k, v.half(), cu, kv, t, 1, 50, 0.1, 5),
        lambda: ops.paged_decode_shared(q, k, v, t, kv, starts[:1], shared, 0.1, 50, 16),
        lambda: ops.paged_decode_shared(q, k, v, t, kv, starts, shared.long(), 0.1, 50, 16),
        lambda: ops.paged_decode_shared(q, k, v, t, kv, starts, shared, 0.1, 50, 65),
        lambda: ops.paged_decode_shared(q, k, v, t, kv, starts, shared, 0.1, 50, -1),
        lambda: ops.varlen_prefill_shared(q, k, v, cu, kv, t, starts, shared.cpu(), 1, 50, 16, 0.1),
        lambda: ops.varlen_prefill_shared(q, k, v, cu, kv, t, starts, shared, 1, 65, 16, 0.1),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(_lib.FlourError):
            f()
            pytest.fail(f"call {i} was not refused")


# ------------------------------------------------------------------ together
def test_a_server_that_shares_a_prompt_and_windows_some_layers():
    """A system prompt written once, chats that share it: their turns prefilled, tokens decoded, one
    layer over everything through the shared calls, one over a window with sinks, through the cache's own
    write and in their order on one stream and workspace."""
    torch.manual_seed(0)
    G, H, D, bs, P = 2, 8, 64, 16, 96
    turns, steps, n = [20, 5, 33], 3, 3
    scale, ws = D ** -0.5, ops.Workspace()
    blocks = P // bs + n * 6
    pools = [[torch.zeros((G, blocks * bs, D), dtype=torch.bfloat16, device="cuda") for _ in range(2)]
             for _ in range(2)]
    tables = torch.zeros((n, P // bs + 6), dtype=torch.int32)
    for s in range(n):
        tables[s, :P // bs] = torch.arange(P // bs)
        tables[s, P // bs:] = P // bs + 6 * s + torch.arange(6)
    lens = [0] * n
    starts, shared = i32([0, n]), i32([P])

    def forward(layer, rows, kv):
        T = sum(rows)
        q, k, v = (torch.randn((T, h, D), device="cuda").to(torch.bfloat16) for h in (H, G, G))
        slots = []
        for s, (r, L) in enumerate(zip(rows, kv)):
            j = torch.arange(L - r, L)
            slots.append(tables[s].long()[j // bs] * bs + j % bs)
        ops.kv_write(k, v, *pools[layer], torch.cat(slots).to(torch.int32).cuda())
        cu = [0]
        for r in rows:
            cu.append(cu[-1] + r)
        b = R.Batch(q.cpu(), pools[layer][0].cpu(), pools[layer][1].cpu(), cu, list(kv), tables, bs, [], [])
        d, t, L = (q, *pools[layer]), tables.cuda(), i32(kv)
        if layer == 0 and max(rows) == 1:
            got = ops.paged_decode_shared(*d, t, L, starts, shared, scale, max(kv), P, workspace=ws)
        elif layer == 0:
            got = ops.varlen_prefill_shared(*d, i32(cu), L, t, starts, shared, max(rows), max(kv), P,
                                            scale, workspace=ws)
        elif max(rows) == 1:
            got = ops.paged_decode_window(*d, t, L, scale, max(kv), 30, 4, workspace=ws)
        else:
            got = ops.varlen_prefill_window(*d, i32(cu), L, t, max(rows), max(kv), scale, 30, 4,
                                            workspace=ws)
        check(got, b, scale, 2.0 ** -11, 30 if layer else R.EVERY, 4 if layer else 0)

    for layer in range(2):
        forward(layer, [P] + [0] * (n - 1), [P] + [0] * (n - 1))  # the prompt, through the first chat
    lens = [P + r for r in turns]
    for layer in range(2):
        forward(layer, turns, lens)
    for _ in range(steps):
        lens = [L + 1 for L in lens]
        for layer in range(2):
            forward(layer, [1] * n, lens)
