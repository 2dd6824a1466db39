"""Batches over shared prefixes in which some sequences have more positions of their own than the bounds on the
lengths say of those with the longest prefix: in no group, or in one with a shorter prefix."""
from __future__ import annotations

import math

import pytest
import torch

import _ranged as R
from flour_amd import _lib, ops
from test_ranged_gpu import DT, TILE_EPS, check, i32, run

pytestmark = pytest.mark.gpu


def every_way(b, dt, scale, decode, modes=(1,)):
    """The prefixes once for their groups, by a wave a column and by two for some and for all."""
    lib = _lib.lib()
    want, mag, top, seen = R.expected(b, scale)
    err = R.bound(mag, top, seen, b.q.shape[2], TILE_EPS[dt], float(b.v_pool.double().abs().max()))
    try:
        for mode in modes:
            assert lib.flour_hip_set_shared_prefix(mode) == 0
            for halves in (1, 2, 3, 0):
                assert lib.flour_hip_set_tile_halves(halves) == 0
                R.close(run(b, scale, decode=decode), want, err)
    finally:
        lib.flour_hip_set_tile_halves(0)
        lib.flour_hip_set_shared_prefix(-1)


HEADS = [(14, 2, 64), (32, 8, 128), (40, 2, 128), (3, 3, 64)]
# (starts, prefixes, lengths)
BATCHES = [
    ([0, 4], [1600], [1610, 1640, 1601, 1630, 1640]),              # one of none, as long as any
    ([1, 4], [1600], [1600, 1610, 1640, 1601, 900, 33]),           # before and behind the group
    ([0, 3, 5, 6], [1600, 70, 0], [1610, 1640, 1601, 1000, 71, 1640]),  # shorter prefixes
    ([0, 1], [1300], [1333, 1200, 1333, 800, 2, 0, 1111, 1333]),   # most of none
]


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("heads", HEADS, ids=str)
@pytest.mark.parametrize("batch", BATCHES, ids=range(len(BATCHES)))
@pytest.mark.parametrize("rows", [0, 7, 130], ids=["decode", "few", "many"])
def test_long_parts_of_their_own(dt, heads, batch, rows):
    starts, shared, kv = batch
    n = [1] * len(kv) if rows == 0 else [min(L, 1 + (rows * (s + 2) // 3) % rows) for s, L in enumerate(kv)]
    b = R.batch(DT[dt], *heads, 16, n, kv, seed=40, starts=starts, shared=shared)
    every_way(b, dt, heads[2] ** -0.5, rows == 0, (1, -1))


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("n,groups", [(70, 2), (150, 70)])
def test_long_parts_in_batches_beyond_a_wave(dt, n, groups):
    """More sequences than a wave's lanes, and more groups."""
    starts = [5 + (g * (n - 10)) // groups for g in range(groups)] + [n - 5]
    shared = [(1024, 16, 40)[g % 3] if g else 1024 for g in range(groups)]
    kv = [1000 + s for s in range(n)]
    for s in range(starts[0], starts[-1]):
        g = max(i for i in range(groups) if starts[i] <= s)
        kv[s] = shared[g] + 1 + s % 30 if s % 11 else 1056
    for decode in (True, False):
        rows = [1] * n if decode else [s % 4 for s in range(n)]
        b = R.batch(DT[dt], 4, 2, 64, 16, rows, kv, seed=41, starts=starts, shared=shared)
        every_way(b, dt, 0.125, decode)


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("n", [12, 40, 64])
def test_more_long_parts_than_a_chip_has_workgroups_for(dt, n):
    """Two sequences of a prefix, the others of none: 96 to 512 items of their own, all longer than planned."""
    kv = [1030, 1056] + [1056 - 7 * s for s in range(n)]
    for decode in (True, False):
        b = R.batch(DT[dt], 8, 8, 64, 16, [1] * (n + 2) if decode else [1 + s % 3 for s in range(n + 2)], kv,
                    seed=44, starts=[0, 2], shared=[1024])
        every_way(b, dt, 0.125, decode)


@pytest.mark.parametrize("value", [math.nan, math.inf])
@pytest.mark.parametrize("dt", DT)
def test_bad_rows_in_long_parts(dt, value):
    """Pieces of numbers that are not finite."""
    starts, shared, kv = BATCHES[1]
    for rows in ([1] * 6, [30, 1, 40, 3, 70, 1]):
        b = R.batch(DT[dt], 8, 2, 64, 16, rows, kv, seed=42, starts=starts, shared=shared)
        b.v_pool[1, b.slots(0, 1600)[1580], 5] = value
        b.v_pool[0, b.slots(4, 900)[300], 7] = value
        want, mag, top, seen = R.expected(b, 0.125)
        bad = ~torch.isfinite(want).all(2).all(1)
        assert bool(bad[b.cu[4]:b.cu[5]].all()) and not bool(bad[b.cu[1]:b.cu[4]].any())
        err = R.bound(torch.nan_to_num(mag, nan=0.0, posinf=0.0), top, seen, 64, TILE_EPS[dt], 8.0)
        lib = _lib.lib()
        try:
            for mode in (1, -1):
                assert lib.flour_hip_set_shared_prefix(mode) == 0
                R.close(run(b, 0.125, decode=max(rows) == 1), want, err)
        finally:
            lib.flour_hip_set_shared_prefix(-1)


@pytest.mark.parametrize("dt", DT)
def test_a_graph_replayed_with_other_groups(dt):
    """Where the groups start and how long their prefixes are is the device's: the same graph, with long parts and
    without, equals eager calls."""
    lib = _lib.lib()
    starts, shared, kv = BATCHES[0]
    b = R.batch(DT[dt], 8, 2, 128, 16, [1] * 5, kv, seed=43, starts=starts, shared=shared)
    d = [b.q.cuda(), b.k_pool.cuda(), b.v_pool.cuda(), b.tables.cuda(), i32(b.kv), i32(starts), i32(shared)]
    try:
        assert lib.flour_hip_set_shared_prefix(1) == 0
        out, ws = torch.zeros_like(d[0]), ops.Workspace()

        def call(o, w):
            return ops.paged_decode_shared(*d, 0.09, b.max_kv, 1600, out=o, workspace=w)

        call(out, ws)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call(out, ws)
        for first, last, P in ((0, 4, 1600), (1, 4, 1600), (0, 4, 16), (4, 4, 1600), (0, 4, 1600)):
            d[5].copy_(i32([first, last])), d[6].copy_(i32([P]))
            out.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, call(None, ops.Workspace()))
            check(out, b, 0.09, TILE_EPS[dt])
    finally:
        lib.flour_hip_set_shared_prefix(-1)


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("heads", [(8, 8, 64), (32, 8, 128), (40, 2, 128)], ids=str)
@pytest.mark.parametrize("n", [1, 16, 64])
def test_packed_calls_of_one_row_a_sequence(dt, heads, n):
    """In the way that the library chooses for them, with the workspace that it asks for; as a step too."""
    for P, own in ((64, 16), (512, 64)):
        b = R.batch(DT[dt], *heads, 16, [1] * n, [P + 1 + s % own for s in range(n)], seed=45, starts=[0, n],
                    shared=[P])
        every_way(b, dt, heads[2] ** -0.5, False, (1, 0, -1))
        every_way(b, dt, heads[2] ** -0.5, True, (-1,))
