"""Numbers that are not finite, and of very different sizes, in every form of the attention over windows and over
shared prefixes, against the 64-bit forms."""
from __future__ import annotations

import math

import pytest
import torch

import _ranged as R
from flour_amd import _lib
from test_ranged_gpu import DECODE_EPS, DT, TILE_EPS, check, run

pytestmark = pytest.mark.gpu

SHARED, PAIRS = "flour_hip_set_shared_prefix", "flour_hip_set_window_pairs"


def each_way(f, decode, window):
    """f(weight eps of a 16-bit call) in every form that the library has for the call: windows by workgroups of a
    (sequence, kv head), by ranges of chunks, by its choice; prefixes for their groups, by sequences, by its
    choice."""
    lib = _lib.lib()
    name = (PAIRS if decode else None) if window else SHARED
    try:
        for mode in (1, 0, -1):
            if name:
                assert getattr(lib, name)(mode) == 0
            f(DECODE_EPS if decode and (window or mode == 0) else TILE_EPS)
    finally:
        if name:
            getattr(lib, name)(-1)


HEADS = [(14, 2, 64), (32, 8, 128), (6, 3, 96)]


# ------------------------------------------------------------------ scores of -inf
@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("heads", HEADS, ids=str)
@pytest.mark.parametrize("kind", ["window", "shared"])
@pytest.mark.parametrize("decode", [True, False], ids=["decode", "prefill"])
def test_rows_without_a_score_above_minus_infinity_are_zero(dt, heads, kind, decode, bad):
    """Whatever the values there hold. Lengths within one chunk of a step's stream, and over many."""
    scale = heads[2] ** -0.5
    for kv in ([9, 40, 9, 12], [2500, 1300, 700, 3]):
        n = len(kv)
        rows = [1] * n if decode else [min(7, L) for L in kv]
        b = R.batch(DT[dt], *heads, 16, rows, kv, seed=30, starts=[0, 2], shared=[8 if kv[0] == 9 else 800])
        b.q[:] = b.q.abs() + 0.1
        for s, v in ((0, bad), (1, bad), (3, 1.0)):
            b.k_pool[:, b.slots(s, kv[s])] = -math.inf
            b.v_pool[:, b.slots(s, kv[s])] = v
        windows = [(5, 0), (1000, 2)] if kind == "window" else [(R.EVERY, 0)]
        for window, sinks in windows:
            want, mag, _, seen = R.expected(b, scale, window, sinks)
            for s in (0, 1, 3):
                assert not bool(want[b.cu[s]:b.cu[s + 1]].any())
            top = torch.zeros_like(mag[..., 0])  # (rows of scores of -inf alone have no error)
            i = slice(b.cu[2], b.cu[3])
            _, mag[i], top[i], seen[i] = R.attend(b.q[i].double(), *b.rows(2, kv[2]), scale, window, sinks)
            mag = torch.nan_to_num(mag, nan=0.0, posinf=0.0)

            def one(eps):
                got = run(b, scale, decode=decode, **(dict(window=window, sinks=sinks) if kind == "window" else {}))
                R.close(got, want, R.bound(mag, top, seen, heads[2], eps[dt], 8.0))

            each_way(one, decode, kind == "window")


# ------------------------------------------------------------------ NaN and infinities behind shared prefixes
# Prefixes that end inside a page, sequences longer and shorter than theirs, one of no group, one without rows.
STARTS, PREFIX, LENS = [0, 4, 5], [245, 77], [300, 250, 100, 246, 500, 40, 120]


def grouped(dt, heads, decode, seed):
    rows = [1, 1, 1, 1, 1, 1, 0] if decode else [9, 5, 40, 2, 70, 40, 0]
    if decode:
        return R.batch(DT[dt], *heads, 16, rows[:6], LENS[:6], seed=seed, starts=STARTS, shared=PREFIX)
    return R.batch(DT[dt], *heads, 16, rows, LENS, seed=seed, starts=STARTS, shared=PREFIX)


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("heads", HEADS, ids=str)
@pytest.mark.parametrize("decode", [True, False], ids=["decode", "prefill"])
def test_positions_behind_sequences_do_not_matter_to_shared_calls(dt, heads, decode, value):
    b = grouped(dt, heads, decode, 31)
    keep = torch.zeros(b.k_pool.shape[1], dtype=torch.bool)
    for s, L in enumerate(b.kv):
        if b.cu[s + 1] > b.cu[s]:
            keep[b.slots(s, L)] = True
    for s, P in zip(b.starts, b.shared):  # (the first table names all of the prefix)
        keep[b.slots(s, P)] = True
    b.k_pool[:, ~keep], b.v_pool[:, ~keep] = value, value
    scale = heads[2] ** -0.5
    each_way(lambda eps: check(run(b, scale, decode=decode), b, scale, eps[dt]), decode, False)


@pytest.mark.parametrize("value", [math.nan, math.inf])
@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("heads", HEADS, ids=str)
@pytest.mark.parametrize("where", ["k", "v"])
@pytest.mark.parametrize("decode", [True, False], ids=["decode", "prefill"])
def test_a_bad_row_of_a_prefix_or_of_a_sequence_spoils_those_who_see_it(dt, heads, decode, where, value):
    """In the first group's prefix behind its third sequence's end, in that prefix's last page (of which each
    sequence has its own), in own positions."""
    scale = heads[2] ** -0.5
    for s_bad, j in (((0, 1, 2, 3), 150), ((0, 1, 3), 242), ((4,), 480), ((5,), 3)):
        b = grouped(dt, heads, decode, 32)
        pool = b.k_pool if where == "k" else b.v_pool
        for s in s_bad:
            if j < b.kv[s]:
                pool[0, b.slots(s, b.kv[s])[j], 3 if where == "v" else slice(None)] = value
        if where == "k" and value == math.inf:  # scores of +inf
            b.q[:, :, 0] = b.q[:, :, 0].abs() + 1
            b.q[:, :, 1:] = 0
        want, mag, top, seen = R.expected(b, scale)
        assert not bool(torch.isfinite(want).all()) and bool(torch.isfinite(want[b.cu[2]]).all() or s_bad[0] == 5)
        mag, top = (torch.nan_to_num(x, nan=0.0, posinf=0.0) for x in (mag, top))

        def one(eps):
            R.close(run(b, scale, decode=decode), want, R.bound(mag, top, seen, heads[2], eps[dt], 8.0))

        each_way(one, decode, False)


# ------------------------------------------------------------------ values of many sizes in one row
@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("heads", [(14, 2, 64), (32, 8, 128)], ids=str)
@pytest.mark.parametrize("kind", ["window", "shared"])
@pytest.mark.parametrize("decode", [True, False], ids=["decode", "prefill"])
def test_dims_of_very_different_sizes(dt, heads, kind, decode):
    """V rows whose dims are 1, 2^-7, 2^-14 and 2^-21 apart. Every dim is as near as its own size allows, but for
    the f16 numbers of 16-bit tiles: a value is off by 2^-25 at most, and a weight (the step of f16 at 0 is 2^-24)."""
    scale = heads[2] ** -0.5
    b = grouped(dt, heads, decode, 33)
    b.v_pool *= (2.0 ** (-7.0 * (torch.arange(heads[2]) % 4))).to(DT[dt])
    kw = dict(window=60, sinks=3) if kind == "window" else {}
    want, mag, top, seen = R.expected(b, scale, kw.get("window", R.EVERY), kw.get("sinks", 0))
    v_max = b.v_pool.double().abs().amax((0, 1))  # of a dim

    def one(eps):
        err = R.bound(mag, top, seen, heads[2], 0.0, 0.0) + 2 * eps[dt] * mag
        if dt == "f16":  # weights in f16 numbers, two of them in a step's stream
            err = err + seen[:, None, None] * 2.0 ** -25 * v_max
        elif dt == "bf16" and eps is TILE_EPS:
            err = err + seen[:, None, None] * 2.0 ** -25 * v_max + 2.0 ** -25
        got = run(b, scale, decode=decode, out_dtype=torch.float32, **kw)
        R.close(got, want, err)

    each_way(one, decode, kind == "window")


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("heads", HEADS, ids=str)
def test_steps_streamed_by_sequences_keep_both_parts_of_their_weights(dt, heads):
    scale = heads[2] ** -0.5
    b = R.batch(DT[dt], *heads, 16, [1] * 5, [450, 33, 0, 161, 1200], seed=34, starts=[0, 5], shared=[160])
    each_way(lambda eps: check(run(b, scale, decode=True, out_dtype=torch.float32), b, scale, eps[dt]), True, False)


@pytest.mark.parametrize("value", [math.nan, math.inf])
@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("heads", [(8, 2, 64), (7, 1, 128)], ids=str)
def test_bad_rows_in_items_cut_along_the_positions(dt, heads, value):
    """Few rows over a long window: pieces of numbers that are not finite, rows beside them that see them no more."""
    scale, lib = heads[2] ** -0.5, _lib.lib()
    b = R.batch(DT[dt], *heads, 16, [5, 0, 1, 20], [5000, 9, 4100, 20], seed=35)
    b.v_pool[0, b.slots(0, 5000)[1998], 9] = value  # the first three rows' windows hold it
    b.v_pool[0, b.slots(2, 4100)[10], 3] = value    # a sink
    b.k_pool[0, b.slots(0, 5000)[500]] = value      # nobody's
    want, mag, top, seen = R.expected(b, scale, 3000, 20)
    bad = ~torch.isfinite(want).all(2).all(1)
    assert bad.tolist() == [True] * 3 + [False] * 2 + [True] + [False] * 20
    mag, top = (torch.nan_to_num(x, nan=0.0, posinf=0.0) for x in (mag, top))
    err = R.bound(mag, top, seen, heads[2], TILE_EPS[dt], 8.0)
    try:
        for halves in (1, 2, 0):
            assert lib.flour_hip_set_tile_halves(halves) == 0
            R.close(run(b, scale, 3000, 20), want, err)
    finally:
        lib.flour_hip_set_tile_halves(0)
