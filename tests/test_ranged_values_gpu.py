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
