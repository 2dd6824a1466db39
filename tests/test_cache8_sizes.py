"""Workspace sizes of the 8-bit cache's operators, without a GPU."""
from __future__ import annotations

import ctypes

import pytest
import torch

from flour_amd import _lib, ops

BF, HF, F = torch.bfloat16, torch.float16, torch.float32


def asked(name, *shape):
    n = ctypes.c_size_t(0)
    _lib.check(getattr(_lib.lib(), name)(*shape, ctypes.byref(n)))
    return n.value


def test_sizes_follow_the_switches():
    """A size that was asked for before a switch was set is asked for again."""
    shape = (3, 16, 1, 128, 500)
    name = "flour_hip_decode_weights_workspace_size"
    first = ops.decode_weights_workspace_bytes(*shape, True)
    assert first == asked(name, *shape, 1)
    try:
        assert _lib.lib().flour_hip_set_decode_workgroups(4096) == 0
        assert asked(name, *shape, 1) > first
        assert ops.decode_weights_workspace_bytes(*shape, True) == asked(name, *shape, 1)
    finally:
        _lib.lib().flour_hip_set_decode_workgroups(0)
    assert ops.decode_weights_workspace_bytes(*shape, True) == first

    shape = (8, 600, 4800, 4096, 32, 8, 128, 16)
    name = "flour_hip_varlen_prefill_q8_workspace_size"
    by_rule = ops.prefill_q8_workspace_bytes(*shape, F)
    try:
        assert _lib.lib().flour_hip_set_prefill_q8(2) == 0  # staged
        assert _lib.lib().flour_hip_set_prefill_f32_mfma(0) == 0
        off = ops.prefill_q8_workspace_bytes(*shape, F)
        assert off == asked(name, *shape, _lib.F32)
        assert _lib.lib().flour_hip_set_prefill_f32_mfma(1) == 0
        assert asked(name, *shape, _lib.F32) > off
        assert ops.prefill_q8_workspace_bytes(*shape, F) == asked(name, *shape, _lib.F32)
    finally:
        _lib.lib().flour_hip_set_prefill_f32_mfma(1)
        _lib.lib().flour_hip_set_prefill_q8(0)
    assert ops.prefill_q8_workspace_bytes(*shape, F) == by_rule


MB = 1 << 20
# the pieces of a streamed call: two of 32 columns for each of 4 waves a CU (256), or of 16 for each of 8,
# at head_dim 128 a row of 128 numbers and three more each in fp32
STREAMED = 2 * 1024 * 32 * (128 + 3) * 4 + 64 * 1024


def prefill_size(seqs, max_q, total, max_kv, H=32, G=8, D=128, bs=16, dtype=BF):
    return ops.prefill_q8_workspace_bytes(seqs, max_q, total, max_kv, H, G, D, bs, dtype)


@pytest.mark.parametrize("dtype", [BF, HF, F])
def test_prefill_of_few_rows_asks_for_no_staged_copy(dtype):
    """Drafted rows, one row of a long context, one row of each of many: they run streamed."""
    for seqs, rows, max_kv in ((32, 8, 4096), (1, 1, 131072), (64, 1, 32768), (32, 3, 4096)):
        n = prefill_size(seqs, rows, seqs * rows, max_kv, dtype=dtype)
        assert 0 < n <= STREAMED, (seqs, rows, max_kv, n / MB)


@pytest.fixture
def staged():
    _lib.lib().flour_hip_set_prefill_q8(2)
    yield
    _lib.lib().flour_hip_set_prefill_q8(0)


def test_staged_prefill_asks_for_its_copy(staged):
    """K and V of the sequences in the queries' type; with 1,536 rows in the mean or more at head_dim 128
    in 16 bits, V once more; slices of 1 GiB."""
    for (seqs, rows, max_kv, G, D, dtype), copies in (
            ((16, 512, 1536, 8, 128, BF), 2), ((4, 2048, 2048, 8, 128, HF), 3),
            ((2, 8192, 8192, 8, 128, F), 2), ((8, 2048, 2048, 2, 64, BF), 2)):
        n = prefill_size(seqs, rows, seqs * rows, max_kv, H=4 * G, G=G, D=D, dtype=dtype)
        copy = copies * seqs * max_kv * G * D * dtype.itemsize
        assert copy <= max(n, STREAMED) <= max(copy + 64 * 1024, STREAMED)
    # 128 x 8,192 positions of 32 KB: 4 GiB, in slices of 1 GiB
    assert prefill_size(128, 1024, 128 * 1024, 8192) <= (1 << 30) + MB
    assert prefill_size(128, 2048, 128 * 2048, 8192) <= (3 << 29) + MB


def test_a_smaller_workspace_is_refused():
    n = prefill_size(2, 5, 9, 60, H=4, G=2)
    args = [4096, _lib.BF16, 512, 128, 4096, 512, 128, _lib.BF16, 4096, 4096, 4096, 4096, _lib.I8, 4096,
            4096, 4096, 4, 2, 5, 9, 4, 2, 128, 16, 64, 60, 1.0]
    for ws, size in ((None, 1 << 30), (4096, n - 1), (4096 + 128, 1 << 30)):
        rc = _lib.lib().flour_hip_varlen_prefill_q8(*args, ws, size, None)
        assert rc == _lib.ERR_WORKSPACE and "workspace" in _lib.last_error()


def test_cold_prompts_are_staged():
    """A prompt without cached positions has half the products of its rows times its positions (fp32 ones
    were taken for streamed, at up to twice the time)."""
    for seqs, rows, H, G, D in ((10, 1185, 8, 8, 64), (4, 2048, 32, 8, 128), (64, 506, 14, 2, 64)):
        n = prefill_size(seqs, rows, seqs * rows, rows, H=H, G=G, D=D, dtype=F)
        assert n >= 2 * seqs * rows * G * D * 4, (seqs, rows)
    # few rows behind as many positions: as before
    assert prefill_size(10, 16, 160, 1185, H=8, G=8, D=64, dtype=F) < 2 * 10 * 1185 * 8 * 64 * 4
