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
    try:
        assert _lib.lib().flour_hip_set_prefill_f32_mfma(0) == 0
        off = ops.prefill_q8_workspace_bytes(*shape, F)
        assert off == asked(name, *shape, _lib.F32)
        assert _lib.lib().flour_hip_set_prefill_f32_mfma(1) == 0
        assert asked(name, *shape, _lib.F32) > off
        assert ops.prefill_q8_workspace_bytes(*shape, F) == asked(name, *shape, _lib.F32)
    finally:
        _lib.lib().flour_hip_set_prefill_f32_mfma(1)
