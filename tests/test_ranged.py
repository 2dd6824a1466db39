"""Attention over windows and shared prefixes without a GPU: what the C entries and the Python ones refuse
before any launch, and calls of no work."""
from __future__ import annotations

import ctypes

import pytest
import torch

from flour_amd import _lib, ops

P = 4096  # a pointer that no host check follows
BF16 = _lib.BF16

COMMON = dict(H=4, G=2, D=128, bs=16, slots=64)
DECODE = dict(out=P, od=BF16, q=P, kp=P, vp=P, bt=P, mb=4, kv=P, batch=2, **COMMON, most=60)
PACKED = dict(out=P, od=BF16, ost=512, osh=128, q=P, qst=512, qsh=128, kp=P, vp=P, cu=P, kv=P, bt=P,
              mb=4, seqs=2)
END = dict(scale=1.0, dtype=BF16, ws=P, wsb=1 << 40, stream=None)
ENTRIES = {
    "flour_hip_paged_decode_window": dict(DECODE, window=9, sinks=2, **END),
    "flour_hip_varlen_prefill_window": dict(PACKED, mq=5, total=9, **COMMON, most=60, window=9,
                                            sinks=2, **END),
    "flour_hip_paged_decode_shared": dict(out=P, od=BF16, q=P, kp=P, vp=P, bt=P, mb=4, kv=P, batch=2,
                                          starts=P, shared=P, groups=1, **COMMON, most=60, mosts=32,
                                          **END),
    "flour_hip_varlen_prefill_shared": dict(PACKED, starts=P, shared=P, groups=1, mq=5, total=9,
                                            **COMMON, most=60, mosts=32, **END),
}


def call(name, **change):
    args = ENTRIES[name]
    assert not set(change) - set(args), (name, change)
    return getattr(_lib.lib(), name)(*{**args, **change}.values())


BAD = [dict(dtype=9), dict(od=7), dict(dtype=_lib.E4M3), dict(od=_lib.I8), dict(H=5), dict(H=0),
       dict(G=0), dict(D=0), dict(bs=0), dict(slots=63), dict(slots=0), dict(mb=0), dict(most=65),
       dict(most=-1), dict(out=None), dict(q=None), dict(kp=None), dict(vp=None), dict(kv=None),
       dict(bt=None)]
WINDOW = [dict(window=0), dict(window=-1), dict(sinks=-1)]
SHARED = [dict(groups=-1), dict(mosts=-1), dict(mosts=65), dict(starts=None), dict(shared=None)]


@pytest.mark.parametrize("name", ENTRIES)
def test_refusals(name):
    bad = BAD + (WINDOW if name.endswith("window") else SHARED)
    bad += [dict(batch=-1)] if "decode" in name else [dict(seqs=-1), dict(total=-1), dict(mq=-1),
                                                      dict(cu=None)]
    for change in bad:
        assert call(name, **change) == _lib.ERR_INVALID_ARGUMENT, change
        assert _lib.last_error(), change


@pytest.mark.parametrize("name", ENTRIES)
def test_head_dims_beyond_the_kernels_are_refused(name):
    assert call(name, D=513, slots=64) == _lib.ERR_UNSUPPORTED
    assert "head_dim" in _lib.last_error()
    assert call(name, H=131072, G=65536) == _lib.ERR_UNSUPPORTED


def test_no_work_is_no_launch():
    for name in ENTRIES:
        for change in ([dict(batch=0)] if "decode" in name else [dict(seqs=0), dict(total=0)]):
            assert call(name, out=None, q=None, kp=None, bt=None, ws=None, wsb=0, **change) == 0


def test_workspace_sizes():
    lib, n = _lib.lib(), ctypes.c_size_t(0)
    size = lib.flour_hip_window_workspace_size
    assert size(2, 5, 9, 4, 2, 128, 60, 9, 2, BF16, ctypes.byref(n)) == 0
    for bad in ((-1, 5, 9, 4, 2, 128, 60, 9, 2, BF16), (2, 5, 9, 5, 2, 128, 60, 9, 2, BF16),
                (2, 5, 9, 4, 2, 0, 60, 9, 2, BF16), (2, 5, 9, 4, 2, 128, 60, 0, 2, BF16),
                (2, 5, 9, 4, 2, 128, 60, 9, -1, BF16), (2, 5, 9, 4, 2, 128, 60, 9, 2, _lib.I8)):
        assert size(*bad, ctypes.byref(n)) == _lib.ERR_INVALID_ARGUMENT, bad
    assert size(2, 5, 9, 4, 2, 128, 60, 9, 2, BF16, None) == _lib.ERR_INVALID_ARGUMENT
    size = lib.flour_hip_shared_workspace_size
    assert size(2, 1, 5, 9, 4, 2, 128, 60, 32, BF16, ctypes.byref(n)) == 0
    for bad in ((2, -1, 5, 9, 4, 2, 128, 60, 32, BF16), (2, 1, 5, 9, 4, 2, 128, 60, -1, BF16),
                (2, 1, 5, -9, 4, 2, 128, 60, 32, BF16), (2, 1, 5, 9, 4, 2, 128, 60, 32, 9)):
        assert size(*bad, ctypes.byref(n)) == _lib.ERR_INVALID_ARGUMENT, bad


def test_ops_refuse_cpu_tensors():
    p = torch.zeros((2, 64, 128))
    t, n = torch.zeros((1, 4), dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    q, c = torch.zeros((1, 4, 128)), torch.zeros(2, dtype=torch.int32)
    for f in (lambda: ops.paged_decode_window(q, p, p, t, n, 1.0, 64, 8),
              lambda: ops.varlen_prefill_window(q, p, p, c, n, t, 1, 64, 1.0, 8),
              lambda: ops.paged_decode_shared(q, p, p, t, n, c, n, 1.0, 64, 16),
              lambda: ops.varlen_prefill_shared(q, p, p, c, n, t, c, n, 1, 64, 16, 1.0)):
        with pytest.raises(_lib.FlourError, match="device tensors"):
            f()


@pytest.mark.parametrize("more", [0, 1, 2 ** 31, 2 ** 31 + 5, 2 ** 40, 2 ** 62])
def test_windows_and_sinks_beyond_32_bits_are_everything(more):
    """(A C int would hold their lowest 32 bits: a window of 2^32 + 4 as one of 4.)"""
    def size(window, sinks):
        return ops.window_workspace_bytes(2, 8, 16, 8, 2, 64, 5000, window, sinks, torch.bfloat16)

    every = 2 ** 31 - 1
    assert size(every, 0) != size(4, 0)
    assert size(every + more, 0) == size(every, 0) and size(4, every + more) == size(4, every)
    for bad in ((0 - more, 0), (1, -1 - more)):
        with pytest.raises(_lib.FlourError) as e:
            size(*bad)
        assert e.value.code == _lib.ERR_INVALID_ARGUMENT
