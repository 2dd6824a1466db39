"""The 8-bit cache and the eviction without a GPU: what their C entries refuse before any launch, calls
of no work, and the tables that tests/_cache8.py goes by."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from _cache8 import E4M3, scale_for, to8
from flour_amd import _lib, ops

P = 4096  # a pointer that no host check follows
BF16, E4M3_T, I8 = _lib.BF16, _lib.E4M3, _lib.I8


def call(name, args, **change):
    """The entry with `args` (in order), some of them changed."""
    lib = _lib.lib()
    assert not set(change) - set(args), name
    return getattr(lib, name)(*{**args, **change}.values())


WRITE = dict(k=P, v=P, st=256, sh=128, dtype=BF16, kp=P, vp=P, ks=P, vs=P, pool=E4M3_T, cu=P, kv=P,
             bt=P, mb=4, seqs=2, total=9, G=2, D=128, bs=16, slots=64, stream=None)
DEQUANT = dict(ko=P, vo=P, dtype=BF16, ot=P, omb=4, oslots=64, kp=P, vp=P, ks=P, vs=P, pool=I8, bt=P,
               mb=4, kv=P, seqs=2, most=60, G=2, D=128, bs=16, slots=64, stream=None)
DECODE = dict(out=P, od=BF16, q=P, dtype=BF16, kp=P, vp=P, ks=P, vs=P, pool=I8, bt=P, mb=4, kv=P,
              batch=2, H=4, G=2, D=128, bs=16, slots=64, most=60, scale=1.0, w=None, width=0, wr=None,
              rows=0, ws=None, wsb=0, stream=None)
WEIGHTS = dict(out=P, od=BF16, q=P, kp=P, vp=P, bt=P, mb=4, kv=P, batch=2, H=4, G=2, D=128, bs=16,
               slots=64, most=60, scale=1.0, dtype=BF16, w=P, width=60, wr=None, rows=2, ws=None,
               wsb=0, stream=None)
PREFILL = dict(out=P, od=BF16, ost=512, osh=128, q=P, qst=512, qsh=128, dtype=BF16, kp=P, vp=P, ks=P,
               vs=P, pool=I8, cu=P, kv=P, bt=P, mb=4, seqs=2, mq=5, total=9, H=4, G=2, D=128, bs=16,
               slots=64, most=60, scale=1.0, ws=None, wsb=0, stream=None)
EVICT = dict(kp=P, vp=P, ks=None, vs=None, pool=BF16, w=P, wo=P, width=60, wr=None, rows=2, bt=P, mb=4,
             kv=P, keep=P, ot=P, omb=2, kept=P, batch=2, G=2, D=128, bs=16, slots=64, most=60,
             mostk=20, recent=4, stream=None)

POOL = [dict(pool=BF16), dict(pool=9), dict(G=0), dict(D=0), dict(bs=0), dict(slots=63), dict(slots=0),
        dict(kp=None), dict(ks=None), dict(slots=1 << 31)]


@pytest.mark.parametrize("name,args,bad", [
    ("flour_hip_kv_write_q8", WRITE, POOL + [dict(dtype=E4M3_T), dict(seqs=-1), dict(total=-1),
                                             dict(mb=0), dict(k=None), dict(cu=None)]),
    ("flour_hip_kv_dequant", DEQUANT, POOL + [dict(dtype=I8), dict(most=65), dict(omb=3),
                                              dict(oslots=40), dict(vo=None), dict(ot=None),
                                              dict(seqs=-1)]),
    ("flour_hip_paged_decode_q8", DECODE, POOL + [dict(dtype=I8), dict(od=7), dict(H=3), dict(H=0),
                                                  dict(most=65), dict(batch=-1), dict(q=None),
                                                  dict(w=P, width=59, rows=2),
                                                  dict(w=P, width=60, rows=1)]),
    ("flour_hip_paged_decode_weights", WEIGHTS, [dict(w=None), dict(dtype=I8), dict(H=5),
                                                 dict(slots=40), dict(most=61), dict(rows=1),
                                                 dict(kp=None), dict(mb=0)]),
    ("flour_hip_varlen_prefill_q8", PREFILL, POOL + [dict(dtype=I8), dict(od=I8), dict(H=3),
                                                     dict(total=-1), dict(most=65), dict(mq=-1),
                                                     dict(q=None), dict(cu=None)]),
    ("flour_hip_kv_evict", EVICT, [dict(pool=9), dict(G=0), dict(bs=0), dict(slots=40), dict(most=61),
                                   dict(mostk=33), dict(recent=-1), dict(rows=1), dict(w=None),
                                   dict(kept=None), dict(ot=None), dict(ks=P), dict(pool=I8),
                                   dict(pool=I8, ks=P), dict(batch=-1)]),
])
def test_refusals(name, args, bad):
    for change in bad:
        assert call(name, args, **change) == _lib.ERR_INVALID_ARGUMENT, change
        assert _lib.last_error(), change


def test_workspaces_are_asked_for_and_checked():
    n = ctypes.c_size_t(0)
    size = _lib.lib().flour_hip_decode_weights_workspace_size
    assert size(2, 4, 2, 128, 60, 1, ctypes.byref(n)) == 0 and n.value >= 2 * 4 * 60 * 4
    for ws, b in ((None, 1 << 30), (P, n.value - 1), (P + 128, 1 << 30)):
        assert call("flour_hip_paged_decode_weights", WEIGHTS, ws=ws, wsb=b) == _lib.ERR_WORKSPACE
        assert "workspace" in _lib.last_error()
    assert size(2, 4, 3, 128, 60, 1, ctypes.byref(n)) == _lib.ERR_INVALID_ARGUMENT
    assert size(2, 4, 2, 128, 60, 1, None) == _lib.ERR_INVALID_ARGUMENT
    size = _lib.lib().flour_hip_varlen_prefill_q8_workspace_size
    assert size(2, 5, 9, 60, 4, 2, 128, 16, BF16, ctypes.byref(n)) == 0
    assert size(2, 5, 9, 60, 4, 2, 128, 16, I8, ctypes.byref(n)) == _lib.ERR_INVALID_ARGUMENT
    assert size(2, 5, 9, 60, 5, 2, 128, 16, BF16, ctypes.byref(n)) == _lib.ERR_INVALID_ARGUMENT


def test_no_work_is_no_launch():
    for name, args, change in (
            ("flour_hip_kv_write_q8", WRITE, dict(total=0)), ("flour_hip_kv_write_q8", WRITE, dict(seqs=0)),
            ("flour_hip_kv_dequant", DEQUANT, dict(seqs=0)), ("flour_hip_kv_dequant", DEQUANT, dict(most=0)),
            ("flour_hip_paged_decode_q8", DECODE, dict(batch=0)),
            ("flour_hip_paged_decode_weights", WEIGHTS, dict(batch=0)),
            ("flour_hip_varlen_prefill_q8", PREFILL, dict(total=0)),
            ("flour_hip_kv_evict", EVICT, dict(batch=0))):
        assert call(name, args, **change) == 0, name


def test_plain_functions_refuse_the_8_bit_types():
    lib = _lib.lib()
    for t in (E4M3_T, I8):
        assert lib.flour_hip_kv_write(P, P, 0, 0, P, P, P, 4, 2, 8, 16, t, None) == \
            _lib.ERR_INVALID_ARGUMENT
        n = ctypes.c_size_t(0)
        assert lib.flour_hip_varlen_prefill_workspace_size(1, 1, 16, 1, 128, t, ctypes.byref(n)) == \
            _lib.ERR_INVALID_ARGUMENT


def test_ops_refuse_cpu_tensors():
    p = torch.zeros((2, 64, 128), dtype=torch.int8)
    s, t, n = torch.ones((2, 4)), torch.zeros((1, 4), dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    q, w = torch.zeros((1, 4, 128)), torch.zeros((1, 2, 64))
    for f in (lambda: ops.kv_write_q8(q[:, :2], q[:, :2], p, p, s, s, n, n, t),
              lambda: ops.kv_dequant(p, p, s, s, t, n, p.float(), p.float(), t, 64),
              lambda: ops.paged_decode_q8(q, p, p, s, s, t, n, 1.0, 64),
              lambda: ops.paged_decode_weights(q, p.float(), p.float(), t, n, 1.0, 64, w),
              lambda: ops.varlen_prefill_q8(q, p, p, s, s, n, n, t, 1, 64, 1.0),
              lambda: ops.kv_evict(p.float(), p.float(), w, t, n, n, t, 64, 16)):
        with pytest.raises(_lib.FlourError, match="device tensors"):
            f()


def test_the_tables_of_the_64_bit_form():
    t = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(t, E4M3)
    x = torch.randn(4096, generator=torch.Generator().manual_seed(0)) * 3
    x = torch.cat([x, torch.arange(-64, 65) / 1024.0, torch.tensor([448.0, -448.0, 0.0])])
    assert np.array_equal(to8(x.double().numpy(), torch.float8_e4m3fn),
                          x.to(torch.float8_e4m3fn).double().numpy())
    for d, top in ((torch.int8, 127.0), (torch.float8_e4m3fn, 448.0)):
        for e in (-100, -7, 0, 30):
            assert scale_for(top * 2.0 ** e, d) == 2.0 ** e
            assert scale_for(top * 2.0 ** e * (1 + 2.0 ** -20), d) == 2.0 ** (e + 1)


def test_shapes_beyond_the_kernels_counts_are_refused():
    for name, args in (("flour_hip_kv_write_q8", WRITE), ("flour_hip_paged_decode_q8", DECODE),
                       ("flour_hip_varlen_prefill_q8", PREFILL), ("flour_hip_kv_dequant", DEQUANT)):
        # a block of 2^23 x 256 = 2^31 elements
        assert call(name, args, bs=1 << 23, D=256, slots=1 << 24) == _lib.ERR_INVALID_ARGUMENT, name
    for change in (dict(batch=65536, rows=65536), dict(G=65536, H=65536)):
        assert call("flour_hip_paged_decode_weights", WEIGHTS, **change) == _lib.ERR_UNSUPPORTED
        assert "too many" in _lib.last_error()
    assert call("flour_hip_kv_evict", EVICT, batch=65536, rows=65536) == _lib.ERR_UNSUPPORTED
