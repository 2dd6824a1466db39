"""Tensor-level entry points of the three kernels (device tensors in, device tensors out).

PyTorch only supplies device memory and the current HIP stream; every operation here is one
call into libflour_hip.so. Shapes follow the C-ABI (include/flour_hip.h):

* KV pool of one layer: ``k_pool``/``v_pool`` of shape (kv_heads, num_slots, head_dim),
  exactly PagedKvPool::new (src/models/common/paged.rs:124-167).
* ``kv_write``        <- PagedKvPool::write (paged.rs:186-204), scatter semantics.
* ``paged_decode``    <- paged_attention (src/backend/cpu.rs:57-112) for seq_q == 1, batched.
* ``varlen_prefill``  <- paged_attention for seq_q >= 1, batched over packed sequences.

A cache in 8 bits (``kv_write_q8``, ``kv_dequant``, ``paged_decode_q8``, ``varlen_prefill_q8``) has
pools of torch.float8_e4m3fn or torch.int8 and fp32 scales (kv_heads, num_blocks);
``paged_decode_weights`` and ``kv_evict`` sum attention weights and evict by them. These have no
counterpart in the reference.
"""
from __future__ import annotations

import ctypes
import functools

import torch

from . import _lib
from ._lib import check, lib, switches

_DT = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}


def dtype_code(dt: torch.dtype) -> int:
    try:
        return _DT[dt]
    except KeyError:
        raise _lib.FlourError(_lib.ERR_INVALID_ARGUMENT, f"unsupported dtype {dt}") from None


def _stream() -> ctypes.c_void_p:
    return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)


def _ptr(t: torch.Tensor | None) -> ctypes.c_void_p:
    return ctypes.c_void_p(0 if t is None else t.data_ptr())


def _need_cuda(*ts: torch.Tensor) -> None:
    for t in ts:
        if t is not None and not t.is_cuda:
            raise _lib.FlourError(_lib.ERR_INVALID_ARGUMENT,
                                  "flour_amd ops take device tensors (got a CPU tensor)")


def _need_i32(*ts: torch.Tensor) -> None:
    for t in ts:
        if t.dtype != torch.int32 or not t.is_contiguous():
            raise _lib.FlourError(_lib.ERR_INVALID_ARGUMENT,
                                  "index tensors must be contiguous int32")


def kv_write(k: torch.Tensor, v: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor,
             slot_mapping: torch.Tensor) -> None:
    """pool[h, slot_mapping[t], :] = k[t, h, :] for every token t with slot >= 0.

    ``k``/``v`` are (num_tokens, kv_heads, head_dim) views with a unit last stride (the
    reference's (kv_heads, seq, head_dim) is ``k.transpose(0, 1)`` of that). The pools are
    contiguous (kv_heads, num_slots, head_dim).
    """
    _need_cuda(k, v, k_pool, v_pool, slot_mapping)
    _need_i32(slot_mapping)
    T, G, D = k.shape
    if v.shape != k.shape or v.stride() != k.stride() or k.stride(2) != 1:
        raise _lib.FlourError(_lib.ERR_INVALID_ARGUMENT, "k/v must share shape and strides, unit last stride")
    if k_pool.shape != v_pool.shape or k_pool.shape[0] != G or k_pool.shape[2] != D or \
            not k_pool.is_contiguous() or not v_pool.is_contiguous():
        raise _lib.FlourError(_lib.ERR_INVALID_ARGUMENT, "pools must be contiguous (kv_heads, num_slots, head_dim)")
    if k.dtype != k_pool.dtype or v.dtype != k_pool.dtype or v_pool.dtype != k_pool.dtype:
        raise _lib.FlourError(_lib.ERR_INVALID_ARGUMENT, "k/v and pools must share a dtype")
    if slot_mapping.numel() != T:
        raise _lib.FlourError(_lib.ERR_INVALID_ARGUMENT, "slot_mapping needs one slot per token")
    check(lib().flour_hip_kv_write(_ptr(k), _ptr(v), k.stride(0), k.stride(1), _ptr(k_pool),
                                   _ptr(v_pool), _ptr(slot_mapping), T, G, D, k_pool.shape[1],
                                   dtype_code(k.dtype), _stream()))


def rope_tables(max_pos: int, head_dim: int, rope_theta: float, dtype: torch.dtype,
                device: torch.device | str = "cpu") -> tuple[torch.Tensor, torch.Tensor]:
    """The cos / sin tables of Cache::new (src/models/common/cache.rs:377-393), each
    (max_pos, head_dim / 2): theta_i = 1 / rope_theta^(2i / head_dim) and angle = pos * theta_i
    in fp32, cos / sin in fp32, then cast to ``dtype``. Computed with torch's fp32 CPU math
    (the reference uses Rust's f32 powf / cos / sin, which may differ in the last fp32 bit)."""
    half = head_dim // 2
    i = torch.arange(half, dtype=torch.float32)
    theta = 1.0 / torch.pow(torch.tensor(rope_theta, dtype=torch.float32), (2 * i) / head_dim)
    pos = torch.arange(max_pos, dtype=torch.float32).reshape(max_pos, 1)
    ang = pos * theta.reshape(1, half)
    return (ang.cos().to(dtype).contiguous().to(device),
            ang.sin().to(dtype).contiguous().to(device))


def rope_kv_write(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_pool: torch.Tensor,
                  v_pool: torch.Tensor, slot_mapping: torch.Tensor, positions: torch.Tensor,
                  cos: torch.Tensor, sin: torch.Tensor, q_out: torch.Tensor | None = None
                  ) -> torch.Tensor:
    """RoPE on q and k (rotate-half form, each product and sum in the tensor dtype), then
    k_pool[h, slot_mapping[t], :] = rope(k[t, h, :]) and v_pool[h, slot_mapping[t], :] =
    v[t, h, :]; returns rope(q) in ``q_out`` (default: a new tensor; ``q_out=q`` rotates in
    place). ``q`` is (num_tokens, num_heads, head_dim), ``k``/``v`` (num_tokens, kv_heads,
    head_dim), all with a unit last stride; ``positions`` holds each token's table row."""
    _need_cuda(q, k, v, k_pool, v_pool, slot_mapping, positions, cos, sin)
    _need_i32(slot_mapping, positions)
    T, H, D = q.shape
    if k.dim() != 3 or k.shape[0] != T or k.shape[2] != D or v.shape != k.shape or \
            v.stride() != k.stride() or k.stride(2) != 1 or q.stride(2) != 1:
        raise _lib.FlourError(_lib.ERR_INVALID_ARGUMENT,
                              "q (T, H, D), k/v (T, G, D) sharing strides, unit last strides")
    G = k.shape[1]
    if q_out is None:
        q_out = torch.empty_strided(q.shape, q.stride(), dtype=q.dtype, device=q.device)
    if q_out.shape != q.shape or q_out.stride() != q.stride() or q_out.dtype != q.dtype:
        raise _lib.FlourError(_lib.ERR_INVALID_ARGUMENT, "q_out must match q's shape and strides")
    if k_pool.shape != v_pool.shape or k_pool.shape[0] != G or k_pool.shape[2] != D or \
            not k_pool.is_contiguous() or not v_pool.is_contiguous():
        raise _lib.FlourError(_lib.ERR_INVALID_ARGUMENT, "pools must be contiguous (kv_heads, num_slots, head_dim)")
    dts = {q.dtype, k.dtype, v.dtype, k_pool.dtype, v_pool.dtype, cos.dtype, sin.dtype}
    if len(dts) != 1:
        raise _lib.FlourError(_lib.ERR_INVALID_ARGUMENT, "q, k, v, pools and tables must share a dtype")
    if cos.shape != sin.shape or cos.dim() != 2 or cos.shape[1] != D // 2 or \
            not cos.is_contiguous() or not sin.is_contiguous():
        raise _lib.FlourError(_lib.ERR_INVALID_ARGUMENT, "tables must be contiguous (max_pos, head_dim / 2)")
    if slot_mapping.numel() != T or positions.numel() != T:
        raise _lib.FlourError(_lib.ERR_INVALID_ARGUMENT, "one slot and one position per token")
    check(lib().flour_hip_rope_kv_write(_ptr(q_out), _ptr(q), q.stride(0), q.stride(1), H,
                                        _ptr(k), _ptr(v), k.stride(0), k.stride(1),
                                        _ptr(k_pool), _ptr(v_pool), _ptr(slot_mapping),
                                        _ptr(positions), _ptr(cos), _ptr(sin), cos.shape[0], T,
                                        G, D, k_pool.shape[1], dtype_code(q.dtype), _stream()))
    return q_out


def decode_workspace_bytes(batch: int, num_heads: int, kv_heads: int, head_dim: int,
                           max_context_len: int) -> int:
    n = ctypes.c_size_t(0)
    check(lib().flour_hip_paged_decode_workspace_size(batch, num_heads, kv_heads, head_dim,
                                                      max_context_len, ctypes.byref(n)))
    return n.value


class Workspace:
    """Device scratch for the kernels that take a workspace (split-context decode partials,
    the prefill V staging copy); grows on demand and is reused.

    Calls sharing one workspace must not overlap in time (one stream, or explicit ordering).
    A buffer that a captured graph uses stays with the workspace when it grows.
    """

    def __init__(self, device: torch.device | str = "cuda"):
        self.device = torch.device(device)
        self.buf: torch.Tensor | None = None
        self.captured: list[torch.Tensor] = []

    def get(self, nbytes: int) -> torch.Tensor:
        if self.buf is None or self.buf.numel() < nbytes:
            self.buf = torch.empty(max(nbytes, 256), dtype=torch.uint8, device=self.device)
        if self.buf.is_cuda and torch.cuda.is_current_stream_capturing() and \
                not any(self.buf is t for t in self.captured):
            self.captured.append(self.buf)
        return self.buf


DecodeWorkspace = Workspace


_default_ws: dict[int, DecodeWorkspace] = {}


def paged_decode(q: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor,
                 block_tables: torch.Tensor, context_lens: torch.Tensor, scale: float,
                 max_context_len: int, block_size: int = 16,
                 out_dtype: torch.dtype | None = None, out: torch.Tensor | None = None,
                 workspace: DecodeWorkspace | None = None) -> torch.Tensor:
    """One decode step for a batch: q (batch, num_heads, head_dim) -> (batch, num_heads, head_dim).

    ``block_tables`` is (batch, max_blocks_per_seq) int32, ``context_lens`` (batch,) int32;
    ``max_context_len`` bounds context_lens (it sizes the split-context grid); block_size is
    the cache's page size (BLOCK_SIZE = 16 in the reference, cache.rs:10).
    """
    _need_cuda(q, k_pool, v_pool, block_tables, context_lens)
    _need_i32(block_tables, context_lens)
    B, H, D = q.shape
    G, num_slots, Dk = k_pool.shape
    if Dk != D or not q.is_contiguous() or not k_pool.is_contiguous() or not v_pool.is_contiguous():
        raise _lib.FlourError(_lib.ERR_INVALID_ARGUMENT, "q and pools must be contiguous with matching head_dim")
    if q.dtype != k_pool.dtype:
        raise _lib.FlourError(_lib.ERR_INVALID_ARGUMENT, "q and pools must share a dtype")
    _check_block_size(num_slots, block_size)
    out_dtype = out_dtype or q.dtype
    if out is None:
        out = torch.empty((B, H, D), dtype=out_dtype, device=q.device)
    if workspace is None and q.dtype == torch.float32:
        # Scratch of its own, in the current stream's order: fp32 steps without a workspace
        # argument share nothing between streams. Steps that the library never splits (shorter
        # than this, other heads) pass none, and run on the vector kernel.
        may_split = max_context_len * D >= 16384 and D in (64, 128) and H <= 16 * G
        ws = torch.empty(decode_workspace_bytes(B, H, G, D, max_context_len), dtype=torch.uint8,
                         device=q.device) if may_split else None
    else:
        if workspace is None:
            workspace = _default_ws.setdefault(q.device.index or 0, DecodeWorkspace(q.device))
        ws = workspace.get(decode_workspace_bytes(B, H, G, D, max_context_len))
    check(lib().flour_hip_paged_decode(_ptr(out), dtype_code(out.dtype), _ptr(q), _ptr(k_pool),
                                       _ptr(v_pool), _ptr(block_tables), block_tables.shape[1],
                                       _ptr(context_lens), B, H, G, D, block_size, num_slots,
                                       max_context_len, float(scale), dtype_code(q.dtype),
                                       _ptr(ws), 0 if ws is None else ws.numel(), _stream()))
    return out


def prepare_paged_decode(q: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor,
                         block_tables: torch.Tensor, context_lens: torch.Tensor, scale: float,
                         max_context_len: int, out: torch.Tensor, workspace: DecodeWorkspace,
                         block_size: int = 16):
    """Validates the arguments of paged_decode once and returns a callable that relaunches the
    same decode step (same tensors, current stream at preparation time) with no per-call
    Python work beyond the C call, as a serving loop that reuses its buffers would. The callable
    keeps the workspace's present buffer alive, also when the workspace grows or goes; the
    caller keeps the tensors."""
    _need_cuda(q, k_pool, v_pool, block_tables, context_lens, out)
    _need_i32(block_tables, context_lens)
    B, H, D = q.shape
    G, num_slots, Dk = k_pool.shape
    if Dk != D or not q.is_contiguous() or not k_pool.is_contiguous() or not v_pool.is_contiguous():
        raise _lib.FlourError(_lib.ERR_INVALID_ARGUMENT, "q and pools must be contiguous with matching head_dim")
    if q.dtype != k_pool.dtype or out.shape != q.shape or not out.is_contiguous():
        raise _lib.FlourError(_lib.ERR_INVALID_ARGUMENT, "q, pools and out must agree")
    _check_block_size(num_slots, block_size)
    ws = workspace.get(decode_workspace_bytes(B, H, G, D, max_context_len))
    args = (_ptr(out), dtype_code(out.dtype), _ptr(q), _ptr(k_pool), _ptr(v_pool),
            _ptr(block_tables), block_tables.shape[1], _ptr(context_lens), B, H, G, D,
            block_size, num_slots, max_context_len, float(scale), dtype_code(q.dtype), _ptr(ws),
            ws.numel(), _stream())
    fn = lib().flour_hip_paged_decode

    def run() -> None:
        rc = fn(*args)
        if rc:
            check(rc)

    run.workspace = ws  # the buffer whose address args holds
    return run


def prefill_workspace_bytes(num_seqs: int, max_blocks_per_seq: int, block_size: int,
                            kv_heads: int, head_dim: int, dtype: torch.dtype) -> int:
    """Bytes of the V staging copy that varlen_prefill's long-prompt path reads (0 when no
    call of this shape can take that path)."""
    n = ctypes.c_size_t(0)
    check(lib().flour_hip_varlen_prefill_workspace_size(num_seqs, max_blocks_per_seq, block_size,
                                                        kv_heads, head_dim, dtype_code(dtype),
                                                        ctypes.byref(n)))
    return n.value


def varlen_prefill(q: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor,
                   cu_seqlens_q: torch.Tensor, kv_lens: torch.Tensor, block_tables: torch.Tensor,
                   max_seqlen_q: int, scale: float, block_size: int = 16,
                   out_dtype: torch.dtype | None = None,
                   out: torch.Tensor | None = None,
                   workspace: Workspace | None = None) -> torch.Tensor:
    """Causal attention of packed query rows q (total_q, num_heads, head_dim) over the cache.

    Sequence s owns rows cu_seqlens_q[s]:cu_seqlens_q[s+1] and kv_lens[s] cached positions
    (its own new rows last). q may be any view with a unit last stride, e.g. the reference's
    head-major (num_heads, seq, head_dim) transposed to (seq, num_heads, head_dim).

    Without ``workspace`` the call goes to flour_hip_varlen_prefill, which needs no device
    memory beyond its arguments. With one, flour_hip_varlen_prefill_ws may stage V in it for
    long prompts (the workspace grows to the size the call needs).
    """
    _need_cuda(q, k_pool, v_pool, cu_seqlens_q, kv_lens, block_tables)
    _need_i32(cu_seqlens_q, kv_lens, block_tables)
    T, H, D = q.shape
    G, num_slots, Dk = k_pool.shape
    if Dk != D or q.stride(2) != 1 or not k_pool.is_contiguous() or not v_pool.is_contiguous():
        raise _lib.FlourError(_lib.ERR_INVALID_ARGUMENT, "bad q / pool layout")
    if q.dtype != k_pool.dtype:
        raise _lib.FlourError(_lib.ERR_INVALID_ARGUMENT, "q and pools must share a dtype")
    _check_block_size(num_slots, block_size)
    out_dtype = out_dtype or q.dtype
    if out is None:
        out = torch.empty((T, H, D), dtype=out_dtype, device=q.device)
    num_seqs = cu_seqlens_q.numel() - 1
    args = (_ptr(out), dtype_code(out.dtype), out.stride(0), out.stride(1), _ptr(q), q.stride(0),
            q.stride(1), _ptr(k_pool), _ptr(v_pool), _ptr(cu_seqlens_q), _ptr(kv_lens),
            _ptr(block_tables), block_tables.shape[1], num_seqs, max_seqlen_q, T, H, G, D,
            block_size, num_slots, float(scale), dtype_code(q.dtype))
    if workspace is None:
        check(lib().flour_hip_varlen_prefill(*args, _stream()))
    else:
        nbytes = prefill_workspace_bytes(num_seqs, block_tables.shape[1], block_size, G, D,
                                         q.dtype)
        ws = workspace.get(nbytes)
        check(lib().flour_hip_varlen_prefill_ws(*args, _ptr(ws), ws.numel(), _stream()))
    return out


def _check_block_size(num_slots: int, block_size: int) -> None:
    """Pools hold whole blocks: num_slots is a multiple of block_size (cache.rs:21-23)."""
    if block_size <= 0 or num_slots % block_size != 0:
        raise _lib.FlourError(_lib.ERR_INVALID_ARGUMENT,
                              f"num_slots {num_slots} is not a multiple of block_size {block_size}")


# ------------------------------------------------------------------ caches kept small
# 8-bit pools (an element stands for itself times its (kv head, block)'s scale) and eviction by
# accumulated attention weight. These run on the tensors' own device, on its current stream.
_POOL_DT = {torch.float8_e4m3fn: _lib.E4M3, torch.int8: _lib.I8}


def _invalid(msg: str) -> _lib.FlourError:
    return _lib.FlourError(_lib.ERR_INVALID_ARGUMENT, msg)


def _same_device(*ts: torch.Tensor | None) -> int:
    """The index of the one device that all tensors are on."""
    dev = ts[0].get_device()
    for t in ts:
        if dev < 0 or t is not None and t.get_device() != dev:
            if not all(x is None or x.is_cuda for x in ts):
                raise _invalid("flour_amd ops take device tensors (got a CPU tensor)")
            raise _invalid(f"tensors on {ts[0].device} and {t.device}")
    return dev


def _at(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


# (a call's host time is longer than its kernels' for small batches: no attribute is looked up twice)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def _launch(fn, dev: int, *args) -> None:
    """fn(*args, stream) on the device's current stream."""
    stream = _raw_stream(dev) if _raw_stream else torch.cuda.current_stream(dev).cuda_stream
    if dev == _current_device():
        rc = fn(*args, stream)
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, stream)
    if rc:
        check(rc)


def _table(t: torch.Tensor, rows: int, what: str) -> int:
    """The table's blocks of a sequence."""
    shape = t.shape
    if len(shape) != 2 or shape[0] != rows:
        raise _invalid(f"{what} must be (sequences, blocks), got {tuple(t.shape)} for {rows}")
    return shape[1]


def _lens(t: torch.Tensor, n: int, what: str) -> None:
    if t.dim() != 1 or t.numel() != n:
        raise _invalid(f"{what} must hold {n} lengths, got {tuple(t.shape)}")


def _pools(k_pool: torch.Tensor, v_pool: torch.Tensor, block_size: int,
           what: str = "pools") -> tuple[int, int, int]:
    shape = k_pool.shape
    if len(shape) != 3 or v_pool.shape != shape or v_pool.dtype != k_pool.dtype or \
            not k_pool.is_contiguous() or not v_pool.is_contiguous():
        raise _invalid(f"{what} must be contiguous (kv_heads, num_slots, head_dim) of one dtype")
    if block_size <= 0 or shape[1] % block_size != 0:
        _check_block_size(shape[1], block_size)
    return shape


def _pools8(k_pool: torch.Tensor, v_pool: torch.Tensor, k_scale: torch.Tensor,
            v_scale: torch.Tensor, block_size: int) -> tuple[int, int, int, int]:
    """(dtype code, kv_heads, num_slots, head_dim) of an 8-bit cache's pools."""
    G, slots, D = _pools(k_pool, v_pool, block_size)
    code = _POOL_DT.get(k_pool.dtype)
    if code is None:
        raise _invalid(f"8-bit pools are torch.float8_e4m3fn or torch.int8, not {k_pool.dtype}")
    shape = (G, slots // block_size)
    for t in (k_scale, v_scale):
        if t is None or t.dtype != torch.float32 or t.shape != shape or not t.is_contiguous():
            raise _invalid(f"scales must be contiguous fp32 (kv_heads, num_blocks) = {shape}")
    return code, G, slots, D


def _out(out: torch.Tensor | None, shape, dtype: torch.dtype, device) -> torch.Tensor:
    if out is None:
        return torch.empty(shape, dtype=dtype, device=device)
    if out.shape != shape or out.device != device:
        raise _invalid(f"out must be {tuple(shape)} on {device}")
    return out


def _weights_args(weights: torch.Tensor | None, weight_rows: torch.Tensor | None, kv_heads: int,
                  batch: int, max_len: int, what: str = "weights") -> tuple:
    """(pointer, width, row pointer, rows) of the sums of attention weights."""
    if weights is None:
        if weight_rows is not None:
            raise _invalid("weight_rows without weights")
        return None, 0, None, 0
    if weights.dtype != torch.float32 or weights.dim() != 3 or weights.shape[1] != kv_heads or \
            not weights.is_contiguous() or weights.shape[2] < max_len:
        raise _invalid(f"{what} must be contiguous fp32 (rows, {kv_heads} kv heads, positions >= "
                       f"{max_len}), got {tuple(weights.shape)} {weights.dtype}")
    if weight_rows is not None:
        _need_i32(weight_rows)
        _lens(weight_rows, batch, "weight_rows")
    elif weights.shape[0] < batch:
        raise _invalid(f"{what} has {weights.shape[0]} rows for {batch} sequences")
    return weights.data_ptr(), weights.shape[2], _at(weight_rows), weights.shape[0]


def kv_write_q8(k: torch.Tensor, v: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor,
                k_scale: torch.Tensor, v_scale: torch.Tensor, cu_seqlens_q: torch.Tensor,
                kv_lens: torch.Tensor, block_tables: torch.Tensor, block_size: int = 16) -> None:
    """Quantises new K/V rows into the blocks of an 8-bit cache.

    ``k``/``v`` are (num_tokens, kv_heads, head_dim) of f32, bf16 or f16 with a unit last stride;
    sequence s brings rows cu_seqlens_q[s]:cu_seqlens_q[s+1] as its positions up to kv_lens[s].
    Each written block's scale becomes the smallest power of two with which its new rows and the
    rows it holds of the sequence from before fit the 8-bit type (those are requantised if it
    grows); a non-finite row gives NaN. A block written by one call belongs to one sequence of it.
    """
    dev = _same_device(k, v, k_pool, v_pool, k_scale, v_scale, cu_seqlens_q, kv_lens, block_tables)
    _need_i32(cu_seqlens_q, kv_lens, block_tables)
    code, G, slots, D = _pools8(k_pool, v_pool, k_scale, v_scale, block_size)
    shape, strides = k.shape, k.stride()
    if len(shape) != 3 or shape[1] != G or shape[2] != D or v.shape != shape or \
            v.stride() != strides or v.dtype != k.dtype or strides[2] != 1:
        raise _invalid("k/v must be (num_tokens, kv_heads, head_dim) sharing dtype and strides, "
                       "unit last stride")
    n = cu_seqlens_q.numel() - 1
    _lens(kv_lens, n, "kv_lens")
    width = _table(block_tables, n, "block_tables")
    _launch(lib().flour_hip_kv_write_q8, dev, k.data_ptr(), v.data_ptr(), strides[0], strides[1],
            dtype_code(k.dtype), k_pool.data_ptr(), v_pool.data_ptr(), k_scale.data_ptr(),
            v_scale.data_ptr(), code, cu_seqlens_q.data_ptr(), kv_lens.data_ptr(),
            block_tables.data_ptr(), width, n, shape[0], G, D, block_size, slots)


def kv_dequant(k_pool: torch.Tensor, v_pool: torch.Tensor, k_scale: torch.Tensor,
               v_scale: torch.Tensor, block_tables: torch.Tensor, kv_lens: torch.Tensor,
               k_out: torch.Tensor, v_out: torch.Tensor, out_tables: torch.Tensor,
               max_kv_len: int, block_size: int = 16) -> None:
    """The values of sequences in an 8-bit cache, into the blocks that ``out_tables`` gives them in
    the plain pools ``k_out``/``v_out`` (kv_heads, out_slots, head_dim) of f32, bf16 or f16.
    ``max_kv_len`` bounds kv_lens."""
    dev = _same_device(k_pool, v_pool, k_scale, v_scale, block_tables, kv_lens, k_out, v_out, out_tables)
    _need_i32(block_tables, kv_lens, out_tables)
    code, G, slots, D = _pools8(k_pool, v_pool, k_scale, v_scale, block_size)
    Go, out_slots, Do = _pools(k_out, v_out, block_size, "k_out and v_out")
    if (Go, Do) != (G, D):
        raise _invalid("k_out and v_out must have the cache's kv_heads and head_dim")
    n = kv_lens.numel()
    width = _table(block_tables, n, "block_tables")
    out_width = _table(out_tables, n, "out_tables")
    _launch(lib().flour_hip_kv_dequant, dev, k_out.data_ptr(), v_out.data_ptr(),
            dtype_code(k_out.dtype), out_tables.data_ptr(), out_width, out_slots,
            k_pool.data_ptr(), v_pool.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), code,
            block_tables.data_ptr(), width, kv_lens.data_ptr(), n, max_kv_len, G, D, block_size,
            slots)


@functools.lru_cache(maxsize=1024)
def _size(query: str, dev: int, set_count: int, *shape: int) -> int:
    """The library's size query for device dev (-1: the current one, none being in use). A size goes by
    the shape, the device's CUs and the library's switches (set_count: settings of them so far)."""
    n = ctypes.c_size_t(0)
    fn = getattr(lib(), query)
    if dev < 0 or dev == _current_device():
        check(fn(*shape, ctypes.byref(n)))
    else:
        with torch.cuda.device(dev):
            check(fn(*shape, ctypes.byref(n)))
    return n.value


def _decode_size(dev: int, batch: int, num_heads: int, kv_heads: int, head_dim: int,
                 max_context_len: int, with_weights: bool) -> int:
    return _size("flour_hip_decode_weights_workspace_size", dev, switches(), batch, num_heads,
                 kv_heads, head_dim, max_context_len, int(with_weights))


def _device_in_use() -> int:
    return torch.cuda.current_device() if torch.cuda.is_initialized() else -1


def decode_weights_workspace_bytes(batch: int, num_heads: int, kv_heads: int, head_dim: int,
                                   max_context_len: int, with_weights: bool) -> int:
    """Bytes of workspace of paged_decode_q8 and paged_decode_weights on the current device."""
    return _decode_size(_device_in_use(), batch, num_heads, kv_heads, head_dim, max_context_len,
                        with_weights)


def _scratch(workspace: Workspace | None, nbytes: int, q: torch.Tensor) -> torch.Tensor:
    # Without a caller's workspace each call has scratch of its own, in its stream's order.
    if workspace is None:
        return torch.empty(max(nbytes, 256), dtype=torch.uint8, device=q.device)
    ws = workspace.get(nbytes)
    if ws.get_device() != q.get_device():
        raise _invalid(f"workspace on {ws.device}, tensors on {q.device}")
    return ws


def _decode_q(q: torch.Tensor, D: int, G: int) -> tuple[int, int]:
    shape = q.shape
    if len(shape) != 3 or shape[2] != D or not q.is_contiguous() or shape[1] == 0 or \
            shape[1] % G != 0:
        raise _invalid("q must be contiguous (batch, num_heads, head_dim), num_heads a multiple "
                       "of the pools' kv_heads")
    return shape[0], shape[1]


def _decode_out(out: torch.Tensor | None, q: torch.Tensor,
                dtype: torch.dtype | None) -> torch.Tensor:
    if out is None:
        return torch.empty_like(q, dtype=dtype)
    out = _out(out, q.shape, q.dtype, q.device)
    if not out.is_contiguous():
        raise _invalid("out must be contiguous")
    return out


def paged_decode_q8(q: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor,
                    k_scale: torch.Tensor, v_scale: torch.Tensor, block_tables: torch.Tensor,
                    context_lens: torch.Tensor, scale: float, max_context_len: int,
                    block_size: int = 16, out_dtype: torch.dtype | None = None,
                    out: torch.Tensor | None = None, workspace: Workspace | None = None,
                    weights: torch.Tensor | None = None,
                    weight_rows: torch.Tensor | None = None) -> torch.Tensor:
    """paged_decode over an 8-bit cache: q (batch, num_heads, head_dim) of f32, bf16 or f16. With
    ``weights`` the step's attention weights are added to it, as paged_decode_weights does."""
    dev = _same_device(q, k_pool, v_pool, k_scale, v_scale, block_tables, context_lens, out, weights,
                 weight_rows)
    _need_i32(block_tables, context_lens)
    code, G, slots, D = _pools8(k_pool, v_pool, k_scale, v_scale, block_size)
    B, H = _decode_q(q, D, G)
    _lens(context_lens, B, "context_lens")
    width = _table(block_tables, B, "block_tables")
    wargs = _weights_args(weights, weight_rows, G, B, max_context_len)
    out = _decode_out(out, q, out_dtype)
    ws = _scratch(workspace, _decode_size(dev, B, H, G, D, max_context_len, weights is not None), q)
    _launch(lib().flour_hip_paged_decode_q8, dev, out.data_ptr(), dtype_code(out.dtype),
            q.data_ptr(), dtype_code(q.dtype), k_pool.data_ptr(), v_pool.data_ptr(),
            k_scale.data_ptr(), v_scale.data_ptr(), code, block_tables.data_ptr(), width,
            context_lens.data_ptr(), B, H, G, D, block_size, slots, max_context_len, float(scale),
            *wargs, ws.data_ptr(), ws.numel())
    return out


def paged_decode_weights(q: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor,
                         block_tables: torch.Tensor, context_lens: torch.Tensor, scale: float,
                         max_context_len: int, weights: torch.Tensor, block_size: int = 16,
                         out_dtype: torch.dtype | None = None, out: torch.Tensor | None = None,
                         workspace: Workspace | None = None,
                         weight_rows: torch.Tensor | None = None) -> torch.Tensor:
    """paged_decode that also adds the step's attention weights to ``weights``, fp32 (rows,
    kv_heads, positions): weights[r, g, j] += the sum over kv head g's query heads of their softmax
    weight on position j, r = weight_rows[b] or b. Rows of one call must differ; one outside the
    tensor adds nothing. A score of NaN or +inf makes its (row, kv head)'s sums NaN, for good."""
    dev = _same_device(q, k_pool, v_pool, block_tables, context_lens, out, weights, weight_rows)
    _need_i32(block_tables, context_lens)
    G, slots, D = _pools(k_pool, v_pool, block_size)
    B, H = _decode_q(q, D, G)
    if q.dtype != k_pool.dtype:
        raise _invalid("q and pools must share a dtype")
    if weights is None:
        raise _invalid("paged_decode_weights needs weights")
    _lens(context_lens, B, "context_lens")
    width = _table(block_tables, B, "block_tables")
    wargs = _weights_args(weights, weight_rows, G, B, max_context_len)
    out = _decode_out(out, q, out_dtype)
    ws = _scratch(workspace, _decode_size(dev, B, H, G, D, max_context_len, True), q)
    _launch(lib().flour_hip_paged_decode_weights, dev, out.data_ptr(), dtype_code(out.dtype),
            q.data_ptr(), k_pool.data_ptr(), v_pool.data_ptr(), block_tables.data_ptr(), width,
            context_lens.data_ptr(), B, H, G, D, block_size, slots, max_context_len, float(scale),
            dtype_code(q.dtype), *wargs, ws.data_ptr(), ws.numel())
    return out


def _prefill_size(dev: int, *shape: int) -> int:
    return _size("flour_hip_varlen_prefill_q8_workspace_size", dev, switches(), *shape)


def prefill_q8_workspace_bytes(num_seqs: int, max_seqlen_q: int, total_q: int, max_kv_len: int,
                               num_heads: int, kv_heads: int, head_dim: int, block_size: int,
                               dtype: torch.dtype) -> int:
    """Bytes of workspace of varlen_prefill_q8 on the current device."""
    return _prefill_size(_device_in_use(), num_seqs, max_seqlen_q, total_q, max_kv_len, num_heads,
                         kv_heads, head_dim, block_size, dtype_code(dtype))


def varlen_prefill_q8(q: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor,
                      k_scale: torch.Tensor, v_scale: torch.Tensor, cu_seqlens_q: torch.Tensor,
                      kv_lens: torch.Tensor, block_tables: torch.Tensor, max_seqlen_q: int,
                      max_kv_len: int, scale: float, block_size: int = 16,
                      out_dtype: torch.dtype | None = None, out: torch.Tensor | None = None,
                      workspace: Workspace | None = None) -> torch.Tensor:
    """varlen_prefill over an 8-bit cache that already holds the rows' K/V (kv_write_q8): packed q
    (total_q, num_heads, head_dim), any view with a unit last stride. ``max_seqlen_q`` bounds the
    rows of a sequence, ``max_kv_len`` kv_lens; rows of q behind the last sequence's (a padded
    batch) leave ``out`` as it was. Calls of many rows round each value of the cache once to q's type,
    exact for the scales that kv_write_q8 stores."""
    dev = _same_device(q, k_pool, v_pool, k_scale, v_scale, cu_seqlens_q, kv_lens, block_tables, out)
    _need_i32(cu_seqlens_q, kv_lens, block_tables)
    code, G, slots, D = _pools8(k_pool, v_pool, k_scale, v_scale, block_size)
    shape, strides = q.shape, q.stride()
    if len(shape) != 3 or shape[2] != D or strides[2] != 1 or shape[1] == 0 or shape[1] % G != 0:
        raise _invalid("q must be (total_q, num_heads, head_dim) with a unit last stride, "
                       "num_heads a multiple of the pools' kv_heads")
    T, H, _ = shape
    n = cu_seqlens_q.numel() - 1
    _lens(kv_lens, n, "kv_lens")
    width = _table(block_tables, n, "block_tables")
    out = _out(out, shape, out_dtype or q.dtype, q.device)
    out_strides = out.stride()
    if out_strides[2] != 1:
        raise _invalid("out must have a unit last stride")
    ws = _scratch(workspace, _prefill_size(dev, n, max_seqlen_q, T, max_kv_len, H, G, D, block_size,
                                           dtype_code(q.dtype)), q)
    _launch(lib().flour_hip_varlen_prefill_q8, dev, out.data_ptr(), dtype_code(out.dtype),
            out_strides[0], out_strides[1], q.data_ptr(), strides[0], strides[1],
            dtype_code(q.dtype), k_pool.data_ptr(), v_pool.data_ptr(), k_scale.data_ptr(),
            v_scale.data_ptr(), code, cu_seqlens_q.data_ptr(), kv_lens.data_ptr(),
            block_tables.data_ptr(), width, n, max_seqlen_q, T, H, G, D, block_size, slots,
            max_kv_len, float(scale), ws.data_ptr(), ws.numel())
    return out


def kv_evict(k_pool: torch.Tensor, v_pool: torch.Tensor, weights: torch.Tensor,
             block_tables: torch.Tensor, context_lens: torch.Tensor, keep_lens: torch.Tensor,
             out_tables: torch.Tensor, max_context_len: int, max_keep_len: int, recent: int = 0,
             block_size: int = 16, k_scale: torch.Tensor | None = None,
             v_scale: torch.Tensor | None = None, weights_out: torch.Tensor | None = None,
             weight_rows: torch.Tensor | None = None,
             kept: torch.Tensor | None = None) -> torch.Tensor:
    """Gathers, for every sequence and kv head, the ``recent`` latest positions and the heaviest
    of the others by ``weights`` (rows, kv_heads, positions) into the blocks of ``out_tables``:
    n = min(keep_lens[b], context_lens[b]) in all, in their order, ties to the lower position.
    ``weights_out`` (default: ``weights`` itself) takes the kept positions' sums in front, zeros up
    to the old length behind; ``weight_rows`` gives each sequence a row of its own. Pools are plain, or 8-bit with ``k_scale``/``v_scale``. Destination
    blocks must be new: in no sequence of the call and not twice among themselves.

    Returns the kept positions (batch, kv_heads, max_keep_len) int32, -1 behind the n-th.
    """
    dev = _same_device(k_pool, v_pool, weights, block_tables, context_lens, keep_lens, out_tables,
                 k_scale, v_scale, weights_out, weight_rows, kept)
    _need_i32(block_tables, context_lens, keep_lens, out_tables)
    if k_pool.dtype in _POOL_DT:
        code, G, slots, D = _pools8(k_pool, v_pool, k_scale, v_scale, block_size)
    else:
        G, slots, D = _pools(k_pool, v_pool, block_size)
        code = dtype_code(k_pool.dtype)
        if k_scale is not None or v_scale is not None:
            raise _invalid("scales go with 8-bit pools")
    B = context_lens.numel()
    _lens(context_lens, B, "context_lens")
    _lens(keep_lens, B, "keep_lens")
    _table(block_tables, B, "block_tables")
    _table(out_tables, B, "out_tables")
    w, width, rows, n_rows = _weights_args(weights, weight_rows, G, B, max_context_len)
    if weights_out is None:
        weights_out = weights
    elif weights_out.shape != weights.shape or weights_out.dtype != torch.float32 or \
            not weights_out.is_contiguous():
        raise _invalid("weights_out must be contiguous fp32 of the shape of weights")
    shape = (B, G, max(max_keep_len, 0))
    if kept is None:
        kept = torch.empty(shape, dtype=torch.int32, device=k_pool.device)
    else:
        _need_i32(kept)
        if kept.shape != shape:
            raise _invalid(f"kept must be {shape}")
    _launch(lib().flour_hip_kv_evict, dev, _at(k_pool), _at(v_pool), _at(k_scale),
            _at(v_scale), code, w, _at(weights_out), width, rows, n_rows, _at(block_tables),
            block_tables.shape[1], _at(context_lens), _at(keep_lens), _at(out_tables),
            out_tables.shape[1], _at(kept), B, G, D, block_size, slots, max_context_len,
            max_keep_len, recent)
    return kept
