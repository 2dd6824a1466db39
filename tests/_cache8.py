"""64-bit restatement of the 8-bit cache, the attention over it and the eviction, in numpy on the
CPU: the definitions that the tests of those operators compare with."""
from __future__ import annotations

import math

import numpy as np
import torch

QMAX = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}

# the values of e4m3's bytes 0 .. 126 (127 is NaN; the sign bit negates)
E4M3 = np.array([(b & 7) * 2.0 ** -9 if b < 8 else (8 + (b & 7)) * 2.0 ** ((b >> 3) - 10)
                 for b in range(127)])


def values(pool: torch.Tensor) -> np.ndarray:
    """The numbers that an 8-bit tensor's bytes are, in 64 bits."""
    b = pool.detach().cpu().contiguous().view(torch.uint8).numpy()
    if pool.dtype == torch.int8:
        return b.view(np.int8).astype(np.float64)
    mag = np.append(E4M3, np.nan)[b & 127]
    return np.where(b & 128, -mag, mag)


def to8(x: np.ndarray, dtype: torch.dtype) -> np.ndarray:
    """x rounded to the 8-bit type's nearest number, ties to even, as a number."""
    if dtype == torch.int8:
        return np.rint(x)
    a = np.abs(x)
    hi = np.clip(np.searchsorted(E4M3, a), 1, 126)
    lo = hi - 1
    dl, dh = a - E4M3[lo], E4M3[hi] - a
    pick = np.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), E4M3[lo], E4M3[hi])
    return np.copysign(pick, x)


def scale_for(amax: float, dtype: torch.dtype) -> float:
    if amax == 0.0:
        return 0.0
    if not math.isfinite(amax):
        return math.nan
    e = -126
    while amax > QMAX[dtype] * 2.0 ** e:
        e += 1
    return 2.0 ** e


def quantised(x: np.ndarray, s: float, dtype: torch.dtype) -> np.ndarray:
    return to8(x / s, dtype) if s > 0 else np.zeros_like(x)


class Cache:
    """Host copies, in 64 bits, of one of an 8-bit cache's pools: q (G, blocks, bs, D), S (G, blocks)."""

    def __init__(self, pool: torch.Tensor, scale: torch.Tensor, bs: int):
        G, slots, D = pool.shape
        self.dtype, self.bs = pool.dtype, bs
        self.q = values(pool).reshape(G, slots // bs, bs, D)
        self.s = scale.detach().cpu().double().numpy().copy()

    def write(self, x: np.ndarray, block_ids, kv: int) -> None:
        """Rows x (n, G, D) as the last n of a sequence's kv positions."""
        n, bs = x.shape[0], self.bs
        if n == 0 or kv < n:
            return
        for lb in range((kv - n) // bs, (kv + bs - 1) // bs):
            if lb >= len(block_ids) or not 0 <= block_ids[lb] < self.s.shape[1]:
                continue
            b = block_ids[lb]
            lo, hi = max(kv - n - lb * bs, 0), min(kv - lb * bs, bs)
            rows = x[lb * bs + lo - (kv - n):lb * bs + hi - (kv - n)]
            for g in range(x.shape[1]):
                old = self.s[g, b] if lo > 0 else 0.0
                new = scale_for(float(np.abs(rows[:, g]).max()), self.dtype)
                s = math.nan if math.isnan(old) or math.isnan(new) else max(old, new)
                if s != old and s > 0:
                    self.q[g, b, :lo] = to8(self.q[g, b, :lo] * (old / s), self.dtype)
                self.q[g, b, lo:hi] = quantised(rows[:, g], s, self.dtype)
                self.s[g, b] = s

    def rows(self, block_ids, n: int) -> np.ndarray:
        """The values (n, G, D) of a sequence's first n positions."""
        j = np.arange(n)
        b = np.clip(np.asarray(block_ids)[j // self.bs], 0, self.s.shape[1] - 1)
        y = self.q[:, b, j % self.bs] * self.s[:, b][:, :, None]
        return y.transpose(1, 0, 2)


def attend(q: np.ndarray, k: np.ndarray, v: np.ndarray, scale: float):
    """Causal attention of the last rows q (n, H, D) of a sequence with k, v (L, G, D): the output,
    the weights (n, H, L) and a bound per (row, head) of the relative error that fp32 arithmetic
    makes on a weight and on an output (of the largest |v|): twice the score's (its products' sum in
    fp32, D + 8 roundings, and q in 22 bits) and one rounding per position summed and 64 for the
    exponential, the rescaling and the merge, all of 2^-23."""
    n, H, D = q.shape
    L, G, _ = k.shape
    out, w, err = np.zeros((n, H, D)), np.zeros((n, H, L)), np.zeros((n, H))
    for i in range(n):
        see = L - n + i + 1
        for h in range(H):
            if see <= 0:
                continue
            kk, vv = k[:see, h // (H // G)], v[:see, h // (H // G)]
            s = kk @ q[i, h] * scale
            e = np.exp(s - s.max())
            w[i, h, :see] = e / e.sum()
            out[i, h] = w[i, h, :see] @ vv
            sabs = float((np.abs(kk) @ np.abs(q[i, h])).max()) * abs(scale)
            err[i, h] = 2 * (D + 8) * 2.0 ** -24 * sabs + (see + 64) * 2.0 ** -23
    return out, w, err


def close(got: torch.Tensor, want: np.ndarray, bound: np.ndarray) -> None:
    """got within half a step of its type and `bound` of want; NaN where want is."""
    eps = torch.finfo(got.dtype).eps
    tiny = {torch.float16: 2.0 ** -25}.get(got.dtype, 0.0)  # half of f16's smallest step
    g = got.detach().cpu().double().numpy()
    assert np.array_equal(np.isnan(g), np.isnan(want))
    off = np.abs(g - want) - (eps / 2 * (np.abs(want) + bound) + bound + tiny)
    off = off[~np.isnan(off)]
    assert off.size == 0 or off.max() <= 0, f"over the bound by {off.max()}"


def evicted(w: np.ndarray, L: int, keep: int, recent: int) -> np.ndarray:
    """The positions that one kv head keeps, in order."""
    n = min(keep, L)
    late = min(recent, n)
    key = w[:L - late].astype(np.float64)
    order = sorted(range(L - late),
                   key=lambda j: (1, 0, j) if math.isnan(key[j]) else (0, -key[j], j))
    return np.array(sorted(order[:n - late]) + list(range(L - late, L)), dtype=np.int64)
