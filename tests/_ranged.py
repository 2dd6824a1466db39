"""64-bit restatement of the attention over a sliding window with sinks and over shared prefixes, and
batches for its tests."""
from __future__ import annotations

import math
import random
from dataclasses import dataclass

import torch

EVERY = 0x7fffffff  # a window over all positions


def attend(q, k, v, scale, window=EVERY, sinks=0):
    """The last rows q (n, H, D) of a sequence with k, v (L, G, D), all float64: row i at p = L - n + i
    sees j <= p with p - j < window or j < sinks. The output, and per (row, head) the sum of weight times
    |v| (n, H, D), the largest |score|'s bound sum |k q| |scale| and the number of positions seen, for
    bounds of the error."""
    n, H, D = q.shape
    L, G, _ = k.shape
    rep = H // G
    p = torch.arange(L - n, L)[:, None]
    j = torch.arange(L)[None]
    seen = (j <= p) & ((p - j < window) | (j < sinks))  # (n, L)
    out, mag = torch.zeros_like(q), torch.zeros_like(q)
    top = torch.zeros((n, H), dtype=torch.float64)
    clean = bool(torch.isfinite(v).all())
    for h in range(H):
        kk, vv = k[:, h // rep], v[:, h // rep]
        s = (q[:, h] @ kk.t()) * scale
        s = torch.where(seen, s, -math.inf)
        m = s.amax(1, keepdim=True)
        none = m == -math.inf  # no position, or no score above -inf
        e = torch.exp(s - torch.where(none, 0.0, m))
        w = e / torch.where(none, 1.0, e.sum(1, keepdim=True))
        if clean:
            out[:, h], mag[:, h] = w @ vv, w @ vv.abs()
        else:
            for i in range(n):
                x = torch.where(seen[i][:, None] & ~none[i], w[i][:, None] * vv, 0.0)
                out[i, h], mag[i, h] = x.sum(0), x.abs().sum(0)
        a = torch.where(seen, q[:, h].abs() @ kk.abs().t(), 0.0)
        top[:, h] = a.amax(1) * abs(scale)
    return out, mag, top, seen.sum(1)


@dataclass
class Batch:
    """Sequences over a pool of pages, on the CPU."""
    q: torch.Tensor             # (rows, H, D)
    k_pool: torch.Tensor
    v_pool: torch.Tensor
    cu: list
    kv: list
    tables: torch.Tensor
    bs: int
    starts: list
    shared: list

    @property
    def max_rows(self):
        return max((b - a for a, b in zip(self.cu, self.cu[1:])), default=0)

    @property
    def max_kv(self):
        return max(self.kv + [0])

    def slots(self, s, n):
        j = torch.arange(n)
        return self.tables[s].long()[j // self.bs] * self.bs + j % self.bs

    def rows(self, s, n):
        """K and V (n, G, D) of the sequence's first n positions, in 64 bits."""
        sl = self.slots(s, n)
        return (self.k_pool[:, sl].double().transpose(0, 1), self.v_pool[:, sl].double().transpose(0, 1))


def batch(dtype, heads, kv_heads, dim, bs, rows, kv, seed=0, starts=(), shared=(), spare=3,
          v_scale=1.0):
    """rows[s] new rows of kv[s] positions a sequence, over shuffled pages; sequences of group g share
    the whole blocks of their first shared[g] positions, and copies of the rest of them."""
    g = torch.Generator().manual_seed(seed)
    rng = random.Random(seed)
    n = len(kv)
    front, lead = [0] * n, [0] * n
    for i, P in enumerate(shared):
        for s in range(starts[i], starts[i + 1]):
            front[s], lead[s] = P, starts[i]
    need = [(max(kv[s], front[s]) + bs - 1) // bs for s in range(n)]
    total = sum(need) + spare
    free = list(range(total))
    rng.shuffle(free)
    width = max(need + [1])
    tables = torch.zeros((n, width), dtype=torch.int32)
    for s in range(n):
        for b in range(need[s]):
            whole = (b + 1) * bs <= front[s]
            tables[s, b] = tables[lead[s], b] if whole and lead[s] != s else free.pop()
    T = sum(rows)
    q = torch.randn((T, heads, dim), generator=g)
    k = torch.randn((kv_heads, total * bs, dim), generator=g)
    v = torch.randn((kv_heads, total * bs, dim), generator=g) * v_scale
    cu = [0]
    for r in rows:
        cu.append(cu[-1] + r)
    b = Batch(q.to(dtype), k.to(dtype), v.to(dtype), cu, list(kv), tables, bs, list(starts),
              list(shared))
    for s in range(n):  # a prefix that ends inside a block: the same rows in each one's own
        if lead[s] != s and front[s] % bs:
            src, dst = b.slots(lead[s], front[s]), b.slots(s, front[s])
            b.k_pool[:, dst], b.v_pool[:, dst] = b.k_pool[:, src], b.v_pool[:, src]
    return b


def expected(b: Batch, scale, window=EVERY, sinks=0):
    """Outputs (rows, H, D) in 64 bits, and what their bounds go by."""
    T, H, D = b.q.shape
    out, mag = torch.zeros((T, H, D), dtype=torch.float64), torch.zeros((T, H, D), dtype=torch.float64)
    top, seen = torch.zeros((T, H), dtype=torch.float64), torch.zeros(T)
    for s, L in enumerate(b.kv):
        r0, r1 = b.cu[s], b.cu[s + 1]
        if L < r1 - r0 or r1 == r0:
            continue
        k, v = b.rows(s, L)
        out[r0:r1], mag[r0:r1], top[r0:r1], seen[r0:r1] = attend(b.q[r0:r1].double(), k, v, scale,
                                                                 window, sinks)
    return out, mag, top, seen


def bound(mag, top, seen, dim, weight_eps, v_max):
    """How far fp32 arithmetic may be off: a score is a sum of D products (D + 8 roundings of 2^-24 of
    the sum of their magnitudes, in the exponent of numerator and denominator: twice), the weights'
    sums, rescalings and exponentials come to 2^-23 for each position and 64 more; a weight is rounded to
    weight_eps of itself in the products and at most that in the sum (twice); weights below f16's normal
    numbers are off by 2^-25 of the largest at most, values by 2^-25."""
    rel = 2 * (dim + 8) * 2.0 ** -24 * top[..., None] + (seen[:, None, None] + 64) * 2.0 ** -23
    rel = rel + 2 * weight_eps
    return rel * mag + (weight_eps > 0) * (seen[:, None, None] * 2.0 ** -25 * v_max + 2.0 ** -25)


def close(got, want, err):
    """got within half a step of its type and err of want; NaN where want is NaN, or infinite (an infinite
    V row times weights of either rounding: the outputs' own infinities may be NaN)."""
    eps = torch.finfo(got.dtype).eps
    tiny = 2.0 ** -25 if got.dtype == torch.float16 else 0.0  # half of f16's smallest step
    g = got.detach().cpu().double()
    assert g.shape == want.shape
    bad = ~torch.isfinite(want)
    assert torch.equal(~torch.isfinite(g), bad), "non-finite outputs in other places"
    off = (g - want).abs() - (eps / 2 * (want.abs() + err) + err + tiny)
    off = off[~bad]
    assert off.numel() == 0 or float(off.max()) <= 0, f"over the bound by {float(off.max())}"
