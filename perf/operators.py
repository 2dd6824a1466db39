"""Calls of the operators that keep a paged KV cache small: a cache in 8 bits with one scale per
block of tokens and kv head, and eviction by accumulated attention weight.

Five kinds of call:

  write    new K/V rows quantised into 8-bit blocks (ops.kv_write_q8), and the written blocks read
           back as the values they stand for (ops.kv_dequant)
  decode   one new token per sequence over an 8-bit cache (ops.paged_decode_q8)
  prefill  packed rows of several new tokens per sequence over an 8-bit cache
           (ops.varlen_prefill_q8)
  weights  a decode step that adds its attention weights to the sequences' sums, over a plain
           cache (ops.paged_decode_weights) or an 8-bit one (ops.paged_decode_q8)
  evict    the heaviest and the latest positions of every sequence and kv head gathered into new
           blocks (ops.kv_evict), over a plain or an 8-bit cache

An 8-bit element stands for itself times its block's scale, a power of two: the smallest with
which no element of the block exceeds the type's largest (448 for e4m3, 127 for int8).

`run` computes either the operators' plain form or, with `own`, makes the library's calls. Block
tables are random permutations of a pool with a quarter more blocks than the batch needs.
"""
import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16,
          "e4m3": torch.float8_e4m3fn, "i8": torch.int8}
BS = 16  # tokens per block
QMAX = {"e4m3": 448.0, "i8": 127.0}


def listed():
    return [
        # one generated token for each of 64 chats, most of them into a block that is partly full
        dict(name="write_e4m3_append_b64", kind="write", pool="e4m3", dtype="bf16", seqs=64,
             heads=32, kv_heads=8, dim=128, lo=512, hi=4096, rows_lo=1, rows_hi=1),
        # a batch of prompts, each after a cached turn that ended inside a block
        dict(name="write_i8_prompts_b8", kind="write", pool="i8", dtype="bf16", seqs=8, heads=32,
             kv_heads=8, dim=128, lo=256, hi=2048, rows_lo=256, rows_hi=2040),
        # one user's chat: all latency
        dict(name="decode_e4m3_b1", kind="decode", pool="e4m3", dtype="bf16", seqs=1, heads=32,
             kv_heads=8, dim=128, lo=2000, hi=2000),
        # the batch that a server of an 8B model runs
        dict(name="decode_e4m3_b64_h32", kind="decode", pool="e4m3", dtype="bf16", seqs=64,
             heads=32, kv_heads=8, dim=128, lo=512, hi=4096),
        # long documents and a large model's 64 heads
        dict(name="decode_i8_long_h64", kind="decode", pool="i8", dtype="f16", seqs=8, heads=64,
             kv_heads=8, dim=128, lo=16384, hi=32768),
        # a small fp32 model, short chats
        dict(name="decode_i8_f32_d64", kind="decode", pool="i8", dtype="f32", seqs=16, heads=8,
             kv_heads=8, dim=64, lo=16, hi=1024),
        # user turns over one cached system prompt
        dict(name="prefill_e4m3_prefix_h28", kind="prefill", pool="e4m3", dtype="bf16", seqs=16,
             heads=28, kv_heads=4, dim=128, lo=1152, hi=1536, rows_lo=128, rows_hi=512),
        # a few drafted tokens per chat, checked in one step
        dict(name="prefill_i8_drafts_h32", kind="prefill", pool="i8", dtype="f16", seqs=32,
             heads=32, kv_heads=8, dim=128, lo=512, hi=4096, rows_lo=3, rows_hi=8),
        # the batch of chats, with the weights that a later eviction goes by
        dict(name="weights_bf16_b64_h32", kind="weights", pool="bf16", dtype="bf16", seqs=64,
             heads=32, kv_heads=8, dim=128, lo=512, hi=4096),
        # the same over 8 bits: few long sequences of a small model
        dict(name="weights_i8_b4_d64", kind="weights", pool="i8", dtype="bf16", seqs=4, heads=14,
             kv_heads=2, dim=64, lo=2048, hi=16384),
        # chats that reached their limit go back to a quarter of it
        dict(name="evict_bf16_b16", kind="evict", pool="bf16", dtype="bf16", seqs=16, heads=32,
             kv_heads=8, dim=128, lo=2048, hi=4096, keep=1000, recent=250),
        # long documents in 8 bits
        dict(name="evict_e4m3_long", kind="evict", pool="e4m3", dtype="bf16", seqs=4, heads=64,
             kv_heads=8, dim=128, lo=16384, hi=32768, keep=4096, recent=512),
    ]


HEADS = [(8, 8, 64), (14, 2, 64), (32, 32, 64), (28, 4, 128), (32, 8, 128), (64, 8, 128),
         (16, 16, 128)]  # (query heads, kv heads, head_dim)


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    while True:
        heads, kv_heads, dim = rng.choice(HEADS)
        kind = rng.choice(["write", "decode", "decode", "prefill", "weights", "evict"])
        pool = rng.choice(["e4m3", "i8"])
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
        if kind in ("weights", "evict") and rng.random() < 0.5:
            pool = dtype
        c = dict(kind=kind, pool=pool, dtype=dtype, heads=heads, kv_heads=kv_heads, dim=dim,
                 seqs=log(1, 128), hi=log(16, 32768))
        c["lo"] = max(1, int(c["hi"] * rng.choice([0.02, 0.125, 0.5, 1.0])))
        if kind in ("write", "prefill"):
            c["rows_hi"] = min(c["lo"], log(1, 2048))
            c["rows_lo"] = max(1, int(c["rows_hi"] * rng.choice([0.125, 0.5, 1.0])))
        if kind == "evict":
            c["keep"] = max(1, int(c["hi"] * rng.uniform(0.1, 0.6)))
            c["recent"] = int(c["keep"] * rng.choice([0.0, 0.1, 0.25, 0.5]))
        padded = c["seqs"] * c["hi"] * kv_heads * dim
        pairs = c["seqs"] * c.get("rows_hi", 1) * c["hi"] * heads
        w = work(c)
        if padded < 2.7e8 and pairs < 2.2e8 and 2e4 < w["bytes"] < 5.5e8 and w["flops"] < 9e10:
            return c


# ------------------------------------------------------------------ sizes and inputs
def _lens(case):
    """The lengths of a case's sequences (cached positions, the new rows among them)."""
    rng = random.Random(1000003 * case["seqs"] + 1009 * case["hi"] + case["lo"])
    return [rng.randint(case["lo"], case["hi"]) for _ in range(case["seqs"])]


def _rows(case):
    """How many of each sequence's positions are new rows."""
    rng = random.Random(7919 * case["seqs"] + 31 * case.get("rows_hi", 1) + case.get("rows_lo", 1))
    return [min(n, rng.randint(case.get("rows_lo", 1), case.get("rows_hi", 1)))
            for n in _lens(case)]


def _blocks(n):
    return (n + BS - 1) // BS


def _table(lens, at, perm):
    """Rows of block ids: sequence s holds the next _blocks(lens[s]) of perm, from perm[at] on."""
    n = torch.tensor([_blocks(x) for x in lens])
    col = torch.arange(int(n.max()))
    idx = at + (torch.cumsum(n, 0) - n)[:, None] + col
    return torch.where(col < n[:, None], perm[idx.clamp(max=len(perm) - 1)], 0).to(torch.int32)


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _pool(g, blocks, case, outliers):
    """(kv_heads, slots, dim) elements and, in 8 bits, (kv_heads, blocks) scales, of normal rows;
    one in 500 of the channels of a K pool six times as large, as trained projections have them."""
    G, D = case["kv_heads"], case["dim"]
    x = torch.randn((G, blocks, BS, D), generator=g, device="cuda", dtype=torch.float32)
    x *= torch.exp(0.4 * torch.randn((G, blocks, 1, 1), generator=g, device="cuda"))
    if outliers:
        big = torch.rand((G, 1, 1, D), generator=g, device="cuda") < 1 / 500
        x = torch.where(big, 6.0 * x, x)
    if case["pool"] not in QMAX:
        return x.reshape(G, blocks * BS, D).to(DTYPES[case["pool"]]), None
    s = _need(x.abs().amax((2, 3)), case["pool"])
    return _to8(x, s[:, :, None, None], case["pool"]).reshape(G, blocks * BS, D), s


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    host = torch.Generator()
    host.manual_seed(seed)
    lens, rows, kind = _lens(case), _rows(case), case["kind"]
    G, D, dt = case["kv_heads"], case["dim"], DTYPES[case["dtype"]]
    kept = [min(n, case["keep"]) for n in lens] if kind == "evict" else []
    used = sum(_blocks(n) for n in lens)
    need = used + sum(_blocks(n) for n in kept)
    blocks = need + (need + 3) // 4
    perm = torch.randperm(blocks, generator=host)
    st = dict(case=case, max_len=max(lens), scale=1.0 / math.sqrt(D), kv_lens=_i32(lens),
              table=_table(lens, 0, perm).cuda())
    st["k_pool"], st["k_scale"] = _pool(g, blocks, case, True)
    st["v_pool"], st["v_scale"] = _pool(g, blocks, case, False)

    def randn(n, heads):
        return torch.randn((n, heads, D), generator=g, device="cuda", dtype=torch.float32).to(dt)

    def plain_pool(n):
        shape = (G, n * BS, D)
        return (torch.zeros(shape, dtype=dt, device="cuda"),
                torch.zeros(shape, dtype=dt, device="cuda"))

    if kind in ("write", "prefill"):
        cu = torch.tensor([0] + rows).cumsum(0)
        st.update(cu=cu.to(torch.int32).cuda(), max_rows=max(rows))
    if kind == "write":
        # new rows a little larger than the cached ones, so that some blocks' scales grow
        st["k"], st["v"] = 1.5 * randn(sum(rows), G), 1.5 * randn(sum(rows), G)
        # the blocks that the call writes, read back: the sequences' tails from the first of them
        first = [(n - r) // BS for n, r in zip(lens, rows)]
        tail = [n - BS * f for n, f in zip(lens, first)]
        col = torch.arange(_blocks(max(tail))) + torch.tensor(first)[:, None]
        table = st["table"].cpu()
        back = torch.gather(table, 1, col.clamp(max=table.shape[1] - 1))
        st.update(back_table=back.contiguous().cuda(), back_lens=_i32(tail), back_max=max(tail))
        n = sum(_blocks(x) for x in tail)
        st["out_table"] = _table(tail, 0, torch.arange(n)).cuda()
        st["k_out"], st["v_out"] = plain_pool(n)
    elif kind == "evict":
        # sums of weights as decode steps leave them: a few heavy positions, a long light tail
        w = torch.randn((len(lens), G, max(lens)), generator=g, device="cuda")
        st["weights"] = torch.exp(2.0 * w - 4.0)
        st["weights_out"] = torch.zeros_like(st["weights"])
        st.update(keep_lens=_i32(kept), max_keep=max(kept),
                  out_table=_table(kept, used, perm).cuda())
        if case["pool"] in QMAX:
            n = sum(_blocks(x) for x in kept)
            st["plain_table"] = _table(kept, 0, torch.arange(n)).cuda()
            st["k_out"], st["v_out"] = plain_pool(n)
    else:
        st["q"] = randn(sum(rows), case["heads"])
        if kind == "weights":
            w = torch.randn((len(lens), G, max(lens)), generator=g, device="cuda")
            st["before"] = torch.exp(w - 5.0)
            st["weights"] = torch.empty_like(st["before"])
    return st


# ------------------------------------------------------------------ the plain forms
def _need(amax, pool):
    """The smallest power of two with amax <= QMAX * scale; 0 for 0."""
    f, e = torch.frexp(amax)
    top, bits = (0.875, 9) if pool == "e4m3" else (127 / 128, 7)
    e = torch.where(f <= top, e - bits, e - bits + 1).clamp(min=-126)
    # (2^e from its bits: ldexp's power of two may be a bit off on a GPU)
    return torch.where(amax > 0, ((e.to(torch.int32) + 127) << 23).view(torch.float32), 0.0)


def _to8(x, s, pool):
    """x / s to the nearest 8-bit value, ties to even (0 where s is 0)."""
    y = torch.where(s > 0, x / torch.where(s > 0, s, 1.0), 0.0)
    return y.to(torch.float8_e4m3fn) if pool == "e4m3" else torch.round(y).to(torch.int8)


def _at(pool, slot):
    """The 8-bit rows pool[:, slot] as fp32 (indexed as bytes)."""
    return pool.view(torch.int8)[:, slot].view(pool.dtype).float()


def _slots(table, pos):
    """The pool slots of positions pos (..., n) of the sequences of table rows (n_seqs, width)."""
    lb = (pos // BS).clamp(0, table.shape[1] - 1)
    return torch.gather(table.long(), 1, lb) * BS + pos % BS


def _values(st, table, n):
    """fp32 K and V (seqs, kv_heads, n, dim) of the first n positions of the sequences."""
    pos = torch.arange(n, device="cuda").expand(table.shape[0], n)
    slot = _slots(table, pos)

    def read(pool, scale):  # (kv_heads, seqs, n, dim), transposed
        if scale is None:
            return pool[:, slot].float().transpose(0, 1)
        x = _at(pool, slot) * scale[:, slot // BS, None]
        return x.transpose(0, 1)

    return read(st["k_pool"], st["k_scale"]), read(st["v_pool"], st["v_scale"])


def _softmax(s):
    e = torch.exp(s - s.amax(-1, keepdim=True).clamp(min=-3e38))
    return e / e.sum(-1, keepdim=True)


def _plain_attention(st, n_rows, row_of):
    """Attention of padded query rows (seqs, n_rows): row_of[b, i] is the packed row or -1. The
    output in the packed layout, and the weights (seqs, kv_heads, rep, n_rows, positions)."""
    case = st["case"]
    H, G, D, L = case["heads"], case["kv_heads"], case["dim"], st["max_len"]
    B = row_of.shape[0]
    k, v = _values(st, st["table"], L)
    q = st["q"][row_of.clamp(min=0)].float()  # (seqs, n_rows, H, D)
    q = q.view(B, n_rows, G, H // G, D).permute(0, 2, 3, 1, 4).reshape(B, G, -1, D)
    s = torch.matmul(q, k.transpose(2, 3).contiguous()) * st["scale"]
    s = s.view(B, G, H // G, n_rows, L)
    count = (row_of >= 0).sum(1, keepdim=True)
    seen = st["kv_lens"][:, None] - count + 1 + torch.arange(n_rows, device="cuda")
    hide = torch.arange(L, device="cuda") >= seen[:, :, None]  # (seqs, n_rows, positions)
    s.masked_fill_(hide[:, None, None], float("-inf"))
    p = _softmax(s)
    o = torch.matmul(p.view(B, G, -1, L), v).view(B, G, H // G, n_rows, D)
    o = o.permute(0, 3, 1, 2, 4).reshape(B, n_rows, H, D)
    return o[row_of >= 0].to(st["q"].dtype), p


def _plain_write(st):
    case = st["case"]
    T, B = st["k"].shape[0], st["table"].shape[0]
    cu, kv = st["cu"].long(), st["kv_lens"].long()
    n = cu[1:] - cu[:-1]
    seq = torch.repeat_interleave(torch.arange(B, device="cuda"), n, output_size=T)
    start = kv - n
    pos = start[seq] + torch.arange(T, device="cuda") - cu[seq]
    slot = _slots(st["table"][seq], pos[:, None])[:, 0]
    # the block that each sequence's first new row goes to, and its rows that stay
    first = _slots(st["table"], start[:, None])[:, 0]
    blk, kept = first // BS, torch.arange(BS, device="cuda") < (first % BS)[:, None]
    has = kept.any(1)
    rows = (blk * BS)[:, None] + torch.arange(BS, device="cuda")  # (seqs, BS)

    def write(x, pool, scale):
        x = x.float()
        top = torch.zeros_like(scale).index_reduce_(1, slot // BS, x.abs().amax(-1).t(), "amax")
        old = torch.zeros_like(scale)
        old[:, blk] = torch.where(has, scale[:, blk], 0.0)
        new = torch.maximum(old, _need(top, case["pool"]))
        touched = torch.zeros(scale.shape[1], dtype=torch.bool, device="cuda")
        touched[slot // BS] = True
        y = _to8(_at(pool, rows) * old[:, blk, None, None], new[:, blk, None, None],
                 case["pool"])
        keep = kept[None, :, :, None]
        bits = torch.where(keep, y.view(torch.int8), pool.view(torch.int8)[:, rows])
        pool.view(torch.int8)[:, rows] = bits
        pool.view(torch.int8)[:, slot] = _to8(x.transpose(0, 1), new[:, slot // BS, None],
                                              case["pool"]).view(torch.int8)
        scale.copy_(torch.where(touched, new, scale))

    write(st["k"], st["k_pool"], st["k_scale"])
    write(st["v"], st["v_pool"], st["v_scale"])
    _plain_dequant(st, st["back_table"], st["back_lens"], st["back_max"], st["out_table"])


def _plain_dequant(st, table, lens, longest, out_table):
    k, v = _values(st, table, longest)
    pos = torch.arange(longest, device="cuda").expand(table.shape[0], longest)
    real = pos < lens[:, None]
    to = _slots(out_table, pos)[real]
    st["k_out"][:, to] = k.transpose(0, 1)[:, real].to(st["k_out"].dtype)
    st["v_out"][:, to] = v.transpose(0, 1)[:, real].to(st["v_out"].dtype)


def _plain_evict(st):
    case, L, K = st["case"], st["max_len"], st["max_keep"]
    G, D, B = case["kv_heads"], case["dim"], st["table"].shape[0]
    j = torch.arange(L, device="cuda")
    n, kv = st["keep_lens"].long()[:, None, None], st["kv_lens"].long()[:, None, None]
    late = j >= kv - torch.clamp(n, max=case["recent"])
    key = torch.where(late, float("inf"), st["weights"])
    key = torch.where(j < kv, key, float("-inf"))
    order = torch.sort(key, dim=-1, descending=True, stable=True).indices
    rank = torch.empty_like(order).scatter_(2, order, j.expand(B, G, L).contiguous())
    chosen = torch.where(rank < n, j, L)
    kept = torch.sort(chosen, dim=-1).values[:, :, :K]  # L beyond a sequence's own n
    real = kept < L
    src_pos = torch.where(real, kept, 0)
    w = torch.gather(st["weights"], 2, src_pos)
    st["weights_out"].copy_(torch.where(j < kv, 0.0, st["weights_out"]))
    st["weights_out"][:, :, :K] = torch.where(real, w, st["weights_out"][:, :, :K])
    head = torch.arange(G, device="cuda")[:, None]
    src = _slots(st["table"], src_pos.view(B, G * K)).view(B, G, K)
    i = torch.arange(K, device="cuda").expand(B, K)
    dst = _slots(st["out_table"], i)[:, None].expand(B, G, K)

    def move(pool, scale):
        if scale is None:
            h = head.expand(B, G, K)[real]
            pool[h, dst[real]] = pool[h, src[real]]
            return
        x = pool.view(torch.int8)[head, src].view(pool.dtype).float()  # (seqs, kv_heads, K, dim)
        x = torch.where(real[..., None], x * scale[head, src // BS][..., None], 0.0)
        pad = torch.nn.functional.pad(x, (0, 0, 0, _blocks(K) * BS - K))
        new = _need(pad.view(B, G, -1, BS, D).abs().amax((3, 4)), case["pool"])  # (B, G, blocks)
        each = new.repeat_interleave(BS, 2)[:, :, :K]
        h = head.expand(B, G, K)[real]
        bits = _to8(x, each[..., None], case["pool"]).view(torch.int8)
        pool.view(torch.int8)[h, dst[real]] = bits[real]
        scale[h, dst[real] // BS] = each[real]

    move(st["k_pool"], st["k_scale"])
    move(st["v_pool"], st["v_scale"])
    if case["pool"] in QMAX:
        _plain_dequant(st, st["out_table"], st["keep_lens"], K, st["plain_table"])
    return torch.where(real, kept, -1).to(torch.int32)


def run(st):
    case = st["case"]
    kind = case["kind"]
    if own:
        return _run_own(st, case, kind)
    if kind == "write":
        _plain_write(st)
        return [st["k_scale"], st["v_scale"], st["k_out"], st["v_out"]]
    if kind == "evict":
        return _evict_outputs(st, _plain_evict(st))
    if kind == "prefill":
        cu, n = st["cu"].long(), st["max_rows"]
        i = torch.arange(n, device="cuda")
        row_of = torch.where(i < (cu[1:] - cu[:-1])[:, None], cu[:-1, None] + i, -1)
        return _plain_attention(st, n, row_of)[0]
    row_of = torch.arange(st["q"].shape[0], device="cuda")[:, None]
    out, p = _plain_attention(st, 1, row_of)
    if kind == "decode":
        return out
    st["weights"].copy_(st["before"])
    st["weights"] += p[:, :, :, 0].sum(2)
    return [out, st["weights"]]


def _evict_outputs(st, kept):
    if st["case"]["pool"] in QMAX:
        return [kept, st["weights_out"], st["k_scale"], st["v_scale"], st["k_out"], st["v_out"]]
    return [kept, st["weights_out"], st["k_pool"], st["v_pool"]]


def _run_own(st, case, kind):
    from flour_amd import ops

    if "workspace" not in st:
        st["workspace"] = ops.Workspace()
    pools = (st["k_pool"], st["v_pool"])
    if case["pool"] in QMAX:
        pools += (st["k_scale"], st["v_scale"])
    if kind == "write":
        ops.kv_write_q8(st["k"], st["v"], *pools, st["cu"], st["kv_lens"], st["table"])
        ops.kv_dequant(*pools, st["back_table"], st["back_lens"], st["k_out"], st["v_out"],
                       st["out_table"], st["back_max"])
        return [st["k_scale"], st["v_scale"], st["k_out"], st["v_out"]]
    if kind == "decode":
        return ops.paged_decode_q8(st["q"], *pools, st["table"], st["kv_lens"], st["scale"],
                                   st["max_len"], workspace=st["workspace"])
    if kind == "prefill":
        return ops.varlen_prefill_q8(st["q"], *pools, st["cu"], st["kv_lens"], st["table"],
                                     st["max_rows"], st["max_len"], st["scale"],
                                     workspace=st["workspace"])
    if kind == "weights":
        st["weights"].copy_(st["before"])
        if case["pool"] in QMAX:
            out = ops.paged_decode_q8(st["q"], *pools, st["table"], st["kv_lens"], st["scale"],
                                      st["max_len"], workspace=st["workspace"],
                                      weights=st["weights"])
        else:
            out = ops.paged_decode_weights(st["q"], *pools, st["table"], st["kv_lens"],
                                           st["scale"], st["max_len"], st["weights"],
                                           workspace=st["workspace"])
        return [out, st["weights"]]
    kept = ops.kv_evict(*pools[:2], st["weights"], st["table"], st["kv_lens"], st["keep_lens"],
                        st["out_table"], st["max_len"], st["max_keep"], recent=case["recent"],
                        k_scale=st["k_scale"], v_scale=st["v_scale"],
                        weights_out=st["weights_out"])
    if case["pool"] in QMAX:
        ops.kv_dequant(*pools, st["out_table"], st["keep_lens"], st["k_out"], st["v_out"],
                       st["plain_table"], st["max_keep"])
    return _evict_outputs(st, kept)


# ------------------------------------------------------------------ what a call cannot do without
def work(case):
    H, G, D = case["heads"], case["kv_heads"], case["dim"]
    lens, rows, kind = _lens(case), _rows(case), case["kind"]
    es = 4 if case["dtype"] == "f32" else 2
    q8 = case["pool"] in QMAX
    row = G * D * (1 if q8 else es)  # one position's K or V
    n, T = sum(lens), sum(rows)
    blocks = sum(_blocks(x) for x in lens)
    scales = 8 * G if q8 else 0  # a block's two
    if kind == "write":
        # new rows in, their 8 bits out; the written blocks' values out
        tail = sum(x - (x - r) // BS * BS for x, r in zip(lens, rows))
        return dict(bytes=2 * T * (G * D * es + row) + 2 * tail * G * D * es,
                    flops=2 * (T + tail) * G * D)
    if kind == "evict":
        kept = sum(min(x, case["keep"]) for x in lens)
        plain = 2 * kept * G * D * es if q8 else 0  # read back as values
        return dict(bytes=4 * n * G + 4 * kept * row + 4 * n * G + 4 * kept * G + plain +
                    2 * scales * kept // BS, flops=n * G)
    pairs = sum(r * (x - r) + r * (r + 1) // 2 for x, r in zip(lens, rows))
    cache = 2 * n * row + scales * blocks + 4 * blocks
    more = 8 * n * G if kind == "weights" else 0
    return dict(bytes=cache + 2 * T * H * D * es + more, flops=4 * pairs * H * D)


# ------------------------------------------------------------------ 64-bit results
def exact(case, seed):
    st = prepare(case, seed)
    lens, rows, kind = _lens(case), _rows(case), case["kind"]
    H, G, D = case["heads"], case["kv_heads"], case["dim"]
    top = QMAX.get(case["pool"])

    def slots(table, s, a, b):
        j = torch.arange(a, b, device="cuda")
        return table[s].long()[j // BS] * BS + j % BS

    def two_to(e):  # exact, unlike exp2 and ldexp
        return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)

    def rounded(x):  # 64-bit values to the 8-bit type's nearest, ties to even
        if case["pool"] == "i8":
            return torch.round(x)
        _, e = torch.frexp(x)
        step = two_to((e - 4).clamp(min=-9))
        return torch.round(x / step) * step

    k64 = v64 = None
    if kind in ("write", "evict") and top:
        def spread(p, s):
            return p.double() * s.double().repeat_interleave(BS, 1)[:, :, None]
        k64, v64 = spread(st["k_pool"], st["k_scale"]), spread(st["v_pool"], st["v_scale"])
        k_scale, v_scale = st["k_scale"].double(), st["v_scale"].double()

    if kind == "write":
        outs = []
        for x, vals, scale in ((st["k"], k64, k_scale), (st["v"], v64, v_scale)):
            out, at, to = torch.zeros(st["k_out"].shape, dtype=torch.float64, device="cuda"), 0, 0
            for s, (n, r) in enumerate(zip(lens, rows)):
                f = (n - r) // BS * BS
                sl = slots(st["table"], s, f, n)
                y = vals[:, sl].clone()
                y[:, n - r - f:] = x[at:at + r].double().transpose(0, 1)
                nb = _blocks(n - f)
                z = torch.nn.functional.pad(y, (0, 0, 0, nb * BS - (n - f))).view(G, nb, BS, D)
                new = z.clone()
                new[:, 0, :n - r - f] = 0.0
                a = new.abs().amax((2, 3))
                e = torch.ceil(torch.log2(torch.where(a > 0, a, 1.0) / top))
                e = torch.where(a > top * two_to(e), e + 1, e)
                e = torch.where((a <= top * two_to(e - 1)), e - 1, e).clamp(min=-126)
                sc = torch.where(a > 0, two_to(e), 0.0)
                ids = st["table"][s].long()[f // BS:f // BS + nb]
                if n - r > f:
                    sc[:, 0] = torch.maximum(sc[:, 0], scale[:, ids[0]])
                scale[:, ids] = sc
                d = torch.where(sc > 0, sc, 1.0)[:, :, None, None]
                w = (rounded(z / d) * d).view(G, nb * BS, D)[:, :n - f]
                out[:, slots(st["out_table"], s, 0, n - f)] = w
                at += r
            outs.append(out)
        return [k_scale, v_scale] + outs

    if kind == "evict":
        K = st["max_keep"]
        kept = torch.full((len(lens), G, K), -1, dtype=torch.int32, device="cuda")
        w_out = st["weights_out"].double()
        if top:
            plain = [torch.zeros(st["k_out"].shape, dtype=torch.float64, device="cuda")
                     for _ in range(2)]
        else:
            k64, v64 = st["k_pool"].double(), st["v_pool"].double()
            src = [k64.clone(), v64.clone()]
        for s, n in enumerate(lens):
            m = min(n, case["keep"])
            late = min(m, case["recent"])
            w = st["weights"][s, :, :n - late].cpu().numpy()
            w_out[s, :, :n] = 0.0
            for h in range(G):
                heavy = (-w[h]).argsort(kind="stable")[:m - late]
                pos = sorted(heavy.tolist()) + list(range(n - late, n))
                p = torch.tensor(pos, device="cuda")
                kept[s, h, :m] = p.int()
                w_out[s, h, :m] = st["weights"][s, h, p].double()
                sl = st["table"][s].long()[p // BS] * BS + p % BS
                to = slots(st["out_table"], s, 0, m)
                if not top:
                    k64[h, to], v64[h, to] = src[0][h, sl], src[1][h, sl]
                    continue
                ids, into = to[::BS] // BS, slots(st["plain_table"], s, 0, m)
                for vals, scale, o in ((k64, k_scale, plain[0]), (v64, v_scale, plain[1])):
                    y = torch.nn.functional.pad(vals[h, sl], (0, 0, 0, _blocks(m) * BS - m))
                    y = y.view(-1, BS, D)
                    a = y.abs().amax((1, 2))
                    e = torch.ceil(torch.log2(torch.where(a > 0, a, 1.0) / top))
                    e = torch.where(a > top * two_to(e), e + 1, e)
                    e = torch.where(a <= top * two_to(e - 1), e - 1, e).clamp(min=-126)
                    sc = torch.where(a > 0, two_to(e), 0.0)
                    scale[h, ids] = sc
                    d = torch.where(sc > 0, sc, 1.0)[:, None, None]
                    o[h, into] = (rounded(y / d) * d).view(-1, D)[:m]
        if top:
            return [kept, w_out, k_scale, v_scale] + plain
        return [kept, w_out, k64, v64]

    out = torch.empty(st["q"].shape, dtype=torch.float64, device="cuda")
    sums = st["before"].double() if kind == "weights" else None
    at = 0
    for s, (n, r) in enumerate(zip(lens, rows)):
        sl = slots(st["table"], s, 0, n)
        hide = (torch.arange(n, device="cuda")[None, :] >
                torch.arange(n - r, n, device="cuda")[:, None])
        for h in range(G):
            k, v = st["k_pool"][h, sl].double(), st["v_pool"][h, sl].double()
            if top:
                k = k * st["k_scale"][h, sl // BS].double()[:, None]
                v = v * st["v_scale"][h, sl // BS].double()[:, None]
            q = st["q"][at:at + r, h * (H // G):(h + 1) * (H // G)].double()
            x = torch.mm(q.reshape(-1, D), k.t().contiguous()).view(r, H // G, n) * st["scale"]
            p = torch.softmax(x.masked_fill_(hide[:, None], float("-inf")), dim=-1)
            o = torch.mm(p.view(-1, n), v)
            out[at:at + r, h * (H // G):(h + 1) * (H // G)] = o.view(r, H // G, D)
            if sums is not None:
                sums[s, h, :n] += p.sum((0, 1))
        at += r
    return [out, sums] if kind == "weights" else out
