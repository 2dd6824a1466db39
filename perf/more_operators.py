"""Calls of paged attention that looks at parts of the cache: a sliding window with a few first tokens
that stay visible (sinks), and batches whose sequences share a long prefix, attended once for all.

Four kinds of call:

  decode_window   one new token per sequence, over the last `window` positions and the first `sinks`
                  ones (ops.paged_decode_window)
  prefill_window  packed rows of several new tokens per sequence, the same visibility for each row
                  behind the causal rule (ops.varlen_prefill_window)
  decode_shared   one new token per sequence; consecutive sequences form groups whose tables start with
                  the same blocks (ops.paged_decode_shared)
  prefill_shared  packed rows of several new tokens per sequence over such groups
                  (ops.varlen_prefill_shared)

`run` computes either the operators' plain form or, with `own`, makes the library's calls. Block
tables are random permutations of a pool with a quarter more blocks than the batch needs.
"""
import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BS = 16  # tokens per block


def listed():
    return [
        # a small fp32 model's chats with a short window: all latency
        dict(name="decode_window_f32_d64_b4", kind="decode_window", dtype="f32", heads=8,
             kv_heads=8, dim=64, seqs=4, lo=1, hi=1024, window=128, sinks=4),
        # the batch that a server of an 8B model runs, the window about a third of the contexts
        dict(name="decode_window_bf16_b64", kind="decode_window", dtype="bf16", heads=32,
             kv_heads=8, dim=128, seqs=64, lo=512, hi=4096, window=1024, sinks=4),
        # long documents and a large model's 64 heads
        dict(name="decode_window_f16_long_h64", kind="decode_window", dtype="f16", heads=64,
             kv_heads=8, dim=128, seqs=8, lo=16384, hi=32768, window=4096, sinks=16),
        # a small fp32 model's prompts
        dict(name="prefill_window_f32_d64", kind="prefill_window", dtype="f32", heads=8,
             kv_heads=8, dim=64, seqs=4, lo=128, hi=512, rows_lo=128, rows_hi=512, window=100,
             sinks=1),
        # a batch of prompts
        dict(name="prefill_window_bf16_b8", kind="prefill_window", dtype="bf16", heads=32,
             kv_heads=8, dim=128, seqs=8, lo=256, hi=2048, rows_lo=256, rows_hi=2048, window=512,
             sinks=4),
        # later turns of chats with a small model
        dict(name="prefill_window_f16_turns_d64", kind="prefill_window", dtype="f16", heads=14,
             kv_heads=2, dim=64, seqs=16, lo=1024, hi=4096, rows_lo=50, rows_hi=300, window=256,
             sinks=8),
        # one long document
        dict(name="prefill_window_bf16_long", kind="prefill_window", dtype="bf16", heads=28,
             kv_heads=4, dim=128, seqs=1, lo=16384, hi=16384, rows_lo=16384, rows_hi=16384,
             window=2048, sinks=4),
        # chats under one long system prompt
        dict(name="decode_shared_bf16_b64", kind="decode_shared", dtype="bf16", heads=32,
             kv_heads=8, dim=128, seqs=64, groups=1, shared_lo=8192, shared_hi=8192, own_lo=16,
             own_hi=512),
        # samples of a few questions each, a small model
        dict(name="decode_shared_f16_groups_d64", kind="decode_shared", dtype="f16", heads=14,
             kv_heads=2, dim=64, seqs=32, groups=4, shared_lo=512, shared_hi=4096, own_lo=1,
             own_hi=256),
        # samples of one question, a small fp32 model
        dict(name="decode_shared_f32_b16", kind="decode_shared", dtype="f32", heads=8, kv_heads=8,
             dim=64, seqs=16, groups=1, shared_lo=2048, shared_hi=2048, own_lo=16, own_hi=256),
        # a few drafted tokens per chat, checked in one step, under one system prompt
        dict(name="prefill_shared_bf16_drafts", kind="prefill_shared", dtype="bf16", heads=32,
             kv_heads=8, dim=128, seqs=32, groups=1, shared_lo=4096, shared_hi=4096, own_lo=64,
             own_hi=1024, rows_lo=3, rows_hi=8),
        # user turns over two cached system prompts
        dict(name="prefill_shared_bf16_turns_h28", kind="prefill_shared", dtype="bf16", heads=28,
             kv_heads=4, dim=128, seqs=16, groups=2, shared_lo=1024, shared_hi=2048, own_lo=128,
             own_hi=512, rows_lo=128, rows_hi=512),
    ]


HEADS = [(8, 8, 64), (14, 2, 64), (32, 32, 64), (28, 4, 128), (32, 8, 128), (64, 8, 128),
         (16, 16, 128)]  # (query heads, kv heads, head_dim)


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    while True:
        heads, kv_heads, dim = rng.choice(HEADS)
        kind = rng.choice(["decode_window", "prefill_window", "decode_shared", "prefill_shared"])
        c = dict(kind=kind, dtype=rng.choice(["bf16", "bf16", "f16", "f32"]), heads=heads,
                 kv_heads=kv_heads, dim=dim, seqs=log(1, 128))
        if kind.endswith("window"):
            c["hi"] = log(16, 32768)
            c["lo"] = max(1, int(c["hi"] * rng.choice([0.02, 0.125, 0.5, 1.0])))
            c["window"] = min(log(1, 8192), c["hi"])
            c["sinks"] = rng.choice([0, 1, 4, 16, 100])
            room = c["lo"]
        else:
            c["groups"] = min(c["seqs"], log(1, 16))
            c["shared_hi"] = log(16, 32768)
            c["shared_lo"] = max(1, int(c["shared_hi"] * rng.choice([0.125, 0.5, 1.0])))
            c["own_hi"] = log(1, 2048)
            c["own_lo"] = max(1, int(c["own_hi"] * rng.choice([0.02, 0.125, 0.5, 1.0])))
            room = c["own_hi"]
        if kind.startswith("prefill"):
            c["rows_hi"] = min(room, log(2, 2048))
            c["rows_lo"] = max(1, int(c["rows_hi"] * rng.choice([0.125, 0.5, 1.0])))
        w = work(c)
        positions = sum(_lens(c))  # in 32 bits while the pool is made
        if positions * kv_heads * dim < 2.7e8 and 2e4 < w["bytes"] < 5.5e8 and \
                w["flops"] < 3e11 and _padded(c) < 2e9:
            return c


# ------------------------------------------------------------------ sizes and inputs
def _rng(case, what):
    return random.Random("%s %s" % (what, sorted((k, v) for k, v in case.items() if k != "name")))


def _groups(case):
    """Where each group of sequences starts, and the prefixes' lengths in positions."""
    if not case["kind"].endswith("shared"):
        return [0], []
    rng = _rng(case, "groups")
    starts = [0] + sorted(rng.sample(range(1, case["seqs"]), case["groups"] - 1))
    shared = [rng.randint(case["shared_lo"], case["shared_hi"]) for _ in starts]
    return starts + [case["seqs"]], [max(BS, n // BS * BS) for n in shared]  # whole blocks


def _lens(case):
    """The lengths of a case's sequences (cached positions, the new rows among them)."""
    rng = _rng(case, "lens")
    if case["kind"].endswith("window"):
        return [rng.randint(case["lo"], case["hi"]) for _ in range(case["seqs"])]
    starts, shared = _groups(case)
    return [n + rng.randint(case["own_lo"], case["own_hi"])
            for g, n in enumerate(shared) for _ in range(starts[g], starts[g + 1])]


def _rows(case):
    """How many of each sequence's positions are new rows."""
    rng = _rng(case, "rows")
    lens = _lens(case)
    if case["kind"].startswith("decode"):
        return [1] * len(lens)
    starts, shared = _groups(case)
    room = list(lens)
    for g, n in enumerate(shared):
        for s in range(starts[g], starts[g + 1]):
            room[s] -= n
    return [min(n, rng.randint(case["rows_lo"], case["rows_hi"])) for n in room]


def _blocks(n):
    return (n + BS - 1) // BS


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    host = random.Random(seed)
    lens, rows = _lens(case), _rows(case)
    starts, shared = _groups(case)
    G, D, dt = case["kv_heads"], case["dim"], DTYPES[case["dtype"]]
    # each sequence's blocks: its group's prefix and its own
    front = [0] * len(lens)
    for i, n in enumerate(shared):
        for s in range(starts[i], starts[i + 1]):
            front[s] = n // BS
    used = sum(_blocks(n) - f for n, f in zip(lens, front)) + sum(n // BS for n in shared)
    blocks = used + (used + 3) // 4
    free = list(range(blocks))
    host.shuffle(free)
    prefix = [[free.pop() for _ in range(n // BS)] for n in shared]
    width = max(_blocks(n) for n in lens)
    table = []
    for s, n in enumerate(lens):
        ids = []
        for i in range(len(shared)):
            if starts[i] <= s < starts[i + 1]:
                ids = list(prefix[i])
        ids += [free.pop() for _ in range(_blocks(n) - len(ids))]
        table.append(ids + [0] * (width - len(ids)))

    def pool(outliers):
        x = torch.randn((G, blocks * BS, D), generator=g, device="cuda", dtype=torch.float32)
        if outliers:  # a few large channels, as trained projections have them
            big = torch.rand((G, 1, D), generator=g, device="cuda") < 1 / 500
            x = torch.where(big, 6.0 * x, x)
        return x.to(dt)

    st = dict(case=case, max_len=max(lens), max_rows=max(rows), scale=1.0 / math.sqrt(D),
              kv_lens=_i32(lens), table=_i32(table), k_pool=pool(True), v_pool=pool(False),
              cu=_i32([0] + torch.tensor(rows).cumsum(0).tolist()))
    if shared:
        st.update(starts=_i32(starts), shared=_i32(shared), max_shared=max(shared))
    st["q"] = torch.randn((sum(rows), case["heads"], D), generator=g, device="cuda",
                          dtype=torch.float32).to(dt)
    return st


# ------------------------------------------------------------------ the plain forms
def _values(st, table, pos):
    """fp32 K and V (kv_heads, n, positions, dim) of positions pos (n, positions) of the sequences of
    table rows (n, width)."""
    lb = (pos // BS).clamp(0, table.shape[1] - 1)
    slot = torch.gather(table.long(), 1, lb) * BS + pos % BS
    return st["k_pool"][:, slot].float(), st["v_pool"][:, slot].float()


def _softmax(s):
    e = torch.exp(s - s.amax(-1, keepdim=True).clamp(min=-3e38))
    return e / e.sum(-1, keepdim=True).clamp(min=1e-38)


def _by_head(st, q):
    """Query rows (n, rows, heads, dim) as (kv_heads, n, rows * rep, dim) in fp32."""
    n, r, H, D = q.shape
    G = st["case"]["kv_heads"]
    return q.float().view(n, r, G, H // G, D).permute(2, 0, 1, 3, 4).reshape(G, n, -1, D)


def _by_row(st, o, r):
    """The way back, in the queries' type."""
    G, n, _, D = o.shape
    o = o.view(G, n, r, -1, D).permute(1, 2, 0, 3, 4)
    return o.reshape(n, r, -1, D).to(st["q"].dtype)


def _attend(st, q, table, pos, seen):
    """Query rows q (n, rows, heads, dim) over positions pos (n, positions) where seen (n, rows,
    positions)."""
    n, r = q.shape[:2]
    rep = st["case"]["heads"] // st["case"]["kv_heads"]
    k, v = _values(st, table, pos)
    s = torch.matmul(_by_head(st, q), k.transpose(2, 3).contiguous()) * st["scale"]
    s.masked_fill_(~seen.repeat_interleave(rep, 1)[None], float("-inf"))
    return _by_row(st, torch.matmul(_softmax(s), v), r)


def _plain_decode_window(st):
    case, n = st["case"], st["kv_lens"].long()[:, None]
    W = min(case["window"], st["max_len"])
    front = torch.arange(min(case["sinks"], st["max_len"]), device="cuda").expand(len(n), -1)
    tail = n - W + torch.arange(W, device="cuda")
    pos = torch.cat([front, tail], 1)
    seen = torch.cat([front < n, tail >= case["sinks"]], 1)
    return _attend(st, st["q"][:, None], st["table"], pos.clamp(min=0), seen[:, None])[:, 0]


def _plain_prefill_window(st):
    case = st["case"]
    lens, rows, W, S = _lens(case), _rows(case), case["window"], case["sinks"]
    out, at = torch.empty_like(st["q"]), 0
    for s, (n, r) in enumerate(zip(lens, rows)):
        for i in range(0, r, 512):  # so many rows at a time, and the positions that they see
            m = min(512, r - i)
            first = n - r + i
            lo = max(0, first - W + 1)
            row = first + torch.arange(m, device="cuda")[:, None]
            pos = torch.cat([torch.arange(min(S, lo), device="cuda"),
                             torch.arange(lo, first + m, device="cuda")])
            seen = (pos <= row) & ((row - pos < W) | (pos < S))
            out[at + i:at + i + m] = _attend(st, st["q"][None, at + i:at + i + m],
                                             st["table"][s:s + 1], pos[None], seen[None])[0]
        at += r
    return out


def _plain_shared(st):
    """A group at a time: scores of all its rows over the prefix, of each sequence's over its own
    positions, one softmax over both."""
    starts, shared = _groups(st["case"])
    lens, rows = _lens(st["case"]), _rows(st["case"])
    rep = st["case"]["heads"] // st["case"]["kv_heads"]
    out, cu = torch.empty_like(st["q"]), [0]
    for r in rows:
        cu.append(cu[-1] + r)
    for a, b, P in zip(starts, starts[1:], shared):
        n, r, own_len = b - a, max(rows[a:b]), max(lens[a:b]) - P
        i = torch.arange(r, device="cuda")
        count = (st["cu"][a + 1:b + 1] - st["cu"][a:b]).long()[:, None]
        at = torch.where(i < count, st["cu"][a:b].long()[:, None] + i, cu[a])
        q = _by_head(st, st["q"][at])  # (kv_heads, n, r * rep, dim)
        G, _, c, D = q.shape
        k1, v1 = _values(st, st["table"][a:a + 1], torch.arange(P, device="cuda")[None])
        pos = P + torch.arange(own_len, device="cuda").expand(n, own_len)
        k2, v2 = _values(st, st["table"][a:b], pos)
        s1 = torch.matmul(q.reshape(G, n * c, D), k1[:, 0].transpose(1, 2).contiguous())
        s2 = torch.matmul(q, k2.transpose(2, 3).contiguous())
        row = st["kv_lens"][a:b].long()[:, None] - count + i  # the rows' own positions
        seen = (pos[:, None] <= row[:, :, None]).repeat_interleave(rep, 1)
        s2 = s2.masked_fill_(~seen[None], float("-inf"))
        p = _softmax(torch.cat([s1.view(G, n, c, P), s2], -1) * st["scale"])
        o = torch.matmul(p[..., :P].reshape(G, n * c, P), v1[:, 0]).view(G, n, c, D)
        o = o + torch.matmul(p[..., P:].contiguous(), v2)
        out[cu[a]:cu[b]] = _by_row(st, o, r)[i < count]
    return out


def run(st):
    case = st["case"]
    if own:
        return _run_own(st, case)
    if case["kind"] == "decode_window":
        return _plain_decode_window(st)
    if case["kind"] == "prefill_window":
        return _plain_prefill_window(st)
    return _plain_shared(st)


def _run_own(st, case):
    from flour_amd import ops

    if "workspace" not in st:
        st["workspace"] = ops.Workspace()
    cache, ws = (st["q"], st["k_pool"], st["v_pool"]), st["workspace"]
    if case["kind"] == "decode_window":
        return ops.paged_decode_window(*cache, st["table"], st["kv_lens"], st["scale"],
                                       st["max_len"], case["window"], case["sinks"], workspace=ws)
    if case["kind"] == "prefill_window":
        return ops.varlen_prefill_window(*cache, st["cu"], st["kv_lens"], st["table"],
                                         st["max_rows"], st["max_len"], st["scale"],
                                         case["window"], case["sinks"], workspace=ws)
    if case["kind"] == "decode_shared":
        return ops.paged_decode_shared(*cache, st["table"], st["kv_lens"], st["starts"],
                                       st["shared"], st["scale"], st["max_len"],
                                       st["max_shared"], workspace=ws)
    return ops.varlen_prefill_shared(*cache, st["cu"], st["kv_lens"], st["table"], st["starts"],
                                     st["shared"], st["max_rows"], st["max_len"],
                                     st["max_shared"], st["scale"], workspace=ws)


# ------------------------------------------------------------------ what a call cannot do without
def _padded(case):
    """Scores that the plain form holds at a time."""
    starts, shared = _groups(case)
    lens, rows = _lens(case), _rows(case)
    if case["kind"] == "decode_window":
        return case["heads"] * len(lens) * (case["window"] + case["sinks"])
    if case["kind"] == "prefill_window":
        return case["heads"] * 512 * min(max(lens), case["window"] + 512)
    return max(case["heads"] * (b - a) * max(rows[a:b]) * max(lens[a:b])
               for a, b in zip(starts, starts[1:]))


def _seen(case, n, r):
    """Visible positions, summed over the last r rows of n positions; how many any of them sees."""
    if case["kind"].endswith("shared"):
        return r * (n - r) + r * (r + 1) // 2, n
    W, S = case["window"], case["sinks"]
    pairs = sum(min(p + 1, W) + min(S, max(0, p + 1 - W)) for p in range(n - r, n))
    lo = max(0, n - r - W + 1)  # the first row's window starts here
    return pairs, n - lo + min(S, lo)


def work(case):
    H, G, D = case["heads"], case["kv_heads"], case["dim"]
    es = 4 if case["dtype"] == "f32" else 2
    lens, rows = _lens(case), _rows(case)
    starts, shared = _groups(case)
    pairs = positions = 0
    for n, r in zip(lens, rows):
        p, m = _seen(case, n, r)
        pairs, positions = pairs + p, positions + m
    for a, b, n in zip(starts, starts[1:], shared):  # a group's prefix is read once
        positions -= (b - a - 1) * n
    return dict(bytes=2 * positions * G * D * es + 4 * (positions // BS) + 2 * sum(rows) * H * D * es,
                flops=4 * pairs * H * D)


# ------------------------------------------------------------------ 64-bit results
def exact(case, seed):
    st = prepare(case, seed)
    lens, rows = _lens(case), _rows(case)
    H, G, D = case["heads"], case["kv_heads"], case["dim"]
    rep = H // G
    W = case.get("window", 1 << 40)
    S = case.get("sinks", 0)
    out = torch.empty(st["q"].shape, dtype=torch.float64, device="cuda")
    at = 0
    for s, (n, r) in enumerate(zip(lens, rows)):
        for i in range(0, r, 1024):
            m = min(1024, r - i)
            p = torch.arange(n - r + i, n - r + i + m, device="cuda")[:, None]
            j = torch.arange(n - r + i + m, device="cuda")[None, :]
            # (positions that some row of these sees)
            j = j[:, ((j < S) | (j > n - r + i - W))[0]]
            hide = (j > p) | ((j <= p - W) & (j >= S))
            slot = st["table"][s].long()[j[0] // BS] * BS + j[0] % BS
            for h in range(G):
                k, v = st["k_pool"][h, slot].double(), st["v_pool"][h, slot].double()
                q = st["q"][at + i:at + i + m, h * rep:(h + 1) * rep].double()
                x = torch.mm(q.reshape(-1, D), k.t().contiguous()).view(m, rep, -1) * st["scale"]
                w = torch.softmax(x.masked_fill_(hide[:, None], float("-inf")), dim=-1)
                o = torch.mm(w.view(m * rep, -1), v)
                out[at + i:at + i + m, h * rep:(h + 1) * rep] = o.view(m, rep, D)
        at += r
    return out
