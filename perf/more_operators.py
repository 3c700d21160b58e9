"""Prefill of chunks over shared pages of a latent cache, as timed cases.

A case names an operator and its sizes:

  attend   attention of a chunk of new tokens over a paged cache in the expanded form: each key's
           latent row gives every head a key (W_uk) and a value (W_uv) of its own, and queries come
           per head, unabsorbed; the cache in 16 bits, or in 8 bits with block scales
  fork     requests continue other requests' first tokens: whole pages are shared, a page that two
           requests would write gets a copy, pages that nobody holds any more are freed
  copy     pages copied within pools, as `fork` and `compact` ask for
  compact  pages in use moved to the low end of the pool: tables, ring of free pages, copies
  step     a shared prompt forked to its requests, pages copied, new tokens' pages, their cache
           rows, their queries and their attention

B requests of up to Sq new tokens; Sk is the longest one's keys, the new ones included.
"""

from __future__ import annotations

import math
import os
import random
import sys

import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(ROOT, "mla-cuda_amd")

DEVICE = "cuda:0"
EPS = 1e-6
HIDDEN, QL, HEADS, R, D, V, NOPE = 7168, 1536, 128, 512, 64, 128, 128
SCALE = math.sqrt(NOPE + D)
DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16}
PAGE = 64
E4M3 = torch.float8_e4m3fn


def attend(name, dtype, B, Sq, Sk, block=0, heads=HEADS):
    """block: 0 for a cache in the queries' type, else tokens a scale of the 8-bit one."""
    return {"name": name, "op": "attend", "dtype": dtype, "B": B, "Sq": Sq, "Sk": Sk,
            "block": block, "heads": heads}


def pages(name, op, B, Sk, spare, layers=1, dtype="bfloat16"):
    """spare: free pages for each page in use (the pool's size); layers: of copied pools."""
    return {"name": name, "op": op, "dtype": dtype, "B": B, "Sk": Sk, "spare": spare, "layers": layers}


def listed():
    return [
        # a follow-up question early in a chat: the smallest chunk
        attend("attend_chunk_short_bf16", "bfloat16", 1, 64, 512),
        # one long prompt, cut into chunks of the usual size; this is its first
        attend("attend_prompt_bf16", "bfloat16", 1, 4096, 4096),
        # and this one further into the document, one device's share of the heads
        attend("attend_document_bf16", "bfloat16", 1, 2048, 32768, heads=16),
        # a batch of ragged chunks beside what is in the cache, in the other 16-bit type
        attend("attend_batch_f16", "float16", 4, 517, 6001),
        # the same work over the cache in 8 bits
        attend("attend_blocked_bf16", "bfloat16", 3, 1024, 8192, block=32),
        # beams of one request change places
        pages("fork_beams", "fork", 8, 700, 0.5),
        # a busy server: some requests continue others' prefixes, some are cut back, some end
        pages("fork_serving", "fork", 256, 16384, 0.25),
        # a small pool made dense again
        pages("compact_small", "compact", 16, 2011, 1.0),
        # a large one, after many requests ended
        pages("compact_pool", "compact", 256, 32768, 0.7),
        # what a compaction moves, in every layer
        pages("copy_compacted_bf16", "copy", 32, 4096, 1.0, layers=4),
        # the open pages of forked requests, in every layer
        pages("copy_forked_f16", "copy", 64, 300, 0.5, layers=8, dtype="float16"),
        # forks of a shared prompt with a ragged chunk each, from the tables to the attention
        {"name": "step_shared_prompt_bf16", "op": "step", "dtype": "bfloat16", "B": 6, "Sq": 300,
         "Sk": 1801, "block": 0, "heads": HEADS},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def _cost(c):
    w = work(c)
    return w["flops"] / 1e15 + w["bytes"] / 4e12


def draw(rng):
    most = max(_cost(c) for c in listed())
    while True:
        op = rng.choice(["attend", "attend", "attend", "attend", "fork", "compact", "copy", "step"])
        dtype = rng.choice(["bfloat16", "bfloat16", "float16"])
        if op in ("attend", "step"):
            B, Sq = _log_int(rng, 1, 8), _log_int(rng, 16, 4096)
            Sk = Sq + rng.choice([0, _log_int(rng, 64, 32768)])
            heads = rng.choice([HEADS, HEADS, 16, 32])
            block = rng.choice([0, 0, 16, 32, 64])
            if op == "step":
                Sq, block, heads = min(Sq, 1024), 0, HEADS
                Sk = max(Sk, Sq + 64)
            c = {"op": op, "dtype": dtype, "B": B, "Sq": Sq, "Sk": Sk, "block": block, "heads": heads}
            if B * (Sk + PAGE) * 2 * heads * V * 4 > 2e10 or B * Sq * heads * 4 * Sk > 4e11:
                continue
        else:
            B, Sk = _log_int(rng, 1, 256), _log_int(rng, 1, 32768)
            c = {"op": op, "dtype": dtype, "B": B, "Sk": Sk, "spare": rng.choice([0.25, 0.7, 1.0]),
                 "layers": _log_int(rng, 1, 8) if op == "copy" else 1}
            if op == "copy" and pool_pages(c) * c["layers"] * PAGE * (R + D) * 2 > 1.5e9:
                continue
        if _cost(c) <= most:
            return c


def lengths(c):
    """Tokens of each request, the new ones included: the longest has Sk, the others spread below."""
    r = random.Random(c["B"] * 1000003 + c["Sk"])
    low = c.get("Sq", 1)
    return [c["Sk"]] + [r.randint(low, c["Sk"]) for _ in range(c["B"] - 1)]


def new_tokens(c):
    """New tokens of each request: Sq, but in ragged batches some bring fewer (or none)."""
    r = random.Random(c["B"] * 7919 + c["Sq"])
    return [c["Sq"] if b == 0 or r.random() < 0.6 else r.randint(0, c["Sq"]) for b in range(c["B"])]


def pool_pages(c):
    used = sum(-(-n // PAGE) for n in lengths(c))
    return used + max(2 * c["B"], int(c["spare"] * used))


def fork_plan(c):
    """Parents and tokens kept: half of the requests stay as they are, the others continue a
    prefix of another one, are cut back, or end."""
    lens = lengths(c)
    r = random.Random(c["B"] * 31 + c["Sk"])
    parents, keep = [], []
    for b, n in enumerate(lens):
        kind = r.random()
        if kind < 0.5:
            p, k = b, n
        elif kind < 0.8:
            p = r.randrange(len(lens))
            k = r.choice([lens[p], r.randint(0, lens[p])])
        elif kind < 0.9:
            p, k = b, r.randint(0, n)
        else:
            p, k = b, 0
        parents.append(p)
        keep.append(k)
    return parents, keep


def shared(c):
    """Tokens of the prompt that a step's requests share: its longest keys without the new ones."""
    return c["Sk"] - c["Sq"]


def _two(e):
    """2^e in 32 bits, exact for -126 <= e <= 127."""
    return ((e.int() + 127) << 23).view(torch.float32)


def prepare(c, seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    dt, B, op = DTYPES[c["dtype"]], c["B"], c["op"]

    def normal(*shape, std=1.0):
        return torch.randn(*shape, generator=g, dtype=torch.float32, device=DEVICE).mul_(std).to(dt)

    def ints(v):
        return torch.tensor(v, dtype=torch.int32, device=DEVICE)

    s = {"case": dict(c)}
    if op == "step":        # before the call row 0 holds the prompt, the others nothing
        lens = [shared(c)] + [0] * (B - 1)
        max_pages = -(-c["Sk"] // PAGE)
        P = -(-shared(c) // PAGE) + B * (c["Sq"] // PAGE + 2) + 3
    elif op == "attend":
        lens = lengths(c)
        max_pages = -(-c["Sk"] // PAGE)
        P = sum(-(-n // PAGE) for n in lens) + 5
    else:
        lens = lengths(c)
        max_pages = -(-c["Sk"] // PAGE)
        P = pool_pages(c)
    need = [-(-n // PAGE) for n in lens]
    pool = torch.randperm(P, generator=g, device=DEVICE).int()
    first = torch.cumsum(ints([0] + need), 0)[:-1]
    j = torch.arange(max_pages, device=DEVICE)[None]
    mine = j < ints(need)[:, None]
    s["block_table"] = torch.where(mine, pool[(first[:, None] + j).clamp(max=P - 1).long()], 0)
    s["seq_lens"] = ints(lens)
    free = pool[sum(need):]
    ring = torch.full((P,), -1, dtype=torch.int32, device=DEVICE)
    head = int(torch.randint(0, P, (1,), generator=g, device=DEVICE))
    ring[(head + torch.arange(free.numel(), device=DEVICE)) % P] = free
    s["free_pages"], s["free_state"] = ring, ints([head, free.numel()])
    if op == "compact":
        return s
    if op == "fork":
        parents, keep = fork_plan(c)
        s["parents"], s["keep_lens"] = ints(parents), ints(keep)
        return s
    if op == "copy":        # destinations are free pages, as both operators give them
        n = min(free.numel(), sum(need))
        pairs = torch.stack((pool[:n], free[:n]), 1)
        gone = torch.rand(n, generator=g, device=DEVICE) < 0.25    # requests without a copy
        s["copies"] = torch.where(gone[:, None], -1, pairs).contiguous()
        s["pools"] = [normal(c["layers"], P, PAGE, w) for w in (R, D)]
        return s

    Sq, H = c["Sq"], c["heads"]
    s["W_uk"] = normal(H, NOPE, R, std=R ** -0.5)
    s["W_uv"] = normal(H, V, R, std=R ** -0.5)
    new = new_tokens(c)
    s["new_lens"] = ints(new)
    # rows that no request holds are whatever the memory held before
    pos = torch.arange(max_pages * PAGE, device=DEVICE)[None]
    slot = s["block_table"].long()[:, pos[0] // PAGE] * PAGE + pos % PAGE
    valid = torch.zeros(P * PAGE, dtype=torch.bool, device=DEVICE)
    valid[slot[pos < s["seq_lens"][:, None]]] = True
    if c["block"]:
        G = c["block"]
        valid = valid.view(P, PAGE // G, G)
        s["scales"] = torch.randint(0, 256, (P, PAGE // G, 2), generator=g, device=DEVICE).to(torch.uint8)
        for part, (name, width) in enumerate((("c_kv", R), ("pe", D))):
            v = torch.randn(P, PAGE // G, G, width, generator=g, device=DEVICE)
            v.mul_(torch.exp(0.5 * torch.randn(P, PAGE // G, 1, 1, generator=g, device=DEVICE)))
            v.mul_(valid[..., None])
            m, e = torch.frexp(v.abs().amax((2, 3)))
            e = e - 9 + (m > 0.875).int()
            v = (v * _two(-e)[..., None, None]).to(E4M3).view(torch.uint8)
            s[name] = torch.where(valid[..., None], v, 0x7F).view(P, PAGE, width).view(E4M3)
            s["scales"][..., part] = torch.where(valid.any(2), (e + 127).to(torch.uint8), s["scales"][..., part])
    else:
        for name, width in (("c_kv", R), ("pe", D)):
            v = normal(P * PAGE, width)
            s[name] = torch.where(valid[:, None], v, math.nan).view(P, PAGE, width)
    if op == "attend":
        s["q_nope"] = normal(B, Sq, H, NOPE)
        s["q_rope"] = normal(B, Sq, H, D)
        return s
    s["parents"] = ints([0] * B)
    s["keep_lens"] = ints([shared(c)] * B)
    s["x"] = normal(B, Sq, HIDDEN)
    s["W_q_a"] = normal(HIDDEN, QL, std=HIDDEN ** -0.5)
    s["q_norm_w"] = (1.0 + 0.1 * torch.randn(QL, generator=g, device=DEVICE)).to(dt)
    s["W_q_b"] = normal(QL, H * (NOPE + D), std=QL ** -0.5)
    s["W_kv_a"] = normal(HIDDEN, R + D, std=HIDDEN ** -0.5)
    s["kv_norm_w"] = (1.0 + 0.1 * torch.randn(R, generator=g, device=DEVICE)).to(dt)
    return s


# ------------------------------------------------------------------ the plain forms

def _pages_of(n):
    return (n + PAGE - 1) // PAGE


def _spread(size, where, index, value, fill, dtype=torch.int64):
    """A vector of `size` fills with value[where] at index[where]."""
    t = torch.full((size + 1,), fill, dtype=dtype, device=index.device)
    t.scatter_(0, torch.where(where, index, size).flatten(), value.expand(where.shape).to(dtype).flatten())
    return t[:size]


def _fork(s):
    table, ring = s["block_table"].long(), s["free_pages"]
    B, max_pages = table.shape
    N, dev = ring.numel(), ring.device
    head, count = s["free_state"].long()
    L = s["seq_lens"].long().clamp(0, max_pages * PAGE)
    parent = s["parents"].long()
    src = parent.clamp(0, B - 1)
    n = torch.minimum(s["keep_lens"].long().clamp(min=0), L[src])
    n = torch.where(parent == src, n, 0)
    rows = table[src]
    j = torch.arange(max_pages, device=dev)[None]
    whole = j < (n // PAGE)[:, None]
    opened = (j == (n // PAGE)[:, None]) & (n % PAGE > 0)[:, None]
    valid = (rows >= 0) & (rows < N)
    held = (j < _pages_of(L)[:, None]) & (table >= 0) & (table < N)
    one = torch.ones((), dtype=torch.int64, device=dev)
    was = _spread(N, held, table, one, 0) > 0
    fixed = _spread(N, whole & valid, rows, one, 0) > 0
    lowest = torch.full((N + 1,), B, dtype=torch.int64, device=dev)
    b = torch.arange(B, device=dev)[:, None].expand(B, max_pages)
    lowest.scatter_reduce_(0, torch.where(opened & valid, rows, N).flatten(), b.flatten(), "amin")
    lowest = lowest[:N]
    at = rows.clamp(0, N - 1)
    need = (opened & valid & (fixed[at] | (lowest[at] != b))).any(1)
    order = torch.cumsum(need, 0) - need.long()
    given = need & (order < count)
    fresh = ring.long()[(head + order) % N]
    old = rows.gather(1, (n // PAGE).clamp(max=max_pages - 1)[:, None])[:, 0]
    copies = torch.where(given[:, None], torch.stack((old, fresh), 1), -1)
    n = torch.where(need & ~given, n // PAGE * PAGE, n)
    opened &= (n % PAGE > 0)[:, None]
    out = torch.where(whole | opened, rows, 0)
    out = torch.where(opened & given[:, None], fresh[:, None], out)
    freed = was & ~fixed & (lowest == B)
    rank = torch.cumsum(freed, 0) - 1
    spill = torch.cat((ring, ring[:1]))
    spill.scatter_(0, torch.where(freed, (head + count + rank) % N, N), torch.arange(N, device=dev).int())
    ring.copy_(spill[:N])
    state = torch.stack(((head + given.sum()) % N, (count - given.sum() + freed.sum()).clamp(max=N)))
    return {"seq_lens": n.int(), "block_table": out.int(), "free_state": state.int(),
            "copies": copies.int(), "free_pages": ring}


def _compact(s):
    table, ring = s["block_table"].long(), s["free_pages"].long()
    B, max_pages = table.shape
    N, dev = ring.numel(), ring.device
    head, count = s["free_state"].long()
    L = s["seq_lens"].long().clamp(0, max_pages * PAGE)
    held = torch.arange(max_pages, device=dev)[None] < _pages_of(L)[:, None]
    valid = held & (table >= 0) & (table < N)
    one = torch.ones((), dtype=torch.int64, device=dev)
    used = _spread(N, valid, table, one, 0) > 0
    i = torch.arange(N, device=dev)
    ringed = ring[(head + i) % N]
    free = (_spread(N, (i < count) & (ringed >= 0) & (ringed < N), ringed, one, 0) > 0) & ~used
    both = used | free
    rank = torch.cumsum(both, 0) - 1
    U = used.sum()
    move, hole = used & (rank >= U), free & (rank < U)
    km, kh = torch.cumsum(move, 0) - 1, torch.cumsum(hole, 0) - 1
    room = max(1, N // 2)
    copies = torch.stack((_spread(room, move, km, i, -1), _spread(room, hole, kh, i, -1)), 1)
    to = torch.where(move, copies[km.clamp(0, room - 1), 1], i)
    out = torch.where(valid, to[table.clamp(0, N - 1)], torch.where(held, table, 0))
    left = both & (rank >= U)
    new_ring = _spread(N, left, rank - U, i, -1)
    state = torch.stack((0 * U, left.sum()))
    return {"block_table": out.int(), "free_pages": new_ring.int(), "free_state": state.int(),
            "copies": copies.int()}


def _copy(copies, pools):
    """Pools [layers, pages, ...]; pairs of -1 copy a source, which no pair writes, to itself."""
    src, dst = copies.long().unbind(1)
    there = (src >= 0) & (dst >= 0)
    still = src.max().clamp(min=0)
    src, dst = torch.where(there, src, still), torch.where(there, dst, still)
    for p in pools:
        p[:, dst] = p[:, src]


def _rows(s, table):
    """The cache rows of a table in 32 bits."""
    key = torch.arange(table.size(1) * PAGE, device=table.device)
    slot = table.long()[:, key // PAGE] * PAGE + key % PAGE
    if not s["case"]["block"]:
        return s["c_kv"].view(-1, R)[slot].float(), s["pe"].view(-1, D)[slot].float()
    e = s["scales"].view(-1, 2)[slot // s["case"]["block"]].int() - 127
    lat = s["c_kv"].view(torch.uint8).view(-1, R)[slot].view(E4M3).float()
    rot = s["pe"].view(torch.uint8).view(-1, D)[slot].view(E4M3).float()
    return lat * _two(e[..., :1]), rot * _two(e[..., 1:])


def _attend(s, q_nope, q_rope, table, lens, new):
    B, Sq, H, _ = q_nope.shape
    lat, rot = _rows(s, table)
    span = lat.size(1)
    key = torch.arange(span, device=table.device)
    there = (key[None] < lens[:, None])[..., None]
    lat, rot = torch.where(there, lat, 0), torch.where(there, rot, 0)
    i = torch.arange(Sq, device=table.device)[None]
    last = torch.where(i >= Sq - new[:, None], lens[:, None] - Sq + i, -1)
    hidden = (key[None, None] > last[..., None])[:, None]           # [B, 1, Sq, span]
    out = torch.empty(B, Sq, H, V, dtype=q_nope.dtype, device=table.device)
    step = max(1, min(H, (1 << 30) // (B * Sq * span)))
    for h in range(0, H, step):
        k = min(step, H - h)
        wk = s["W_uk"][h:h + k].float().view(k * NOPE, R).t()
        wv = s["W_uv"][h:h + k].float().view(k * V, R).t()
        keys = torch.matmul(lat, wk).view(B, span, k, NOPE).permute(0, 2, 3, 1)
        values = torch.matmul(lat, wv).view(B, span, k, V).permute(0, 2, 1, 3)
        t = torch.matmul(q_nope[:, :, h:h + k].float().transpose(1, 2), keys)
        t += torch.matmul(q_rope[:, :, h:h + k].float().transpose(1, 2), rot.transpose(1, 2)[:, None])
        t.div_(SCALE).masked_fill_(hidden, -math.inf)
        top = t.amax(-1, keepdim=True)
        t.sub_(torch.where(torch.isfinite(top), top, 0)).exp_()
        total = t.sum(-1, keepdim=True)
        o = torch.matmul(t, values)
        out[:, :, h:h + k] = torch.where(total > 0, o / total, 0).transpose(1, 2).to(out.dtype)
    return out


def _angles(pos):
    inv = 1.0 / 10000 ** (torch.arange(0, D, 2, dtype=torch.float32) / D)
    return (pos[..., None].float() * inv.to(pos.device)).double()


def _rotate(x, pos):
    a = _angles(pos)
    cos, sin = a.cos().float(), a.sin().float()
    while cos.dim() < x.dim():
        cos, sin = cos.unsqueeze(-2), sin.unsqueeze(-2)
    even, odd = x[..., 0::2], x[..., 1::2]
    return torch.stack((even * cos - odd * sin, even * sin + odd * cos), -1).flatten(-2)


def _norm(x, w):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w.float()


def _q_heads(s, pos):
    dt = s["x"].dtype
    B, Sq, _ = s["x"].shape
    lat = _norm(torch.matmul(s["x"].float(), s["W_q_a"].float()), s["q_norm_w"]).to(dt)
    q = torch.matmul(lat.float(), s["W_q_b"].float()).view(B, Sq, HEADS, NOPE + D)
    return q[..., :NOPE].to(dt), _rotate(q[..., NOPE:], pos).to(dt)


def _append(s, table, pos):
    dt = s["x"].dtype
    kv = torch.matmul(s["x"].float(), s["W_kv_a"].float())
    lat, rot = _norm(kv[..., :R], s["kv_norm_w"]).to(dt), _rotate(kv[..., R:], pos).to(dt)
    p = pos.clamp(min=0)
    rows = s["c_kv"].numel() // R
    slot = torch.where(pos >= 0, table.long().gather(1, p // PAGE) * PAGE + p % PAGE, rows).flatten()
    for name, v, w in (("c_kv", lat, R), ("pe", rot, D)):
        flat = s[name].view(-1, w)
        spill = torch.cat((flat, flat[:1]))
        spill[slot] = v.view(-1, w)
        flat.copy_(spill[:rows])


def _grow(s, lens, table, state):
    """Pages of the new tokens (all of them fit): table and lengths with them, positions."""
    ring = s["free_pages"].long()
    N, Sq = ring.numel(), s["case"]["Sq"]
    L, n = lens.long(), s["new_lens"].long()
    take = _pages_of(L + n) - _pages_of(L)
    before = torch.cumsum(take, 0) - take
    j = torch.arange(table.size(1), device=table.device)[None]
    k = j - _pages_of(L)[:, None]
    fresh = ring[(state.long()[0] + before[:, None] + k) % N]
    table = torch.where((k >= 0) & (k < take[:, None]), fresh.int(), table)
    pos = (L + n)[:, None] - Sq + torch.arange(Sq, device=table.device)[None]
    state = torch.stack(((state.long()[0] + take.sum()) % N, state.long()[1] - take.sum())).int()
    return (L + n).int(), table, state, torch.where(pos >= L[:, None], pos, -1)


# ------------------------------------------------------------------ one pass

def run(s):
    c = s["case"]
    op = c["op"]
    if own:
        if PKG not in sys.path:
            sys.path.insert(0, PKG)
        import mla_custom_cuda as mla
    if op == "fork" or op == "step":
        if own:
            lens, table, state, copies = mla.cache_fork(
                s["parents"], s["keep_lens"], s["seq_lens"], s["block_table"], s["free_pages"],
                s["free_state"], PAGE)
            out = {"seq_lens": lens, "block_table": table, "free_state": state, "copies": copies,
                   "free_pages": s["free_pages"]}
        else:
            out = _fork(s)
        if op == "fork":
            return out
    if op == "compact":
        if own:
            table, ring, state, copies = mla.cache_compact(
                s["seq_lens"], s["block_table"], s["free_pages"], s["free_state"], PAGE)
            return {"block_table": table, "free_pages": ring, "free_state": state, "copies": copies}
        return _compact(s)
    if op == "copy":
        if own:
            mla.cache_copy_pages(s["copies"], s["pools"], layered=True)
        else:
            _copy(s["copies"], s["pools"])
        return list(s["pools"])
    if op == "attend":
        if not own:
            return _attend(s, s["q_nope"], s["q_rope"], s["block_table"], s["seq_lens"], s["new_lens"])
        if c["block"]:
            return mla.mla_attention_paged_fp8blk_expanded(
                s["q_nope"], s["q_rope"], s["c_kv"], s["pe"], s["scales"], s["block_table"],
                s["seq_lens"], s["W_uk"], s["W_uv"], SCALE, causal=True, new_lens=s["new_lens"])
        return mla.mla_attention_paged_expanded(
            s["q_nope"], s["q_rope"], s["c_kv"], s["pe"], s["block_table"], s["seq_lens"],
            s["W_uk"], s["W_uv"], SCALE, causal=True, new_lens=s["new_lens"])
    # step: `out` holds the forked tables
    if own:
        mla.cache_copy_pages(out["copies"], [s["c_kv"], s["pe"]])
        lens, state, new, pos, _ = mla.cache_extend(
            s["new_lens"], out["seq_lens"], out["block_table"], s["free_pages"], out["free_state"],
            c["Sq"], PAGE)
        table = out["block_table"]
        mla.kv_append_paged(s["x"], s["W_kv_a"], s["kv_norm_w"], pos, table, s["c_kv"], s["pe"], EPS)
        q_nope, q_rope = mla.q_heads(s["x"], s["W_q_a"], s["q_norm_w"], s["W_q_b"], pos, NOPE, D, EPS)
        attn = mla.mla_attention_paged_expanded(q_nope, q_rope, s["c_kv"], s["pe"], table, lens,
                                                s["W_uk"], s["W_uv"], SCALE, causal=True, new_lens=new)
    else:
        _copy(out["copies"], [s["c_kv"][None], s["pe"][None]])
        lens, table, state, pos = _grow(s, out["seq_lens"], out["block_table"], out["free_state"])
        _append(s, table, pos)
        q_nope, q_rope = _q_heads(s, pos)
        attn = _attend(s, q_nope, q_rope, table, lens, s["new_lens"])
    return {"seq_lens": lens, "block_table": table, "free_state": state, "copies": out["copies"],
            "positions": pos, "q_nope": q_nope, "q_rope": q_rope, "attn": attn}


def work(c):
    op, B = c["op"], c["B"]
    if op == "copy":
        used = sum(-(-n // PAGE) for n in lengths(c))
        moved = 0.75 * min(used, pool_pages(c) - used)
        return {"bytes": int(2 * moved * c["layers"] * PAGE * (R + D) * 2), "flops": 0}
    if op in ("fork", "compact"):
        used, P = sum(-(-n // PAGE) for n in lengths(c)), pool_pages(c)
        span = B * -(-c["Sk"] // PAGE)
        if op == "fork":    # tables in and out, a word a request for each of six vectors
            return {"bytes": 4 * (used + span + 7 * B) + 16, "flops": span}
        return {"bytes": 4 * (used + span + B + P - used + P + 2 * (P // 2)) + 16, "flops": P}
    Sq, H = c["Sq"], c["heads"]
    new = new_tokens(c)
    lens = [shared(c) + k for k in new] if op == "step" else lengths(c)
    new = [min(k, n) for k, n in zip(new, lens)]
    tokens, keys = sum(new), sum(lens)
    pairs = sum(k * n - k * (k - 1) // 2 for k, n in zip(new, lens))
    distinct = shared(c) + tokens if op == "step" else keys     # rows, shared ones counted once
    # the cheaper of the two forms: keys and values per head, or queries and sums per latent
    expanded = 2 * distinct * H * (NOPE + V) * R + 2 * pairs * H * (NOPE + D + V)
    absorbed = 2 * tokens * H * (NOPE + V) * R + 2 * pairs * H * (2 * R + D)
    size = 1 if c["block"] else 2
    nbytes = distinct * (R + D) * size + 4 * (keys // PAGE + B) + 2 * H * (NOPE + V) * R
    nbytes += tokens * H * (NOPE + D) * 2 + B * Sq * H * V * 2
    flops = min(expanded, absorbed)
    if op == "step":
        weights = HIDDEN * QL + QL * H * (NOPE + D) + HIDDEN * (R + D)
        nbytes += 2 * (weights + tokens * HIDDEN)
        flops += 2 * tokens * weights
    return {"bytes": nbytes, "flops": flops}


# ------------------------------------------------------------------ from the definitions, in 64 bits

def _exact_fork(s):
    """Request by request, page by page, on the host."""
    table, ring = s["block_table"].tolist(), s["free_pages"].tolist()
    lens, N = s["seq_lens"].tolist(), len(ring)
    head, count = s["free_state"].tolist()
    plan, fixed, open_of = [], set(), {}
    for b, (p, k) in enumerate(zip(s["parents"].tolist(), s["keep_lens"].tolist())):
        n = min(max(k, 0), lens[p]) if 0 <= p < len(lens) else 0
        row = table[p][:-(-n // PAGE)] if n else []
        fixed.update(row[:n // PAGE])
        if n % PAGE:
            open_of.setdefault(row[-1], []).append(b)
        plan.append((n, row))
    out = torch.zeros_like(s["block_table"], device="cpu")
    copies, after, taken = [], [], 0
    held = set(fixed)
    for b, (n, row) in enumerate(plan):
        pair = [-1, -1]
        if n % PAGE:
            page = row[-1]
            if page not in fixed and open_of[page][0] == b:
                held.add(page)
            elif taken < count:
                pair = [page, ring[(head + taken) % N]]
                row = row[:-1] + [pair[1]]
                taken += 1
            else:
                n, row = n // PAGE * PAGE, row[:-1]
        out[b, :len(row)] = torch.tensor(row, dtype=torch.int32)
        copies.append(pair)
        after.append(n)
    was = {p for row, n in zip(table, lens) for p in row[:-(-n // PAGE)]}
    for i, page in enumerate(sorted(was - held)):
        ring[(head + count + i) % N] = page
    i32 = torch.int32
    return {"seq_lens": torch.tensor(after, dtype=i32), "block_table": out,
            "free_state": torch.tensor([(head + taken) % N, count - taken + len(was - held)], dtype=i32),
            "copies": torch.tensor(copies, dtype=i32), "free_pages": torch.tensor(ring, dtype=i32)}


def _exact_compact(s):
    table, ring = s["block_table"].tolist(), s["free_pages"].tolist()
    lens, N = s["seq_lens"].tolist(), len(ring)
    head, count = s["free_state"].tolist()
    rows = [row[:-(-n // PAGE)] for row, n in zip(table, lens)]
    used = {p for row in rows for p in row}
    free = {ring[(head + i) % N] for i in range(count)}
    order = sorted(used | free)
    low, rest = order[:len(used)], order[len(used):]
    pairs = list(zip((p for p in rest if p in used), (p for p in low if p in free)))
    to = dict(pairs)
    out = torch.zeros_like(s["block_table"], device="cpu")
    for b, row in enumerate(rows):
        out[b, :len(row)] = torch.tensor([to.get(p, p) for p in row], dtype=torch.int32)
    copies = torch.full((max(1, N // 2), 2), -1, dtype=torch.int32)
    if pairs:
        copies[:len(pairs)] = torch.tensor(pairs, dtype=torch.int32)
    i32 = torch.int32
    return {"block_table": out, "free_pages": torch.tensor(rest + [-1] * (N - len(rest)), dtype=i32),
            "free_state": torch.tensor([0, len(rest)], dtype=i32), "copies": copies}


def _exact_rows(s, row, n):
    """Latent and rope rows of one request's n keys in 64 bits."""
    k = torch.arange(n, device=DEVICE)
    slot = row.to(DEVICE).long()[k // PAGE] * PAGE + k % PAGE
    lat, rot = s["c_kv"].view(-1, R)[slot], s["pe"].view(-1, D)[slot]
    if not s["case"]["block"]:
        return lat.double(), rot.double()
    e = torch.exp2(s["scales"].view(-1, 2)[slot // s["case"]["block"]].double() - 127)
    return lat.float().double() * e[:, :1], rot.float().double() * e[:, 1:]


def _exact_attend(s, q_nope, q_rope, rows, new):
    """Through absorbed queries, request by request; rows: (latent, rope) of each."""
    B, Sq, H, _ = q_nope.shape
    out = torch.zeros(B, Sq, H, V, dtype=torch.float64, device=DEVICE)
    wk, wv = s["W_uk"].double(), s["W_uv"].double().transpose(1, 2).contiguous()
    for b, ((lat, rot), m) in enumerate(zip(rows, new)):
        n = lat.size(0)
        kt = torch.cat((lat, rot), 1).t().contiguous()
        step = max(1, (1 << 27) // (H * max(1, n)))
        for i in range(Sq - m, Sq, step):
            z = min(Sq, i + step)
            qa = torch.matmul(q_nope[b, i:z].double().transpose(0, 1).contiguous(), wk)     # [H, rows, R]
            q = torch.cat((qa, q_rope[b, i:z].double().transpose(0, 1)), -1)
            t = torch.matmul(q, kt) / SCALE
            see = torch.arange(n, device=DEVICE)[None] <= torch.arange(n - Sq + i, n - Sq + z, device=DEVICE)[:, None]
            t = torch.softmax(t.masked_fill(~see, -math.inf), -1).nan_to_num()
            out[b, i:z] = torch.matmul(torch.matmul(t, lat), wv).transpose(0, 1)
    return out


def exact(c, seed):
    s = prepare(c, seed)
    op = c["op"]
    if op == "fork":
        return _exact_fork(s)
    if op == "compact":
        return _exact_compact(s)
    if op == "copy":
        out = [p.double() for p in s["pools"]]
        for a, b in s["copies"].tolist():
            if a >= 0:
                for o, p in zip(out, s["pools"]):
                    o[:, b] = p[:, a]
        return out
    if op == "attend":
        lens, new = s["seq_lens"].tolist(), s["new_lens"].tolist()
        rows = [_exact_rows(s, s["block_table"][b], n) for b, n in enumerate(lens)]
        return _exact_attend(s, s["q_nope"], s["q_rope"], rows, new)
    prompt = _exact_rows(s, s["block_table"][0], shared(c))
    f = _exact_fork(s)
    table, lens, new = f["block_table"], f["seq_lens"].tolist(), s["new_lens"].tolist()
    ring, (head, count) = f["free_pages"].tolist(), f["free_state"].tolist()
    B, Sq, taken = c["B"], c["Sq"], 0
    pos = torch.full((B, Sq), -1, dtype=torch.int64)
    for b, (n, k) in enumerate(zip(lens, new)):
        for j in range(-(-n // PAGE), -(-(n + k) // PAGE)):
            table[b, j] = ring[(head + taken) % len(ring)]
            taken += 1
        if k:
            pos[b, Sq - k:] = torch.arange(n, n + k)

    def norm(v, w):
        return v / torch.sqrt((v * v).mean(-1, keepdim=True) + EPS) * w.double()

    def turn(v):                                # [B, Sq, ..., D]
        z = torch.view_as_complex(v.reshape(*v.shape[:-1], D // 2, 2).contiguous())
        a = _angles(pos.to(DEVICE))
        a = a.view(B, Sq, *([1] * (v.dim() - 3)), D // 2)
        return torch.view_as_real(z * torch.polar(torch.ones_like(a), a)).reshape(v.shape)

    x = s["x"].double()
    q = (norm(x @ s["W_q_a"].double(), s["q_norm_w"]) @ s["W_q_b"].double()).view(B, Sq, HEADS, NOPE + D)
    q_nope, q_rope = q[..., :NOPE].contiguous(), turn(q[..., NOPE:])
    kv = x @ s["W_kv_a"].double()
    lat, rot = norm(kv[..., :R], s["kv_norm_w"]), turn(kv[..., R:])
    rows = [(torch.cat((prompt[0], lat[b, Sq - k:])), torch.cat((prompt[1], rot[b, Sq - k:])))
            for b, k in enumerate(new)]
    i32 = torch.int32
    return {"seq_lens": torch.tensor([n + k for n, k in zip(lens, new)], dtype=i32), "block_table": table,
            "free_state": torch.tensor([(head + taken) % len(ring), count - taken], dtype=i32),
            "copies": f["copies"], "positions": pos, "q_nope": q_nope, "q_rope": q_rope,
            "attn": _exact_attend(s, q_nope, q_rope, rows, new)}
