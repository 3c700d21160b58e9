"""Plain restatements, in 64 bits and on the CPU, of the operators of the paged 8-bit cache with
block scales, and the inputs their tests share -- TEST INFRASTRUCTURE ONLY.

A cache is a dict: codes ``c_kv`` [P, page, 512] and ``pe`` [P, page, 64] (uint8, e4m3), scales
[P, page / block, 2] (uint8, E8M0), value = code * 2^(byte - 127).
"""

from __future__ import annotations

import math

import torch

from oracle import mla_ref as R

D = R.DSV3
KV, ROPE = 512, 64
F64 = torch.float64
EMIN = -100
INT_MIN = -2 ** 31


# ------------------------------------------------------------------ block tables and slots

def extend(new_lens, seq_lens, table, ring, state, Sq, page):
    """Request by request; returns everything that the call leaves (lists and new tensors)."""
    table, old, ring = table.clone(), ring, ring.clone()
    N, span = ring.numel(), table.size(1) * page
    head, count = int(state[0]) % N, min(max(int(state[1]), 0), N)
    pos = torch.full((len(seq_lens), Sq), -1, dtype=torch.int64)
    slots = pos.clone()
    granted, after, asked, taken, pushed = [], [], 0, 0, 0
    up = lambda n: -(-n // page)  # noqa: E731
    for b, (L, n) in enumerate(zip(seq_lens, new_lens)):
        L = min(max(L, 0), span)
        if n > 0:
            need = up(L + n) - up(L)
            ok = n <= Sq and L + n <= span
            if ok:
                asked += need
            if not ok or (need > 0 and asked > count):
                n = 0
            for i in range(need if n else 0):
                table[b, up(L) + i] = old[(head + taken) % N]
                taken += 1
            for i in range(n):
                p = L + i
                pos[b, Sq - n + i] = p
                slots[b, Sq - n + i] = int(table[b, p // page]) * page + p % page
        else:
            n = max(n, -L)
            for j in range(up(L + n), up(L)):
                if count + pushed < N:   # a place that holds no free page
                    ring[(head + count + pushed) % N] = table[b, j]
                    pushed += 1
        granted.append(n)
        after.append(L + n)
    return {"seq_lens": after, "granted": granted, "positions": pos, "slots": slots, "table": table,
            "ring": ring, "state": [(head + taken) % N, count - taken + pushed]}


# ------------------------------------------------------------------ codes

def code_values():
    return R.e4m3_values().double()


def two(e):
    return torch.ldexp(torch.ones((), dtype=F64), torch.as_tensor(e))


def round_code(x, e):
    """x rounded to the nearest value code * 2^e (ties to even; |x| <= 448 * 2^e); NaN stays."""
    y = x / two(e)
    _, ex = torch.frexp(y)
    step = torch.ldexp(torch.ones_like(y), (ex - 4).clamp(min=-9))
    return torch.round(y / step) * step * two(e)


def half_step(x, e):
    """Half the distance of the codes around |x| under the scale 2^e: at most |x| 2^-4."""
    _, ex = torch.frexp(x.abs() / two(e))
    return torch.ldexp(torch.ones_like(x), (ex - 4).clamp(min=-9)) / 2 * two(e)


def exponent(amax):
    """Smallest e >= EMIN with amax <= 448 * 2^e."""
    if amax == 0:
        return EMIN
    e = math.frexp(amax)[1] - 10
    while amax > 448 * 2.0 ** e:
        e += 1
    return max(e, EMIN)


def decode(cache):
    """The pool's rows in 64 bits: [P * page, 512], [P * page, 64]."""
    out = []
    for name, part in (("c_kv", 0), ("pe", 1)):
        v = code_values()[cache[name].view(torch.uint8).long()]
        s = cache["scales"].view(torch.uint8)[..., part].int() - 127
        P, page, w = v.shape
        out.append((v.view(P, s.size(1), -1) * two(s)[..., None]).view(P * page, w))
    return out


def encode(rows, e):
    """uint8 codes of rows [.., block, w] under exponents e [..]."""
    return (rows / two(e)[..., None, None]).float().to(torch.float8_e4m3fn).view(torch.uint8)


def new_pool(P, page, block, g, spread=0.5):
    """A pool of unit-spread rows whose scale wanders from block to block, and its exponents."""
    cache = {"scales": torch.zeros(P, page // block, 2, dtype=torch.uint8)}
    for name, part, w in (("c_kv", 0, KV), ("pe", 1, ROPE)):
        v = torch.randn(P, page // block, block, w, generator=g, dtype=F64)
        v *= torch.exp(spread * torch.randn(P, page // block, 1, 1, generator=g, dtype=F64))
        amax = v.abs().amax((2, 3))
        e = torch.ceil(torch.log2(amax / 448)).int()
        cache[name] = encode(v, e).view(P, page, w)
        cache["scales"][..., part] = (e + 127).to(torch.uint8)
    return cache


def slots_of(table, b, lo, hi, page):
    p = torch.arange(lo, hi)
    return table[b].long()[p // page] * page + p % page


def poison(cache, table, lens, page, block):
    """Every row without a key, and every scale of a block without one, as memory that was never
    written: NaN codes and byte 255."""
    held = torch.zeros(cache["c_kv"].size(0) * page, dtype=torch.bool)
    for b, n in enumerate(lens):
        held[slots_of(table, b, 0, n, page)] = True
    held = held.view(-1, page)
    for name in ("c_kv", "pe"):
        cache[name][~held] = 0x7F
    cache["scales"][~held.view(held.size(0), -1, block).any(2)] = 255


# ------------------------------------------------------------------ append

def kv_rows(x, W, gain, positions, eps=1e-6, inv_freq=None):
    """The cache rows of tokens x [n, hidden] in 64 bits, and a bound on what float32 sums and
    roundings may move each value by: the product's K * 2^-24 * sum |x w| (any order of K float32
    additions), carried through the norm and the rotation, and 2^-20 of the value for the norm's
    and the rotation's own few operations (sin and cos: 4 ulp of 1 on each of the two values)."""
    x, W, gain = x.double(), W.double(), gain.double()
    kv, E = x @ W, x.size(1) * 2.0 ** -24 * (x.abs() @ W.abs())
    lat, e = kv[:, :KV], E[:, :KV]
    inv = 1 / torch.sqrt((lat * lat).mean(1, keepdim=True) + eps)
    rel = e.norm(dim=1, keepdim=True) / lat.norm(dim=1, keepdim=True).clamp(min=1e-300)
    lat = lat * inv * gain
    e_lat = e * inv * gain.abs() + lat.abs() * (rel + 2.0 ** -20)
    if inv_freq is None:
        inv_freq = 1.0 / 10000 ** (torch.arange(0, ROPE, 2, dtype=torch.float32) / ROPE)
    a = (positions[:, None].float() * inv_freq).double()
    p, q = kv[:, KV::2], kv[:, KV + 1::2]
    rot = torch.stack((p * a.cos() - q * a.sin(), p * a.sin() + q * a.cos()), -1).flatten(1)
    ee = (E[:, KV::2] + E[:, KV + 1::2] + 2.0 ** -20 * (p.abs() + q.abs()))
    return lat, rot, e_lat, ee.repeat_interleave(2, 1)


def append(cache, x, W, gain, seq_lens, new_lens, table, page, block, eps=1e-6, inv_freq=None):
    """What the append leaves: for each part the rows' unrounded values, bounds on the kernel's
    distance from them, the exponents, and which pool rows and blocks were written (new), kept
    beside new ones (old), or not touched."""
    P = cache["c_kv"].size(0)
    Sq = x.size(1)
    want = {"new": torch.zeros(P * page, dtype=torch.bool), "old": torch.zeros(P * page, dtype=torch.bool),
            "e": cache["scales"].view(torch.uint8).view(-1, 2).int() - 127,
            "touched": torch.zeros(P * page // block, dtype=torch.bool),
            "value": [torch.zeros(P * page, w, dtype=F64) for w in (KV, ROPE)],
            "bound": [torch.zeros(P * page, w, dtype=F64) for w in (KV, ROPE)]}
    before = want["e"].clone()
    for b, (L, n) in enumerate(zip(seq_lens, new_lens)):
        L = min(max(L, 0), table.size(1) * page)
        n = min(max(n, 0), Sq, L)
        if n == 0:
            continue
        lat, rot, el, er = kv_rows(x[b, Sq - n:], W, gain, torch.arange(L - n, L), eps, inv_freq)
        for lo in range((L - n) // block * block, L, block):
            pg = int(table[b, lo // page])
            if not 0 <= pg < P:
                continue
            row0 = pg * page + lo % page
            first, hi = max(lo, L - n), min(lo + block, L)
            rows = slice(row0 + first - lo, row0 + hi - lo)
            mine = slice(first - (L - n), hi - (L - n))
            want["new"][rows] = True
            want["old"][row0:row0 + first - lo] = True
            want["touched"][row0 // block] = True
            for part, (v, bd) in enumerate(((lat, el), (rot, er))):
                want["value"][part][rows], want["bound"][part][rows] = v[mine], bd[mine]
                t = v[mine].abs()
                e = exponent(float(t[torch.isfinite(t)].max()) if torch.isfinite(t).any() else 0.0)
                if first > lo:
                    e = max(e, int(before[row0 // block, part]))
                want["e"][row0 // block, part] = e
    return want


# ------------------------------------------------------------------ attention

def attention(qa, qr, rows, table, seq_lens, W_uv, scale, causal, page, P):
    """Over decoded rows, in 64 bits; a page outside the pool counts as rows of zeros."""
    B, Sq, H, _ = qa.shape
    out = torch.zeros(B, Sq, H, W_uv.size(1), dtype=F64)
    for b in range(B):
        n = min(max(int(seq_lens[b]), 0), table.size(1) * page)
        if n == 0:
            continue
        p = torch.arange(n)
        pg = table[b].long()[p // page]
        there = (pg >= 0) & (pg < P)
        slot = torch.where(there, pg, 0) * page + p % page
        lat, rot = (torch.where(there[:, None], r[slot], 0) for r in rows)
        t = (qa[b].double().reshape(Sq * H, -1) @ lat.T + qr[b].double().reshape(Sq * H, -1) @ rot.T) / scale
        t = t.view(Sq, H, n)
        if causal:
            hidden = p[None] > (n - Sq + torch.arange(Sq))[:, None]
            t = t.masked_fill(hidden[:, None], -math.inf)
        w = torch.nan_to_num(torch.softmax(t, -1))
        ctx = (w.view(Sq * H, n) @ lat).view(Sq, H, -1)
        out[b] = torch.einsum("shr,hvr->shv", ctx, W_uv.double())
    return out


def queries(B, Sq, H, V, g, dt):
    """With the spread that the layer's projections give (scores of unit spread over unit rows)."""
    qa = torch.randn(B, Sq, H, KV, generator=g) * math.sqrt(D.nope / D.kv_rank)
    qr = torch.randn(B, Sq, H, ROPE, generator=g)
    w = torch.randn(H, V, KV, generator=g) / math.sqrt(KV)
    return qa.to(dt), qr.to(dt), w.to(dt)


def tables(lens, page, P, g, max_pages=None):
    """A shuffled pool's table for sequences of these lengths; unused entries are no pages."""
    need = [-(-n // page) for n in lens]
    mp = max_pages or max(1, max(need))
    order = torch.randperm(P, generator=g).int()
    table = torch.full((len(lens), mp), -7, dtype=torch.int32)
    at = 0
    for b, k in enumerate(need):
        table[b, :k] = order[at:at + k]
        at += k
    assert at <= P
    return table
