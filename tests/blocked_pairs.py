"""Inputs on which the outputs of the blocked 8-bit cache's attention are decided by the low bits of
the rows between the softmax and W_uv -- TEST INFRASTRUCTURE ONLY.

Queries of zeros give every key the weight 1 exactly, and latents that are multiples of 2^-11 below 2
have sums that float32 holds exactly, in any order: a row is the mean of the keys that its token sees,
known but for the last operations.  The latents' columns come in pairs that differ in few keys and by
one code step there, and every output takes one pair, with weights w and -w.  So it is w times the
difference of two neighbouring values of about 1, some 2^-8 of them: a row rounded once to 16 bits, or
with a low term that is another row's, is off by a multiple of what its own format allows.
"""

from __future__ import annotations

import torch

import blocked_cache as K

F64 = torch.float64


def case(lens, Sq, H, V, dt, seed, page=64, block=32):
    """(qa, qr, W_uv, cache, table, pair [H, V], w [H, V])"""
    g = torch.Generator().manual_seed(seed)
    P = sum(-(-n // page) for n in lens) + 2
    if P > 500:   # pages that sequences share
        P = 100
        table = torch.randint(0, P, (len(lens), -(-max(lens) // page)), generator=g).int()
    else:
        table = K.tables(lens, page, P, g)
    # codes 0x30 .. 0x3E, and one up: 0.5 .. 1.875 in steps of 2^-4 (below 1) and 2^-3, in about half of the
    # blocks times 2^-7 (3,000 of them are below 2^24 of the smallest step, 2^-11)
    first = torch.randint(0x30, 0x3F, (P, page, K.KV // 2), generator=g)
    second = first + (torch.rand(first.shape, generator=g) < 1 / 16)
    cache = {"c_kv": torch.stack((first, second), -1).view(P, page, K.KV).to(torch.uint8),
             "pe": torch.randint(0, 0x70, (P, page, K.ROPE), generator=g).to(torch.uint8),
             "scales": 127 - 7 * torch.randint(0, 2, (P, page // block, 2), generator=g).to(torch.uint8)}
    B = len(lens)
    pair = torch.randint(0, K.KV // 2, (H, V), generator=g)
    w = ((1 + torch.rand(H, V, generator=g)) * (torch.randint(0, 2, (H, V), generator=g) * 2 - 1)).to(dt)
    W = torch.zeros(H, V, K.KV, dtype=dt)
    W.scatter_(2, 2 * pair[..., None], w[..., None])
    W.scatter_(2, 2 * pair[..., None] + 1, -w[..., None])
    return torch.zeros(B, Sq, H, K.KV, dtype=dt), torch.zeros(B, Sq, H, K.ROPE, dtype=dt), W, cache, table, pair, w


def rows(cache, table, lens, Sq, page=64):
    """[B, Sq, 512]: the mean latent of the keys that each token sees (causal), in 64 bits; zeros
    where it sees none."""
    lat = K.decode(cache)[0]
    out = torch.zeros(len(lens), Sq, K.KV, dtype=F64)
    for b, n in enumerate(lens):
        if n == 0:
            continue
        total = torch.cumsum(lat[K.slots_of(table, b, 0, n, page)], 0)
        for s in range(Sq):
            k = n - Sq + s + 1
            if k > 0:
                out[b, s] = total[k - 1] / k
    return out


def outputs(ctx, pair, w):
    """[B, Sq, H, V] of rows [B, Sq, 512], in 64 bits."""
    a, b = ctx[..., 2 * pair], ctx[..., 2 * pair + 1]
    return w.double() * (a - b)


def bound(ctx, pair, w, dt, packed):
    """How far an output may be off.  Each of the two values enters with
      merged rows (two terms of dt): u^2, u = eps / 2 of dt -- what is left of the second term --
        and, in fp16, half a subnormal step, 2^-25;
      packed rows: bf16 u(fp16) = 2^-11 of itself (f16 numbers under a float32 scale); fp16 half a step of
        the integers, 2^-16 of the largest of its 128 columns, and the two terms' u^2;
    and 2^-17 of itself for float32 work: a rounding of 2^-24 for each chunk that is merged (at most 94, the
    blocks of 3,000 keys), the division and the scales' own.  The output is rounded to dt."""
    u = torch.finfo(dt).eps / 2
    top = ctx.view(*ctx.shape[:2], 4, 128).abs().amax(3).repeat_interleave(128, 2)
    if not packed:
        each = ctx.abs() * u * u + (2.0 ** -25 if dt == torch.float16 else 0)
    elif dt == torch.float16:
        each = ctx.abs() * u * u + top * 2.0 ** -16 + 2.0 ** -25
    else:
        each = ctx.abs() * 2.0 ** -11
    each = each + ctx.abs() * 2.0 ** -17
    out = outputs(ctx, pair, w)
    off = w.double().abs() * (each[..., 2 * pair] + each[..., 2 * pair + 1])
    return off + u * (out.abs() + off) + 1e-30


def two_terms(ctx, dt, mistake=None):
    """Rows as two terms of dt: hi + lo, or with lo left out, or with the lo of the token before."""
    hi = ctx.to(dt).double()
    lo = (ctx - hi).to(dt).double()
    if mistake == "no_low":
        lo = torch.zeros_like(lo)
    elif mistake == "other_low":
        lo = lo.reshape(-1, K.KV).roll(1, 0).view_as(lo)
    return hi + lo


def packed(ctx, dt, mistake=None):
    """Packed rows: f16 numbers (bf16) or integers (fp16) under their 128 columns' largest / 32767; the
    mistake: rows rounded to dt as other 3d engines take them, or fp16's two terms with a mistake."""
    if mistake == "rounded":
        return ctx.to(dt).double()
    s = (ctx.view(*ctx.shape[:2], 4, 128).abs().amax(3).repeat_interleave(128, 2) / 32767).clamp(min=1e-30)
    if dt == torch.float16:
        return two_terms(torch.round(ctx / s) * s, dt, mistake)
    return (ctx / s).to(torch.float16).double() * s
