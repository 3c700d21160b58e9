"""GPU checks of the blocked 8-bit cache at the ends of its scales' range."""

from __future__ import annotations

import pytest
import torch

import blocked_cache as K
from test_gpu_blocked_cache import (BF, DEV, DT, F32, SCALE, append_inputs, attention_case, check_append,  # noqa: F401
                                    ext, i32, run_append)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("block", [16, 32, 64])
@pytest.mark.parametrize("byte", [253, 254])
def test_append_under_the_largest_scales(ext, dt, block, byte):  # noqa: F811
    """New rows in blocks that already have the scale 2^126 or 2^127, their values up to 2^124 (gain and
    W's rope columns times 2^122): codes under that scale, not zeros."""
    lens, new, Sq = [block // 2 + 9, block + 8], [9, 5], 9
    cache, x, W, gain, table = append_inputs(lens, new, Sq, block, 64, F32, byte)
    W[:, K.KV:] *= 2.0 ** 122
    x, W, gain = x.to(DT[dt]), W.to(DT[dt]), (gain * 2.0 ** 122).to(DT[dt])
    for b in range(2):     # the block that keeps rows: the first of sequence 0, the second of sequence 1
        row = int(K.slots_of(table, b, lens[b] - new[b], lens[b] - new[b] + 1, 64)[0])
        cache["scales"].view(-1, 2)[row // block] = byte
    after = run_append(ext, cache, x, W, gain, lens, new, table)
    want = K.append(cache, x, W, gain, lens, new, table, 64, block)
    kept = want["touched"] & (want["e"][:, 0] == byte - 127)
    assert int(kept.sum()) >= 1
    check_append(cache, after, want, block)


@pytest.mark.parametrize("up,w_up", [(114, -110), (114, 5), (-95, 100), (-60, -20)])
@pytest.mark.parametrize("B,Sq", [(1, 1), (3, 20), (3, 70), (140, 1)])
def test_attention_wide_powers_of_two(ext, up, w_up, B, Sq):  # noqa: F811
    """bf16 values times 2^up and each output column's W_uv times a power of two of its own: the bits but
    for the exponent, whatever the number of tokens -- nothing behind the softmax leaves float32's range
    where the output does not.  (Queries of zeros: weights of 1, whose sums stay inside it.  Outputs down to
    2^-100: what makes their last bit is normal too.)"""
    g = torch.Generator().manual_seed(Sq)
    lens = [70, 300, 1200] if B == 3 else [Sq + 200] * B
    qa, qr, w, cache, table = attention_case(lens, Sq, 32, 64, BF, 3, H=16)
    qa.zero_(), qr.zero_()
    moved = {**cache, "scales": cache["scales"].clone()}
    held = moved["scales"][..., 0] != 255
    moved["scales"][..., 0][held] = (moved["scales"][..., 0][held].int() + up).to(torch.uint8)
    e = torch.randint(min(0, w_up), max(0, w_up) + 1, (16, 128), generator=g).double()

    def attend(c, w, scale):
        return ext.mla_attention_paged_fp8blk(qa.to(DEV), qr.to(DEV), c["c_kv"].to(DEV), c["pe"].to(DEV),
                                              c["scales"].to(DEV), table.to(DEV), i32(lens).to(DEV), w.to(DEV),
                                              scale, True).cpu()

    base = attend(cache, w, SCALE)
    out = attend(moved, (w.double() * 2.0 ** e[..., None]).to(BF), SCALE * 2.0 ** up)
    want = base.double() * 2.0 ** (up + e)
    assert want.abs().max() < torch.finfo(BF).max
    assert torch.equal(out.double(), want)


@pytest.mark.parametrize("dt,up,code", [("f16", 13, 0x50), ("f16", 13, 0xFE), ("f16", 24, 0x02), ("bf16", 120, 0x78),
                                        ("bf16", 120, 0xFE)])
@pytest.mark.parametrize("Sq,H,lens,at", [(4, 16, [300, 33, 4], 2), (3, 3, [500, 17], 1), (20, 10, [500, 33, 64], 18),
                                          (50, 16, [50, 100, 900], 17), (70, 3, [700, 70], 1)])
def test_attention_hidden_values_past_the_range(ext, dt, up, code, Sq, H, lens, at):  # noqa: F811
    """A value of 2^16 or more in fp16 (2^128 in bf16) in a token's latent row: the queries in front of it,
    which do not see it, keep their bits, in its block and in the blocks beside it."""
    dt, page, block = DT[dt], 64, 16
    g = torch.Generator().manual_seed(Sq)
    P = sum(-(-n // page) for n in lens) + 2
    table = K.tables(lens, page, P, g)
    # codes under 2^0 are values of unit spread (at most 7, so that 2^13 of them stay in fp16's range)
    cache = {"c_kv": K.encode(torch.randn(P, 4, 16, K.KV, generator=g, dtype=K.F64).clamp(-7, 7),
                              torch.zeros(P, 4)).view(P, page, K.KV),
             "pe": K.encode(torch.randn(P, 4, 16, K.ROPE, generator=g, dtype=K.F64), torch.zeros(P, 4)).view(P, page, -1),
             "scales": torch.full((P, page // block, 2), 127, dtype=torch.uint8)}
    if up == 24:   # under 2^24 the code 1 is 2^15, and 2 is past the range
        cache["c_kv"] = torch.tensor([0, 1, 0x81], dtype=torch.uint8)[torch.randint(0, 3, cache["c_kv"].shape, generator=g)]
    cache["scales"][..., 0] += up
    qa, qr, w = K.queries(len(lens), Sq, H, 64, g, dt)
    w = (w.double() * 2.0 ** -{13: 13, 24: 8, 120: 100}[up]).to(dt)

    def attend(c):
        return ext.mla_attention_paged_fp8blk(qa.to(DEV), qr.to(DEV), c["c_kv"].to(DEV), c["pe"].to(DEV),
                                              c["scales"].to(DEV), table.to(DEV), i32(lens).to(DEV), w.to(DEV),
                                              SCALE * 2.0 ** up, True).cpu()

    clean = attend(cache)
    assert torch.isfinite(clean).all()
    for column in (3, 300):
        bad = {k: v.clone() for k, v in cache.items()}
        for b, n in enumerate(lens):
            slot = int(K.slots_of(table, b, n - Sq + at, n - Sq + at + 1, page)[0])
            bad["c_kv"].view(-1, K.KV)[slot, column] = code
        out = attend(bad)
        assert torch.equal(out[:, :at], clean[:, :at])
        assert not torch.equal(out[:, at:], clean[:, at:])
