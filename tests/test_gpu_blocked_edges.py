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
