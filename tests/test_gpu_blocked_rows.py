"""GPU checks of the rows between the softmax and W_uv in the blocked 8-bit cache's attention: the
merged rows' two terms (up to 8 tokens, up to 128) and the packed rows past that, on inputs whose
outputs their low bits decide (tests/blocked_pairs.py; tests/test_blocked_pairs_cpu.py shows that
the bound rejects rows without them)."""

from __future__ import annotations

import pytest
import torch

import blocked_pairs as R
from test_blocked_pairs_cpu import DT, FEW, MANY, TILES, lens_of
from test_gpu_blocked_cache import DEV, SCALE, ext, i32  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("B,Sq,H,V,lens", FEW + TILES + MANY)
def test_attention_keeps_its_rows_low_bits(ext, dt, B, Sq, H, V, lens):  # noqa: F811
    dt, lens = DT[dt], lens_of(B, Sq, lens)
    qa, qr, W, cache, table, pair, w = R.case(lens, Sq, H, V, dt, B + Sq)
    out = ext.mla_attention_paged_fp8blk(qa.to(DEV), qr.to(DEV), *(cache[k].to(DEV) for k in ("c_kv", "pe", "scales")),
                                         table.to(DEV), i32(lens).to(DEV), W.to(DEV), SCALE, True).cpu()
    ctx = R.rows(cache, table, lens, Sq)
    off = (out.double() - R.outputs(ctx, pair, w)).abs()
    over = off / R.bound(ctx, pair, w, dt, B * Sq > 128)
    assert float(over.max()) <= 1, (float(over.max()), int((over > 1).sum()), over.argmax())
