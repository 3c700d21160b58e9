"""CPU checks that the bound of the GPU tests of 3d's rows (tests/test_gpu_blocked_rows.py) accepts
rows as the kernels hold them and rejects rows that lose their low bits, on those tests' inputs."""

from __future__ import annotations

import pytest
import torch

import blocked_pairs as R

DT = {"bf16": torch.bfloat16, "f16": torch.float16}
FEW = [(1, 1, 3, 64, [3000]), (4, 2, 3, 132, [2000, 90, 7, 700]), (8, 1, 2, 128, [5, 64, 65, 300, 1, 33, 900, 100])]
TILES = [(3, 3, 3, 64, [3000, 100, 3]), (40, 3, 2, 132, None), (128, 1, 2, 128, None), (60, 2, 4, 128, (2000, 3000))]
MANY = [(3, 50, 3, 132, [3000, 300, 50]), (140, 1, 2, 128, None), (2, 200, 20, 64, [201, 1500])]


def lens_of(B, Sq, lens):
    if lens is None:
        lens = torch.randint(Sq, 300, (B,), generator=torch.Generator().manual_seed(B)).tolist()
        lens[0], lens[B // 2] = 1500, 0
    if isinstance(lens, tuple):
        lens = torch.randint(*lens, (B,), generator=torch.Generator().manual_seed(B)).tolist()
    return lens


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("B,Sq,H,V,lens", FEW + TILES + MANY)
def test_the_bound_tells_lost_low_bits(dt, B, Sq, H, V, lens):
    dt, lens = DT[dt], lens_of(B, Sq, lens)
    _, _, _, cache, table, pair, w = R.case(lens, Sq, H, V, dt, B + Sq)
    ctx = R.rows(cache, table, lens, Sq)
    many = B * Sq > 128
    want, bound = R.outputs(ctx, pair, w), R.bound(ctx, pair, w, dt, many)
    form = R.packed if many else R.two_terms

    def beyond(mistake):
        off = (R.outputs(form(ctx.float().double(), dt, mistake), pair, w).to(dt).double() - want).abs()
        seen = want.abs().sum(-1) > 0
        return float((off > bound)[seen].double().mean())

    assert beyond(None) == 0
    for mistake in (["rounded"] if many else []) + (["no_low", "other_low"] if not many or dt == torch.float16 else []):
        if mistake == "other_low" and B * Sq == 1:
            continue   # the token's own
        assert beyond(mistake) > 0.25, (mistake, beyond(mistake))
