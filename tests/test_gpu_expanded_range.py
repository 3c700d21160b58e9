"""GPU checks of the expanded attention where values and scores lie far apart (bounds of tests/expanded_ref.py)."""

from __future__ import annotations

import math

import pytest
import torch

import expanded_ref as E
from test_gpu_expanded import BF, DEV, DT, SCALE, ext, make, rows_of, run_paged  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("Sq,n", [(40, 40), (140, 700)])
@pytest.mark.parametrize("power", [0, 2, 6])
def test_scores_past_float32s_steps(ext, dtype, Sq, n, power):
    """Scores of 2^25 and more, where float32 has steps of more than one: a weight of one for the largest score, where
    it is further from the others than keys' and queries' roundings, 2^-11 of sum |q k| / scale each, can bring it."""
    dt = DT[dtype]
    t = make(53, 1, Sq, [n], 2, dt)
    wide = dt is BF
    for k in ("q_nope", "q_rope"):
        t[k] *= 2.0 ** (13 + (power if wide else 0))
    for k in ("c_kv", "pe"):
        t[k] *= 2.0 ** (12 + (power if wide else 0))
    got = run_paged(ext, t, True)[0].double()
    assert torch.isfinite(got).all()
    lat, rot = (x.double() for x in rows_of(t, 0, n))
    hide = torch.arange(n, device=DEV)[None] > torch.as_tensor(E.limits(Sq, n, Sq, True), device=DEV)[:, None]
    tested = 0
    for h in range(2):
        k, v = lat @ t["W_uk"][h].double().t(), lat @ t["W_uv"][h].double().t()
        q, qr = t["q_nope"][0, :, h].double(), t["q_rope"][0, :, h].double()
        s = ((q @ k.t() + qr @ rot.t()) / SCALE).masked_fill(hide, -math.inf)
        off = 2.0 ** -10 * (q.abs() @ k.abs().t() + qr.abs() @ rot.abs().t()) / SCALE
        best = s.argmax(-1)
        low = s.gather(1, best[:, None]) - off.gather(1, best[:, None])
        rest = (s + off).scatter(1, best[:, None], -math.inf)
        sure = low[:, 0] > rest.amax(-1) + 200
        tested += int(sure.sum())
        d, size = (got[sure, h] - v[best[sure]]).norm(dim=-1), v[best[sure]].norm(dim=-1)
        assert (d <= 2 ** -7 * size).all()
    assert tested > Sq
