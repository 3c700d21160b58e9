"""GPU checks of the expanded attention where values and scores lie far apart: what a query does not see costs
it nothing (bounds of tests/expanded_ref.py)."""

from __future__ import annotations

import math

import pytest
import torch

import expanded_ref as E
from test_gpu_expanded import BF, DEV, DT, SCALE, ext, make, rows_of, run_paged  # noqa: F401

pytestmark = pytest.mark.gpu

MOST = 3.3e38                                    # near bf16's end


def visible(t, got, at, dtype=BF):
    """The queries in front of key `at` of the one sequence, against the keys in front of it."""
    Sq, n = got.size(1), int(t["lens"][0])
    first = max(0, at - (n - Sq))
    lat, rot = (x[:at] for x in rows_of(t, 0, n))
    lims = E.limits(Sq, n, Sq, True)[:first]
    ref = E.attention(t["q_nope"][0, :first], t["q_rope"][0, :first], lat, rot, t["W_uk"], t["W_uv"], SCALE, lims, dtype)
    return (got[0, :first],) + ref


@pytest.mark.parametrize("splits", [1, 3])
@pytest.mark.parametrize("Sq", [60, 140])
@pytest.mark.parametrize("at", [255, 257, 290, 299])
@pytest.mark.parametrize("size", [1.0, 2.0 ** -9, 2.0 ** -30])
@pytest.mark.parametrize("what", ["latent", "rope"])
def test_a_hidden_row_near_the_end_of_the_type(ext, what, size, at, Sq, splits, monkeypatch):
    """A key whose values are near bf16's largest, behind ordinary and behind small ones: queries that do not see
    it keep the bounds that they have over the keys they see."""
    monkeypatch.setenv("MLA_EXPAND_SPLITS", str(splits))
    t = make(50 + Sq, 1, Sq, [300], 2, BF)
    t["c_kv"] *= size
    t["pe"] *= size
    t["q_nope"] /= size
    t["q_rope"] /= size
    page, row = t["table"][0, at // 64].item(), at % 64
    n = "c_kv" if what == "latent" else "pe"
    t[n][page, row] = MOST * torch.sign(t[n][page, row].float()).to(BF)
    E.check(*visible(t, run_paged(ext, t, True), at), name=f"{what} {at}")


@pytest.mark.parametrize("Sq", [60, 140])
@pytest.mark.parametrize("at", [257, 290, 299])
def test_a_hidden_row_behind_rows_of_zeros(ext, at, Sq):
    """The same where the keys of its 64 in front of it have latent rows of zeros."""
    t = make(51, 1, Sq, [300], 2, BF)
    page, row = t["table"][0, at // 64].item(), at % 64
    t["c_kv"][page, :row] = 0
    t["c_kv"][page, row] = MOST
    E.check(*visible(t, run_paged(ext, t, True), at), name=str(at))


@pytest.mark.parametrize("at", [129, 161, 250, 299])
@pytest.mark.parametrize("size", [2.0 ** 13, 2.0 ** 14, 2.0 ** 40, 1e30])
@pytest.mark.parametrize("what", ["latent", "rope"])
def test_a_far_larger_row_costs_no_bits(ext, what, size, at):
    """A key that is far larger than the others leaves the queries in front of it within the bounds over their own
    keys, which do not know of it."""
    t = make(52, 1, 140, [300], 2, BF)
    page, row = t["table"][0, at // 64].item(), at % 64
    t["c_kv" if what == "latent" else "pe"][page, row] *= size
    E.check(*visible(t, run_paged(ext, t, True), at), name=f"{what} {at}")


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
