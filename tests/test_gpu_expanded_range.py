"""GPU checks of the expanded attention where values, weights and scores lie far apart: what a query does not see
costs it nothing, and powers of two in the weights cost no bits (bounds of tests/expanded_ref.py)."""

from __future__ import annotations

import math
import random

import pytest
import torch

import expanded_ref as E
from test_gpu_expanded import BF, DEV, DT, N, SCALE, ext, make, rows_of, run_paged  # noqa: F401

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


def columns(got, ref, name):
    """E.check's 2-norms, of every head and output column of its own."""
    out, _, usual = ref
    d = (got.double() - out).norm(dim=0)
    assert torch.isfinite(got).all(), name
    assert (d <= usual.norm(dim=0)).all(), f"{name}: {(d / usual.norm(dim=0)).max().item():.3f} of the bound"


@pytest.mark.parametrize("uk,uv", [(0, -30), (0, -12), (0, 12), (0, 60), (-30, 0), (-12, 0), (12, 0), (60, 0), (-40, 40), (5, 5)])
@pytest.mark.parametrize("Sq,lens,splits", [(60, [300], 1), (140, [300], 3), (140, [140, 400], 1)])
def test_powers_of_two_in_the_weights(ext, uk, uv, Sq, lens, splits, monkeypatch):
    """W_uk under 2^uk, with queries under 2^-uk, and W_uv under 2^uv: the same function, and the same bits of it."""
    monkeypatch.setenv("MLA_EXPAND_SPLITS", str(splits))
    t = make(54, len(lens), Sq, lens, 3, BF)
    t["W_uk"] *= 2.0 ** uk
    t["q_nope"] *= 2.0 ** -uk
    t["W_uv"] *= 2.0 ** uv
    got = run_paged(ext, t, True)
    for b, n in enumerate(lens):
        ref = E.attention(t["q_nope"][b], t["q_rope"][b], *rows_of(t, b, n), t["W_uk"], t["W_uv"], SCALE,
                          E.limits(Sq, n, Sq, True), BF)
        columns(got[b], ref, f"{uk} {uv} {b}")


@pytest.mark.parametrize("Sq,n", [(64, 64), (200, 333)])
@pytest.mark.parametrize("most", [8, 40])
def test_weights_of_rows_far_apart(ext, Sq, n, most):
    """Every row of W_uk and W_uv under a power of two of its own, some rows zeros, in some of the heads."""
    t = make(55, 1, Sq, [n], 4, BF)
    g = torch.Generator(device=DEV)
    g.manual_seed(most)
    for name in ("W_uk", "W_uv"):
        e = torch.randint(-most, most + 1, (4, N), generator=g, device=DEV).float()
        e[1] = 0
        t[name] *= torch.exp2(e)[..., None].to(BF)
        if name == "W_uk":
            t["q_nope"] *= torch.exp2(-e).to(BF)[None, None]
        t[name][2, 5] = 0
    got = run_paged(ext, t, True)
    ref = E.attention(t["q_nope"][0], t["q_rope"][0], *rows_of(t, 0, n), t["W_uk"], t["W_uv"], SCALE,
                      E.limits(Sq, n, Sq, True), BF)
    columns(got[0], ref, f"{Sq} {n}")


@pytest.mark.parametrize("uk", [-30, -12, 20])
def test_rows_of_zeros_among_scaled_weights(ext, uk):
    """Query columns that meet rows of zeros, with the size of the others' scaled ones, cost those no bits."""
    t = make(61, 1, 70, [200], 3, BF)
    t["W_uk"] *= 2.0 ** uk
    t["q_nope"] *= 2.0 ** -uk
    t["W_uk"][1, 5], t["W_uk"][2, 64:], t["W_uv"][0, 3:90] = 0, 0, 0
    got = run_paged(ext, t, True)
    ref = E.attention(t["q_nope"][0], t["q_rope"][0], *rows_of(t, 0, 200), t["W_uk"], t["W_uv"], SCALE,
                      E.limits(70, 200, 70, True), BF)
    columns(got[0], ref, str(uk))


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("Sq,n,splits", [(64, 200, 1), (70, 200, 1), (130, 700, 2), (30, 20, 1)])
def test_weights_that_are_not_finite(ext, dtype, Sq, n, splits, monkeypatch):
    """A weight that is not finite makes its output column (W_uv) or its head (W_uk) NaN where a query sees a key, and
    changes nothing else."""
    monkeypatch.setenv("MLA_EXPAND_SPLITS", str(splits))
    t = make(56, 1, max(Sq, n), [n], 3, DT[dtype])
    for k in ("q_nope", "q_rope"):
        t[k] = t[k][:, -Sq:].contiguous()
    want = run_paged(ext, t, True)
    empty = max(0, Sq - n)
    t["W_uv"][1, 7, 100] = math.inf
    t["W_uk"][2, 9, 3] = math.nan
    got = run_paged(ext, t, True)
    assert not got[:, :empty].any()
    assert torch.equal(got[:, :, 0], want[:, :, 0])
    assert got[:, empty:, 1, 7].isnan().all()
    keep = [i for i in range(N) if i != 7]
    assert torch.equal(got[:, :, 1, keep], want[:, :, 1, keep])
    assert got[:, empty:, 2].isnan().all()


def own(t):
    """Weights and queries of their own memory."""
    return {**t, "W_uk": t["W_uk"].clone(), "W_uv": t["W_uv"].clone(), "q_nope": t["q_nope"].clone()}


def scaled(t, uk, uv):
    """Heads of W_uk and W_uv under powers of two of their own, the queries' columns under W_uk's inverse."""
    u = own(t)
    k, v = (torch.exp2(torch.tensor(e, dtype=torch.float32, device=DEV)).to(BF) for e in (uk, uv))
    u["W_uk"] *= k[:, None, None]
    u["q_nope"] /= k[:, None]
    u["W_uv"] *= v[:, None, None]
    return u, v[:, None]


@pytest.mark.parametrize("B,Sq,lens,span", [(1, 130, [300], 1400000), (40, 3, [3 + 5 * b for b in range(40)], 0), (2, 64, [64, 1000], 0)])
def test_heads_under_powers_of_their_own(ext, B, Sq, lens, span):
    """Groups of heads, more sequences than heads, few queries: the outputs are those of ordinary weights under W_uv's
    powers of two, bit for bit (every rounding on the way is under powers of two that are taken out again)."""
    t = make(57, B, Sq, lens, 5, BF)
    t["q_rope"].zero_()             # (whose scores lie beside those of scaled columns)
    if span:                        # 2 GiB hold three heads of that many keys
        table = torch.zeros(1, span // 64, dtype=torch.int32, device=DEV)
        table[:, :t["table"].size(1)] = t["table"]
        t["table"] = table
    want = run_paged(ext, t, True)
    u, v = scaled(t, [0, 20, -20, 0, -14], [0, 0, 30, -30, 14])
    assert torch.equal(run_paged(ext, u, True), want * v)


def test_weights_change_between_replays(ext):
    """A captured call looks at its weights in every replay; eager calls in between."""
    t = make(58, 2, 70, [200, 130], 5, BF)
    t["q_rope"].zero_()
    u = own(t)
    steps = [([0] * 5, [0] * 5), ([0, 20, -20, 0, -14], [0, 0, 30, -30, 14]), ([0] * 5, [0] * 5), ([-20] * 5, [14, 0, 0, 0, 0])]
    want = run_paged(ext, t, True)
    run_paged(ext, u, True)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run_paged(ext, u, True)
    for uk, uv in steps:
        s, v = scaled(t, uk, uv)
        for k in ("W_uk", "W_uv", "q_nope"):
            u[k].copy_(s[k])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want * v)
        assert torch.equal(run_paged(ext, s, True), want * v)
        torch.cuda.synchronize()


@pytest.mark.parametrize("block", [0, 32])
def test_scaled_weights_over_other_caches(ext, block):
    """The dense cache and the one in 8 bits."""
    t = make(59, 2, 40, [128, 128], 4, BF)
    t["q_rope"].zero_()
    u, v = scaled(t, [20, 0, -20, 1], [30, -30, 0, 1])
    if block:
        codes = [torch.nan_to_num(t[n].float()).mul(40).to(torch.float8_e4m3fn) for n in ("c_kv", "pe")]
        scales = torch.full((t["c_kv"].size(0), 64 // block, 2), 122, dtype=torch.uint8, device=DEV)
        call = lambda x: ext.mla_attention_paged_fp8blk_expanded(x["q_nope"], x["q_rope"], *codes, scales, t["table"], t["lens"],
                                                                 x["W_uk"], x["W_uv"], SCALE, True)
    else:
        rows = [torch.stack([rows_of(t, b, 128)[i] for b in range(2)]).contiguous() for i in range(2)]
        call = lambda x: ext.mla_attention_expanded(x["q_nope"], x["q_rope"], *rows, x["W_uk"], x["W_uv"], SCALE, True)
    assert torch.equal(call(u), call(t) * v)


@pytest.mark.parametrize("weight", [2.0 ** -9, 255 / 256, 1.0, 255 / 128, 255.0])
@pytest.mark.parametrize("Sq,n", [(64, 64), (130, 200)])
def test_the_largest_values(ext, Sq, n, weight):
    """Latent rows along the weights' rows, each at its largest: 512 products of one sign, 65,025 in the scale that fp16
    holds them in."""
    t = make(60, 1, Sq, [n], 2, BF)
    sign = torch.sign(t["W_uv"][0, 0].float()).to(BF)
    t["W_uv"][0] = weight * sign
    for j in range(-(-n // 64)):
        t["c_kv"][t["table"][0, j]] = 127.5 * sign
    got = run_paged(ext, t, True)
    assert (got[0, :, 0] == torch.tensor(512 * 127.5 * weight, device=DEV).to(BF)).all()


@pytest.mark.parametrize("seed", range(24))
def test_rows_weights_and_units_of_any_size(ext, seed, monkeypatch):
    """Rows, units or a few rows under powers of two of their own, in half of the batches the weights' rows too: every
    query of every head keeps the bounds' 2-norm, its columns each in its W_uv row's unit."""
    r = random.Random(seed)
    Sq = r.choice([5, 33, 60, 64, 65, 140, 300])
    n = Sq + r.choice([0, 1, 30, 64, 200, 500])
    monkeypatch.setenv("MLA_EXPAND_SPLITS", str(r.choice([1, 1, 2, 5])))
    span, mode = r.choice([3, 10, 14, 40, 60]), r.choice(["rows", "units", "a few"])
    t = make(70 + seed, 1, Sq, [n], 3, BF)
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    P = t["c_kv"].size(0)
    powers = {}
    for k in ("c_kv", "pe"):
        e = torch.randint(-span, span + 1, (P, 1 if mode == "units" else 64), generator=g, device=DEV).float().expand(P, 64)
        if mode == "a few":
            e = torch.where(torch.rand(P, 64, generator=g, device=DEV) < 0.03, float(span), 0.0)
        powers[k] = powers["c_kv"] if mode == "units" and k == "pe" else e
        t[k] *= torch.exp2(powers[k])[..., None].to(BF)
    t["q_nope"] *= 2.0 ** -span
    t["q_rope"] *= 2.0 ** -span
    if r.random() < 0.5:
        for k in ("W_uk", "W_uv"):
            e = torch.randint(-30, 31, (3, N), generator=g, device=DEV).float()
            t[k] *= torch.exp2(e)[..., None].to(BF)
            if k == "W_uk":
                t["q_nope"] *= torch.exp2(-e)[None, None].to(BF)
    got = run_paged(ext, t, True)[0]
    out, _, usual = E.attention(t["q_nope"][0], t["q_rope"][0], *rows_of(t, 0, n), t["W_uk"], t["W_uv"], SCALE,
                                E.limits(Sq, n, Sq, True), BF)
    assert torch.isfinite(got).all()
    unit = t["W_uv"].double().norm(dim=-1)
    assert (((got.double() - out) / unit).norm(dim=-1) <= (usual / unit).norm(dim=-1)).all()
