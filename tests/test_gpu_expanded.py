"""GPU checks of the expanded attention (dense, paged, paged in 8 bits) and of the queries per head
that it takes, against 64-bit plain forms (tests/expanded_ref.py, which derives the tolerances)."""

from __future__ import annotations

import math
import random

import pytest
import torch

import blocked_cache as K
import expanded_ref as E

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
BF, H16 = torch.bfloat16, torch.float16
DT = {"bf16": BF, "f16": H16}
R, D, N = 512, 64, 128
SCALE = math.sqrt(N + D)
NAN, INF = math.nan, math.inf


@pytest.fixture(scope="module")
def ext():
    if not torch.cuda.is_available():
        pytest.fail("GPU tests need a ROCm GPU")
    import mla_custom_cuda
    return mla_custom_cuda


def normal(g, *shape, dtype, std=1.0):
    return (torch.randn(*shape, generator=g, device=DEV) * std).to(dtype)


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def make(seed, B, Sq, lens, H, dtype, page=64, spare=3, shared=None, spread=1.0):
    """Queries, weights and a paged cache of random pages; rows that no sequence holds are NaN.
    shared: {b: (c, pages)} makes the first pages of b those of c."""
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    max_pages = max(1, -(-max(max(lens), Sq) // page))
    need = [-(-n // page) for n in lens]
    P = sum(need) + spare
    order = torch.randperm(P, generator=g, device=DEV).tolist()
    table = torch.zeros(B, max_pages, dtype=torch.int32)
    for b in range(B):
        for j in range(need[b]):
            table[b, j] = order.pop()
        if shared and b in shared:
            c, k = shared[b]
            table[b, :k] = table[c, :k]
    t = {"c_kv": torch.full((P, page, R), NAN, dtype=dtype, device=DEV),
         "pe": torch.full((P, page, D), NAN, dtype=dtype, device=DEV)}
    for b in range(B):
        for j in range(need[b]):
            n = min(page, lens[b] - j * page)
            if shared and b in shared and j < shared[b][1]:
                continue
            t["c_kv"][table[b, j], :n] = normal(g, n, R, dtype=dtype)
            t["pe"][table[b, j], :n] = normal(g, n, D, dtype=dtype)
    t["table"], t["lens"] = table.to(DEV), i32(lens)
    t["q_nope"] = normal(g, B, Sq, H, N, dtype=dtype, std=spread)
    t["q_rope"] = normal(g, B, Sq, H, D, dtype=dtype, std=spread)
    t["W_uk"] = normal(g, H, N, R, dtype=dtype, std=R ** -0.5)
    t["W_uv"] = normal(g, H, N, R, dtype=dtype, std=R ** -0.5)
    return t


def rows_of(t, b, n):
    page = t["c_kv"].size(1)
    j = torch.arange(n, device=DEV)
    p = t["table"][b].long()[j // page]
    return t["c_kv"][p, j % page], t["pe"][p, j % page]


def run_paged(ext, t, causal, new=None):
    return ext.mla_attention_paged_expanded(
        t["q_nope"], t["q_rope"], t["c_kv"], t["pe"], t["table"], t["lens"], t["W_uk"], t["W_uv"],
        SCALE, causal=causal, new_lens=None if new is None else i32(new))


def check_all(t, got, lens, causal, new=None, rows=rows_of):
    B, Sq = t["q_nope"].shape[:2]
    parts = [[], [], [], []]
    for b in range(B):
        k = Sq if new is None else max(0, min(Sq, new[b]))
        assert not got[b, :Sq - k].any(), f"padding rows of sequence {b}"
        lat, rot = rows(t, b, lens[b])
        ref = E.attention(t["q_nope"][b, Sq - k:], t["q_rope"][b, Sq - k:], lat, rot, t["W_uk"], t["W_uv"],
                          SCALE, E.limits(Sq, lens[b], k, causal), got.dtype)
        for p, x in zip(parts, (got[b, Sq - k:],) + ref):
            p.append(x)
    E.check(*(torch.cat(p) for p in parts))


# Sq around a wave's 32 rows, a workgroup's 128 and past two of those; keys around the 64-key step;
# odd heads and head counts that do not divide by the XCDs
PAGED = [
    (1, 1, [1], 1), (1, 1, [64], 3), (2, 1, [65, 200], 8), (1, 2, [2], 5), (3, 31, [31, 64, 130], 2),
    (2, 33, [33, 63], 16), (1, 127, [500], 3), (1, 128, [128], 8), (2, 129, [129, 700], 2),
    (1, 257, [1000], 4), (4, 64, [64, 1000, 64, 127], 3), (1, 300, [2300], 9), (5, 70, [70, 71, 90, 128, 333], 1),
]


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("B,Sq,lens,H", PAGED)
def test_paged_causal(ext, dtype, B, Sq, lens, H):
    t = make(Sq + sum(lens), B, Sq, lens, H, DT[dtype])
    check_all(t, run_paged(ext, t, True), lens, True)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("B,Sq,lens,H,page", [(2, 40, [3, 300], 2, 64), (1, 5, [1], 3, 128), (3, 140, [0, 64, 257], 2, 192)])
def test_paged_full(ext, dtype, B, Sq, lens, H, page):
    """Not causal: every key visible; a sequence without keys gives zeros; larger pages."""
    t = make(7 + Sq, B, Sq, lens, H, DT[dtype], page=page)
    check_all(t, run_paged(ext, t, False), lens, False)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("causal", [True, False])
def test_ragged_new_tokens(ext, dtype, causal):
    """Fewer new tokens than Sq, none, more than Sq and below zero (clamped); rows in front are zeros;
    queries that see no key give zeros."""
    lens, new, Sq = [400, 64, 10, 200, 150, 3], [150, 0, 10, 999, -5, 20], 150
    t = make(3, 6, Sq, lens, 3, DT[dtype])
    got = run_paged(ext, t, causal, new)
    check_all(t, got, lens, causal, new)
    if causal:      # sequence 5 has 3 keys: of its 20 queries the first 17 see none
        assert not got[5, Sq - 20:Sq - 3].any() and got[5, Sq - 3:].any(-1).all()


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_lengths_past_the_table(ext, dtype):
    """Lengths are clamped to the table's span."""
    t = make(4, 2, 16, [128, 128], 2, DT[dtype])
    want = run_paged(ext, t, True)
    t["lens"] = i32([2 ** 31 - 1, 128])
    assert torch.equal(run_paged(ext, t, True), want)
    t["lens"] = i32([-7, 128])
    got = run_paged(ext, t, True)
    assert not got[0].any() and torch.equal(got[1], want[1])


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("page", [64, 128])
def test_shared_pages(ext, dtype, page):
    """Pages shared with another sequence, whole, partly past one's end, or with different lengths."""
    k = page // 64
    lens = [700, 650, 300, 20, 700, 128]
    shared = {1: (0, 10 // k), 2: (0, 4 // k), 4: (2, 2 // k), 5: (0, 2 // k)}
    t = make(9, 6, 130, lens, 2, DT[dtype], page=page, shared=shared)
    check_all(t, run_paged(ext, t, True), lens, True)


def test_same_page_past_one_end(ext):
    """A page that one sequence holds in part and another whole is not taken for a shared unit."""
    t = make(11, 2, 8, [64, 40], 2, BF)
    t["table"][1, 0] = t["table"][0, 0]
    check_all(t, run_paged(ext, t, True), [64, 40], True)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_pages_outside_the_pool(ext, dtype):
    """Entries outside the pool read as zero rows and are never followed."""
    t = make(12, 2, 20, [200, 64], 2, DT[dtype])
    t["table"][0, 1], t["table"][1, 0] = -1, t["c_kv"].size(0)

    def rows(t, b, n):
        u = dict(t, table=t["table"].clamp(0, t["c_kv"].size(0) - 1))
        lat, rot = (x.clone() for x in rows_of(u, b, n))
        if b == 0:
            lat[64:128], rot[64:128] = 0, 0
        else:
            lat.zero_(), rot.zero_()
        return lat, rot
    check_all(t, run_paged(ext, t, True), [200, 64], True, rows=rows)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("bad", [NAN, INF, -INF])
def test_rows_that_are_not_finite(ext, dtype, bad):
    """A latent value that is not finite makes the rows that see it NaN and touches no other; so
    does a rope value of NaN; an infinite rope value gives NaN or a weight of zero."""
    Sq, lens = 140, [300, 140]
    t = make(13, 2, Sq, lens, 2, DT[dtype])
    want = run_paged(ext, t, True)
    page, at = t["table"][0, 250 // 64].item(), 250 % 64
    t["c_kv"][page, at, 17] = bad
    got = run_paged(ext, t, True)
    first = 250 - (300 - Sq)                  # the query whose own key is 250
    assert torch.equal(got[0, :first], want[0, :first]) and torch.equal(got[1], want[1])
    assert got[0, first:].isnan().all()
    t["c_kv"][page, at, 17] = 0
    t["pe"][page, at, 5] = bad
    got = run_paged(ext, t, True)
    assert torch.equal(got[0, :first], want[0, :first]) and torch.equal(got[1], want[1])
    if math.isnan(bad):
        assert got[0, first:].isnan().all()
    else:
        down = t["q_rope"][0, first:, :, 5].double() * bad < 0
        assert torch.equal(got[0, first:].isnan().any(-1), ~down)
        assert torch.equal(got[0, first:].isnan().all(-1), ~down)


def test_values_past_fp16(ext):
    """An expanded value past fp16's range stays finite and hidden from queries in front of it."""
    t = make(14, 1, 70, [70], 2, H16)
    want = run_paged(ext, t, True)
    t["c_kv"][t["table"][0, 0], 40] = 60000.0 * torch.sign(t["W_uv"][0, 0].float()).to(H16)
    got = run_paged(ext, t, True)
    assert torch.equal(got[0, :40], want[0, :40])
    assert torch.isfinite(got).all()


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("spread", [8.0, 30.0])
def test_large_scores(ext, dtype, spread):
    """Scores that climb far from one key step to the next: references move, sums stay."""
    t = make(15, 1, 130, [900], 2, DT[dtype], spread=spread)
    check_all(t, run_paged(ext, t, True), [900], True)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("B,Sq,Sk,H,causal", [(1, 1, 1, 1, False), (2, 50, 77, 3, True), (1, 200, 641, 8, True), (2, 130, 64, 2, False)])
def test_dense(ext, dtype, B, Sq, Sk, H, causal):
    g = torch.Generator(device=DEV)
    g.manual_seed(Sk)
    dt = DT[dtype]
    t = make(16, B, Sq, [Sk] * B, H, dt)
    ckv, pe = normal(g, B, Sk, R, dtype=dt), normal(g, B, Sk, D, dtype=dt)
    got = ext.mla_attention_expanded(t["q_nope"], t["q_rope"], ckv, pe, t["W_uk"], t["W_uv"], SCALE, causal)
    check_all(t, got, [Sk] * B, causal, rows=lambda _, b, n: (ckv[b], pe[b]))
    absorbed = torch.einsum("bshn,hnr->bshr", t["q_nope"].float(), t["W_uk"].float()).to(dt)
    other = ext.mla_attention(absorbed.contiguous(), t["q_rope"], ckv, pe, t["W_uv"], SCALE, causal)
    # the two forms round different things: keys and values here, absorbed queries and ctx there
    assert (got.double() - other.double()).norm() <= 8 * torch.finfo(dt).eps * other.double().norm()


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("block", [16, 32, 64])
@pytest.mark.parametrize("page", [64, 128])
def test_blocked_cache(ext, dtype, block, page):
    """Over the 8-bit cache: its decoded values, exact in the queries' type."""
    dt, Sq, lens, new = DT[dtype], 75, [200, 64, 129], [75, 3, 40]
    t = make(17, 3, Sq, lens, 3, dt, page=page)
    P = t["c_kv"].size(0)
    g = torch.Generator(device=DEV)
    g.manual_seed(block)
    scales = torch.randint(119, 127, (P, page // block, 2), generator=g, device=DEV).to(torch.uint8)
    codes = {n: torch.nan_to_num(t[n].float()).mul(40).to(torch.float8_e4m3fn) for n in ("c_kv", "pe")}

    def value(n, part):
        f = torch.exp2(scales[..., part].double() - 127).repeat_interleave(block, 1)[..., None]
        return codes[n].float().double() * f
    plain = dict(t, c_kv=value("c_kv", 0), pe=value("pe", 1))
    got = ext.mla_attention_paged_fp8blk_expanded(
        t["q_nope"], t["q_rope"], codes["c_kv"], codes["pe"], scales, t["table"], t["lens"], t["W_uk"],
        t["W_uv"], SCALE, True, i32(new))
    check_all(dict(t), got, lens, True, new, rows=lambda _, b, n: rows_of(plain, b, n))
    same = ext.mla_attention_paged_expanded(
        t["q_nope"], t["q_rope"], plain["c_kv"].to(dt), plain["pe"].to(dt), t["table"], t["lens"],
        t["W_uk"], t["W_uv"], SCALE, True, i32(new))
    assert torch.equal(got, same)
    # a NaN code reaches only the queries that see it
    codes["c_kv"].view(torch.uint8)[t["table"][0, 190 // page], 190 % page, 3] = 0x7F
    hurt = ext.mla_attention_paged_fp8blk_expanded(
        t["q_nope"], t["q_rope"], codes["c_kv"], codes["pe"], scales, t["table"], t["lens"], t["W_uk"],
        t["W_uv"], SCALE, True, i32(new))
    first = 190 - (200 - Sq)
    assert torch.equal(hurt[0, :first], got[0, :first]) and hurt[0, first:].isnan().all()
    assert torch.equal(hurt[1:], got[1:])


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("rows,H,ragged", [(1, 4, False), (3, 128, True), (128, 6, False), (300, 16, True), (2050, 2, False)])
def test_q_heads(ext, dtype, rows, H, ragged):
    """q_rope has q_absorbed's bits, and q_nope times W_uk is what q_absorbed makes of it: with W_uk
    an identity, q_nope itself."""
    dt = DT[dtype]
    g = torch.Generator(device=DEV)
    g.manual_seed(rows + H)
    B, Sq = (3, rows // 3) if ragged and rows >= 3 else (1, rows)
    x = normal(g, B, Sq, 1024, dtype=dt)
    wa, wb = normal(g, 1024, 256, dtype=dt, std=1 / 32), normal(g, 256, H * 192, dtype=dt, std=1 / 16)
    gain = (1 + 0.1 * torch.randn(256, generator=g, device=DEV)).to(dt)
    pos = torch.randint(-1, 30000, (B, Sq) if ragged else (Sq,), generator=g, device=DEV)
    eye = torch.eye(N, dtype=dt, device=DEV).expand(H, N, N).contiguous()
    qa, qr = ext.q_absorbed(x, wa, gain, wb, eye, pos, N, D, 1e-6)
    qn, qr2 = ext.q_heads(x, wa, gain, wb, pos, N, D, 1e-6)
    assert qn.shape == (B, Sq, H, N) and qr2.shape == (B, Sq, H, D)
    assert torch.equal(qr, qr2) and torch.equal(qa, qn)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_head_groups(ext, dtype):
    """A span whose keys and values need several groups of heads."""
    H, Sq, n = 5, 130, 1000
    t = make(18, 1, Sq, [n], H, DT[dtype])
    span = 1400000          # 2 GiB hold three heads of that many keys
    table = torch.zeros(1, span // 64, dtype=torch.int32, device=DEV)
    table[:, :t["table"].size(1)] = t["table"]
    t["table"] = table
    check_all(t, run_paged(ext, t, True), [n], True)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("splits", [1, 2, 5, 64])
def test_key_splits(ext, dtype, splits, monkeypatch):
    """Any number of key splits, empty ones among them; NaN and padding rows through the merge."""
    monkeypatch.setenv("MLA_EXPAND_SPLITS", str(splits))
    lens, new, Sq = [700, 64, 10, 330], [150, 64, 0, 150], 150
    t = make(22, 4, Sq, lens, 3, DT[dtype])
    t["new"] = new
    got = run_paged(ext, t, True, new)
    check_all(t, got, lens, True, new)
    t["c_kv"][t["table"][0, 10], 0] = NAN           # key 640: seen by queries from 90 on
    hurt = run_paged(ext, t, True, new)
    assert torch.equal(hurt[0, :90], got[0, :90]) and hurt[0, 90:].isnan().all() and torch.equal(hurt[1:], got[1:])


def test_strided_and_other_stream(ext):
    """Non-contiguous queries, and a call on a stream of its own."""
    t = make(19, 2, 40, [100, 70], 4, BF)
    want = run_paged(ext, t, True)
    wide = torch.empty(2, 40, 4, N + D, dtype=BF, device=DEV)
    wide[..., :N], wide[..., N:] = t["q_nope"], t["q_rope"]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = ext.mla_attention_paged_expanded(wide[..., :N], wide[..., N:], t["c_kv"], t["pe"], t["table"],
                                               t["lens"], t["W_uk"], t["W_uv"], SCALE, causal=True)
    s.synchronize()
    assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_graph_replay(ext, dtype):
    """Captured once, replayed with other lengths, rows and queries in the same tensors, beside eager
    calls; each replay equals the eager call."""
    lens, new = [300, 129], [100, 60]
    t = make(20, 2, 100, lens, 4, DT[dtype])
    fresh = i32(new)

    def call():
        return ext.mla_attention_paged_expanded(t["q_nope"], t["q_rope"], t["c_kv"], t["pe"], t["table"],
                                                t["lens"], t["W_uk"], t["W_uv"], SCALE, True, fresh)
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for i in range(4):
        if i:
            t["q_nope"].mul_(-1.0)
            t["lens"].copy_(i32([300 - 40 * i, 129 - i]))
            fresh.copy_(i32([100 - i, 60 + i]))
        if i == 2:
            t["c_kv"][t["table"][0, 2], 3, 3] = NAN        # key 131 of sequence 0
        if i == 3:
            t["c_kv"][t["table"][0, 2], 3, 3] = 0.5
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        want = call()
        torch.cuda.synchronize()
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(), want.nan_to_num())
        assert bool(got.isnan().any()) == (i == 2)


def test_same_result_twice(ext):
    t = make(21, 3, 200, [700, 200, 333], 6, BF)
    a, b = run_paged(ext, t, True), run_paged(ext, t, True)
    assert torch.equal(a, b)


@pytest.mark.parametrize("seed", range(6))
def test_random_batches(ext, seed):
    r = random.Random(seed)
    B, Sq, H = r.randint(1, 5), r.randint(1, 280), r.choice([1, 2, 3, 7])
    lens = [r.randint(0, 900) for _ in range(B)]
    new = [r.randint(0, Sq) for _ in range(B)]
    page = r.choice([64, 128, 256])
    t = make(seed, B, Sq, lens, H, r.choice([BF, H16]), page=page)
    causal = r.random() < 0.7
    check_all(t, run_paged(ext, t, causal, new), lens, causal, new)


@pytest.mark.parametrize("at", [0, 40, 129, 250, 299])
@pytest.mark.parametrize("size", [2.0 ** 14, 2.0 ** 40, 1e30])
def test_a_row_far_larger(ext, at, size):
    """One key with a latent row or a rope row that is far larger than the others, seen or not: no
    query loses bits by it, those that do not see it not one."""
    Sq, lens = 140, [300]
    t = make(23, 1, Sq, lens, 2, BF)
    want = run_paged(ext, t, True)
    check_all(t, want, lens, True)
    page, row = t["table"][0, at // 64].item(), at % 64
    first = max(0, at - (300 - Sq))             # the first query that sees it
    old = t["c_kv"][page, row].clone(), t["pe"][page, row].clone()
    t["c_kv"][page, row] *= size
    got = run_paged(ext, t, True)
    assert (got[0, :first].double() - want[0, :first].double()).norm() <= 2 ** -8 * want[0, :first].double().norm()
    ref = E.attention(t["q_nope"][0], t["q_rope"][0], *rows_of(t, 0, 300), t["W_uk"], t["W_uv"], SCALE,
                      E.limits(Sq, 300, Sq, True), BF)[0]
    # with scores of such size a row's weights are nothing but 0 and 1, where the score is further from the others
    # than the rounding of its key's components, 2^-11 of each, can bring it: 2^-11 sum |q k| / scale
    big = t["c_kv"][page, row].double() @ t["W_uk"].double().transpose(1, 2)        # [H, 128]
    s = (t["q_nope"][0, first:].double() * big[None]).sum(-1) / SCALE               # [rows, H]
    off = 200 + 2.0 ** -11 * (t["q_nope"][0, first:].double() * big[None]).abs().sum(-1) / SCALE
    gone, all_ = s < -off, s > off
    d = (got[0, first:].double() - ref[first:]).norm(dim=-1)
    n = ref[first:].norm(dim=-1)
    assert (gone | all_).double().mean() > (0.9 if size > 1e5 else 0.5)
    assert (d[gone | all_] <= 2 ** -7 * n[gone | all_]).all()
    t["c_kv"][page, row], t["pe"][page, row] = old[0], old[1] * size
    got = run_paged(ext, t, True)
    assert (got[0, :first].double() - want[0, :first].double()).norm() <= 2 ** -8 * want[0, :first].double().norm()
    ref = E.attention(t["q_nope"][0], t["q_rope"][0], *rows_of(t, 0, 300), t["W_uk"], t["W_uv"], SCALE,
                      E.limits(Sq, 300, Sq, True), BF)[0]
    s = (t["q_rope"][0, first:].double() * t["pe"][page, row].double()).sum(-1) / SCALE
    # (rope components are exact; their float32 sums are off by less than 2^-18 of the sum of magnitudes)
    sure = s.abs() > 200 + 2.0 ** -18 * (t["q_rope"][0, first:].double() * t["pe"][page, row].double()).abs().sum(-1) / SCALE
    d, n = (got[0, first:].double() - ref[first:]).norm(dim=-1), ref[first:].norm(dim=-1)
    assert (d[sure] <= 2 ** -7 * n[sure]).all()


@pytest.mark.parametrize("B", [1, 2])
def test_dense_rows_that_are_not_finite(ext, B):
    t = make(24, B, 100, [130] * B, 3, BF)
    g = torch.Generator(device=DEV)
    g.manual_seed(1)
    ckv, pe = normal(g, B, 130, R, dtype=BF), normal(g, B, 130, D, dtype=BF)
    call = lambda: ext.mla_attention_expanded(t["q_nope"], t["q_rope"], ckv, pe, t["W_uk"], t["W_uv"], SCALE, True)
    want = call()
    ckv[0, 90, 3] = INF
    got = call()
    assert torch.equal(got[0, :60], want[0, :60]) and got[0, 60:].isnan().all() and torch.equal(got[1:], want[1:])


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("lens", [[0], [0, 0, 0]])
def test_no_keys_at_all(ext, dtype, lens):
    t = make(25, len(lens), 5, [1] * len(lens), 2, DT[dtype])
    t["lens"].zero_()
    assert not run_paged(ext, t, True).any()


def test_small_units_behind_large_ones(ext):
    """Units of very different size in one sequence, in either order, weights split over keys."""
    t = make(26, 1, 64, [640], 2, BF, spread=0.01)
    for j in range(10):
        page = t["table"][0, j].item()
        t["c_kv"][page] *= 2.0 ** [0, 3, 11, -2, -20, 0, -30, 12, -9, 1][j]
        t["pe"][page] *= 2.0 ** [0, 3, 11, -2, -20, 0, -30, 12, -9, 1][j]
    t["q_nope"] *= 2.0 ** -10
    t["q_rope"] *= 2.0 ** -10
    check_all(t, run_paged(ext, t, False), [640], False)


def test_beyond_four_gib(ext):
    """Pages behind the pool's first 2^32 bytes, and their copies."""
    P, dt = 70000, BF
    t = make(27, 1, 70, [200], 2, dt)
    pools = [torch.empty(P, 64, w, dtype=dt, device=DEV) for w in (R, D)]
    last = [P - 1, P - 3, 65600, 3]
    for n, pool in zip(("c_kv", "pe"), pools):
        pool[last] = t[n][t["table"][0, :4].long()]
    want = run_paged(ext, t, True)
    t.update(c_kv=pools[0], pe=pools[1], table=i32([last]))
    assert torch.equal(run_paged(ext, t, True), want)
    to = [P - 2, 1, 69000, 65537]
    ext.cache_copy_pages(i32(list(zip(last, to))), pools)
    for pool in pools:
        for a, b in zip(last, to):
            pool[a] = 0
    t["table"] = i32([to])
    assert torch.equal(run_paged(ext, t, True), want)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("what", ["queries", "keys", "both", "latent rows", "half the keys"])
def test_zeros(ext, dtype, what):
    """Queries, keys or both of zeros: averages of what a row sees, and never NaN."""
    t = make(28, 2, 70, [150, 40], 2, DT[dtype])
    if what in ("queries", "both"):
        t["q_nope"][:, ::2], t["q_rope"][:, ::2] = 0, 0
    if what in ("keys", "both", "latent rows"):
        t["c_kv"].zero_()
    if what in ("keys", "both"):
        t["pe"].zero_()
    if what == "half the keys":
        t["c_kv"][t["table"][0, 0].item()], t["c_kv"][:, 32:] = 0, 0
        t["pe"] *= 2.0 ** 9
    got = run_paged(ext, t, True)
    if what in ("keys", "both", "latent rows"):
        assert not got.any()
    else:
        check_all(t, got, [150, 40], True)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_head_groups_by_eight(ext, dtype):
    """Groups of 8, 8 and 3 heads."""
    H, Sq, n = 19, 70, 300
    t = make(29, 1, Sq, [n], H, DT[dtype])
    table = torch.zeros(1, 6250, dtype=torch.int32, device=DEV)     # 2 GiB hold ten heads of 400,000 keys
    table[:, :t["table"].size(1)] = t["table"]
    t["table"] = table
    check_all(t, run_paged(ext, t, True), [n], True)


def test_two_streams_at_once(ext):
    """Calls that overlap, with workspaces of their own."""
    ts = [make(30 + i, 2, 130, [400 - 50 * i, 200], 4, BF) for i in range(2)]
    ts[1]["c_kv"][ts[1]["table"][1, 0], 3] = NAN
    want = [run_paged(ext, t, True) for t in ts]
    streams = [torch.cuda.Stream() for _ in ts]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(run_paged(ext, ts[i], True))
    torch.cuda.synchronize()
    for w, gs in zip(want, got):
        for g in gs:
            assert torch.equal(g.isnan(), w.isnan()) and torch.equal(g.nan_to_num(), w.nan_to_num())


def test_two_graphs_share_a_workspace(ext):
    """Graphs of one memory pool, of other shapes, types and paths (alone, planned, split), in any order."""
    ts = [make(32, 1, 64, [300], 2, BF), make(33, 3, 100, [500, 100, 130], 3, H16), make(34, 1, 40, [6000], 2, BF)]
    ts[1]["c_kv"][ts[1]["table"][0, 7], 0] = NAN
    want = [run_paged(ext, t, True) for t in ts]
    torch.cuda.synchronize()
    graphs, outs, pool = [], [], torch.cuda.graph_pool_handle()
    for t in ts:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], pool=pool):
            out = run_paged(ext, t, True)
            outs.append(out)
    for i in (0, 1, 2, 1, 0, 2, 2, 0, 1, 1):
        graphs[i].replay()
        torch.cuda.synchronize()
        g = outs[i].clone()
        assert torch.equal(g.isnan(), want[i].isnan()) and torch.equal(g.nan_to_num(), want[i].nan_to_num())
        run_paged(ext, ts[(i + 1) % 3], True)
        torch.cuda.synchronize()


def test_many_sequences_of_one_prompt(ext):
    """More sequences behind one first page than a plan compares with each other, and none of them wrong."""
    B = 1100
    t = make(35, 1, 2, [64], 1, BF)
    g = torch.Generator(device=DEV)
    g.manual_seed(36)
    P = 1 + 2 * B
    c_kv, pe = normal(g, P, 64, R, dtype=BF), normal(g, P, 64, D, dtype=BF)
    table = torch.arange(1, P, dtype=torch.int32, device=DEV).reshape(B, 2)
    table[:, 0] = 0
    table[1::2, 1] = 2                                  # and half of them behind a second page too
    t.update(c_kv=c_kv, pe=pe, table=table, lens=i32([70 + b % 59 if b % 2 == 0 else 128 for b in range(B)]),
             q_nope=normal(g, B, 2, 1, N, dtype=BF), q_rope=normal(g, B, 2, 1, D, dtype=BF))
    got = run_paged(ext, t, True)
    for b in (0, 1, 2, 3, 500, 501, 1023, 1024, 1025, 1026, 1098, 1099):
        one = {**t, "table": table[b:b + 1].clone(), "lens": t["lens"][b:b + 1].clone(), "q_nope": t["q_nope"][b:b + 1],
               "q_rope": t["q_rope"][b:b + 1]}
        assert torch.equal(run_paged(ext, one, True)[0], got[b]), b


def test_most_sequences(ext):
    """As many sequences as a call takes, all behind one page or none, one key each or a page and one."""
    B = 65535
    g = torch.Generator(device=DEV)
    g.manual_seed(37)
    t = make(38, 1, 1, [64], 1, BF)
    P = 3000
    table = torch.stack((torch.zeros(B, dtype=torch.int32, device=DEV),
                         torch.arange(B, dtype=torch.int32, device=DEV) % (P - 1) + 1), 1).contiguous()
    lens = i32([65, 1, 0] * (B // 3))
    t.update(c_kv=normal(g, P, 64, R, dtype=BF), pe=normal(g, P, 64, D, dtype=BF), table=table, lens=lens,
             q_nope=normal(g, B, 1, 1, N, dtype=BF), q_rope=normal(g, B, 1, 1, D, dtype=BF))
    got = run_paged(ext, t, True)
    assert not got[2::3].any()
    for b in (0, 1, 3, 4, 1500, 1501, 4095, 32768, 65532, 65533):
        one = {**t, "table": table[b:b + 1].clone(), "lens": lens[b:b + 1].clone(),
               "q_nope": t["q_nope"][b:b + 1], "q_rope": t["q_rope"][b:b + 1]}
        assert torch.equal(run_paged(ext, one, True)[0], got[b]), b


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("rows", [5, 128, 700])
def test_q_heads_apart(ext, dtype, rows, monkeypatch):
    """With RoPE in a launch of its own the same queries, bit for bit."""
    g = torch.Generator(device=DEV)
    g.manual_seed(39)
    H, hidden, ql, dt = 16, 512, 256, DT[dtype]
    args = (normal(g, 1, rows, hidden, dtype=dt), normal(g, hidden, ql, dtype=dt, std=hidden ** -0.5),
            torch.ones(ql, dtype=dt, device=DEV), normal(g, ql, H * (N + D), dtype=dt, std=ql ** -0.5),
            torch.arange(rows, device=DEV) + 40, N, D, 1e-6)
    want = ext.q_heads(*args)
    monkeypatch.setenv("MLA_QUP_FUSE", "0")
    got = ext.q_heads(*args)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("Sq", [1, 33, 64, 65])
@pytest.mark.parametrize("at", [0, 31, 32, 200, 270, 299])
@pytest.mark.parametrize("splits", [1, 3])
def test_a_large_row_and_few_queries(ext, Sq, at, splits, monkeypatch):
    """A key whose latent row is 2^13 times the others', under queries that are as much smaller, so that
    scores are ordinary and the row shows in its values.  A row's distance is at most its output's rounding
    (2^-9), twice what the scores are off (2^-11 sum |q k| / scale, some 2^-11 * 6, in weights and in their sum), and
    a half step of 11 bits for weights and values each: 0.0088."""
    monkeypatch.setenv("MLA_EXPAND_SPLITS", str(splits))
    t = make(40 + Sq, 1, Sq, [300], 2, BF)
    t["q_nope"] *= 2.0 ** -13
    page, row = t["table"][0, at // 64].item(), at % 64
    t["c_kv"][page, row] *= 2.0 ** 13
    got = run_paged(ext, t, True)[0]
    ref = E.attention(t["q_nope"][0], t["q_rope"][0], *rows_of(t, 0, 300), t["W_uk"], t["W_uv"], SCALE,
                      E.limits(Sq, 300, Sq, True), BF)[0]
    d, n = (got.double() - ref).norm(dim=-1), ref.norm(dim=-1)
    assert (d <= 2 ** -6 * n).all()


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("B,Sq,lens,H,splits", [(1, 64, [64], 3, 1), (2, 64, [65, 1000], 8, 4), (3, 17, [32, 33, 700], 2, 64),
                                                (1, 3, [31], 16, 2), (4, 50, [500, 0, 51, 640], 5, 3)])
def test_few_queries(ext, dtype, B, Sq, lens, H, splits, monkeypatch):
    monkeypatch.setenv("MLA_EXPAND_SPLITS", str(splits))
    t = make(60 + Sq, B, Sq, lens, H, DT[dtype])
    for causal in (True, False):
        got = run_paged(ext, t, causal)
        check_all(t, got, lens, causal)
    t["c_kv"][t["table"][0, 0], 5] = INF
    hurt = run_paged(ext, t, False)
    assert hurt[0].isnan().all() and torch.equal(hurt[1:], got[1:])
