"""GPU checks of the paged 8-bit cache with block scales: cache_extend, kv_append_paged_fp8blk,
kv_read_fp8blk and mla_attention_paged_fp8blk, against the plain 64-bit forms of
tests/blocked_cache.py.

Tolerances.  Tables, positions, slots, scales and codes are whole numbers and compared as such.
Where float32 sums come before a code (the append's product and norm), a value may round to the
neighbouring code: its distance from the unrounded 64-bit value is at most half a code step there
plus the bound on the float32 sums that blocked_cache.kv_rows derives.  Attention rounds P, ctx and
the output to 16 bits, each by at most u = eps / 2 relative; the three are independent and zero in
the mean, so the outputs' distance in the 2-norm is at most sqrt(3) u of it (a row of few keys,
where they are not independent, at most 3 u), and single elements keep attn_cases.tol.
"""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

import attn_cases as C
import blocked_cache as K

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
SCALE = C.SCALE
BF, H16, F32 = torch.bfloat16, torch.float16, torch.float32
DT = {"bf16": BF, "f16": H16, "f32": F32}


@pytest.fixture(scope="module")
def ext():
    if not torch.cuda.is_available():
        pytest.fail("GPU tests need a ROCm GPU")
    import mla_custom_cuda
    return mla_custom_cuda


def i32(v):
    return torch.tensor(v, dtype=torch.int32)


def to_gpu(cache):
    return {k: v.to(DEV) for k, v in cache.items()}


# ------------------------------------------------------------------ cache_extend

def check_extend(ext, new, lens, table, ring, state, Sq, page):
    want = K.extend(new, lens, table, ring, state, Sq, page)
    t, r = table.to(DEV), ring.to(DEV)
    got = ext.cache_extend(i32(new).to(DEV), i32(lens).to(DEV), t, r, i32(state).to(DEV), Sq, page)
    got = [x.cpu() for x in got]
    assert got[0].tolist() == want["seq_lens"]
    assert got[1].tolist() == want["state"]
    assert got[2].tolist() == want["granted"]
    assert torch.equal(got[3], want["positions"])
    assert torch.equal(got[4], want["slots"])
    assert torch.equal(t.cpu(), want["table"])
    assert torch.equal(r.cpu(), want["ring"])
    return want


def extend_inputs(B, Sq, page, max_pages, seed, free):
    """Requests of any length, what they ask for now and then more than they may, the pool's other
    pages free (the ring's head anywhere)."""
    g = torch.Generator().manual_seed(seed)
    span = max_pages * page
    lens = torch.randint(0, span + 1, (B,), generator=g)
    lens[torch.rand(B, generator=g) < 0.2] = 0
    new = torch.randint(-8, Sq + 3, (B,), generator=g)
    new = torch.where(torch.rand(B, generator=g) < 0.5, torch.full((B,), Sq), new)
    new = torch.where(torch.rand(B, generator=g) < 0.1, torch.full((B,), K.INT_MIN), new)
    new = torch.where(torch.rand(B, generator=g) < 0.1, torch.full((B,), 2 ** 31 - 1), new)
    need = sum(-(-int(n) // page) for n in lens)
    P = need + free
    table = K.tables(lens.tolist(), page, P, g, max_pages)
    used = set(table[table >= 0].tolist())
    rest = [p for p in range(P) if p not in used]
    head = int(torch.randint(0, P, (1,), generator=g))
    ring = torch.full((P,), -1, dtype=torch.int32)
    for i, p in enumerate(rest):
        ring[(head + i) % P] = p
    return new.tolist(), lens.tolist(), table, ring, [head, len(rest)]


@pytest.mark.parametrize("B,Sq,page,max_pages,free", [
    (1, 1, 64, 1, 1), (1, 1, 64, 3, 0), (3, 4, 64, 5, 2), (61, 1, 64, 40, 7), (130, 4, 128, 9, 20),
    (64, 100, 64, 6, 64), (1023, 2, 64, 3, 300), (1024, 8, 64, 2, 100), (5, 5000, 64, 130, 90),
    (1025, 3, 64, 4, 200), (2500, 1, 64, 2, 500), (40, 300, 192, 20, 33), (2, 20000, 64, 400, 700),
])
def test_extend(ext, B, Sq, page, max_pages, free):
    """One launch, two launches (many requests, many positions), with enough free pages for some."""
    for seed in (0, 1):
        check_extend(ext, *extend_inputs(B, Sq, page, max_pages, 17 * B + seed, max(free, 1)), Sq, page)


def test_extend_limits(ext):
    """A full table, an asked length past Sq, lengths outside the table's span, a request that needs
    no page behind one that could get none, an empty ring with a page coming back, head and count
    outside the ring."""
    table = torch.arange(24, dtype=torch.int32).view(8, 3)
    lens = [192, 100, 60, -5, 1000, 64, 128, 65]
    new = [1, 5, 4, 4, 1, 0, -1, -70]
    ring = torch.arange(100, 130, dtype=torch.int32)
    for state in ([0, 30], [29, 2], [7, 0], [7, 1], [-3, 99], [31, -4]):
        check_extend(ext, new, lens, table, ring, state, 4, 64)


def test_extend_slots_past_32_bits(ext):
    page = 1 << 20
    ring = torch.arange(8000, 0, -1, dtype=torch.int32)
    table = torch.tensor([[7900, -1], [7777, -1]], dtype=torch.int32)
    want = check_extend(ext, [2, 3], [page - 1, 5], table, ring, [0, 10], 3, page)
    assert int(want["slots"].max()) > 2 ** 32


def test_extend_many_rounds(ext):
    """Sixty calls in a row, each on the last one's state: every page stays in exactly one place."""
    g = torch.Generator().manual_seed(5)
    B, Sq, page, mp, P = 37, 3, 64, 6, 120
    lens, state = i32([0] * B).to(DEV), i32([11, P]).to(DEV)
    table = torch.full((B, mp), -1, dtype=torch.int32, device=DEV)
    ring = torch.randperm(P, generator=g).int().to(DEV)
    for step in range(60):
        new = torch.randint(-2, Sq + 1, (B,), generator=g)
        new = torch.where(torch.rand(B, generator=g) < 0.05, torch.full((B,), K.INT_MIN), new).int()
        if step % 7 == 0:
            new = torch.full((B,), Sq, dtype=torch.int32)
        big = 64 if step % 5 == 0 else Sq
        want = K.extend((new * (big // Sq) if step % 5 == 0 and step % 7 else new).tolist(), lens.tolist(),
                        table.cpu(), ring.cpu(), state.tolist(), big, page)
        ask = (new * (big // Sq) if step % 5 == 0 and step % 7 else new).to(DEV)
        lens, state, granted, _, slots = ext.cache_extend(ask, lens, table, ring, state, big, page)
        assert lens.tolist() == want["seq_lens"] and granted.tolist() == want["granted"]
        assert torch.equal(table.cpu(), want["table"]) and torch.equal(slots.cpu(), want["slots"])
        head, count = state.tolist()
        free = [int(ring[(head + i) % P]) for i in range(count)]
        held = [int(p) for b, n in enumerate(lens.tolist()) for p in table[b, :-(-n // page)].tolist()]
        assert sorted(free + held) == list(range(P))


def lib():
    import mla_custom_cuda  # noqa: F401  (one HIP runtime: torch's)
    import os
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    L = ctypes.CDLL(os.path.join(root, "mla-cuda_amd", "libmla_amd.so"))
    L.mla_last_error.restype = ctypes.c_char_p
    L.mla_cache_extend_workspace_bytes.restype = ctypes.c_size_t
    L.mla_kv_append_workspace_bytes.restype = ctypes.c_size_t
    return L


def ptr(t):
    return ctypes.c_void_p(t.data_ptr())


def stream():
    return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)


@pytest.mark.parametrize("B,Sq", [(50, 2), (1100, 2)])
def test_extend_in_place_state(ext, B, Sq):
    """The C entry's outputs may be its inputs: lengths, free state (and what was granted over what
    was asked)."""
    L = lib()
    new, lens, table, ring, state = extend_inputs(B, Sq, 64, 4, 3, 40)
    want = K.extend(new, lens, table, ring, state, Sq, 64)
    n, ln, t, r, st = (x.to(DEV) for x in (i32(new), i32(lens), table, ring, i32(state)))
    pos = torch.empty(B, Sq, dtype=torch.int64, device=DEV)
    slots = torch.empty_like(pos)
    wsb = L.mla_cache_extend_workspace_bytes(B, Sq)
    ws = torch.empty(max(wsb, 1), dtype=torch.uint8, device=DEV)
    st_code = L.mla_cache_extend(B, Sq, 64, 4, ring.numel(), ptr(n), ptr(ln), ptr(st), ptr(t), ptr(r), ptr(ln),
                                 ptr(st), ptr(n), ptr(pos), ptr(slots), ptr(ws), ctypes.c_size_t(wsb), stream())
    assert st_code == 0, L.mla_last_error()
    assert ln.tolist() == want["seq_lens"] and st.tolist() == want["state"] and n.tolist() == want["granted"]
    assert torch.equal(slots.cpu(), want["slots"]) and torch.equal(pos.cpu(), want["positions"])
    assert torch.equal(t.cpu(), want["table"]) and torch.equal(r.cpu(), want["ring"])


# ------------------------------------------------------------------ kv_append_paged_fp8blk

def check_append(before, after, want, block):
    """The cache after the append against its plain form (the module's docstring)."""
    P, page, _ = before["c_kv"].shape
    e = after["scales"].view(-1, 2).int() - 127
    assert torch.equal(e[~want["touched"]], want["e"][~want["touched"]])
    rows = K.decode(after)
    kept = K.decode(before)
    old_e = before["scales"].view(-1, 2).int() - 127
    new, old = want["new"], want["old"]
    for part, name in enumerate(("c_kv", "pe")):
        # a scale may differ only where a border lies within the float32 bound of the maximum
        for i in (torch.nonzero(want["touched"])[:, 0]).tolist():
            if int(e[i, part]) != int(want["e"][i, part]):
                r = slice(i * block, (i + 1) * block)
                v = want["value"][part][r]
                v = torch.where(torch.isfinite(v), v, 0)
                border = 448 * 2.0 ** min(int(e[i, part]), int(want["e"][i, part]))
                assert abs(int(e[i, part]) - int(want["e"][i, part])) == 1
                assert ((v.abs() - border).abs() <= want["bound"][part][r] * (1 + 1e-9)).any(), "wrong scale"
        er = e[:, part].repeat_interleave(block)
        v, got = want["value"][part][new], rows[part][new]
        fine = torch.isfinite(v)
        assert torch.isnan(got[~fine]).all()
        bound = want["bound"][part][new][fine]
        ex = er[new][:, None].expand_as(v)[fine]
        off = (got[fine] - v[fine]).abs()
        assert (off <= K.half_step(v[fine].abs() + bound, ex) + bound).all()
        # rows of before: the same values under a larger scale, rounded once more, exactly
        oe = old_e[:, part].repeat_interleave(block)[old]
        assert (er[old] >= oe).all()
        again = K.round_code(kept[part][old], er[old][:, None])
        assert torch.equal(torch.nan_to_num(rows[part][old], nan=1e30), torch.nan_to_num(again, nan=1e30))
        # everything else keeps its bytes
        rest = ~(new | old)
        w = before[name].size(2)
        assert torch.equal(after[name].view(-1, w)[rest], before[name].view(-1, w)[rest])
        same = (e[:, part] == old_e[:, part]).repeat_interleave(block) & old
        assert torch.equal(after[name].view(-1, w)[same], before[name].view(-1, w)[same])


def append_inputs(lens, new, Sq, block, page, dt, seed, hidden=256, spare=3):
    g = torch.Generator().manual_seed(seed)
    P = sum(-(-n // page) for n in lens) + spare
    table = K.tables(lens, page, P, g)
    cache = K.new_pool(P, page, block, g)
    K.poison(cache, table, [max(0, n - max(0, k)) for n, k in zip(lens, new)], page, block)
    x = torch.randn(len(lens), Sq, hidden, generator=g).to(dt)
    W = (torch.randn(hidden, K.KV + K.ROPE, generator=g) / math.sqrt(hidden)).to(dt)
    gain = (1 + 0.1 * torch.randn(K.KV, generator=g)).to(dt)
    return cache, x, W, gain, table


def run_append(ext, cache, x, W, gain, lens, new, table):
    c = to_gpu(cache)
    ext.kv_append_paged_fp8blk(x.to(DEV), W.to(DEV), gain.to(DEV), i32(lens).to(DEV), i32(new).to(DEV),
                               table.to(DEV), c["c_kv"], c["pe"], c["scales"], 1e-6)
    return {k: v.cpu() for k, v in c.items()}


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("block", [16, 32, 64])
@pytest.mark.parametrize("page,Sq,lens,new", [
    (64, 1, [1, 16, 17, 64, 65, 200], [1, 1, 1, 1, 1, 1]),
    (64, 1, [30, 31, 0, 500], [0, 1, 1, -3]),
    (128, 4, [4, 18, 129, 66, 3, 260], [4, 4, 4, 4, 3, 9]),
    (64, 70, [70, 100, 64, 300, 71], [70, 70, 33, 1, 64]),
    (192, 200, [200, 577], [200, 200]),
])
def test_append(ext, dt, block, page, Sq, lens, new):
    cache, x, W, gain, table = append_inputs(lens, new, Sq, block, page, DT[dt], 3 * block + Sq)
    after = run_append(ext, cache, x, W, gain, lens, new, table)
    want = K.append(cache, x, W, gain, lens, new, table, page, block)
    check_append(cache, after, want, block)


@pytest.mark.parametrize("dt,B,Sq", [("bf16", 128, 1), ("f16", 3, 50), ("f32", 8, 1)])
def test_append_at_the_layers_width(ext, dt, B, Sq):
    """hidden 7168: the product in several splits, summed while the rows are made."""
    g = torch.Generator().manual_seed(B)
    lens = torch.randint(Sq, 400, (B,), generator=g).tolist()
    new = [Sq] * B
    cache, x, W, gain, table = append_inputs(lens, new, Sq, 32, 64, DT[dt], B + 1, hidden=7168)
    after = run_append(ext, cache, x, W, gain, lens, new, table)
    check_append(cache, after, K.append(cache, x, W, gain, lens, new, table, 64, 32), 32)


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("block", [16, 32, 64])
def test_append_long_rows_in_many_splits(ext, dt, block):
    """Many new tokens whose product comes in many splits (the rows are made in a launch of their
    own), with padding, a sequence without new tokens, and blocks that keep rows of before."""
    lens, new, Sq = [90, 170, 20, 33], [40, 37, 0, 33], 40
    cache, x, W, gain, table = append_inputs(lens, new, Sq, block, 64, DT[dt], block, hidden=7168)
    after = run_append(ext, cache, x, W, gain, lens, new, table)
    check_append(cache, after, K.append(cache, x, W, gain, lens, new, table, 64, block), block)


def test_append_scale_grows_and_stays(ext):
    """Token after token into one block, each larger than the last (the rows before are coded again
    every time, down to codes that vanish), then smaller ones, which keep the scale."""
    hidden, page, block = 64, 64, 32
    g = torch.Generator().manual_seed(2)
    W = torch.randn(hidden, K.KV + K.ROPE, generator=g) / 8
    gain = torch.ones(K.KV)
    cache = K.new_pool(2, page, block, g)
    cache["c_kv"].fill_(0x7F), cache["pe"].fill_(0x7F), cache["scales"].fill_(255)
    table = i32([[1]])
    grow = [0.01, 0.02, 0.03, 1.0, 5.0, 600.0, 3e5, 1e-3, 2.0, 0.0]
    for t, s in enumerate(grow):
        x = torch.randn(1, 1, hidden, generator=g) * s
        gain_t = gain * max(s, 1e-3)
        after = run_append(ext, cache, x, W, gain_t, [t + 1], [1], table)
        check_append(cache, after, K.append(cache, x, W, gain_t, [t + 1], [1], table, page, block), block)
        cache = after


def abi_append(L, dt_code, x, W, gain, inv_freq, lens, new, table, c, block, eps=0.0):
    class Dims(ctypes.Structure):
        _fields_ = [(n, ctypes.c_int32) for n in
                    ("batch", "sq", "sk", "hidden", "q_lora", "heads", "nope", "rope", "kv_rank", "v")]
    B, Sq, hidden = x.shape
    P, page, _ = c["c_kv"].shape
    d = Dims(B, Sq, table.size(1) * page, hidden, 0, 0, 0, K.ROPE, K.KV, 0)
    wsb = L.mla_kv_append_workspace_bytes(dt_code, ctypes.byref(d))
    ws = torch.empty(wsb, dtype=torch.uint8, device=DEV)
    t = [a.to(DEV) for a in (x, W, gain, inv_freq, i32(lens), i32(new), table)]
    st = L.mla_kv_append_paged_fp8blk(dt_code, ctypes.byref(d), ptr(t[0]), ptr(t[1]), ptr(t[2]), ptr(t[3]),
                                      ctypes.c_double(eps), ptr(t[4]), ptr(t[5]), ptr(t[6]), page, P, block,
                                      ptr(c["c_kv"]), ptr(c["pe"]), ptr(c["scales"]), ptr(ws),
                                      ctypes.c_size_t(wsb), stream())
    assert st == 0, L.mla_last_error()
    torch.cuda.synchronize()


def test_append_codes_exactly(ext):
    """Where float32 sums are exact the bytes are: one-hot tokens pick rows of W, and a table of zero
    frequencies leaves the rope part as it is.  Values on and past 448 times a power of two, halfway
    between codes, subnormal ones, zeros, blocks of zeros alone and of tiny values."""
    L, block, page, hidden = lib(), 16, 64, 64
    g = torch.Generator().manual_seed(4)
    W = torch.zeros(hidden, K.KV + K.ROPE)
    W[:, :K.KV] = 1.0
    rope = torch.randn(hidden, K.ROPE, generator=g)
    top = torch.full((hidden,), 448.0)
    top[16:32] = 448.0 * (1 + 2.0 ** -23)     # just past the border: a scale more
    top[32:48] = 3.0
    for k in range(hidden):
        mag = rope[k].abs() / rope[k].abs().max()
        rope[k] = torch.copysign(mag.clamp(max=0.99) * top[k], rope[k])
        rope[k, 0] = top[k]
    ties = torch.tensor([17.0, 19.0, 1.0625, 1.1875, 2.0 ** -10, 3 * 2.0 ** -10, 5 * 2.0 ** -11, 0.5, 0.0,
                         -17.0, -2.0 ** -10, 2.0 ** -9, 2.0 ** -6, 15.5 * 2.0 ** -10, 440.0, 447.0])
    rope[3, 1:17] = ties                       # scale 1 (the row's block has 448 as its maximum)
    rope[40, 1:17] = ties * 2.0 ** -8
    rope[48:] = 0.0
    rope[52, 7] = 1e-35                        # at the smallest scale, 2^-100
    W[:, K.KV:] = rope
    x = torch.eye(hidden)[None]
    cache = K.new_pool(2, page, block, g)
    c = to_gpu(cache)
    abi_append(L, 0, x, W, torch.ones(K.KV), torch.zeros(K.ROPE // 2), [64], [64], i32([[1]]), c, block)
    r = rope.double().view(4, block, K.ROPE)
    e = torch.tensor([K.exponent(float(v.abs().max())) for v in r])
    assert e.tolist() == [0, 1, -7, -100]
    got = c["scales"].cpu()[1].int() - 127
    assert torch.equal(got[:, 1], e.int())
    assert got[:, 0].tolist() == [-8] * 4      # a row of ones
    codes = c["pe"].cpu()[1].view(4, block, K.ROPE)
    assert torch.equal(K.code_values()[codes.long()] * K.two(e)[:, None, None], K.round_code(r, e[:, None, None]))
    sign = (codes >> 7).bool()
    assert torch.equal(sign, torch.signbit(rope).view_as(sign))
    assert torch.equal(c["pe"].cpu()[0], cache["pe"][0])


def test_append_values_that_are_not_finite(ext):
    """A token with an infinity or a NaN becomes NaN codes; its neighbours keep their own scale."""
    lens, new = [20, 40], [20, 8]
    cache, x, W, gain, table = append_inputs(lens, new, 20, 16, 64, BF, 8)
    clean = run_append(ext, cache, x, W, gain, lens, new, table)
    x2 = x.clone()
    x2[0, 3, 5], x2[0, 18, 0], x2[1, 15, 9] = math.inf, math.nan, -math.inf
    got = run_append(ext, cache, x2, W, gain, lens, new, table)
    rows, ref = K.decode(got), K.decode(clean)
    bad = torch.zeros(rows[0].size(0), dtype=torch.bool)
    bad[K.slots_of(table, 0, 0, 20, 64)[[3, 18]]] = True
    bad[K.slots_of(table, 1, 32, 40, 64)[[3]]] = True
    for part in (0, 1):
        assert torch.isnan(rows[part][bad]).all()
    want = K.append(cache, x2, W, gain, lens, new, table, 64, 16)
    check_append(cache, got, want, 16)


def test_append_skips_what_is_no_page(ext):
    """Table entries outside the pool: their blocks are skipped, the others written; lengths past the
    table's span and new lengths past Sq or the length are clamped."""
    lens, new = [130, 70, 64], [70, 70, 64]
    cache, x, W, gain, table = append_inputs(lens, new, 70, 32, 64, BF, 9)
    table[0, 1], table[1, 1], table[2, 0] = -1, cache["c_kv"].size(0), 2 ** 31 - 1
    after = run_append(ext, cache, x, W, gain, lens, new, table)
    want = K.append(cache, x, W, gain, lens, new, table, 64, 32)
    assert int(want["new"].sum()) == 2 + 4 + 64   # rows 60..63 and 128, 129 of the first; the second's page
    check_append(cache, after, want, 32)
    lens, new = [5, 10 ** 6, -4], [9, 2 ** 31 - 1, 5]
    cache, x, W, gain, table = append_inputs([64, 128, 64], [64, 8, 64], 8, 16, 64, BF, 10)
    after = run_append(ext, cache, x, W, gain, lens, new, table)
    check_append(cache, after, K.append(cache, x, W, gain, lens, new, table, 64, 16), 16)


# ------------------------------------------------------------------ kv_read_fp8blk

@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("block", [16, 32, 64])
def test_read_every_code(ext, dt, block):
    """All codes under many scales, each the 64-bit value rounded once to the type."""
    g = torch.Generator().manual_seed(block)
    P, page = 5, 64
    cache = {"c_kv": torch.randint(0, 256, (P, page, K.KV), generator=g).to(torch.uint8),
             "pe": torch.randint(0, 256, (P, page, K.ROPE), generator=g).to(torch.uint8),
             "scales": torch.randint(20, 236, (P, page // block, 2), generator=g).to(torch.uint8)}
    if dt == "f16":
        cache["scales"] = torch.randint(97, 140, cache["scales"].shape, generator=g).to(torch.uint8)
    slots = torch.randperm(P * page, generator=g)
    c = to_gpu(cache)
    lat, rot = ext.kv_read_fp8blk(slots.to(DEV), c["c_kv"], c["pe"], c["scales"], DT[dt])
    for got, rows in zip((lat, rot), K.decode(cache)):
        assert got.dtype == DT[dt]
        want = rows[slots].to(DT[dt])
        got = got.cpu()
        nan = torch.isnan(want)
        assert torch.equal(torch.isnan(got), nan)
        assert torch.equal(got[~nan], want[~nan])


@pytest.mark.parametrize("n", [0, 1, 2, 3, 4, 5, 17, 64, 1001])
def test_read_slots(ext, n):
    """Any number of slots, some outside the pool (rows of zeros), the same one twice; the views of
    the types torch has for codes and scales; a two-dimensional index."""
    g = torch.Generator().manual_seed(n)
    P, page = 7, 64
    cache = K.new_pool(P, page, 32, g)
    slots = torch.randint(-3, P * page + 3, (n,), generator=g)
    if n > 4:
        slots[0], slots[1], slots[2], slots[3] = slots[4], -2 ** 62, 2 ** 62, P * page
    c = to_gpu(cache)
    lat, rot = ext.kv_read_fp8blk(slots.to(DEV), c["c_kv"].view(torch.float8_e4m3fn),
                                  c["pe"].view(torch.float8_e4m3fn), c["scales"].view(torch.float8_e8m0fnu), F32)
    in_pool = ((slots >= 0) & (slots < P * page))[:, None]
    for got, rows in zip((lat, rot), K.decode(cache)):
        assert torch.equal(got.cpu().double(), torch.where(in_pool, rows[slots.clamp(0, P * page - 1)], 0.0))
    if n == 64:
        two_d, _ = ext.kv_read_fp8blk(slots.view(4, 16).to(DEV), c["c_kv"], c["pe"], c["scales"], F32)
        assert two_d.shape == (4, 16, 512) and torch.equal(two_d.view(64, 512), lat)


# ------------------------------------------------------------------ attention

def check_attention(out, ref, dt, few=False):
    assert out.dtype == dt and torch.isfinite(out.float()).all()
    u = torch.finfo(dt).eps / 2
    for b in range(out.size(0)):
        r = ref[b]
        off = (out[b].double() - r).norm()
        assert off <= (3 if few else math.sqrt(3)) * u * r.norm(), (b, float(off / r.norm()), u)
    torch.testing.assert_close(out.float(), ref.float(), **C.tol(dt, ref.float()))


def attention_case(lens, Sq, block, page, dt, seed, H=128, V=128, spare=3, spread=0.5):
    g = torch.Generator().manual_seed(seed)
    P = sum(-(-max(0, n) // page) for n in lens) + spare
    table = K.tables(lens, page, P, g)
    cache = K.new_pool(P, page, block, g, spread)
    K.poison(cache, table, lens, page, block)
    return (*K.queries(len(lens), Sq, H, V, g, dt), cache, table)


def attend(ext, qa, qr, w, cache, table, lens, causal):
    c = to_gpu(cache)
    return ext.mla_attention_paged_fp8blk(qa.to(DEV), qr.to(DEV), c["c_kv"], c["pe"], c["scales"],
                                          table.to(DEV), i32(lens).to(DEV), w.to(DEV), SCALE, causal).cpu()


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("block", [16, 32, 64])
@pytest.mark.parametrize("page,Sq,lens,causal", [
    (64, 1, [1, 15, 16, 17, 31, 32, 33], False),
    (64, 1, [0, 63, 64, 65, 700, 0, 2000], False),
    (128, 4, [4, 20, 129, 700], True),
    (192, 1, [577, 192, 193], False),
    (64, 33, [33, 100, 50], True),
    (64, 3, [300, 65], False),
])
def test_attention(ext, dt, block, page, Sq, lens, causal):
    """Rows without a key hold NaN codes and NaN scales, table entries past a sequence no page."""
    qa, qr, w, cache, table = attention_case(lens, Sq, block, page, DT[dt], sum(lens) + block)
    out = attend(ext, qa, qr, w, cache, table, lens, causal)
    rows = [torch.nan_to_num(r) for r in K.decode(cache)]
    ref = K.attention(qa, qr, rows, table, lens, w, SCALE, causal, page, cache["c_kv"].size(0))
    few = min([n for n in lens if n], default=0) < 64
    check_attention(out, ref, DT[dt], few)
    for b, n in enumerate(lens):
        if n == 0:
            assert not out[b].any()


@pytest.mark.parametrize("dt", ["bf16", "f16"])
def test_attention_fewer_keys_than_queries(ext, dt):
    """Causal queries in front of a sequence's first token see nothing: rows of zeros."""
    lens, Sq = [2, 7, 0, 8, 5], 8
    qa, qr, w, cache, table = attention_case(lens, Sq, 16, 64, DT[dt], 6)
    out = attend(ext, qa, qr, w, cache, table, lens, True)
    rows = [torch.nan_to_num(r) for r in K.decode(cache)]
    ref = K.attention(qa, qr, rows, table, lens, w, SCALE, True, 64, cache["c_kv"].size(0))
    for b, n in enumerate(lens):
        assert not out[b, :Sq - n].any()
        if n:
            check_attention(out[b:b + 1, Sq - n:], ref[b:b + 1, Sq - n:], DT[dt], True)


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("Sq,H,lens,at", [(4, 128, [300, 33, 4], 2), (4, 16, [64, 700, 4], 1), (40, 3, [40, 100, 2000], 17),
                                          (33, 128, [500, 33, 64], 32), (7, 200, [90, 7, 4000], 0),
                                          (50, 3, [50, 100, 9000], 17), (64, 16, [900, 64, 2000], 63)])
def test_attention_hidden_nan(ext, monkeypatch, dt, Sq, H, lens, at):
    """A NaN in a token's row (latent, or rope alone): the queries in front of it keep their bits, it
    and the ones behind it are NaN."""
    qa, qr, w, cache, table = attention_case(lens, Sq, 32, 64, DT[dt], Sq, H=H)
    for fused in ("0", "1"):
        monkeypatch.setenv("MLA_OUT_SMALL", fused)
        clean = attend(ext, qa, qr, w, cache, table, lens, True)
        for name, column in (("c_kv", 77), ("c_kv", 500), ("pe", 9)):
            bad = {k: v.clone() for k, v in cache.items()}
            for b, n in enumerate(lens):
                slot = int(K.slots_of(table, b, n - Sq + at, n - Sq + at + 1, 64)[0])
                bad[name].view(-1, bad[name].size(2))[slot, column] = 0xFF if b else 0x7F
            out = attend(ext, qa, qr, w, bad, table, lens, True)
            assert torch.equal(out[:, :at], clean[:, :at])
            assert torch.isnan(out[:, at:]).all()


@pytest.mark.parametrize("H,V", [(1, 4), (3, 128), (16, 64), (65, 132), (200, 128)])
def test_attention_heads(ext, H, V):
    lens = [100, 300, 9]
    qa, qr, w, cache, table = attention_case(lens, 2, 32, 64, BF, H, H=H, V=V)
    out = attend(ext, qa, qr, w, cache, table, lens, True)
    rows = [torch.nan_to_num(r) for r in K.decode(cache)]
    check_attention(out, K.attention(qa, qr, rows, table, lens, w, SCALE, True, 64, cache["c_kv"].size(0)), BF, True)


@pytest.mark.parametrize("B,Sk", [(1, 4989), (40, 1500), (300, 90)])
def test_attention_balanced_list(ext, B, Sk):
    """One sequence cut into many chunks; ragged batches; more sequences than CUs."""
    g = torch.Generator().manual_seed(B)
    lens = [Sk] + torch.randint(0, Sk + 1, (B - 1,), generator=g).tolist()
    qa, qr, w, cache, table = attention_case(lens, 1, 16, 64, BF, B + 5)
    out = attend(ext, qa, qr, w, cache, table, lens, False)
    rows = [torch.nan_to_num(r) for r in K.decode(cache)]
    ref = K.attention(qa, qr, rows, table, lens, w, SCALE, False, 64, cache["c_kv"].size(0))
    check_attention(out, ref, BF, True)


@pytest.mark.parametrize("dt", ["bf16", "f16"])
def test_attention_scales_far_apart(ext, dt):
    """Blocks whose scales lie up to 2^12 apart, small ones first: scores climb from block to block
    (a row then raises its reference and repeats the pass), the two parts' scales unlike."""
    lens, block, page = [400, 130], 16, 64
    qa, qr, w, cache, table = attention_case(lens, 1, block, page, DT[dt], 12)
    for b, n in enumerate(lens):
        for i, lo in enumerate(range(0, n, block)):
            blk = (int(table[b, lo // page]) * page + lo % page) // block
            up = min(i, 8) - 4
            cache["scales"].view(-1, 2)[blk] = torch.tensor([118 + up, 119 - (i % 3) + up], dtype=torch.uint8)
    out = attend(ext, qa, qr, w, cache, table, lens, False)
    rows = [torch.nan_to_num(r) for r in K.decode(cache)]
    ref = K.attention(qa, qr, rows, table, lens, w, SCALE, False, page, cache["c_kv"].size(0))
    check_attention(out, ref, DT[dt], True)


def test_attention_equals_one_scale(ext, monkeypatch):
    """Every scale the same power of two: bit for bit what mla_attention_paged_fp8kv gives, whose
    one scale it is (a power of two moves no rounding), with the merge and 3d as launches of their own
    as that call has them."""
    monkeypatch.setenv("MLA_OUT_SMALL", "0")
    lens = [700, 64, 1, 333]
    qa, qr, w, cache, table = attention_case(lens, 1, 32, 64, BF, 21, spread=0.0)
    table = table.clamp(min=0)
    for e in (-6, 0, 3):
        cache["scales"].fill_(127 + e)
        c = to_gpu(cache)
        args = [t.to(DEV) for t in (qa * 2.0 ** -max(e + 8, 0), qr * 2.0 ** -max(e + 8, 0))]
        a = ext.mla_attention_paged_fp8blk(*args, c["c_kv"], c["pe"], c["scales"], table.to(DEV),
                                           i32(lens).to(DEV), w.to(DEV), SCALE)
        b = ext.mla_attention_paged_fp8kv(*args, c["c_kv"], c["pe"], table.to(DEV), i32(lens).to(DEV),
                                          2.0 ** e, w.to(DEV), SCALE)
        assert torch.equal(a, b) and torch.isfinite(a.float()).all()


@pytest.mark.parametrize("B,Sq,H,Sk,page", [(1, 130, 128, 9000, 64), (2, 128, 64, 6000, 192), (300, 1, 64, 4500, 64)])
def test_attention_long_walks(ext, monkeypatch, B, Sq, H, Sk, page):
    """Workgroups that walk over more pages than a register holds entries of (64), from anywhere in the
    table: again the bits of mla_attention_paged_fp8kv."""
    monkeypatch.setenv("MLA_OUT_SMALL", "0")
    g = torch.Generator().manual_seed(Sk)
    P = 160
    cache = to_gpu(K.new_pool(P, page, 64, g, 0.0))
    cache["scales"].fill_(119)
    table = torch.randint(0, P, (B, -(-Sk // page)), generator=g).int().to(DEV)
    lens = torch.randint(Sk // 2, Sk + 1, (B,), generator=g)
    lens[0] = Sk
    qa, qr, w = (t.to(DEV) for t in K.queries(B, Sq, H, 128, g, BF))
    a = ext.mla_attention_paged_fp8blk(qa, qr, cache["c_kv"], cache["pe"], cache["scales"], table,
                                       lens.int().to(DEV), w, SCALE, Sq > 1)
    b = ext.mla_attention_paged_fp8kv(qa, qr, cache["c_kv"], cache["pe"], table, lens.int().to(DEV), 2.0 ** -8, w,
                                      SCALE, Sq > 1)
    assert torch.equal(a, b) and torch.isfinite(a.float()).all()


def test_attention_pages_outside_the_pool(ext):
    """A table entry that is no page, among a sequence's keys: rows of zeros, no access."""
    lens = [200, 130]
    qa, qr, w, cache, table = attention_case(lens, 1, 64, 64, BF, 14)
    table[0, 1], table[1, 0], table[1, 2] = -1, cache["c_kv"].size(0), 2 ** 31 - 1
    out = attend(ext, qa, qr, w, cache, table, lens, False)
    rows = [torch.nan_to_num(r) for r in K.decode(cache)]
    ref = K.attention(qa, qr, rows, table, lens, w, SCALE, False, 64, cache["c_kv"].size(0))
    check_attention(out, ref, BF, True)


def test_attention_shared_and_far_pages(ext):
    """Two sequences with one prefix, in a pool whose pages lie past 4 GB (row offsets, and the read's
    and the append's, in 64 bits)."""
    page, block, P = 64, 16, 140_000            # 8.96M rows: 4.6 GB of latent codes
    lens = [200, 170]
    g = torch.Generator().manual_seed(3)
    small = K.new_pool(6, page, block, g)
    qa, qr, w = K.queries(2, 1, 128, 128, g, BF)
    far = [P - 1, P - 7, 131_073, 139_000, 5, P - 2]
    table = torch.tensor([[0, 1, 2, 3], [0, 1, 4, 5]], dtype=torch.int32)
    far_table = i32(far)[table.long()].int()
    c = {"c_kv": torch.empty(P, page, K.KV, dtype=torch.uint8, device=DEV),
         "pe": torch.empty(P, page, K.ROPE, dtype=torch.uint8, device=DEV),
         "scales": torch.empty(P, page // block, 2, dtype=torch.uint8, device=DEV)}
    for k in c:
        c[k][torch.tensor(far, device=DEV)] = small[k].to(DEV)
    a = [t.to(DEV) for t in (qa, qr)]
    out = ext.mla_attention_paged_fp8blk(*a, c["c_kv"], c["pe"], c["scales"], far_table.to(DEV),
                                         i32(lens).to(DEV), w.to(DEV), SCALE).cpu()
    check_attention(out, K.attention(qa, qr, K.decode(small), table, lens, w, SCALE, False, page, 6), BF)
    slots = (torch.tensor(far)[:, None] * page + torch.arange(page)).flatten()
    lat, rot = ext.kv_read_fp8blk(slots.to(DEV), c["c_kv"], c["pe"], c["scales"], F32)
    assert torch.equal(lat.cpu().double(), K.decode(small)[0]) and torch.equal(rot.cpu().double(), K.decode(small)[1])
    # the append into the last, unshared pages
    lens, new = [201, 171], [1, 1]
    x = torch.randn(2, 1, 256, generator=g).to(BF)
    W = (torch.randn(256, 576, generator=g) / 16).to(BF)
    gain = torch.ones(512).to(BF)
    ext.kv_append_paged_fp8blk(x.to(DEV), W.to(DEV), gain.to(DEV), i32(lens).to(DEV), i32(new).to(DEV),
                               far_table.to(DEV), c["c_kv"], c["pe"], c["scales"], 1e-6)
    after = {k: c[k][torch.tensor(far, device=DEV)].cpu() for k in c}
    check_append(small, after, K.append(small, x, W, gain, lens, new, table, page, block), block)


def test_attention_strided_inputs_and_streams(ext):
    """Queries, tables and pools as strided views; a call on another stream than the current one's
    tensors were made on; the same bits each time."""
    lens = [300, 77]
    qa, qr, w, cache, table = attention_case(lens, 2, 32, 64, BF, 33)
    base = attend(ext, qa, qr, w, cache, table, lens, True)
    c = to_gpu(cache)
    view = lambda t: t.to(DEV).transpose(1, 2).contiguous().transpose(1, 2)  # noqa: E731
    wide = torch.zeros(2, 2 * table.size(1), dtype=torch.int32, device=DEV)
    wide[:, ::2] = table.to(DEV)
    pool = torch.zeros(c["c_kv"].size(0), 64, 600, dtype=torch.uint8, device=DEV)
    pool[..., 40:552] = c["c_kv"]
    out = ext.mla_attention_paged_fp8blk(view(qa), view(qr), pool[..., 40:552], c["pe"], c["scales"],
                                         wide[:, ::2], i32(lens).to(DEV), view(w), SCALE, True)
    assert torch.equal(out.cpu(), base)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        out2 = ext.mla_attention_paged_fp8blk(view(qa), view(qr), c["c_kv"], c["pe"], c["scales"],
                                              wide[:, ::2], i32(lens).to(DEV), view(w), SCALE, True)
    s.synchronize()
    assert torch.equal(out2.cpu(), base)


# ------------------------------------------------------------------ together

def serving_state(dt, B=5, Sq=4, hidden=256, page=64, block=16, mp=4, P=14, seed=40):
    g = torch.Generator().manual_seed(seed)
    W = (torch.randn(hidden, 576, generator=g) / math.sqrt(hidden)).to(dt)
    gain = (1 + 0.1 * torch.randn(512, generator=g)).to(dt)
    cache = {"c_kv": torch.full((P, page, 512), 0x7F, dtype=torch.uint8),
             "pe": torch.full((P, page, 64), 0x7F, dtype=torch.uint8),
             "scales": torch.full((P, page // block, 2), 255, dtype=torch.uint8)}
    return g, W, gain, cache


def serve(ext, st, new, x, qa, qr, w, Sq, page, scale=SCALE):
    """One step of a server: bookkeeping, write, attention, and the new rows read back."""
    lens, state, granted, pos, slots = ext.cache_extend(new, st["lens"], st["table"], st["ring"], st["state"],
                                                        Sq, page)
    ext.kv_append_paged_fp8blk(x, st["W"], st["gain"], lens, granted, st["table"], st["c_kv"], st["pe"],
                               st["scales"], 1e-6)
    out = ext.mla_attention_paged_fp8blk(qa, qr, st["c_kv"], st["pe"], st["scales"], st["table"], lens, w,
                                         scale, True)
    lat, rot = ext.kv_read_fp8blk(slots, st["c_kv"], st["pe"], st["scales"], F32)
    return lens, state, granted, out, lat, rot, slots


@pytest.mark.parametrize("dt", ["bf16", "f16"])
def test_serving_steps(ext, dt):
    """Twelve steps: prompts, drafts, rejections, a request that ends and one that cannot get a page;
    every step's tables, cache and attention against the plain forms."""
    B, Sq, page, block, mp, P = 5, 4, 64, 16, 4, 9
    g, W, gain, cache = serving_state(DT[dt], P=P)
    lens, state = [0] * B, [3, P]
    table = torch.full((B, mp), -1, dtype=torch.int32)
    ring = torch.randperm(P, generator=g).int()
    st = {"lens": i32(lens).to(DEV), "state": i32(state).to(DEV), "table": table.to(DEV), "ring": ring.to(DEV),
          "W": W.to(DEV), "gain": gain.to(DEV), **to_gpu(cache)}
    plan = [[100, 30, 64, 1, 0], [4, 4, 4, 4, 90], [-2, 0, -3, 4, 1], [4, 4, 4, 4, 4], [-100, -1, 0, 0, 0],
            [4, 1, 2, 3, 4], [120, 0, 0, 0, 0], [1, 1, 1, 1, 1], [K.INT_MIN, 100, 60, 0, 1], [4, 4, 4, 4, 4],
            [60, 100, 4, 3, 2], [1, 1, 1, 1, 1]]
    for new in plan:
        sq = max(Sq, max(new))
        x = torch.randn(B, sq, 256, generator=g).to(DT[dt])
        qa, qr, w = K.queries(B, sq, 128, 128, g, DT[dt])
        want = K.extend(new, lens, table, ring, state, sq, page)
        dest = K.append(cache, x, W, gain, want["seq_lens"], want["granted"], want["table"], page, block)
        got_lens, got_state, granted, out, lat, rot, slots = serve(
            ext, st, i32(new).to(DEV), x.to(DEV), qa.to(DEV), qr.to(DEV), w.to(DEV), sq, page)
        st["lens"], st["state"] = got_lens, got_state
        lens, state, table, ring = want["seq_lens"], want["state"], want["table"], want["ring"]
        assert got_lens.tolist() == lens and got_state.tolist() == state
        assert granted.tolist() == want["granted"] and torch.equal(slots.cpu(), want["slots"])
        assert torch.equal(st["table"].cpu(), table) and torch.equal(st["ring"].cpu(), ring)
        after = {k: st[k].cpu() for k in cache}
        check_append(cache, after, dest, block)
        cache = after
        rows = [torch.nan_to_num(r) for r in K.decode(cache)]
        there = (want["slots"] >= 0)[..., None]
        assert torch.equal(lat.cpu().double(), torch.where(there, rows[0][want["slots"].clamp(min=0)], 0.0))
        assert torch.equal(rot.cpu().double(), torch.where(there, rows[1][want["slots"].clamp(min=0)], 0.0))
        ref = K.attention(qa, qr, rows, table, lens, w, SCALE, True, page, P)
        for b in range(B):
            n = min(sq, lens[b])   # queries in front of the first token give zeros
            assert not out[b, :sq - n].any()
            if n:
                check_attention(out[b:b + 1, sq - n:].cpu(), ref[b:b + 1, sq - n:], DT[dt], True)


def test_serving_step_in_a_graph(ext):
    """A whole step captured, its lengths and free state fed back inside the graph: every replay adds
    a token to each sequence, and equals the eager step on a copy of the state, bit for bit, with
    eager work and synchronisations between the replays."""
    B, Sq, page, P = 5, 2, 64, 24
    g, W, gain, cache = serving_state(BF, P=P)
    def fresh():
        return {"lens": i32([63, 10, 0, 126, 30]).to(DEV), "state": i32([20, 14]).to(DEV),
                "table": i32([[0, -1, -1, -1], [1, -1, -1, -1], [-1] * 4, [2, 3, -1, -1], [4, -1, -1, -1]]).to(DEV),
                "ring": ((torch.arange(P, dtype=torch.int32) + 9) % P).to(DEV), "W": W.to(DEV),
                "gain": gain.to(DEV), **to_gpu(cache)}
    a, b = fresh(), fresh()
    for st in (a, b):   # the tokens that the sequences start with
        x = torch.randn(B, 126, 256, generator=torch.Generator().manual_seed(1)).to(BF).to(DEV)
        ext.kv_append_paged_fp8blk(x, st["W"], st["gain"], st["lens"], st["lens"], st["table"], st["c_kv"],
                                   st["pe"], st["scales"], 1e-6)
    new = i32([2, 1, 2, 2, 0]).to(DEV)
    x = torch.randn(B, Sq, 256, generator=g).to(BF).to(DEV)
    qa, qr, w = (t.to(DEV) for t in K.queries(B, Sq, 128, 128, g, BF))

    def step(st):
        out = serve(ext, st, new, x, qa, qr, w, Sq, page)
        st["lens"].copy_(out[0])
        st["state"].copy_(out[1])
        return out

    warm = fresh()
    step(warm)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(a)
    for i in range(6):
        x.copy_(torch.randn(B, Sq, 256, generator=g).to(BF))
        graph.replay()
        eager = step(b)
        torch.cuda.synchronize()
        for got, want in zip(outs, eager):
            assert torch.equal(got, want), i
        for k in ("table", "ring", "c_kv", "pe", "scales", "lens", "state"):
            assert torch.equal(a[k], b[k]), (i, k)
        step(warm)


@pytest.mark.parametrize("B,Sq,Sk", [(1, 1, 5000), (2, 1, 63), (7, 1, 4989), (16, 4, 1500), (33, 1, 3000),
                                     (64, 1, 900), (64, 2, 130), (3, 20, 700), (1, 70, 70)])
def test_attention_list_without_a_launch(ext, monkeypatch, B, Sq, Sk):
    """Up to 64 sequences the workgroups work the list out themselves: the same bits as from the
    list that is built in a launch of its own, for ragged, equal, empty and unlike lengths."""
    g = torch.Generator().manual_seed(B + Sk)
    page, block = 64, 32
    cache = to_gpu(K.new_pool(300, page, block, g))
    mp = -(-Sk // page)
    table = torch.randint(0, 300, (B, mp), generator=g).int().to(DEV)   # (read only: pages may be shared)
    qa, qr, w = (t.to(DEV) for t in K.queries(B, Sq, 128, 128, g, BF))
    some = torch.randint(0, Sk + 1, (B,), generator=g)
    long = torch.where(torch.arange(B) == B // 2, Sk, torch.ones(B, dtype=torch.long))
    for lens in (some, torch.full((B,), Sk), torch.full((B,), Sk // 3), torch.zeros(B, dtype=torch.long), long,
                 torch.where(torch.arange(B) % 2 == 0, torch.full((B,), Sk), torch.zeros(B, dtype=torch.long)),
                 some - Sk // 2, some + Sk):
        outs = []
        for env in ("0", "1"):
            monkeypatch.setenv("MLA_SMALL_LIST", env)
            outs.append(ext.mla_attention_paged_fp8blk(qa, qr, cache["c_kv"], cache["pe"], cache["scales"], table,
                                                       lens.int().to(DEV), w, SCALE, Sq > 1))
        assert torch.equal(outs[0], outs[1])


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("B,Sq,H,V", [(1, 1, 128, 128), (2, 1, 128, 128), (4, 2, 128, 128), (1, 8, 128, 128),
                                      (8, 1, 128, 128), (3, 1, 1, 4), (5, 1, 16, 100), (7, 1, 33, 256)])
def test_attention_few_tokens(ext, monkeypatch, dt, B, Sq, H, V):
    """Up to eight tokens the merge of the chunks runs inside 3d: chunked, whole and empty sequences
    against the plain form, and close to the two launches of their own (MLA_OUT_SMALL=0)."""
    g = torch.Generator().manual_seed(B * 10 + Sq)
    lens = [3000] + torch.randint(0, 700, (B - 1,), generator=g).tolist()
    if B > 3:
        lens[2], lens[3] = 0, 20
    qa, qr, w, cache, table = attention_case(lens, Sq, 32, 64, DT[dt], B, H=H, V=V)
    rows = [torch.nan_to_num(r) for r in K.decode(cache)]
    ref = K.attention(qa, qr, rows, table, lens, w, SCALE, Sq > 1, 64, cache["c_kv"].size(0))
    out = attend(ext, qa, qr, w, cache, table, lens, Sq > 1)
    check_attention(out, ref, DT[dt], True)
    monkeypatch.setenv("MLA_OUT_SMALL", "0")
    two = attend(ext, qa, qr, w, cache, table, lens, Sq > 1)
    check_attention(two, ref, DT[dt], True)


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("B,Sq,H,V,Sk", [(9, 1, 4, 128, 20000), (13, 1, 128, 128, 2000), (17, 2, 128, 132, 700),
                                         (64, 2, 16, 64, 300), (11, 9, 3, 260, 900), (128, 1, 128, 128, 400),
                                         (129, 1, 128, 128, 200)])
def test_attention_decode_batches(ext, monkeypatch, dt, B, Sq, H, V, Sk):
    """9 to 128 tokens: the chunks' merge runs inside 3d, a tile of tokens at a time (past 64 chunks a
    sequence, odd tiles, columns past a block of 128), and one token past it."""
    g = torch.Generator().manual_seed(B * 10 + Sq)
    lens = [Sk] + torch.randint(0, min(Sk, 700), (B - 1,), generator=g).tolist()
    lens[B // 2] = 0
    qa, qr, w, cache, table = attention_case(lens, Sq, 64, 64, DT[dt], B, H=H, V=V)
    rows = [torch.nan_to_num(r) for r in K.decode(cache)]
    ref = K.attention(qa, qr, rows, table, lens, w, SCALE, Sq > 1, 64, cache["c_kv"].size(0))
    check_attention(attend(ext, qa, qr, w, cache, table, lens, Sq > 1), ref, DT[dt], True)
    monkeypatch.setenv("MLA_OUT_SMALL", "0")
    check_attention(attend(ext, qa, qr, w, cache, table, lens, Sq > 1), ref, DT[dt], True)


@pytest.mark.parametrize("layer", [1, 2])
def test_one_layer_of_layered_pools(ext, layer):
    """Pools of several layers in one tensor: a layer's scale bytes start at any even address (here 6
    and 12 bytes in).  The same bits as pools of its own, and the other layers' bytes stay."""
    lens, new, block, page = [100, 30], [70, 30], 64, 64
    cache, x, W, gain, table = append_inputs(lens, new, 70, block, page, BF, 5, spare=0)
    assert cache["scales"].numel() == 6
    alone = to_gpu(cache)
    stacked = {k: v.unsqueeze(0).repeat(3, *[1] * v.dim()).to(DEV) for k, v in cache.items()}
    before = {k: v.cpu() for k, v in stacked.items()}
    one = {k: v[layer] for k, v in stacked.items()}
    qa, qr, w = (t.to(DEV) for t in K.queries(2, 1, 128, 128, torch.Generator().manual_seed(5), BF))
    args = [t.to(DEV) for t in (x, W, gain, i32(lens), i32(new), table)]
    outs = []
    for c in (alone, one):
        ext.kv_append_paged_fp8blk(*args, c["c_kv"], c["pe"], c["scales"], 1e-6)
        outs.append([ext.mla_attention_paged_fp8blk(qa, qr, c["c_kv"], c["pe"], c["scales"], args[5], args[3], w,
                                                    SCALE, False),
                     *ext.kv_read_fp8blk(torch.arange(3 * page, device=DEV), c["c_kv"], c["pe"], c["scales"], BF)])
    for got, want in zip(outs[1], outs[0]):
        assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(want))
    for k, v in stacked.items():
        assert torch.equal(v[layer], alone[k])
        for other in {0, 1, 2} - {layer}:
            assert torch.equal(v[other].cpu(), before[k][other])


@pytest.mark.parametrize("dt", ["bf16", "f16"])
def test_attention_unrounded_rows_past_128_tokens(ext, monkeypatch, dt):
    """With MLA_OUT_SMALL=0 the large-tile GEMM is 3d, of rows in 16 bits or (MLA_CTX16=0) in float32."""
    g = torch.Generator().manual_seed(129)
    lens = torch.randint(0, 400, (43,), generator=g).tolist()
    lens[0], lens[1] = 3000, 0
    qa, qr, w, cache, table = attention_case(lens, 4, 32, 64, DT[dt], 129)
    rows = [torch.nan_to_num(r) for r in K.decode(cache)]
    ref = K.attention(qa, qr, rows, table, lens, w, SCALE, True, 64, cache["c_kv"].size(0))
    monkeypatch.setenv("MLA_OUT_SMALL", "0")
    check_attention(attend(ext, qa, qr, w, cache, table, lens, True), ref, DT[dt], True)
    monkeypatch.setenv("MLA_CTX16", "0")
    check_attention(attend(ext, qa, qr, w, cache, table, lens, True), ref, DT[dt], True)


def test_steps_on_two_streams(ext):
    """Two servers with pools of their own, a step each at once on two streams: the bits of one after
    the other."""
    B, Sq, page = 5, 4, 64
    cases = []
    for seed, new in ((40, [4, 3, 0, 4, 1]), (41, [1, 4, 4, 2, 3])):
        g, W, gain, cache = serving_state(BF, seed=seed)
        x = torch.randn(B, Sq, 256, generator=g).to(BF).to(DEV)
        cases.append((W.to(DEV), gain.to(DEV), cache, x, [t.to(DEV) for t in K.queries(B, Sq, 128, 128, g, BF)],
                      i32(new).to(DEV)))

    def state(case):
        return {"W": case[0], "gain": case[1], **to_gpu(case[2]), "lens": i32([0] * B).to(DEV),
                "state": i32([3, 14]).to(DEV), "table": torch.full((B, 4), -1, dtype=torch.int32, device=DEV),
                "ring": torch.arange(14, dtype=torch.int32, device=DEV)}

    def steps(case, st):
        outs = []
        for _ in range(6):
            out = serve(ext, st, case[5], case[3], *case[4], Sq, page)
            st["lens"], st["state"] = out[0], out[1]
            outs.append(out)
        return outs

    want = [steps(c, state(c)) for c in cases]
    states = [state(c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[], []]
    for i, s in enumerate(streams):
        with torch.cuda.stream(s):
            got[i] = steps(cases[i], states[i])
    torch.cuda.synchronize()
    for w, o in zip(want, got):
        for a, b in zip(w, o):
            for x, y in zip(a, b):
                assert torch.equal(torch.nan_to_num(x), torch.nan_to_num(y))


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("B,Sq,H,V,lens", [
    (1, 129, 1, 4, [129]), (3, 100, 3, 132, [100, 1000, 101]), (130, 1, 5, 260, None), (2, 300, 16, 64, [7000, 300]),
    (1, 1000, 2, 128, [1500]), (43, 4, 65, 128, None), (300, 1, 128, 128, None)])
def test_attention_many_tokens(ext, dt, B, Sq, H, V, lens):
    """Past 128 tokens the rows go to 3d packed: tiles of tokens that are not full, columns past a block of
    128, sequences in one chunk and in several, empty ones."""
    g = torch.Generator().manual_seed(B + Sq)
    if lens is None:
        lens = torch.randint(0, 300, (B,), generator=g).tolist()
        lens[0], lens[1] = 2000, 0
    qa, qr, w, cache, table = attention_case(lens, Sq, 32, 64, DT[dt], B, H=H, V=V)
    rows = [torch.nan_to_num(r) for r in K.decode(cache)]
    ref = K.attention(qa, qr, rows, table, lens, w, SCALE, True, 64, cache["c_kv"].size(0))
    check_attention(attend(ext, qa, qr, w, cache, table, lens, True), ref, DT[dt], True)


@pytest.mark.parametrize("up,w_up", [(60, 50), (-60, -40), (100, -90)])
@pytest.mark.parametrize("Sq", [1, 70])
def test_attention_powers_of_two(ext, up, w_up, Sq):
    """Values times 2^up (the queries the less) and each output column's W_uv times a power of two of its
    own: the outputs' bits but for the exponent, few tokens or many.  (bf16, whose range holds all of
    them as normal numbers.)"""
    lens = [70, 300, 1200]
    g = torch.Generator().manual_seed(Sq)
    qa, qr, w, cache, table = attention_case(lens, Sq, 32, 64, BF, 3, H=16)
    cache["pe"].zero_()
    base = attend(ext, qa, qr, w, cache, table, lens, True)
    moved = {**cache, "scales": cache["scales"].clone()}
    held = moved["scales"][..., 0] != 255
    moved["scales"][..., 0][held] = (moved["scales"][..., 0][held].int() + up).to(torch.uint8)
    e = torch.randint(min(0, w_up), max(0, w_up) + 1, (16, 128), generator=g).double()
    out = attend(ext, (qa.double() * 2.0 ** -up).to(BF), qr, (w.double() * 2.0 ** e[..., None]).to(BF), moved, table,
                 lens, True)
    assert torch.equal(out.double(), base.double() * 2.0 ** (up + e))


@pytest.mark.parametrize("B,Sq,H,Sk", [(1, 1, 128, 3000), (2, 1, 16, 700), (1, 70, 20, 900), (40, 4, 128, 300),
                                       (1, 3, 3, 65), (130, 2, 128, 200)])
@pytest.mark.parametrize("kind", ["ramp", "steps", "late", "halves"])
def test_attention_scores_that_climb(ext, kind, B, Sq, H, Sk):
    """fp16, whose P ends at 2^16: scores that climb past a row's first reference by hundreds of powers of
    two, again and again, in one key half or the other, for some rows more than for others; few tokens and
    many, in one chunk and in several."""
    page, block = 64, 32
    g = torch.Generator().manual_seed(B + Sk)
    P = B * -(-Sk // page) + 2
    table = K.tables([Sk] * B, page, P, g)
    cache = K.new_pool(P, page, block, g, 0.0)
    key = torch.arange(Sk)
    level = {"ramp": key / Sk * 100, "steps": (key // 150) * 30.0, "late": (key >= Sk - 3) * 200.0,
             "halves": ((key // 16) % 2) * (key // 40) * 9.0}[kind]          # powers of two
    # a column of the rope key carries the level: q_r[0] = 1 (or less, by row) against it
    lev = (level.double() * math.log(2) * SCALE).round()
    e = max(0, math.ceil(math.log2(max(1.0, float(lev.max())) / 448)))
    for b in range(B):
        slots = K.slots_of(table, b, 0, Sk, page)
        pe = cache["pe"].view(-1, 64)
        pe[slots] = 0
        pe[slots, 0] = (lev / 2.0 ** e).float().to(torch.float8_e4m3fn).view(torch.uint8)
    cache["scales"][..., 1] = 127 + e
    qa, qr, w = K.queries(B, Sq, H, 128, g, H16)
    qr.zero_()
    qr[..., 0] = 1.0 - (torch.arange(H) % 3) * 0.25
    lens = [Sk] * B
    rows = [torch.nan_to_num(r) for r in K.decode(cache)]
    ref = K.attention(qa, qr, rows, table, lens, w, SCALE, Sq > 1, page, P)
    check_attention(attend(ext, qa, qr, w, cache, table, lens, Sq > 1), ref, H16, True)
