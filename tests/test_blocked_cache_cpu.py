"""CPU checks of the paged 8-bit cache with block scales: the C ABI's and the binding's refusals
(all made before the first HIP call), the plain forms that the GPU tests compare with, and that
those tests' tolerances tell plausible mistakes from the real thing on their own inputs."""

from __future__ import annotations

import ctypes
import math
import os

import pytest
import torch

import attn_cases as C
import blocked_cache as K
from oracle import mla_ref as R

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
OK, INVALID, UNSUPPORTED, WORKSPACE, HIP = range(5)
F32, BF16, F16, F64 = range(4)
P16 = ctypes.c_void_p(1 << 20)          # aligned, never dereferenced
ODD = ctypes.c_void_p((1 << 20) + 4)
BYTE = ctypes.c_void_p((1 << 20) + 1)
BIG = ctypes.c_size_t(1 << 40)


class Dims(ctypes.Structure):
    _fields_ = [(n, ctypes.c_int32) for n in
                ("batch", "sq", "sk", "hidden", "q_lora", "heads", "nope", "rope", "kv_rank", "v")]


def dims(**kw):
    d = dict(batch=2, sq=1, sk=256, hidden=256, q_lora=0, heads=128, nope=128, rope=64, kv_rank=512, v=128)
    return Dims(**{**d, **kw})


@pytest.fixture(scope="module")
def lib():
    import mla_custom_cuda  # noqa: F401
    L = ctypes.CDLL(os.path.join(ROOT, "mla-cuda_amd", "libmla_amd.so"))
    L.mla_last_error.restype = ctypes.c_char_p
    for n in ("mla_cache_extend_workspace_bytes", "mla_attention_paged_fp8blk_workspace_bytes",
              "mla_kv_append_workspace_bytes", "mla_attention_paged_fp8kv_workspace_bytes"):
        getattr(L, n).restype = ctypes.c_size_t
    return L


# ------------------------------------------------------------------ refusals of the C ABI

EXTEND = dict(batch=2, sq=1, page_size=64, max_pages=4, num_pages=8, new_lens=P16, seq_lens=P16, free_state=P16,
              block_table=P16, free_pages=P16, seq_lens_out=P16, free_state_out=P16, granted=P16, positions=P16,
              slots=P16, workspace=P16, workspace_bytes=BIG, stream=None)


@pytest.mark.parametrize("change,status,word", [
    (dict(batch=0), INVALID, "batch"), (dict(sq=-1), INVALID, "sq"), (dict(max_pages=0), INVALID, "max_pages"),
    (dict(num_pages=0), INVALID, "num_pages"), (dict(num_pages=(1 << 30) + 1), INVALID, "2^30"),
    (dict(page_size=32), INVALID, "page_size"), (dict(page_size=0), INVALID, "page_size"),
    (dict(batch=1 << 20, sq=1 << 11), INVALID, "2^30"), (dict(max_pages=1 << 26), INVALID, "2^31"),
    (dict(batch=1 << 20, max_pages=1 << 12), INVALID, "2^31"),
    *[({k: None}, INVALID, k) for k, v in EXTEND.items() if v is P16 and k != "workspace"],
    *[({k: ODD}, INVALID, k) for k, v in EXTEND.items() if v is P16 and k != "workspace"],
    (dict(batch=2000, workspace=None), WORKSPACE, "workspace"),
    (dict(sq=5000, workspace_bytes=ctypes.c_size_t(47)), WORKSPACE, "small"),
])
def test_extend_refuses(lib, change, status, word):
    assert lib.mla_cache_extend(*{**EXTEND, **change}.values()) == status
    assert word in lib.mla_last_error().decode()


APPEND = dict(dtype=BF16, dims=None, x=P16, W_kv_a=P16, kv_norm_w=P16, inv_freq=P16, eps=ctypes.c_double(1e-6),
              seq_lens=P16, new_lens=P16, block_table=P16, page_size=64, num_pages=8, scale_block=32,
              c_kv_pages=P16, pe_pages=P16, scales=P16, workspace=P16, workspace_bytes=BIG, stream=None)


@pytest.mark.parametrize("change,status,word", [
    (dict(dtype=F64), UNSUPPORTED, "float64"), (dict(dtype=9), INVALID, "dtype"),
    (dict(dims=dims(batch=0)), INVALID, "batch"), (dict(dims=dims(hidden=252)), INVALID, "hidden"),
    (dict(dims=dims(kv_rank=256)), UNSUPPORTED, "kv_rank 512"), (dict(dims=dims(rope=32)), UNSUPPORTED, "rope 64"),
    (dict(dims=dims(sk=100)), INVALID, "page_size"), (dict(page_size=16), INVALID, "page_size"),
    (dict(num_pages=0), INVALID, "num_pages"), (dict(scale_block=8), UNSUPPORTED, "scale_block"),
    (dict(scale_block=48), UNSUPPORTED, "scale_block"), (dict(scale_block=128), UNSUPPORTED, "scale_block"),
    (dict(eps=ctypes.c_double(-1.0)), INVALID, "eps"), (dict(eps=ctypes.c_double(math.nan)), INVALID, "eps"),
    *[({k: None}, INVALID, k) for k, v in APPEND.items() if v is P16 and k != "workspace"],
    (dict(c_kv_pages=ODD), INVALID, "aligned"), (dict(scales=BYTE), INVALID, "scales must be 2-byte aligned"),
    (dict(workspace_bytes=ctypes.c_size_t(16)), WORKSPACE, "small"),
])
def test_append_refuses(lib, change, status, word):
    a = {**APPEND, "dims": dims(), **change}
    a["dims"] = ctypes.byref(a["dims"])
    assert lib.mla_kv_append_paged_fp8blk(*a.values()) == status
    assert word in lib.mla_last_error().decode()


READ = dict(dtype=BF16, slots=P16, n=ctypes.c_int64(5), c_kv_pages=P16, pe_pages=P16, scales=P16, page_size=64,
            num_pages=8, scale_block=16, latent=P16, rope=P16, stream=None)


@pytest.mark.parametrize("change,status,word", [
    (dict(dtype=F64), UNSUPPORTED, "float64"), (dict(n=ctypes.c_int64(-1)), INVALID, "n must"),
    (dict(page_size=65), INVALID, "page_size"), (dict(num_pages=-2), INVALID, "num_pages"),
    (dict(scale_block=0), UNSUPPORTED, "scale_block"),
    *[({k: None}, INVALID, k) for k, v in READ.items() if v is P16],
    *[({k: ODD}, INVALID, k) for k, v in READ.items() if v is P16 and k != "scales"],
    (dict(scales=BYTE), INVALID, "scales must be 2-byte aligned"),
])
def test_read_refuses(lib, change, status, word):
    assert lib.mla_kv_read_fp8blk(*{**READ, **change}.values()) == status
    assert word in lib.mla_last_error().decode()


def test_read_of_nothing(lib):
    assert lib.mla_kv_read_fp8blk(*{**READ, "n": ctypes.c_int64(0), "slots": None, "latent": None}.values()) == OK


ATTEND = dict(dtype=BF16, dims=None, q_absorbed=P16, q_rope=P16, c_kv_pages=P16, pe_pages=P16, scales=P16,
              block_table=P16, seq_lens=P16, page_size=64, num_pages=8, scale_block=64, W_uv=P16,
              scale=ctypes.c_double(13.0), causal=0, out=P16, workspace=P16, workspace_bytes=BIG, stream=None)


@pytest.mark.parametrize("change,status,word", [
    (dict(dtype=F32), UNSUPPORTED, "bf16 or fp16"), (dict(dtype=F64), UNSUPPORTED, "bf16 or fp16"),
    (dict(dims=dims(heads=0)), INVALID, "heads"), (dict(dims=dims(v=6)), INVALID, "dims.v"),
    (dict(dims=dims(kv_rank=256)), UNSUPPORTED, "kv_rank 512"), (dict(dims=dims(rope=128)), UNSUPPORTED, "rope 64"),
    (dict(dims=dims(sk=96)), INVALID, "page_size"), (dict(dims=dims(sq=300), causal=1), INVALID, "sk >= sq"),
    (dict(dims=dims(batch=1, sq=1 << 14)), UNSUPPORTED, "2^31"),
    (dict(dims=dims(v=1 << 18)), UNSUPPORTED, "heads * v"),
    (dict(page_size=0), INVALID, "page_size"), (dict(num_pages=0), INVALID, "num_pages"),
    (dict(scale_block=1), UNSUPPORTED, "scale_block"), (dict(scale=ctypes.c_double(0.0)), INVALID, "scale"),
    *[({k: None}, INVALID, k) for k, v in ATTEND.items() if v is P16 and k != "workspace"],
    (dict(pe_pages=ODD), INVALID, "aligned"), (dict(scales=BYTE), INVALID, "scales must be 2-byte aligned"),
    (dict(workspace=None), WORKSPACE, "workspace"),
    (dict(workspace_bytes=ctypes.c_size_t(256)), WORKSPACE, "small"),
])
def test_attention_refuses(lib, change, status, word):
    a = {**ATTEND, "dims": dims(), **change}
    a["dims"] = ctypes.byref(a["dims"])
    assert lib.mla_attention_paged_fp8blk(*a.values()) == status
    assert word in lib.mla_last_error().decode()


def test_workspace_queries(lib):
    assert lib.mla_cache_extend_workspace_bytes(0, 1) == lib.mla_cache_extend_workspace_bytes(1, 0) == 0
    assert lib.mla_cache_extend_workspace_bytes(64, 8) == 0      # one launch, no workspace
    assert lib.mla_cache_extend_workspace_bytes(2000, 1) >= 2001 * 16
    assert lib.mla_cache_extend_workspace_bytes(1, 100000) >= 2 * 16
    d = dims(batch=8, sk=8192)
    q = lib.mla_attention_paged_fp8blk_workspace_bytes
    assert q(BF16, ctypes.byref(d), 0, 64) == q(F16, ctypes.byref(d), 0, 64) > 0
    assert q(BF16, ctypes.byref(d), 0, 64) <= lib.mla_attention_paged_fp8kv_workspace_bytes(
        BF16, ctypes.byref(d), 0, 64)
    assert q(F32, ctypes.byref(d), 0, 64) == 0 and q(BF16, ctypes.byref(d), 0, 63) == 0
    assert q(BF16, None, 0, 64) == 0


# ------------------------------------------------------------------ refusals of the binding

def pool(P=4, page=64, block=16):
    return (torch.zeros(P, page, 512, dtype=torch.uint8), torch.zeros(P, page, 64, dtype=torch.uint8),
            torch.zeros(P, page // block, 2, dtype=torch.uint8))


def ints(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


@pytest.fixture(scope="module")
def ext():
    import mla_custom_cuda
    return mla_custom_cuda


def test_binding_extend(ext):
    good = dict(new_lens=ints(2), seq_lens=ints(2), block_table=ints(2, 3), free_pages=ints(9), free_state=ints(2),
                Sq=1, page_size=64)
    for change, word in ((dict(new_lens=ints(3)), "new_lens"), (dict(seq_lens=ints(2, 1)), "seq_lens"),
                         (dict(new_lens=torch.zeros(2, dtype=torch.int64)), "int32"),
                         (dict(block_table=ints(6)), "block_table"), (dict(block_table=ints(2, 0)), "block_table"),
                         (dict(block_table=ints(3, 2).T), "contiguous"), (dict(free_pages=ints(18)[::2]), "contiguous"),
                         (dict(free_pages=ints(0)), "free_pages"), (dict(free_state=ints(3)), "free_state"),
                         (dict(Sq=0), "Sq"), (dict(page_size=-64), "page_size"), ({}, "ROCm GPU")):
        with pytest.raises(RuntimeError, match=word):
            ext.cache_extend(**{**good, **change})


def test_binding_append(ext):
    c, p, s = pool()
    x, W, g = torch.zeros(2, 3, 64), torch.zeros(64, 576), torch.zeros(512)
    good = dict(x=x, W_kv_a=W, kv_norm_w=g, seq_lens=ints(2), new_lens=ints(2), block_table=ints(2, 3), c_kv_pages=c,
                pe_pages=p, scales=s, eps=1e-6)
    for change, word in ((dict(x=x[0]), "x must"), (dict(W_kv_a=W[:, :570]), "W_kv_a"), (dict(kv_norm_w=g[:3]), "kv_norm_w"),
                         (dict(W_kv_a=W.half()), "dtype"), (dict(seq_lens=ints(3)), "seq_lens"),
                         (dict(new_lens=ints(2).long()), "int32"), (dict(block_table=ints(3, 3)), "block_table"),
                         (dict(pe_pages=p[:3]), "pe_pages"), (dict(c_kv_pages=c.float()), "e4m3fn or uint8"),
                         (dict(scales=s[:, :3]), "scales"), (dict(scales=s[..., :1]), "scales"),
                         (dict(scales=s.float()), "e8m0fnu or uint8"),
                         (dict(c_kv_pages=torch.zeros(4, 64, 600, dtype=torch.uint8)[..., :512]), "contiguous"),
                         ({}, "ROCm GPU")):
        with pytest.raises(RuntimeError, match=word):
            ext.kv_append_paged_fp8blk(**{**good, **change})


def test_binding_read(ext):
    c, p, s = pool()
    slots = torch.zeros(3, dtype=torch.int64)
    for args, word in (((slots.int(), c, p, s, torch.float32), "int64"), ((slots, c, p[:2], s, torch.float32), "pe_pages"),
                       ((slots, c, p, s, torch.int32), "dtype"), ((slots, c[..., :256], p, s, torch.float32), "kv_rank"),
                       ((slots, c, p, s, torch.float32), "ROCm GPU")):
        with pytest.raises(RuntimeError, match=word):
            ext.kv_read_fp8blk(*args)


def test_binding_attention(ext):
    c, p, s = pool()
    BF = torch.bfloat16
    qa, qr, w = torch.zeros(2, 1, 4, 512, dtype=BF), torch.zeros(2, 1, 4, 64, dtype=BF), torch.zeros(4, 128, 512, dtype=BF)
    good = dict(q_absorbed=qa, q_rope=qr, c_kv_pages=c, pe_pages=p, scales=s, block_table=ints(2, 3), seq_lens=ints(2),
                W_uv=w, scale=1.0)
    for change, word in ((dict(q_rope=qr[:1]), "q_rope"), (dict(q_absorbed=qa.float(), q_rope=qr.float(), W_uv=w.float()),
                                                           "bfloat16 or float16"),
                         (dict(W_uv=w.half()), "dtype"), (dict(seq_lens=ints(3)), "seq_lens"),
                         (dict(block_table=ints(1, 3)), "block_table"), (dict(scales=s[:2]), "scales"),
                         (dict(pe_pages=p.half()), "e4m3fn or uint8"), ({}, "ROCm GPU")):
        with pytest.raises(RuntimeError, match=word):
            ext.mla_attention_paged_fp8blk(**{**good, **change})


# ------------------------------------------------------------------ the plain forms themselves

def test_codes_are_torchs(seed=0):
    """round_code is torch's conversion, e4m3's steps are half_step's, exponent is the smallest."""
    g = torch.Generator().manual_seed(seed)
    v = torch.randn(4000, generator=g) * torch.exp2(torch.randint(-12, 8, (4000,), generator=g).float())
    v = torch.cat((v.clamp(-448, 448), torch.tensor([0.0, 448.0, -448.0, 2.0 ** -10, 3 * 2.0 ** -10, 17.0, 19.0])))
    want = v.to(torch.float8_e4m3fn).double()
    assert torch.equal(K.round_code(v.double(), torch.zeros((), dtype=torch.int32)), want)
    assert ((want - v.double()).abs() <= K.half_step(v.double(), torch.zeros((), dtype=torch.int32))).all()
    for a in (448.0, 448.0 * (1 + 2 ** -23), 1.0, 1e-20, 3.4e38, 5e-324, 224.0, 223.99):
        e = K.exponent(a)
        assert a <= 448 * 2.0 ** e and (e == K.EMIN or a > 448 * 2.0 ** (e - 1))


def test_append_rows_are_the_layers():
    """kv_rows is the paged append's row (the oracle's, in float32) at 64 bits, inside its bound."""
    g = torch.Generator().manual_seed(1)
    x, W = torch.randn(1, 9, 64, generator=g), torch.randn(64, 576, generator=g) / 8
    gain = 1 + 0.1 * torch.randn(512, generator=g)
    table = torch.tensor([[1]], dtype=torch.int32)
    pos = torch.arange(30, 39)[None]
    ck, pe = R.kv_append_paged(x, W, gain, pos, table, torch.zeros(2, 64, 512), torch.zeros(2, 64, 64))
    lat, rot, el, er = K.kv_rows(x[0], W, gain, pos[0])
    assert ((ck[1, 30:39].double() - lat).abs() <= el).all()
    assert ((pe[1, 30:39].double() - rot).abs() <= er).all()


def test_attention_is_the_oracles():
    g = torch.Generator().manual_seed(2)
    lens = [70, 3, 0]
    table = K.tables(lens, 64, 5, g)
    cache = K.new_pool(5, 64, 16, g)
    qa, qr, w = K.queries(3, 2, 4, 8, g, torch.float32)
    rows = K.decode(cache)
    out = K.attention(qa, qr, rows, table, lens, w, C.SCALE, True, 64, 5)
    ref = R.mla_attention_paged(qa[:2], qr[:2], rows[0].float().view(5, 64, -1), rows[1].float().view(5, 64, -1),
                                table[:2].clamp(min=0), torch.tensor(lens[:2], dtype=torch.int32), w, C.SCALE, True)
    torch.testing.assert_close(out[:2].float(), ref, rtol=1e-4, atol=1e-5)
    assert not out[2].any()


@pytest.mark.parametrize("mistake", ["neighbour", "swapped", "no_scale", "whole_block_64", "latent_only"])
@pytest.mark.parametrize("block", [16, 32])
def test_attention_tolerance_tells_wrong_scales(mistake, block):
    """The bound of the GPU attention tests rejects a pass that takes the next block's scale, swaps
    the parts' scales, takes none, one scale for 64 tokens, or the latent's for both parts -- and
    accepts the pass with its three roundings."""
    g = torch.Generator().manual_seed(3)
    lens, page = [700], 64
    table = K.tables(lens, page, 14, g)
    cache = K.new_pool(14, page, block, g)
    dt = torch.bfloat16
    qa, qr, w = K.queries(1, 1, 8, 128, g, dt)
    rows = K.decode(cache)
    ref = K.attention(qa, qr, rows, table, lens, w, C.SCALE, False, page, 14)
    u = torch.finfo(dt).eps / 2
    bad = {k: v.clone() for k, v in cache.items()}
    s = bad["scales"]
    if mistake == "neighbour":
        bad["scales"] = s.view(-1, 2).roll(1, 0).view(s.shape)
    elif mistake == "swapped":
        bad["scales"] = s.flip(2)
    elif mistake == "no_scale":
        s.fill_(120)
    elif mistake == "whole_block_64":
        s[:] = s[:, :1].clone()
    else:
        s[..., 1] = s[..., 0]
    out = K.attention(qa, qr, K.decode(bad), table, lens, w, C.SCALE, False, page, 14)
    assert (out - ref).norm() > 2 * math.sqrt(3) * u * ref.norm()
    # the real thing, rounded where the kernel rounds
    slot = K.slots_of(table, 0, 0, 700, page)
    lat, rot = rows[0][slot], rows[1][slot]
    t = (qa[0, 0].double() @ lat.T + qr[0, 0].double() @ rot.T) / C.SCALE
    p = torch.exp(t - t.amax(1, keepdim=True))
    ctx = (p.to(dt).double() @ lat / p.sum(1, keepdim=True)).to(dt).double()
    near = torch.einsum("hr,hvr->hv", ctx, w.double()).to(dt).double()
    assert (near - ref[0, 0]).norm() <= math.sqrt(3) * u * ref.norm()


# ------------------------------------------------------------------ the work list's item bound

@pytest.mark.parametrize("row_tiles", [1, 2, 3, 8, 40, 86, 300])
def test_sixteen_bit_lists_stay_inside_their_bound(row_tiles, tmp_path):
    """wl_max_items16, which the grid and the partial slots of this cache's attention are sized for,
    covers every 16-bit list that the rules make when nothing limits them."""
    import subprocess

    import numpy as np

    import wl_check as W
    from test_worklist_cpu import distributions

    src = tmp_path / "bound.cpp"
    src.write_text('#include "worklist.h"\nextern "C" int bound(int B, int rt) '
                   '{ return mla::wl_max_items16(B, rt); }\n')
    out = tmp_path / "bound.so"
    subprocess.run(["g++", "-O2", "-std=c++17", "-shared", "-fPIC", "-I", W.CSRC, str(src), "-o", str(out)], check=True)
    bound = ctypes.CDLL(str(out)).bound
    rng = np.random.default_rng(row_tiles)
    for B in (1, 2, 3, 5, 7, 8, 16, 31, 64, 65, 100, 127, 128, 129, 132, 160, 255, 256, 300, 1000):
        most = bound(B, row_tiles)
        assert most % 8 == 0
        for Sk in (64, 128, 640, 4992, 65536):
            for name, lens in distributions(B, Sk, rng):
                wl = W.build_serial(lens, Sk, row_tiles, 32, 40 * B + 4096)
                assert wl[0] <= most, (B, row_tiles, Sk, name, int(wl[0]), most)
                W.check_list(W.build_serial(lens, Sk, row_tiles, 32, most), lens, Sk, 32, most)
