"""Refusals of the expanded attention and of mla_q_heads, which come before any GPU work."""

from __future__ import annotations

import ctypes

import pytest
import torch

from test_abi_cpu import (BF16, F32, LIB, MLA_ERR_INVALID_ARGUMENT as INVALID, MLA_ERR_UNSUPPORTED as UNSUPPORTED,
                          MLA_ERR_WORKSPACE as WORKSPACE, Dims)

F16, F64 = 2, 3
A = [0x10000000 + 0x1000000 * i for i in range(16)]     # addresses that are never followed


def dims(**kw):
    d = Dims(2, 100, 256, 7168, 1536, 4, 128, 64, 512, 128)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


@pytest.fixture(scope="module")
def lib():
    L = ctypes.CDLL(LIB)
    L.mla_last_error.restype = ctypes.c_char_p
    for n in ("mla_attention_expanded_workspace_bytes", "mla_attention_paged_expanded_workspace_bytes",
              "mla_q_heads_workspace_bytes"):
        getattr(L, n).restype = ctypes.c_size_t
    return L


def P(x):
    return ctypes.c_void_p(x)


def dense(lib, dt=BF16, d=None, p=None, scale=13.0, causal=1, ws=A[12], wsb=1 << 40):
    p = p or A[:7]
    return lib.mla_attention_expanded(dt, ctypes.byref(d or dims()), *map(P, p[:6]), ctypes.c_double(scale), causal,
                                      P(p[6]), P(ws), ctypes.c_size_t(wsb), None)


def paged(lib, dt=BF16, d=None, p=None, page=64, pages=20, scale=13.0, causal=1, ws=A[12], wsb=1 << 40):
    p = p or A[:10]
    return lib.mla_attention_paged_expanded(dt, ctypes.byref(d or dims()), *map(P, p[:7]), page, pages, P(p[7]), P(p[8]),
                                            ctypes.c_double(scale), causal, P(p[9]), P(ws), ctypes.c_size_t(wsb), None)


def blocked(lib, dt=BF16, d=None, p=None, page=64, pages=20, block=32, scale=13.0, causal=1, ws=A[12], wsb=1 << 40):
    p = p or A[:11]
    return lib.mla_attention_paged_fp8blk_expanded(
        dt, ctypes.byref(d or dims()), *map(P, p[:8]), page, pages, block, P(p[8]), P(p[9]), ctypes.c_double(scale), causal,
        P(p[10]), P(ws), ctypes.c_size_t(wsb), None)


CALLS = [(dense, 7, ()), (paged, 10, (6,)), (blocked, 11, (4, 7))]


@pytest.mark.parametrize("call,n,special", CALLS)
def test_refusals(lib, call, n, special):
    for dt in (F32, F64):
        assert call(lib, dt=dt) == UNSUPPORTED
    assert call(lib, dt=9) == INVALID
    for kw in ({"kv_rank": 256}, {"rope": 32}, {"nope": 64}, {"v": 64}, {"batch": 65536, "sq": 1, "heads": 1}):
        assert call(lib, d=dims(**kw)) == UNSUPPORTED, kw
    for kw in ({"batch": 0}, {"sq": 0}, {"sk": 0}, {"heads": 0}, {"sq": 257}, {"kv_rank": 0}, {"rope": -8},
               {"batch": 1 << 14, "heads": 1 << 14}):
        assert call(lib, d=dims(**kw)) == INVALID, kw
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        assert call(lib, scale=scale) == INVALID
    for i in range(n):
        p = A[:n]
        p[i] = A[i] + 1
        assert call(lib, p=p) == INVALID, i
        p[i] = None
        if i not in special or (call is blocked and i == 4):
            assert call(lib, p=p) == INVALID, i
    assert call(lib, ws=None) == WORKSPACE and call(lib, wsb=1000) == WORKSPACE and call(lib, ws=A[12] + 16) == WORKSPACE
    assert lib.mla_last_error()


@pytest.mark.parametrize("call", [paged, blocked])
def test_page_refusals(lib, call):
    for kw in ({"page": 0}, {"page": 32}, {"page": -64}, {"page": 192}, {"pages": 0}, {"pages": -1}):
        assert call(lib, **kw) == INVALID, kw


def test_block_refusals(lib):
    assert blocked(lib, block=8) == UNSUPPORTED and blocked(lib, block=128) == UNSUPPORTED


def test_workspace(lib):
    """Keys and values of all heads, or of as many as 2 GiB take."""
    def paged_bytes(d):
        return lib.mla_attention_paged_expanded_workspace_bytes(BF16, ctypes.byref(d), 1, 64)
    rows, part = 2 * 256, 2 * 100 * 4 * (512 + 8)        # and up to 16 key splits' rows
    assert rows * (1152 + 4 * 512) <= paged_bytes(dims()) <= rows * (1152 + 4 * 512) + 16 * part + 16384
    d = dims(batch=1, sk=1 << 20, heads=128)
    assert (2 << 30) < paged_bytes(d) < (2 << 30) + (1 << 20) * 1152 + 16 * 100 * 128 * 520 + (1 << 20)
    d = dims(batch=1, sq=1, sk=1 << 21, heads=2)          # check_attn_dims' limit of keys
    assert paged_bytes(d) == 0
    assert lib.mla_attention_expanded_workspace_bytes(BF16, ctypes.byref(dims(sk=250)), 1) >= 2 * 256 * (1152 + 4 * 512)
    assert lib.mla_attention_expanded_workspace_bytes(F32, ctypes.byref(dims()), 1) == 0
    assert lib.mla_attention_expanded_workspace_bytes(BF16, None, 1) == 0
    assert lib.mla_attention_paged_expanded_workspace_bytes(BF16, ctypes.byref(dims()), 1, 100) == 0


def test_q_heads_refusals(lib):
    def call(dt=BF16, d=None, p=None, eps=1e-6, ws=A[12], wsb=1 << 40):
        p = p or A[:8]
        return lib.mla_q_heads(dt, ctypes.byref(d or dims()), *map(P, p[:5]), 0, P(p[5]), ctypes.c_double(eps), P(p[6]),
                               P(p[7]), P(ws), ctypes.c_size_t(wsb), None)
    for dt in (F32, F64):
        assert call(dt=dt) == UNSUPPORTED
    for kw in ({"batch": 0}, {"hidden": 12}, {"q_lora": 0}, {"heads": -1}, {"nope": 4}, {"rope": 0}, {"rope": 1024}):
        assert call(d=dims(**kw)) == INVALID, kw
    for i in range(8):
        p = A[:8]
        p[i] = None
        assert call(p=p) == INVALID
        p[i] = A[i] + 2
        assert call(p=p) == INVALID
    assert call(eps=-1.0) == INVALID and call(eps=float("nan")) == INVALID
    assert call(wsb=64) == WORKSPACE
    assert lib.mla_q_heads_workspace_bytes(BF16, ctypes.byref(dims(kv_rank=0))) > 0
    assert lib.mla_q_heads_workspace_bytes(F32, ctypes.byref(dims())) == 0


def test_binding_refusals():
    import mla_custom_cuda as ext
    bf = torch.bfloat16
    z = lambda *s, dt=bf: torch.zeros(*s, dtype=dt)
    i = lambda *s: torch.zeros(*s, dtype=torch.int32)
    good = dict(q_nope=z(2, 5, 3, 128), q_rope=z(2, 5, 3, 64), c_kv_pages=z(7, 64, 512), pe_pages=z(7, 64, 64),
                block_table=i(2, 4), seq_lens=i(2), W_uk=z(3, 128, 512), W_uv=z(3, 128, 512), scale=1.0)
    for k, v in (("q_nope", z(2, 5, 128)), ("q_rope", z(2, 5, 2, 64)), ("q_rope", z(2, 5, 3, 64, dt=torch.float16)),
                 ("c_kv_pages", z(7, 64, 500)), ("c_kv_pages", z(7, 64, 512, dt=torch.float32)), ("pe_pages", z(7, 32, 64)),
                 ("pe_pages", z(7, 64, 32)), ("block_table", i(3, 4)), ("block_table", z(2, 4)), ("seq_lens", i(3)),
                 ("seq_lens", z(2)), ("W_uk", z(2, 128, 512)), ("W_uk", z(3, 64, 512)), ("W_uv", z(3, 128, 256)),
                 ("new_lens", i(3)), ("new_lens", z(2))):
        with pytest.raises(RuntimeError):
            ext.mla_attention_paged_expanded(**{**good, k: v})
    with pytest.raises(RuntimeError, match="GPU"):
        ext.mla_attention_paged_expanded(**good)
    codes = dict(good, c_kv_pages=z(7, 64, 512, dt=torch.uint8), pe_pages=z(7, 64, 64, dt=torch.uint8),
                 scales=z(7, 2, 2, dt=torch.uint8))
    for k, v in (("scales", z(7, 2, 3, dt=torch.uint8)), ("scales", z(6, 2, 2, dt=torch.uint8)), ("c_kv_pages", z(7, 64, 512))):
        with pytest.raises(RuntimeError):
            ext.mla_attention_paged_fp8blk_expanded(**{**codes, k: v})
    with pytest.raises(RuntimeError, match="GPU"):
        ext.mla_attention_paged_fp8blk_expanded(**codes)
    flat = dict(q_nope=good["q_nope"], q_rope=good["q_rope"], c_kv=z(2, 9, 512), pe_cache=z(2, 9, 64), W_uk=good["W_uk"],
                W_uv=good["W_uv"], scale=1.0)
    for k, v in (("c_kv", z(1, 9, 512)), ("pe_cache", z(2, 8, 64)), ("pe_cache", z(2, 9, 32))):
        with pytest.raises(RuntimeError):
            ext.mla_attention_expanded(**{**flat, k: v})
    with pytest.raises(RuntimeError, match="GPU"):
        ext.mla_attention_expanded(**flat)
    q = dict(x=z(2, 5, 64), W_q_a=z(64, 32), q_norm_w=z(32), W_q_b=z(32, 3 * 192), positions=torch.arange(5), nope_dim=128,
             rope_dim=64, eps=1e-6)
    for k, v in (("W_q_a", z(32, 32)), ("W_q_b", z(32, 100)), ("W_q_b", z(16, 192)), ("q_norm_w", z(31)),
                 ("positions", torch.arange(6)), ("positions", torch.zeros(5)), ("nope_dim", 0), ("rope_dim", -1), ("rope_dim", 63)):
        with pytest.raises(RuntimeError):
            ext.q_heads(**{**q, k: v})
    with pytest.raises(RuntimeError, match="GPU"):
        ext.q_heads(**q)
