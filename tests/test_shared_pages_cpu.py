"""The host forms of forking and compacting keep every request's tokens (what the GPU tests compare
with), and the refusals of the calls, which come before any GPU work."""

from __future__ import annotations

import ctypes
import random

import pytest
import torch

import shared_pages as S
from test_abi_cpu import LIB, MLA_ERR_INVALID_ARGUMENT as INVALID, MLA_ERR_WORKSPACE as WORKSPACE, MLA_OK


def batch(r, B, max_pages, page, N):
    """A state in which some rows share whole pages."""
    free = list(range(N))
    r.shuffle(free)
    table, lens = [], []
    for b in range(B):
        n = r.choice([0, r.randint(0, max_pages * page), r.randint(0, max_pages) * page])
        row = []
        if b and r.random() < 0.4:
            c = r.randrange(b)
            row = table[c][:min(lens[c] // page, n // page)]
        row = list(row)
        while len(row) < S.pages(n, page):
            if not free:
                n = len(row) * page
                break
            row.append(free.pop())
        table.append(row + [r.randrange(N) for _ in range(max_pages - len(row))])
        lens.append(n)
    head = r.randrange(N)
    ring = [r.randrange(N) for _ in range(N)]
    for i, p in enumerate(free):
        ring[(head + i) % N] = p
    return table, lens, ring, head, len(free)


@pytest.mark.parametrize("seed", range(40))
def test_fork_keeps_tokens(seed):
    r = random.Random(seed)
    B, max_pages, page = r.randint(1, 9), r.randint(1, 6), 64
    N = r.randint(B, B * max_pages + 6)
    table, lens, ring, head, count = batch(r, B, max_pages, page, N)
    parents = [r.choice([b, r.randrange(B), -1, B]) for b in range(B)]
    keep = [r.choice([0, 10 ** 6, r.randint(-5, max_pages * page)]) for _ in range(B)]
    out = S.fork(parents, keep, lens, table, ring, head, count, page)
    pool = {(p, i): (p, i) for p in range(N) for i in range(page)}
    for a, b in out["copies"]:
        if a >= 0:
            for i in range(page):
                pool[b, i] = (a, i)
    held = {}
    for b in range(B):
        n = out["seq_lens"][b]
        p = parents[b] if 0 <= parents[b] < B else b
        want = min(max(keep[b], 0), lens[p]) if 0 <= parents[b] < B else 0
        assert n == want or n == want // page * page
        assert S.contents(out["block_table"][b], n, page, pool) == \
            [(table[p][i // page], i % page) for i in range(n)]
        for j in range(S.pages(n, page)):
            held.setdefault(out["block_table"][b][j], []).append(j < n // page)
    # an open page has one holder; held and free pages are apart, and all pages are one of the two
    assert all(len(v) == 1 or all(v) for v in held.values())
    h, c = out["state"]
    free = [out["ring"][(h + i) % N] for i in range(c)]
    assert sorted(free + list(held)) == list(range(N))


@pytest.mark.parametrize("seed", range(40))
def test_compact_keeps_tokens(seed):
    r = random.Random(seed)
    B, max_pages, page = r.randint(1, 9), r.randint(1, 6), 64
    N = r.randint(B, B * max_pages + 6)
    table, lens, ring, head, count = batch(r, B, max_pages, page, N)
    out = S.compact(lens, table, ring, head, count, page)
    where = list(range(N))
    for a, b in out["copies"]:
        if a >= 0:
            where[b] = a
    used = set()
    for b in range(B):
        k = S.pages(lens[b], page)
        assert [where[p] for p in out["block_table"][b][:k]] == table[b][:k]
        used |= set(out["block_table"][b][:k])
    assert used == set(range(len(used)))
    assert out["ring"][:out["state"][1]] == list(range(len(used), N))


# ------------------------------------------------------------------ refusals

@pytest.fixture(scope="module")
def lib():
    L = ctypes.CDLL(LIB)
    L.mla_last_error.restype = ctypes.c_char_p
    for n in ("mla_cache_fork_workspace_bytes", "mla_cache_compact_workspace_bytes"):
        getattr(L, n).restype = ctypes.c_size_t
    return L


class Pool(ctypes.Structure):
    _fields_ = [("data", ctypes.c_void_p), ("page_bytes", ctypes.c_int64),
                ("layer_bytes", ctypes.c_int64), ("layers", ctypes.c_int32)]


A = [0x10000000 + 0x1000000 * i for i in range(16)]     # addresses that are never followed


def fork_call(lib, batch=4, page=64, max_pages=8, pages=100, p=None, ws=None, wsb=0):
    p = p or A[:10]
    return lib.mla_cache_fork(batch, page, max_pages, pages, *map(ctypes.c_void_p, p), ctypes.c_void_p(ws),
                              ctypes.c_size_t(wsb), None)


def compact_call(lib, batch=4, page=64, max_pages=8, pages=100, p=None, ws=None, wsb=0):
    p = p or A[:8]
    return lib.mla_cache_compact(batch, page, max_pages, pages, *map(ctypes.c_void_p, p), ctypes.c_void_p(ws),
                                 ctypes.c_size_t(wsb), None)


@pytest.mark.parametrize("call,n_in,n", [(fork_call, 6, 10), (compact_call, 4, 8)])
def test_table_refusals(lib, call, n_in, n):
    for kw in ({"batch": 0}, {"batch": -1}, {"batch": (1 << 16) + 1}, {"page": 0}, {"page": 63}, {"page": -64},
               {"max_pages": 0}, {"pages": 0}, {"pages": (1 << 30) + 1}, {"max_pages": 1 << 25, "page": 64},
               {"batch": 1 << 16, "max_pages": 1 << 15}):
        assert call(lib, **kw) == INVALID, kw
        assert lib.mla_last_error()
    for i in range(n):
        p = A[:n]
        p[i] = None
        assert call(lib, p=p) == INVALID
        p[i] = A[i] + 4
        assert call(lib, p=p) == INVALID and b"aligned" in lib.mla_last_error()
    for o in range(n_in, n):
        for i in range(n):
            if i != o:
                p = A[:n]
                p[o] = p[i]
                assert call(lib, p=p) == INVALID and b"overlap" in lib.mla_last_error()
    # a large pool needs a workspace
    assert call(lib, pages=1 << 20) == WORKSPACE
    assert call(lib, pages=1 << 20, ws=A[11], wsb=64) == WORKSPACE


def test_workspace_sizes(lib):
    assert lib.mla_cache_fork_workspace_bytes(4, 100) == 0
    assert lib.mla_cache_compact_workspace_bytes(100) == 0
    assert lib.mla_cache_fork_workspace_bytes(4, 1 << 20) >= 4 << 20
    assert lib.mla_cache_fork_workspace_bytes(5000, 100) >= 400
    assert lib.mla_cache_compact_workspace_bytes(1 << 20) >= 5 << 20
    assert lib.mla_cache_fork_workspace_bytes(0, 5) == 0 and lib.mla_cache_compact_workspace_bytes(-3) == 0


def test_copy_refusals(lib):
    def call(pools, n=3, pages=10, copies=A[0], n_pools=None):
        arr = (Pool * max(1, len(pools)))(*pools)
        return lib.mla_cache_copy_pages(ctypes.c_void_p(copies), ctypes.c_int64(n), pages, arr,
                                        len(pools) if n_pools is None else n_pools, None)
    good = Pool(A[1], 128, 1280, 2)
    assert call([good], n=0) == MLA_OK
    assert call([good], n=0, copies=None) == MLA_OK
    for kw in ({"n": -1}, {"n": 1 << 31}, {"pages": 0}, {"n_pools": 0}, {"copies": None}, {"copies": A[0] + 8}):
        assert call([good], **kw) == INVALID, kw
    assert call([good] * 9) == INVALID
    for bad in (Pool(None, 128, 1280, 2), Pool(A[1], 0, 1280, 2), Pool(A[1], -4, 1280, 2), Pool(A[1], 128, 1279, 2),
                Pool(A[1], 128, 1280, 0), Pool(A[1], 1 << 50, 0, 1), Pool(A[1], 128, 1 << 45, 5), Pool(A[1], 128, 1280, 65536)):
        assert call([bad]) == INVALID
    assert lib.mla_cache_copy_pages(ctypes.c_void_p(A[0]), ctypes.c_int64(1), 10, None, 1, None) == INVALID


def test_binding_refusals():
    import mla_custom_cuda as ext

    def i(*s):
        return torch.zeros(*s, dtype=torch.int32)
    good = dict(parents=i(3), keep_lens=i(3), seq_lens=i(3), block_table=i(3, 4), free_pages=i(9), free_state=i(2),
                page_size=64)
    for k, v in (("parents", i(2)), ("keep_lens", i(3, 1)), ("seq_lens", torch.zeros(3)), ("block_table", i(12)),
                 ("block_table", torch.zeros(3, 4)), ("block_table", i(0, 4)), ("free_pages", i(0)),
                 ("free_pages", torch.zeros(9)), ("free_pages", i(18)[::2]), ("free_state", i(3)), ("page_size", 0)):
        with pytest.raises(RuntimeError):
            ext.cache_fork(**{**good, k: v})
        if k not in ("parents", "keep_lens"):
            if k == "free_pages" and not v.is_contiguous():
                continue
            c = {n: x for n, x in good.items() if n not in ("parents", "keep_lens")}
            with pytest.raises(RuntimeError):
                ext.cache_compact(**{**c, k: v})
    with pytest.raises(RuntimeError, match="GPU"):
        ext.cache_fork(**good)
    pool = torch.zeros(9, 64, 8)
    for copies, pools, layered in ((i(3), [pool], False), (i(3, 3), [pool], False), (torch.zeros(3, 2), [pool], False),
                                   (i(3, 2), [], False), (i(3, 2), [pool] * 9, False), (i(3, 2), [pool, pool[:8]], False),
                                   (i(3, 2), [pool[:, ::2]], False), (i(3, 2), [pool.transpose(0, 1)], True),
                                   (i(3, 2), [torch.zeros(5)], True)):
        with pytest.raises(RuntimeError):
            ext.cache_copy_pages(copies, pools, layered)
    with pytest.raises(RuntimeError, match="GPU"):
        ext.cache_copy_pages(i(3, 2), [pool])
