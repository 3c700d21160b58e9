"""GPU checks of cache_fork, cache_compact and cache_copy_pages against tests/shared_pages.py (whole
numbers and bytes: equal), and of a serving step that runs them with the cache's other operators."""

from __future__ import annotations

import math
import random

import pytest
import torch

import expanded_ref as E
import shared_pages as S
from test_shared_pages_cpu import batch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


@pytest.fixture(scope="module")
def ext():
    if not torch.cuda.is_available():
        pytest.fail("GPU tests need a ROCm GPU")
    import mla_custom_cuda
    return mla_custom_cuda


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def check_fork(ext, parents, keep, lens, table, ring, head, count, page):
    want = S.fork(parents, keep, lens, table, ring, head, count, page)
    tab, r = i32(table), i32(ring)
    got = ext.cache_fork(i32(parents), i32(keep), i32(lens), tab, r, i32([head, count]), page)
    assert got[0].tolist() == want["seq_lens"]
    assert got[1].tolist() == want["block_table"]
    assert got[2].tolist() == want["state"]
    assert got[3].tolist() == want["copies"]
    assert r.tolist() == want["ring"] and tab.tolist() == table


def check_compact(ext, lens, table, ring, head, count, page):
    want = S.compact(lens, table, ring, head, count, page)
    got = ext.cache_compact(i32(lens), i32(table), i32(ring), i32([head, count]), page)
    assert got[0].tolist() == want["block_table"]
    assert got[1].tolist() == want["ring"]
    assert got[2].tolist() == want["state"]
    assert got[3].tolist() == want["copies"]


def plan(r, B, max_pages, page):
    parents = [r.choice([b, b, r.randrange(B), r.randrange(B), -1, B, 2 ** 31 - 1, -2 ** 31]) for b in range(B)]
    keep = [r.choice([0, 2 ** 31 - 1, -2 ** 31, r.randint(0, max_pages * page), r.randint(0, max_pages) * page])
            for _ in range(B)]
    return parents, keep


# a pool past one workgroup's range of 16,384 pages, and more requests than it has threads, take the
# launches apart
SIZES = [(1, 1, 1), (3, 2, 9), (8, 11, 60), (17, 40, 500), (64, 70, 3000), (5, 9, 16384), (5, 9, 16385),
         (40, 300, 40000), (1025, 3, 2600), (1300, 20, 33000)]


@pytest.mark.parametrize("page", [64, 192])
@pytest.mark.parametrize("B,max_pages,N", SIZES)
def test_fork(ext, B, max_pages, N, page):
    r = random.Random(B * 7 + N + page)
    table, lens, ring, head, count = batch(r, B, max_pages, page, N)
    check_fork(ext, *plan(r, B, max_pages, page), lens, table, ring, head, count, page)


@pytest.mark.parametrize("page", [64, 128])
@pytest.mark.parametrize("B,max_pages,N", SIZES)
def test_compact(ext, B, max_pages, N, page):
    r = random.Random(B * 5 + N + page)
    table, lens, ring, head, count = batch(r, B, max_pages, page, N)
    check_compact(ext, lens, table, ring, head, count, page)


@pytest.mark.parametrize("N", [7, 20000])
def test_fork_runs_out(ext, N):
    """More copies than free pages: the later requests are cut back to their whole pages."""
    B, page = 6, 64
    table = [[1, 2, 0]] + [[0, 0, 0]] * 5
    ring = list(range(3, N)) + [0, 1, 2]
    for count in (0, 1, 3, 5):
        check_fork(ext, [0] * B, [100] * B, [100, 0, 0, 0, 0, 0], table, ring, 0, count, page)


@pytest.mark.parametrize("N", [30, 20000])
def test_fork_open_against_whole(ext, N):
    """A page that one request keeps whole and others open: all of those take copies; cut back to
    nothing, to one token, to a whole page."""
    ring = [-1] * N
    for i in range(10):
        ring[(N - 4 + i) % N] = 10 + i
    table = [[5, 6, 7], [8, 9, 0], [0, 0, 0], [0, 0, 0]]
    lens = [150, 70, 0, 0]
    for keep in ([150, 100, 100, 128], [150, 1, 64, 65], [0, 150, 150, 150], [100, 128, 100, 99], [64, 64, 0, 63]):
        check_fork(ext, [0, 0, 0, 0], keep, lens, table, ring, N - 4, 10, 64)
        check_fork(ext, [1, 0, 3, 1], keep, lens, table, ring, N - 4 + N, 10, 64)
        check_fork(ext, [1, 0, 3, 1], keep, lens, table, ring, -4, 10, 64)


@pytest.mark.parametrize("N", [30, 20000])
def test_odd_states(ext, N):
    """Entries outside the pool, lengths past the table or below zero, counts past the ring, a ring that
    names held pages, pages of neither kind."""
    table = [[3, -1, 4], [N, 2 ** 31 - 1, -2 ** 31], [5, 6, 3], [3, 9, 9]]
    ring = [7, 3, -1, N, 8, 7, 2] + [1] * (N - 7)
    for lens in ([150, 150, 192, 70], [2 ** 31 - 1, -5, 64, 1], [0, 0, 0, 0]):
        for head, count in ((0, 7), (N - 2, 5), (5, -3), (0, N)):
            check_compact(ext, lens, table, ring, head, count, 64)
            check_fork(ext, [0, 1, 0, 2], [140, 190, 64, 130], lens, table, ring, head, min(count, 7), 64)


def test_ring_entry_outside_the_pool(ext):
    """A free page that is none goes into the table as it is, where nothing follows it."""
    check_fork(ext, [0, 0, 0], [70, 70, 70], [70, 0, 0], [[1, 2], [0, 0], [0, 0]], [-1, -7, 99, 3, 4, 5, 6, 0], 0, 4, 64)


# ------------------------------------------------------------------ copies

@pytest.mark.parametrize("dtype,shape", [(torch.bfloat16, (64, 512)), (torch.uint8, (64, 576)), (torch.uint8, (4, 2)),
                                         (torch.uint8, (1, 3)), (torch.float32, (5,)), (torch.float8_e4m3fn, (128, 64))])
@pytest.mark.parametrize("n,P", [(1, 2), (5, 40), (700, 1500)])
def test_copy(ext, dtype, shape, n, P):
    g = torch.Generator().manual_seed(n + P)
    order = torch.randperm(P, generator=g)[:2 * n].int()
    k = order.numel() // 2
    pairs = torch.stack((order[:k], order[k:2 * k]), 1)
    junk = torch.tensor([[-1, -1], [0, -1], [P, 0], [-2 ** 31, 1], [1, 2 ** 31 - 1]], dtype=torch.int32)
    pairs = torch.cat((junk, pairs, junk))[torch.randperm(k + 10, generator=g)]
    raw = torch.randint(0, 256, (P, *shape), generator=g, dtype=torch.int32)
    pool = raw.to(torch.uint8).view(dtype) if dtype.itemsize == 1 else raw.to(dtype)
    want = pool.view(torch.uint8).clone()
    for a, b in pairs.tolist():
        if 0 <= a < P and 0 <= b < P:
            want[b] = pool.view(torch.uint8)[a]
    got = pool.to(DEV)
    ext.cache_copy_pages(pairs.to(DEV), [got])
    assert torch.equal(got.cpu().view(torch.uint8), want)


def test_copy_layers_and_pools(ext):
    """Several pools of several layers, layers apart, an odd start, an empty list."""
    P, L = 50, 3
    g = torch.Generator().manual_seed(1)
    a = torch.randint(0, 255, (L, P + 4, 64, 32), generator=g).to(torch.uint8).to(DEV)[:, 2:-2]
    b = torch.randint(0, 255, (L * P * 6 + 1,), generator=g).to(torch.uint8).to(DEV)[1:].view(L, P, 6)
    c = torch.randn(2 * L, P, 64, 16, generator=g).to(torch.bfloat16).to(DEV)[::2]
    pairs = torch.tensor([[4, 7], [0, 49], [-1, -1], [9, 1]], dtype=torch.int32, device=DEV)
    want = [t.clone() for t in (a, b, c)]
    for s, d in ((4, 7), (0, 49), (9, 1)):
        for t in want:
            t[:, d] = t[:, s]
    outer = a._base.clone()
    ext.cache_copy_pages(torch.empty(0, 2, dtype=torch.int32, device=DEV), [a, b, c], layered=True)
    ext.cache_copy_pages(pairs, [a, b, c], layered=True)
    for x, y in zip((a, b, c), want):
        assert torch.equal(x, y)
    assert torch.equal(a._base[:, :2], outer[:, :2]) and torch.equal(a._base[:, -2:], outer[:, -2:])


# ------------------------------------------------------------------ together

@pytest.mark.parametrize("N", [40, 20000])
def test_graph_replay(ext, N):
    """Fork, copies and compaction captured together; replays with other inputs, eager work between."""
    r = random.Random(3)
    B, max_pages, page = 6, 5, 64
    first = batch(r, B, max_pages, page, N)
    t = {k: i32(v) for k, v in zip(("table", "lens", "ring"), first[:3])}
    t["state"] = i32(list(first[3:]))
    p, k = plan(r, B, max_pages, page)
    t["parents"], t["keep"] = i32(p), i32(k)
    pool = torch.zeros(N, 64, 4, dtype=torch.int32, device=DEV)

    def call():
        f = ext.cache_fork(t["parents"], t["keep"], t["lens"], t["table"], t["ring"], t["state"], page)
        ext.cache_copy_pages(f[3], [pool])
        c = ext.cache_compact(f[0], f[1], t["ring"], f[2], page)
        ext.cache_copy_pages(c[3], [pool])
        return f + c
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for i in range(4):
        table, lens, ring, head, count = batch(r, B, max_pages, page, N)
        p, k = plan(r, B, max_pages, page)
        results = []
        for run in (graph.replay, call):
            for name, v in (("table", table), ("lens", lens), ("ring", ring), ("state", [head, count]), ("parents", p), ("keep", k)):
                t[name].copy_(i32(v))
            pool.copy_(torch.arange(N, dtype=torch.int32, device=DEV)[:, None, None].expand_as(pool))
            torch.cuda.synchronize()
            got = run()
            torch.cuda.synchronize()
            results.append([x.clone() for x in (got or out)] + [t["ring"].clone(), pool.clone()])
        assert all(torch.equal(x, y) for x, y in zip(*results))
        f = S.fork(p, k, lens, table, ring, head, count, page)
        c = S.compact(f["seq_lens"], f["block_table"], f["ring"], *f["state"], page)
        assert results[0][4].tolist() == c["block_table"] and results[0][7].tolist() == c["copies"]


@pytest.mark.parametrize("blocked", [False, True])
def test_shared_prompt_step(ext, blocked):
    """As a server runs them: a prompt forked to its requests, a chunk of new tokens appended to each and
    attended to, two requests forked again and others ended, the pool compacted, another chunk: the
    attention of every request is that over the rows that the cache's own reader gives for it."""
    B, page, max_pages, P, H, dt = 4, 64, 8, 60, 2, torch.bfloat16
    g = torch.Generator(device=DEV)
    g.manual_seed(5)

    def normal(*shape, std=1.0):
        return (torch.randn(*shape, generator=g, device=DEV) * std).to(dt)
    hidden = 256
    W = {"kv": normal(hidden, 576, std=1 / 16), "norm": normal(512, std=0.1) + 1, "qa": normal(hidden, 128, std=1 / 16),
         "qn": normal(128, std=0.1) + 1, "qb": normal(128, H * 192, std=1 / 11), "uk": normal(H, 128, 512, std=1 / 22),
         "uv": normal(H, 128, 512, std=1 / 22)}
    if blocked:
        pools = [torch.full((P, page, 512), 0x7F, dtype=torch.uint8, device=DEV),
                 torch.full((P, page, 64), 0x7F, dtype=torch.uint8, device=DEV),
                 torch.full((P, page // 32, 2), 200, dtype=torch.uint8, device=DEV)]
    else:
        pools = [torch.full((P, page, w), math.nan, dtype=dt, device=DEV) for w in (512, 64)]
    table = torch.zeros(B, max_pages, dtype=torch.int32, device=DEV)
    ring, state = torch.randperm(P, generator=g, device=DEV).int(), i32([0, P])
    lens = i32([0] * B)
    seen = {}       # the rows of every request so far, as read back when they were written

    def chunk(new, Sq):
        nonlocal lens, state
        x = normal(B, Sq, hidden)
        lens, state, granted, pos, slots = ext.cache_extend(i32(new), lens, table, ring, state, Sq, page)
        assert granted.tolist() == new
        if blocked:
            ext.kv_append_paged_fp8blk(x, W["kv"], W["norm"], lens, granted, table, *pools, 1e-6)
        else:
            ext.kv_append_paged(x, W["kv"], W["norm"], pos, table, pools[0], pools[1], 1e-6)
        qn, qr = ext.q_heads(x, W["qa"], W["qn"], W["qb"], pos, 128, 64, 1e-6)
        scale = math.sqrt(192)
        if blocked:
            out = ext.mla_attention_paged_fp8blk_expanded(qn, qr, *pools, table, lens, W["uk"], W["uv"], scale, True, granted)
        else:
            out = ext.mla_attention_paged_expanded(qn, qr, *pools, table, lens, W["uk"], W["uv"], scale, True, granted)
        parts = []
        for b, n in enumerate(lens.tolist()):
            k = torch.arange(n, device=DEV)
            slot = table[b].long()[k // page] * page + k % page
            if blocked:
                lat, rot = ext.kv_read_fp8blk(slot, *pools, dt)
            else:
                lat, rot = pools[0].view(-1, 512)[slot], pools[1].view(-1, 64)[slot]
            assert torch.isfinite(lat.float()).all() and torch.isfinite(rot.float()).all()
            old = seen.get(b)
            if old is not None and not blocked:      # what was written stays (8 bits: may be coded again)
                assert torch.equal(lat[:old[0].size(0)], old[0]) and torch.equal(rot[:old[1].size(0)], old[1])
            seen[b] = (lat, rot)
            m = new[b]
            assert not out[b, :Sq - m].any()
            ref = E.attention(qn[b, Sq - m:], qr[b, Sq - m:], lat, rot, W["uk"], W["uv"], scale,
                              E.limits(Sq, n, m, True), dt)
            parts.append((out[b, Sq - m:],) + ref)
        E.check(*(torch.cat(p) for p in zip(*parts)))

    def fork(parents, keep):
        nonlocal lens, state, table
        lens, table, state, copies = ext.cache_fork(i32(parents), i32(keep), lens, table, ring, state, page)
        ext.cache_copy_pages(copies, pools)
        was = dict(seen)
        for b, (p, k) in enumerate(zip(parents, keep)):
            seen[b] = tuple(x[:k] for x in was[p])
        assert lens.tolist() == [x[0].size(0) for x in (seen[b] for b in range(B))]

    def compact():
        nonlocal table, ring, state
        table, ring, state, copies = ext.cache_compact(lens, table, ring, state, page)
        ext.cache_copy_pages(copies, pools)

    chunk([150, 0, 0, 0], 150)
    fork([0, 0, 0, 0], [150, 150, 128, 100])
    chunk([40, 33, 1, 64], 64)
    fork([0, 0, 3, 1], [190, 0, 164, 150])
    chunk([3, 20, 17, 0], 20)
    compact()
    chunk([70, 5, 60, 77], 77)
    fork([0, 1, 2, 3], [0, 25, 0, 200])
    compact()
    chunk([10, 30, 9, 30], 30)
    held = {p for b, n in enumerate(lens.tolist()) for p in table[b, :S.pages(n, page)].tolist()}
    head, count = state.tolist()
    free = [ring[(head + i) % P].item() for i in range(count)]
    assert sorted(free + list(held)) == list(range(P))


# where one workgroup's waves become more, and one launch becomes several
EDGES = [(256, 14, 4096), (257, 14, 4096), (256, 14, 4097), (1024, 14, 16384), (1024, 14, 16385), (1025, 14, 16384),
         (4100, 3, 13000)]


@pytest.mark.parametrize("B,max_pages,N", EDGES)
def test_edges(ext, B, max_pages, N):
    r = random.Random(B + N)
    table, lens, ring, head, count = batch(r, B, max_pages, 64, N)
    check_fork(ext, *plan(r, B, max_pages, 64), lens, table, ring, head, count, 64)
    check_compact(ext, lens, table, ring, head, count, 64)


def test_two_streams_at_once(ext):
    """Large pools' calls that overlap, with workspaces of their own."""
    r = random.Random(3)
    made, streams = [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for N in (20000, 30000):
        table, lens, ring, head, count = batch(r, 40, 100, 64, N)
        parents, keep = plan(r, 40, 100, 64)
        made.append((i32(parents), i32(keep), i32(lens), i32(table), i32(ring), i32([head, count])))

    def calls(m):
        ring = m[4].clone()
        fork = ext.cache_fork(m[0], m[1], m[2], m[3], ring, m[5], 64)
        return [ring] + fork + ext.cache_compact(fork[0], fork[1], ring, fork[2], 64)
    want = [calls(m) for m in made]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(4):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(calls(made[i]))
    torch.cuda.synchronize()
    for w, gs in zip(want, got):
        assert all(torch.equal(a, b) for g in gs for a, b in zip(g, w))
