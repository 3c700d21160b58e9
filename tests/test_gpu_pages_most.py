"""GPU checks of the page operators at the most that their calls take: requests of a fork and a compaction, pairs of a
copy (tests/shared_pages.py: equal)."""

from __future__ import annotations

import random

import pytest
import torch

from test_gpu_pages import DEV, check_compact, check_fork, ext, plan  # noqa: F401
from test_shared_pages_cpu import batch

pytestmark = pytest.mark.gpu


def test_most_requests(ext):
    B, max_pages, N = 1 << 16, 2, 100000
    r = random.Random(1)
    table, lens, ring, head, count = batch(r, B, max_pages, 64, N)
    check_fork(ext, *plan(r, B, max_pages, 64), lens, table, ring, head, count, 64)
    check_compact(ext, lens, table, ring, head, count, 64)


@pytest.mark.parametrize("layers", [1, 3])
def test_more_pairs_than_a_launch_has_threads_for(ext, layers):
    """2^30 pairs and a few: 2^24 workgroups of 256 threads for 64 pairs each would be 2^32 threads."""
    n = (1 << 30) + 65
    copies = torch.full((n, 2), -1, dtype=torch.int32, device=DEV)
    pool = torch.arange(layers * 40 * 4, dtype=torch.int32, device=DEV).view(layers, 40, 4).contiguous()
    want = pool.clone()
    at = [0, 63, 64, 1 << 29, (1 << 30) - 1, 1 << 30, n - 1]
    for i, k in enumerate(at):
        copies[k, 0], copies[k, 1] = 2 * i, 2 * i + 1
        want[:, 2 * i + 1] = want[:, 2 * i]
    ext.cache_copy_pages(copies, [pool], layered=True)
    assert torch.equal(pool, want)
