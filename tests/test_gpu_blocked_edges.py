"""GPU checks of the blocked 8-bit cache at the ends of its scales' range."""

from __future__ import annotations

import pytest
import torch

import blocked_cache as K
from test_gpu_blocked_cache import DT, F32, append_inputs, check_append, ext, run_append  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("block", [16, 32, 64])
@pytest.mark.parametrize("byte", [253, 254])
def test_append_under_the_largest_scales(ext, dt, block, byte):  # noqa: F811
    """New rows in blocks that already have the scale 2^126 or 2^127, their values up to 2^124 (gain and
    W's rope columns times 2^122): codes under that scale, not zeros."""
    lens, new, Sq = [block // 2 + 9, block + 8], [9, 5], 9
    cache, x, W, gain, table = append_inputs(lens, new, Sq, block, 64, F32, byte)
    W[:, K.KV:] *= 2.0 ** 122
    x, W, gain = x.to(DT[dt]), W.to(DT[dt]), (gain * 2.0 ** 122).to(DT[dt])
    for b in range(2):     # the block that keeps rows: the first of sequence 0, the second of sequence 1
        row = int(K.slots_of(table, b, lens[b] - new[b], lens[b] - new[b] + 1, 64)[0])
        cache["scales"].view(-1, 2)[row // block] = byte
    after = run_append(ext, cache, x, W, gain, lens, new, table)
    want = K.append(cache, x, W, gain, lens, new, table, 64, block)
    kept = want["touched"] & (want["e"][:, 0] == byte - 127)
    assert int(kept.sum()) >= 1
    check_append(cache, after, want, block)
