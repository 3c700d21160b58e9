"""CPU checks of the blocked 8-bit cache's item bound over many row tiles: the attention's grid and
partial rows are sized for it, and a prefill batch's partial rows are most of its memory."""

from __future__ import annotations

import ctypes
import os
import subprocess

import numpy as np
import pytest

import wl_check as W
from test_worklist_cpu import distributions

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADS = 128


@pytest.fixture(scope="module")
def bound(tmp_path_factory):
    d = tmp_path_factory.mktemp("bound")
    (d / "bound.cpp").write_text('#include "worklist.h"\nextern "C" int bound(int B, int rt, int Sk) '
                                 '{ return mla::wl_max_items16(B, rt, Sk); }\n')
    subprocess.run(["g++", "-O2", "-std=c++17", "-shared", "-fPIC", "-I", W.CSRC, str(d / "bound.cpp"), "-o",
                    str(d / "bound.so")], check=True)
    return ctypes.CDLL(str(d / "bound.so")).bound


def worst_list(B, rt, Sk, seed):
    """The most items over equal lengths (every dense split that a length up to Sk takes) and over
    ragged draws."""
    most, h = B, W.harness()
    for L in list(range(32, min(Sk, 8192) + 1, 32)) + list(range(8192, Sk + 1, 512)) + [Sk]:
        k = h.wl_harness_dense_keys(L, B * rt, 32)
        most = max(most, B * -(-L // k))
    rng = np.random.default_rng(seed)
    for _, lens in distributions(B, Sk, rng):
        most = max(most, int(W.build_serial(lens, Sk, rt, 32, 40 * B + 4096)[0]))
    return most


@pytest.mark.parametrize("Sk", [2048, 4992, 32768])
@pytest.mark.parametrize("B,Sq", [(1, 2000), (4, 333), (7, 300), (11, 1000), (15, 4000), (32, 512), (100, 700)])
def test_many_row_tiles_have_no_slots_to_spare(bound, B, Sq, Sk):
    """From 600 row tiles up the bound is the longest list there is, in whole eights."""
    rt = W.row_tiles_of(Sq, HEADS)
    assert rt >= 600
    worst = worst_list(B, rt, Sk, B)
    assert bound(B, rt, Sk) == -(-worst // 8) * 8


@pytest.mark.parametrize("row_tiles", [1, 2, 5, 40, 86, 300, 666, 3000])
def test_the_bound_covers_every_list_of_its_span(bound, row_tiles):
    for B in (1, 2, 3, 4, 6, 9, 15, 40, 66, 129, 131, 200, 257, 300):
        for Sk in (64, 640, 4992, 16384, 131072, 2097088):
            assert bound(B, row_tiles, Sk) % 8 == 0
            assert bound(B, row_tiles, Sk) >= worst_list(B, row_tiles, Sk if Sk < 1e6 else 200000, B), (B, Sk)


def test_workspace_of_a_long_prefill():
    """15 sequences of 4,000 queries over up to 32,768 keys: rows in float32 and 16 partial slots."""
    import mla_custom_cuda  # noqa: F401  (torch's HIP runtime first)
    from test_blocked_cache_cpu import BF16, dims

    lib = ctypes.CDLL(os.path.join(ROOT, "mla-cuda_amd", "libmla_amd.so"))
    lib.mla_attention_paged_fp8blk_workspace_bytes.restype = ctypes.c_size_t
    d = dims(batch=15, sq=4000, sk=32768)
    rows = 4000 * HEADS
    got = lib.mla_attention_paged_fp8blk_workspace_bytes(BF16, ctypes.byref(d), 1, 64)
    assert (15 + 16) * rows * 512 * 4 < got < 1.02 * (15 + 16) * rows * 512 * 4
