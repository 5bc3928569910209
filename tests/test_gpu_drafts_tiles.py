"""GPU tests of attention of drafted tokens in every tile that a call may get, over pages of any size, and in calls whose
entries differ much. The tile's rows are read from the workspace that the call asks for."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

import pa_amd
from drafts import Cache, random_tree
from pa_amd import _lib
from test_gpu_drafts import check_attention, cols_for, run_attention

pytestmark = [pytest.mark.gpu, pytest.mark.usefixtures("gpu_device")]


def tile_rows(cache, entries, hq):
    """Rows of the call's tiles: its workspace is 2 slots a block, 130 floats a row, and 32 bytes a block; one block a
    CU, or two where FP8 tiles have 128 rows or fewer."""
    c = _lib.CachedTokens()
    c.num_tokens, c.num_entries = sum(n for _, n in entries), len(entries)
    c.block_table_stride, c.num_table_rows = cache.table.shape[1], cache.table.shape[0]
    c.num_pages, c.page_size, c.num_kv_heads = cache.pages, cache.page, cache.hkv
    dtype = {"fp16": pa_amd.FP16, "fp8": pa_amd.FP8_E4M3, "block": pa_amd.FP8_E4M3_BLOCK}[cache.kind]
    need = ctypes.c_size_t()
    assert _lib.load().pa_tree_attention_workspace(dtype, ctypes.byref(c), hq, ctypes.byref(need)) == _lib.PA_OK
    cus = torch.cuda.get_device_properties(0).multi_processor_count
    for rows in (64, 128, 256):
        grid = cus * (2 if cache.kind != "fp16" and rows <= 128 else 1)
        if need.value == grid * (2 * rows * 130 * 4 + 32):
            return rows
    raise AssertionError(need.value)


# Entries that a tile of 64, 128 and 256 rows is chosen for (with 2 heads a kv head 40, 108 and 329 rows on average),
# with tiles that are cut over blocks and ones that are not full.
SIZES = {64: [(700, 30), (0, 1), (33, 28)], 128: [(45, 30), (700, 70), (1500, 61)], 256: [(45, 30), (700, 130), (2100, 333)]}


@pytest.mark.parametrize("kind,page", [("fp16", 1), ("fp16", 3), ("fp16", 5), ("fp16", 4), ("fp16", 100), ("fp8", 1), ("fp8", 3),
                                       ("fp8", 5), ("fp8", 4), ("block", 8), ("block", 24), ("block", 16)])
@pytest.mark.parametrize("rows", list(SIZES))
@pytest.mark.parametrize("chain", [False, True])
def test_every_tile_over_pages_of_any_size(kind, page, rows, chain):
    entries = SIZES[rows]
    cache = Cache(kind, page, 2, len(entries), cols_for(entries, page), seed=page + rows)
    assert tile_rows(cache, entries, 4) == rows
    trees = None if chain else [random_tree(np.random.default_rng(i), n, spread=20) for i, (_, n) in enumerate(entries)]
    out, q = run_attention(cache, entries, 4, trees)
    check_attention(cache, entries, 4, trees, out, q)


@pytest.mark.parametrize("kind", ["fp16", "fp8", "block"])
@pytest.mark.parametrize("singles,rows", [(60, 64), (20, 128), (6, 256)])
def test_single_tokens_beside_a_piece_of_a_prompt(kind, singles, rows):
    """A server's mixed step: many sequences with one new token, one with a piece of its prompt, which sees its own
    earlier places and in a chain of its own."""
    r = np.random.default_rng(singles)
    entries = [(int(r.integers(0, 400)), 1) for _ in range(singles)]
    entries.insert(singles // 2, (130, 300))
    cache = Cache(kind, 16, 2, len(entries), cols_for(entries, 16), seed=singles)
    assert tile_rows(cache, entries, 16) == rows
    out, q = run_attention(cache, entries, 16, None)
    check_attention(cache, entries, 16, None, out, q)
