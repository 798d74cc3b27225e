"""Workspaces of the cache-budget operators go by what a call can need, not by
how wide its page table is."""
from __future__ import annotations

import copy

import numpy as np
import pytest
import torch

import budget_cases as C
from test_gpu_budget import (DEV, check_o, check_weights, dev, queries, run_evict, spread,
                             tensors)
from turboquant_amd import _lib, ops

pytestmark = pytest.mark.gpu


def widened(c, width):
    """The same sequences with table rows of `width` pages (-1 behind the pages)."""
    d = copy.copy(c)
    need = np.diff(c.indptr)
    d.indices = np.full(len(c.lens) * width, -1, np.int32)
    d.indptr = (np.arange(len(c.lens) + 1) * width).astype(np.int32)
    for b, n in enumerate(need):
        d.indices[b * width:b * width + n] = c.indices[c.indptr[b]:c.indptr[b] + n]
    return d


def peak(call):
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    call()
    torch.cuda.synchronize()
    return torch.cuda.max_memory_allocated() - before


def decode(c, q):
    t = tensors(c)
    o = torch.full(tuple(q.shape), 7.0, dtype=torch.float16, device=DEV)
    return t, o, lambda: ops.decode_paged_tracked(
        q, t["cache"], t["indices"], t["indptr"], t["seq"], c.hkv, c.hd, c.pd, c.scale, t["signs"], o,
        t["weights"], t["positions"], t["ends"])


@pytest.mark.parametrize("hq,hkv,hd,page", [(8, 2, 128, 16), (16, 1, 64, 48), (4, 4, 256, 16)])
def test_decode_over_a_table_wider_than_the_cache(hq, hkv, hd, page):
    """Scores by page of the cache instead of by table entry: the same bits."""
    c = C.make(301 + hd, [700, 33, 0, 129], hq, hkv, hd, page=page)
    wide = widened(c, 1000)
    for d in (c, wide):  # pages outside the cache
        d.indices[d.indptr[0] + 2], d.indices[d.indptr[3] + 1] = -1, c.nb
    assert len(c.indices) < c.nb < len(wide.indices)
    q, qx = queries(c, 4, "fp16")
    got = []
    for d in (c, wide):
        t, o, call = decode(d, q)
        call()
        torch.cuda.synchronize()
        got.append((o, t["weights"], t["positions"]))
    ref_o, ref_w, ref_p = C.attend(wide, qx, np.arange(5), 1, True, decode=True)
    check_weights(c, got[1][1].cpu().numpy(), ref_w, qx, hq // hkv)
    check_o(c, got[1][0], ref_o, qx, "fp16")
    assert np.array_equal(got[1][2].cpu().numpy(), ref_p)
    for a, b in zip(*got):
        assert torch.equal(a, b)


def test_decode_workspace_goes_by_the_cache():
    """256 rows of a table for 131072 tokens each over a cache of 4200 tokens."""
    c = widened(C.make(310, [16] * 255 + [100], 32, 8, 128), 131072 // 16)
    q, _ = queries(c, 256, "fp16")
    _, _, call = decode(c, q)
    # scores of the cache's tokens, and the partial rows of at most 1024 parts
    most = c.nb * 16 * 32 * 4 + 1024 * 32 * (128 * 4 + 2 * 8) + (1 << 20)
    assert peak(call) <= most


def test_decode_refuses_a_workspace_that_is_too_small():
    c = C.make(311, [100, 20], 8, 2, 128)
    lib = _lib.load()
    t = tensors(c)
    q, _ = queries(c, 2, "fp16")
    o = torch.zeros((2, 8, 128), dtype=torch.float16, device=DEV)
    for table in (t["indices"], dev(widened(c, 50).indices)):
        pages = min(table.numel(), c.nb)
        need = lib.tq_decode_tracked_workspace_bytes(2, pages, 8, 2, 128, 16)
        assert need > lib.tq_decode_tracked_workspace_bytes(2, pages - 1, 8, 2, 128, 16)
        ws = torch.empty(need, dtype=torch.uint8, device=DEV)
        for size, want in ((need, 0), (need - 1, -22)):
            rc = lib.tq_decode_paged_tracked(
                q.data_ptr(), 1024, 128, 1, t["cache"].data_ptr(), t["cache"][1].data_ptr(),
                table.data_ptr(), table.numel(), t["indptr"].data_ptr(), t["seq"].data_ptr(), 2, 8, 2,
                128, 128, 16, 80, c.nb, c.scale, None, o.data_ptr(), 1, t["weights"].data_ptr(), None,
                None, ws.data_ptr(), size, torch.cuda.current_stream().cuda_stream)
            assert rc == want
    torch.cuda.synchronize()


@pytest.mark.parametrize("page,packed", [(16, True), (48, False)])
def test_evict_with_lists_by_table_place(page, packed):
    """300 sequences under a budget of 20000: lists of their own for every row
    would be over 64 MiB, so they stand where the sequences' tokens do.  One
    sequence is cut by one entry, one to half, one beyond 32768 tokens."""
    lens = [(7 * b) % 60 for b in range(300)]
    lens[3], lens[100], lens[299] = 20001, 40000, 26017
    if not packed:
        lens[100] = 33000
    c = spread(C.make(320 + page, lens, 2, 2, 64, page=page, packed=packed))
    own = 300 * 2 * 20000 * 8
    assert own > 64 << 20
    got = _lib.load().tq_evict_workspace_bytes(300, 2, len(c.indices), page, 20000)
    assert got < own or not packed
    run_evict(c, 20000, 700, 4)


def test_evict_lists_by_table_place_of_bad_tables():
    """... with pages outside the cache and tokens behind the table."""
    lens = [(7 * b) % 60 for b in range(300)]
    lens[3], lens[299] = 20500, 45000
    c = spread(C.make(331, lens, 2, 2, 64))
    for at in (5, 700, 1290, len(c.indices) - 2, len(c.indices) - 900):
        c.indices[at] = -1 if at % 2 else c.nb
    c.lens[299] = 47000
    run_evict(c, 20000, 300, 4)
