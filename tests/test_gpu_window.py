"""Windowed decode attention on an MI355X against its formula in 64 bits."""
from __future__ import annotations

import copy

import numpy as np
import pytest
import torch

import budget_cases as C
import window_cases as W
from test_gpu_budget import DEV, GEOMETRIES, TYPES, dev, largest_row, queries, tensors
from turboquant_amd import ops

pytestmark = pytest.mark.gpu


def check_o(c, got, ref, q, dtype, window, sink):
    """u = 2^-24.  A score: K levels as fp16 (8.7e-5 relative), q' as a hi + lo
    pair (4 u), a chain of at most 2 pd / 16 fp32 sums and eight roundings, all
    relative to |q| |K| (Cauchy-Schwarz); a probability is off by twice that.
    The output in front of its own rounding: the probability times the V norm as
    fp16 (half a step, 2^-11, of it; below 2^-14 half a step of 2^-24 for each
    of the n tokens in sight, times a level of at most 2.74 and the tables'
    scale 1.481, per coordinate), the V levels as fp16, the partial rows as fp16
    (2^-11) and fp32 sums; no rotation makes an error longer."""
    u = 2.0 ** -24
    half = {"fp16": 2.0 ** -11, "bf16": 2.0 ** -8}[dtype]
    qn = float(np.sqrt((q ** 2).sum(-1)).max()) if q.size else 0.0
    score = qn * largest_row(c, 0) * c.scale * (8.7e-5 + (4 + c.pd / 8 + 8) * u)
    n = min(int(max(c.lens, default=0)), window + sink)
    row = (2 * score + 2.0 ** -11 + 8.7e-5 + 2.0 ** -11 + 64 * u) * largest_row(c, 1)
    row += n * 2.0 ** -25 * 2.74 * 1.481 * c.pd ** 0.5
    tol = half * np.abs(ref) + row * (1 + half) + 2.0 ** -24
    err = np.abs(got.double().cpu().numpy() - ref)
    assert (err <= tol).all(), f"o off by {err.max():.3e}, {(err / tol).max():.2f} x bound"


def call(c, t, q, o, window, sink, signs=True):
    return ops.decode_paged_window(q, t["cache"], t["indices"], t["indptr"], t["seq"], c.hkv, c.hd,
                                   c.pd, c.scale, t["signs"] if signs else None, o, window, sink)


def run(c, window, sink, dtype="fp16", o_dtype=None, q_scale=1.0, signs=True, hide=True):
    """One call, hidden entries and table entries spoiled; (tensors, q, o)"""
    if hide:
        W.poison(W.release(c, window, sink), window, sink)
    t = tensors(c)
    b = len(c.lens)
    q, qx = queries(c, b, dtype, q_scale)
    o = torch.full((b, c.hq, c.hd), 7.0, dtype=TYPES[o_dtype or dtype], device=DEV)
    assert call(c, t, q, o, window, sink, signs) is o
    torch.cuda.synchronize()
    clean = copy.copy(c)
    clean.cache = c.cache.copy()
    norms = clean.cache[..., c.pd // 2:c.pd // 2 + 2].copy().view(np.float16)
    clean.cache[..., c.pd // 2:c.pd // 2 + 2] = np.where(np.isfinite(norms), norms, 0) \
        .astype(np.float16).view(np.uint8)  # (for the bound's largest row)
    check_o(clean, o, W.decode(c, qx, window, sink, signs), qx, o_dtype or dtype, window, sink)
    assert np.array_equal(t["cache"].cpu().numpy(), c.cache)
    return t, q, o


@pytest.mark.parametrize("hq,hkv,hd", GEOMETRIES)
def test_geometries(hq, hkv, hd):
    c = C.make(hq * 1000 + hkv, [1, 37, 300, 16, 171], hq, hkv, hd)
    run(c, 100, 4, "bf16" if hkv % 2 else "fp16")


@pytest.mark.parametrize("window", [1, 2, 15, 16, 17, 31, 32, 33, 48, 100, 2 ** 31 - 1])
@pytest.mark.parametrize("sink", [0, 1, 4, 16, 17, 40, 2 ** 31 - 1])
def test_borders(window, sink):
    """Every place of the window's and the sinks' borders within a tile."""
    lens = [0, 1, 5, 16, 17, 63, 64, 65, 79, 80, 81, 200, 207, 208, 209, 215]
    run(C.make(window % 1000 + sink % 1000, lens, 8, 2, 64), window, sink)


@pytest.mark.parametrize("page", [16, 32, 48])
@pytest.mark.parametrize("packed", [True, False])
def test_pages(page, packed):
    c = C.make(page, [500, 77, 0, 96, 333], 4, 2, 128, page=page, packed=packed)
    run(copy.deepcopy(c), 70, 5)
    run(c, 129, 20, "bf16")


@pytest.mark.parametrize("dtype,o_dtype", [("fp16", "bf16"), ("bf16", "fp16"), ("bf16", "bf16")])
def test_types(dtype, o_dtype):
    run(C.make(7, [129, 500], 16, 4, 128), 64, 4, dtype, o_dtype)


def test_without_rotation_and_extreme_scores():
    run(C.make(8, [129, 40], 8, 2, 64), 50, 3, signs=False)
    run(C.make(10, [700, 64], 8, 2, 128), 300, 4, q_scale=8.0)
    run(C.make(11, [700, 64], 8, 2, 128), 300, 4, q_scale=0.0)


@pytest.mark.parametrize("batch", [65, 130, 1024, 1025, 2100])
def test_many_sequences(batch):
    rng = np.random.default_rng(batch)
    run(C.make(batch, rng.integers(0, 90, batch).tolist(), 4, 2, 64), 30, 2)


@pytest.mark.parametrize("lens,window,sink", [([9001], 1024, 4), ([4000, 3, 2500], 2000, 100),
                                              ([20000] * 3, 5000, 1)])
def test_long(lens, window, sink):
    run(C.make(len(lens), lens, 8, 2, 128), window, sink)


def test_a_window_beyond_the_sequence_is_full_attention():
    """Within the same bounds as the decode over every token (whose split of the
    work, and so its order of the sums, is another)."""
    c = C.make(12, [500, 33, 1, 0, 1200], 32, 8, 128)
    t, q, o = run(c, 2000, 7)
    qx = q.double().cpu().numpy()
    rows = ops.balanced_rows(5, 32, 8, 128)
    full = torch.empty_like(o)
    ops.decode_paged_balanced(q, t["cache"], t["indices"], t["indptr"], t["seq"], 8, 128, 128,
                              c.scale, t["signs"], full,
                              torch.empty((rows, 32, 128), device=DEV),
                              torch.empty((rows, 32), device=DEV),
                              torch.empty(7, dtype=torch.int32, device=DEV))
    ref = W.decode(c, qx, 2000, 7)
    check_o(c, full, ref, qx, "fp16", 2000, 7)
    check_o(c, o, ref, qx, "fp16", 2000, 7)


@pytest.mark.parametrize("hq,hkv,hd", [(8, 1, 64), (16, 2, 96), (12, 6, 128), (8, 8, 256),
                                       (16, 1, 128)])
@pytest.mark.parametrize("window,sink", [(192, 16), (200, 9), (384, 16), (385, 16), (4, 396), (1, 400)])
def test_where_one_launch_ends(hq, hkv, hd, window, sink):
    """Windows on both sides of the sizes that one launch takes, few sequences
    and more than workgroups of it would fit."""
    lens = [1500, 0, window, window + 1, window + sink + 40, 7, 800]
    run(C.make(hq + hd, lens, hq, hkv, hd), window, sink, "bf16")
    run(C.make(hq + hd + 1, lens * 38, hq, hkv, hd), window, sink)


def test_bad_pages_and_short_tables_are_empty():
    c = C.make(13, [200, 90, 64], 8, 2, 128)
    c.indices[11], c.indices[16], c.indices[0] = -1, c.nb, 2 ** 31 - 1
    c.lens[2] = 200  # nine pages behind the table's end
    run(c, 100, 20, hide=False)
    c = C.make(14, [32, 48], 8, 2, 128)
    c.indices[:2] = -1  # a sequence with nothing in the cache
    _, _, o = run(c, 10, 2, hide=False)
    assert (o[0] == 0).all()


def test_nan_and_inf_in_sight_stay_with_their_head():
    c = C.make(15, [100, 80], 8, 2, 128)
    pg, off, _ = C.places(c, 0)
    c.cache[0, pg[95], off[95], 1, 64:68].view(np.float16)[:] = np.nan
    t = tensors(c)
    q, _ = queries(c, 2, "fp16")
    o = torch.empty((2, 8, 128), dtype=torch.float16, device=DEV)
    call(c, t, q, o, 20, 0)
    o = o.float().cpu().numpy()
    assert np.isnan(o[0, 4:]).all() and np.isfinite(o[0, :4]).all() and np.isfinite(o[1]).all()


def test_strides_alignment_and_tables_with_a_start():
    c = W.release(C.make(16, [300, 41], 8, 2, 128), 64, 4)
    t = tensors(c)
    q, qx = queries(c, 2, "bf16")
    first = call(c, t, q, torch.empty_like(q), 64, 4).clone()
    wide = torch.full((2, 11, 200), 5.0, dtype=torch.bfloat16, device=DEV)
    for rows in (wide[:, 3:, 72:], wide[:, :8, 1:129], wide[:, ::1, 8:136][:, 2:10]):
        rows.copy_(q)
        assert torch.equal(call(c, t, rows, torch.empty_like(q), 64, 4), first)
    flip = torch.empty((8, 2, 128), dtype=torch.bfloat16, device=DEV).transpose(0, 1)
    flip.copy_(q)
    assert torch.equal(call(c, t, flip, torch.empty_like(q), 64, 4), first)
    # the second sequence's table further in, the first's behind it
    it = t["indices"]
    t["indices"] = torch.cat((it.new_full((3,), -9), it[19:], it[:19]))
    t["indptr"] = torch.tensor([3 + len(it) - 19, 3], dtype=torch.int32, device=DEV)
    assert torch.equal(call(c, t, q, torch.empty_like(q), 64, 4), first)


def test_repeated_calls_other_streams_and_a_graph():
    c = C.make(17, [900, 300, 64, 1300], 16, 4, 128)
    t = tensors(c)
    q, qx = queries(c, 4, "fp16")
    o = torch.empty_like(q)
    first = call(c, t, q, o, 256, 4).clone()
    for _ in range(3):
        assert torch.equal(call(c, t, q, torch.empty_like(q), 256, 4), first)
    # two calls at once
    s = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    outs = []
    for i in range(6):
        with torch.cuda.stream(s[i % 2]):
            outs.append(call(c, t, q, torch.empty_like(q), 256, 4))
    torch.cuda.synchronize()
    assert all(torch.equal(x, first) for x in outs)
    # captured, replayed with other lengths and eager work in between
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call(c, t, q, o, 256, 4)
    for lens in ([900, 300, 64, 1300], [1, 0, 30, 1299], [899, 257, 2, 40]):
        c.lens[:] = lens
        t["seq"].copy_(dev(c.lens))
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, call(c, t, q, torch.empty_like(q), 256, 4))
        check_o(c, o, W.decode(c, qx, 256, 4), qx, "fp16", 256, 4)


def test_registered_op():
    ops.register_ops()
    c = C.make(18, [100, 40], 8, 2, 64)
    t = tensors(c)
    q, qx = queries(c, 2, "fp16")
    o = torch.zeros_like(q)
    torch.ops.turboquant_v5.decode_paged_window(q, t["cache"], t["indices"], t["indptr"], t["seq"],
                                                2, 64, 64, c.scale, t["signs"], o, 30, 2)
    check_o(c, o, W.decode(c, qx, 30, 2), qx, "fp16", 30, 2)


def test_cache_beyond_32_bit_offsets():
    """Pages whose byte offsets inside a slab pass 2^32, at the table's end and
    at both borders."""
    c = C.make(19, [80, 333], 8, 8, 128)
    far = 440_000  # a page of one slab is 10240 bytes
    nb = far + c.nb
    cache = torch.empty((2, nb, 16, 8, 80), dtype=torch.uint8, device=DEV)
    cache[:, far:].copy_(dev(c.cache))
    t = tensors(c)
    q, qx = queries(c, 2, "fp16")
    o = torch.empty_like(q)
    ops.decode_paged_window(q, cache, t["indices"] + far, t["indptr"], t["seq"], 8, 128, 128,
                            c.scale, t["signs"], o, 100, 20)
    check_o(c, o, W.decode(c, qx, 100, 20), qx, "fp16", 100, 20)


def test_a_long_sequence_among_many():
    """256 sequences, one of 36 million tokens with all of them in its window:
    a unit's share of a pair is a product beyond 2^31."""
    c = C.make(20, [16 * 40 + 9] + [1] * 255, 2, 1, 128)
    entries = 36_000_000 // 16
    length = (entries - 1) * 16 + 9
    at = np.sort(np.concatenate(([entries - 1], c.rng.permutation(entries - 1)[:40])))
    table = np.full(entries + 255, -1, np.int32)
    table[at], table[entries:] = c.indices[:41], c.indices[41:]
    indptr = np.concatenate(([0], entries + np.arange(256))).astype(np.int32)
    t = tensors(c)
    seq = t["seq"].clone()
    seq[0] = length
    q, qx = queries(c, 256, "fp16")
    o = torch.full((256, 2, 128), 7.0, dtype=torch.float16, device=DEV)
    ops.decode_paged_window(q, t["cache"], dev(table), dev(indptr), seq, 1, 128, 128, c.scale,
                            t["signs"], o, 2 ** 31 - 1, 0)
    # the pages that are there, as one sequence
    check_o(c, o, W.decode(c, qx, 2 ** 31 - 1, 0), qx, "fp16", 2 ** 20, 0)
