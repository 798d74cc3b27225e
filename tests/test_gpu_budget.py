"""The cache-budget operators on an MI355X against their formulas in 64 bits:
tracked decode, window weights, eviction, and a run of the three together."""
from __future__ import annotations

import copy
import math

import numpy as np
import pytest
import torch

import budget_cases as C
from turboquant_amd import ops

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).to(DEV)


def tensors(c):
    return dict(cache=dev(c.cache), indices=dev(c.indices), indptr=dev(c.indptr), seq=dev(c.lens),
                weights=dev(c.weights), positions=dev(c.positions), ends=dev(c.ends),
                signs=dev(c.signs))


def queries(c, rows, dtype, scale=1.0):
    """(as the kernel gets them, their exact values)"""
    q = torch.from_numpy(c.rng.standard_normal((rows, c.hq, c.hd)) * scale).to(TYPES[dtype])
    return q.to(DEV), q.double().numpy()


def largest_row(c, slab):
    """Largest 2-norm of a dequantized row of the case's tokens."""
    top = 0.0
    for b in range(len(c.lens)):
        pg, off, ok = C.places(c, b)
        for h in range(c.hkv):
            if ok.any():
                top = max(top, float(np.sqrt((C.rows(c, slab, pg[ok], off[ok], h) ** 2).sum(-1))
                                     .max()))
    return top


def score_error(c, q):
    """Bound on the absolute error of a score (natural units): u = 2^-24.
    Operands are hi + lo pairs, off by 2^-22 = 4 u relative each (8 u together);
    a score is a chain of at most 2 pd / 16 MFMA sums of products in fp32, each
    off by u relative to |q| |K| (Cauchy-Schwarz), and goes through at most
    eight fp32 roundings (norm, constants, log2 units, exp2's argument)."""
    u = 2.0 ** -24
    qn = float(np.sqrt((q ** 2).sum(-1)).max()) if q.size else 0.0
    return qn * largest_row(c, 0) * c.scale * (8 + c.pd / 8 + 8) * u


def check_weights(c, got, ref, q, seen):
    """A probability is exp(s - lse): relative error twice a score's (lse is a
    mean of scores), plus exp2, log2 and sums: a chain of up to 64 fp32
    roundings covers them at these sizes; `seen` queries x heads add up, and one
    rounding of the new sum."""
    u = 2.0 ** -24
    rel = 2 * score_error(c, q) + 64 * u
    added = np.abs(ref - np.where(np.isfinite(c.weights), c.weights, 0))
    tol = rel * np.maximum(np.abs(ref), np.minimum(added, seen)) + 2 * u * np.abs(ref) + 1e-37
    err = np.abs(got.astype(np.float64) - ref)
    assert (err <= tol).all(), f"weights off by {err.max():.3e}, {(err / tol).max():.2f} x bound"


def check_o(c, got, ref, q, dtype):
    """The output's rounding, and in front of it errors that no rotation makes
    longer: the V levels as fp16 (8.7e-5), probabilities as hi + lo pairs
    (2^-22; 2^-11 alone above 8 q heads per kv head) and their own error."""
    half = {"fp16": 2.0 ** -11, "bf16": 2.0 ** -8}[dtype]
    p = (2.0 ** -22 if c.hq // c.hkv <= 8 else 2.0 ** -11) + 2 * score_error(c, q) + 2.0 ** -18
    tol = half * np.abs(ref) + (8.7e-5 + p) * largest_row(c, 1) * (1 + half) + 2.0 ** -24
    err = np.abs(got.double().cpu().numpy() - ref)
    assert (err <= tol).all(), f"o off by {err.max():.3e}, {(err / tol).max():.2f} x bound"


def run_decode(c, dtype="fp16", q_scale=1.0, o_dtype=None, record=True, signs=True):
    t = tensors(c)
    b = len(c.lens)
    q, qx = queries(c, b, dtype, q_scale)
    o = torch.full((b, c.hq, c.hd), 7.0, dtype=TYPES[o_dtype or dtype], device=DEV)
    ops.decode_paged_tracked(q, t["cache"], t["indices"], t["indptr"], t["seq"], c.hkv, c.hd, c.pd,
                             c.scale, t["signs"] if signs else None, o, t["weights"],
                             t["positions"] if record else None, t["ends"] if record else None)
    torch.cuda.synchronize()
    ref_o, ref_w, ref_p = C.attend(c, qx, np.arange(b + 1), 1, signs, decode=True)
    check_weights(c, t["weights"].cpu().numpy(), ref_w, qx, c.hq // c.hkv)
    check_o(c, o, ref_o, qx, o_dtype or dtype)
    if not record:
        ref_p = c.positions
    assert np.array_equal(t["positions"].cpu().numpy(), ref_p)
    assert np.array_equal(t["cache"].cpu().numpy(), c.cache)
    return t, o


GEOMETRIES = [(32, 8, 128), (16, 4, 64), (16, 2, 256), (8, 1, 128), (12, 4, 96), (8, 8, 64),
              (32, 2, 128), (6, 3, 80), (10, 10, 128), (16, 1, 256), (24, 12, 64), (5, 1, 40),
              (4, 4, 256), (2, 2, 128), (12, 1, 64)]


@pytest.mark.parametrize("hq,hkv,hd", GEOMETRIES)
def test_decode_geometries(hq, hkv, hd):
    c = C.make(hq * 1000 + hkv, [1, 37, 300, 16, 17], hq, hkv, hd)
    run_decode(c, "bf16" if hkv % 2 else "fp16")


@pytest.mark.parametrize("lens", [[1], [15], [16], [33], [0, 5, 0], [0], [1000, 1, 31, 32],
                                  [2049, 700]])
@pytest.mark.parametrize("page", [16, 48])
def test_decode_lengths(lens, page):
    run_decode(C.make(len(lens) + page, lens, 8, 2, 128, page=page, packed=page == 16), "fp16")


@pytest.mark.parametrize("dtype,o_dtype", [("fp16", "bf16"), ("bf16", "fp16"), ("bf16", "bf16")])
def test_decode_types(dtype, o_dtype):
    run_decode(C.make(7, [129, 500], 16, 4, 128), dtype, o_dtype=o_dtype)


def test_decode_without_rotation_or_positions():
    run_decode(C.make(8, [129, 40], 8, 2, 64), signs=False)
    run_decode(C.make(9, [129, 40], 8, 2, 64), record=False)


def test_decode_peaked_and_flat():
    """Scores of +-60: one token takes nearly all; and all equal."""
    run_decode(C.make(10, [700, 64], 8, 2, 128), q_scale=8.0)
    c = C.make(11, [700, 64], 8, 2, 128)
    t, _ = run_decode(c, q_scale=0.0)
    w = t["weights"].cpu().numpy()
    pg, off, _ = C.places(c, 1)
    assert np.abs(w[pg[63], 0, off[63]] - 4 / 64) < 1e-6


@pytest.mark.parametrize("batch", [65, 130])
def test_decode_many_short(batch):
    rng = np.random.default_rng(batch)
    run_decode(C.make(batch, rng.integers(0, 70, batch).tolist(), 4, 2, 64))


def test_decode_bad_pages_are_empty():
    """Page ids outside the cache, and tokens behind the table."""
    c = C.make(12, [200, 90, 64], 8, 2, 128)
    c.indices[3], c.indices[7], c.indices[14] = -1, c.nb, 2 ** 31 - 1
    c.lens[2] = 200  # nine pages behind the table's end
    run_decode(c)
    c = C.make(13, [32, 48], 8, 2, 128)
    c.indices[:2] = -1  # a sequence with nothing in the cache
    _, o = run_decode(c)
    assert (o[0] == 0).all()


def test_decode_nan_and_inf_stay_with_their_head():
    c = C.make(14, [100, 80], 8, 2, 128)
    pg, off, _ = C.places(c, 0)
    c.cache[0, pg[5], off[5], 1, 64:68].view(np.float16)[:] = np.nan
    t = tensors(c)
    q, qx = queries(c, 2, "fp16")
    o = torch.empty((2, 8, 128), dtype=torch.float16, device=DEV)
    ops.decode_paged_tracked(q, t["cache"], t["indices"], t["indptr"], t["seq"], 2, 128, 128,
                             c.scale, t["signs"], o, t["weights"], t["positions"], t["ends"])
    w = t["weights"].cpu().numpy()
    assert np.isnan(w[pg, 1, off]).all() and np.isfinite(w[pg, 0, off]).all()
    o = o.float().cpu().numpy()
    assert np.isnan(o[0, 4:]).all() and np.isfinite(o[0, :4]).all() and np.isfinite(o[1]).all()


def test_decode_reads_no_entry_behind_the_last_token():
    """NaN norms and weights behind the sequences' ends change nothing."""
    c = C.make(15, [37, 81], 8, 2, 128)
    for b in range(2):
        last = c.indices[c.indptr[b + 1] - 1]
        n = int(c.lens[b]) % 16
        c.cache[:, last, n:, :, 64:68] = 0xff
        c.weights[last, :, n:] = np.nan
    t, o = run_decode_ignoring_nan(c)
    w = t["weights"].cpu().numpy()
    for b in range(2):
        last = c.indices[c.indptr[b + 1] - 1]
        assert np.isnan(w[last, :, int(c.lens[b]) % 16:]).all()


def run_decode_ignoring_nan(c):
    t = tensors(c)
    q, qx = queries(c, len(c.lens), "fp16")
    o = torch.empty((len(c.lens), c.hq, c.hd), dtype=torch.float16, device=DEV)
    ops.decode_paged_tracked(q, t["cache"], t["indices"], t["indptr"], t["seq"], c.hkv, c.hd, c.pd,
                             c.scale, t["signs"], o, t["weights"], t["positions"], t["ends"])
    ref_o, ref_w, _ = C.attend(c, qx, np.arange(len(c.lens) + 1), 1, True, decode=True)
    got, keep = t["weights"].cpu().numpy(), np.isfinite(c.weights)
    c2 = copy.copy(c)
    c2.weights = np.where(keep, c.weights, 0)
    check_weights(c2, np.where(keep, got, 0), np.where(keep, ref_w, 0), qx, c.hq // c.hkv)
    check_o(c, o, ref_o, qx, "fp16")
    return t, o


def test_decode_strided_q_side_stream_and_graph():
    """q as a slice of fused rows; a captured call replayed with other lengths;
    the same bits every time."""
    c = C.make(16, [300, 90, 1], 16, 4, 128)
    t = tensors(c)
    q, qx = queries(c, 3, "bf16")
    fused = torch.zeros((3, 16 * 128 + 264), dtype=torch.bfloat16, device=DEV)
    fused[:, 8:8 + 2048] = q.reshape(3, -1)
    view = fused[:, 8:8 + 2048].view(3, 16, 128)
    o = torch.empty((3, 16, 128), dtype=torch.bfloat16, device=DEV)
    w0, p0 = t["weights"].clone(), t["positions"].clone()

    def call():
        t["weights"].copy_(w0)
        t["positions"].copy_(p0)
        ops.decode_paged_tracked(view, t["cache"], t["indices"], t["indptr"], t["seq"], 4, 128, 128,
                                 c.scale, t["signs"], o, t["weights"], t["positions"], t["ends"])
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        call()
    st.synchronize()
    ref_o, ref_w, ref_p = C.attend(c, qx, np.arange(4), 1, True, decode=True)
    check_weights(c, t["weights"].cpu().numpy(), ref_w, qx, 4)
    check_o(c, o, ref_o, qx, "bf16")
    first = (o.clone(), t["weights"].clone())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call()
    for lens in ([300, 90, 1], [17, 90, 0], [300, 1, 1], [300, 90, 1]):
        t["seq"].copy_(torch.tensor(lens, dtype=torch.int32))
        g.replay()
        torch.cuda.synchronize()
        got = (o.clone(), t["weights"].clone(), t["positions"].clone())
        call()
        torch.cuda.synchronize()
        for a, b in zip(got, (o, t["weights"], t["positions"])):
            assert torch.equal(a, b)
    assert torch.equal(first[0], o) and torch.equal(first[1], t["weights"])


# ------------------------------------------------------------------ windows

def run_window(c, chunks, window, dtype="fp16", record=True, signs=True, q_scale=1.0):
    t = tensors(c)
    starts = np.concatenate(([0], np.cumsum(chunks))).astype(np.int32)
    q, qx = queries(c, int(starts[-1]), dtype, q_scale)
    ops.track_window(q, dev(starts), window, t["cache"], t["indices"], t["indptr"], t["seq"], c.hkv,
                     c.hd, c.pd, c.scale, t["signs"] if signs else None, t["weights"],
                     t["positions"] if record else None, t["ends"] if record else None)
    torch.cuda.synchronize()
    _, ref_w, ref_p = C.attend(c, qx, starts, window, signs)
    check_weights(c, t["weights"].cpu().numpy(), ref_w, qx, window * c.hq // c.hkv)
    assert np.array_equal(t["positions"].cpu().numpy(), ref_p if record else c.positions)
    return t


@pytest.mark.parametrize("hq,hkv,hd", GEOMETRIES)
def test_window_geometries(hq, hkv, hd):
    c = C.make(hq * 1000 + hkv + 1, [1, 37, 300, 16], hq, hkv, hd)
    run_window(c, [1, 20, 40, 16], 9, "bf16" if hkv % 2 else "fp16")


@pytest.mark.parametrize("window", [1, 2, 31, 64, 256])
def test_window_sizes(window):
    run_window(C.make(window, [700, 33, 90], 8, 2, 128, page=32, packed=False), [300, 33, 1],
               window)


@pytest.mark.parametrize("lens,chunks", [([1], [1]), ([0, 5], [0, 5]), ([100, 50], [0, 50]),
                                         ([2049], [2049]), ([64, 0, 64], [64, 0, 1])])
def test_window_lengths(lens, chunks):
    run_window(C.make(sum(lens) + 1, lens, 12, 4, 96), chunks, 8)


def test_window_without_rotation_or_positions_and_peaked():
    run_window(C.make(21, [129, 40], 8, 2, 64), [50, 40], 8, signs=False)
    run_window(C.make(22, [129, 40], 8, 2, 64), [50, 40], 8, record=False)
    run_window(C.make(23, [700], 8, 2, 128), [700], 16, q_scale=8.0)


def test_window_bad_pages_are_empty():
    c = C.make(24, [200, 90, 64], 8, 2, 128)
    c.indices[3], c.indices[7], c.indices[14] = -1, c.nb, 2 ** 31 - 1
    c.lens[2] = 200
    run_window(c, [40, 90, 30], 16)


def test_window_of_one_is_the_decode_record():
    c = C.make(25, [333, 65], 8, 2, 128)
    t = run_window(c, [1, 1], 1)
    u = tensors(c)
    c2 = C.make(25, [333, 65], 8, 2, 128)
    q, _ = queries(c2, 2, "fp16")
    o = torch.empty((2, 8, 128), dtype=torch.float16, device=DEV)
    ops.decode_paged_tracked(q, u["cache"], u["indices"], u["indptr"], u["seq"], 2, 128, 128,
                             c.scale, u["signs"], o, u["weights"], u["positions"], u["ends"])
    assert torch.equal(t["positions"], u["positions"])
    assert torch.allclose(t["weights"], u["weights"], rtol=1e-4, atol=0)


# ------------------------------------------------------------------ eviction

def run_evict(c, budget, recent=0, sink=0, record=True):
    t = tensors(c)
    new = torch.full((len(c.lens),), -9, dtype=torch.int32, device=DEV)
    pos = t["positions"] if record else None
    ops.evict_paged(t["cache"], t["weights"], pos, t["indices"], t["indptr"], t["seq"],
                    t["ends"] if record else None, budget, recent, sink, new)
    torch.cuda.synchronize()
    d = c
    if not record:
        d = copy.copy(c)
        d.positions = np.zeros_like(c.positions)
    cache, acc, p, lens = C.evict(d, budget, recent, sink)
    assert np.array_equal(new.cpu().numpy(), lens)
    assert np.array_equal(t["weights"].cpu().numpy().view(np.int32), acc.view(np.int32))
    if record:
        assert np.array_equal(t["positions"].cpu().numpy(), p)
    assert np.array_equal(t["cache"].cpu().numpy(), cache)
    return t


def spread(c):
    """Positions as an earlier cut may have left them: any order, all different."""
    for b in range(len(c.lens)):
        pg, off, ok = C.places(c, b)
        for h in range(c.hkv):
            x = c.rng.permutation(int(c.ends[b]))[:len(pg)]
            c.positions[pg[ok], h, off[ok]] = x[ok]
    return c


@pytest.mark.parametrize("hq,hkv,hd", [(8, 8, 128), (4, 4, 64), (2, 2, 256), (1, 1, 96)])
@pytest.mark.parametrize("budget,recent,sink", [(64, 0, 0), (100, 20, 4), (1, 0, 0), (1, 1, 0),
                                                (300, 150, 150), (33, 0, 33), (1000, 10, 0)])
def test_evict(hq, hkv, hd, budget, recent, sink):
    run_evict(spread(C.make(budget + hkv, [300, 64, 1, 0, 65, 301], hq, hkv, hd)), budget, recent,
              sink)


@pytest.mark.parametrize("page", [32, 48])
def test_evict_pages_and_padded_tables(page):
    run_evict(spread(C.make(page, [500, 77, 96], 4, 2, 128, page=page, packed=False)), 90, 10, 2)


@pytest.mark.parametrize("n,budget", [(1023, 1000), (1024, 1023), (1025, 512), (5000, 4999),
                                      (32768, 8000), (32769, 8000), (40000, 39990)])
def test_evict_long(n, budget):
    run_evict(spread(C.make(n, [n, 900], 1, 1, 64)), budget, 100, 4)


def test_evict_ties_nan_and_infinities():
    c = spread(C.make(31, [400, 200], 2, 2, 128))
    w = c.weights
    w[c.rng.random(w.shape) < 0.3] = 0.0
    w[c.rng.random(w.shape) < 0.1] = -0.0
    w[c.rng.random(w.shape) < 0.1] = np.nan
    w[c.rng.random(w.shape) < 0.05] = np.inf
    w[c.rng.random(w.shape) < 0.05] = -np.inf
    w[c.rng.random(w.shape) < 0.1] = -1.5
    w[c.rng.random(w.shape) < 0.05] = 1e-42
    for budget in (50, 150, 199, 390):
        run_evict(copy.deepcopy(c), budget, 10, 3)
    c.weights[:] = 0.25  # all equal: the first ones stay, nothing moves
    t = run_evict(copy.deepcopy(c), 128, record=False)
    assert np.array_equal(t["cache"].cpu().numpy(), c.cache)
    c.weights[:] = np.nan
    run_evict(c, 128, record=False)


def test_evict_bad_pages_and_tables():
    c = spread(C.make(32, [200, 90, 64], 2, 2, 128))
    c.indices[3], c.indices[7], c.indices[14] = -1, c.nb, 2 ** 31 - 1
    c.lens[2] = 3000
    run_evict(copy.deepcopy(c), 60, 5, 1)
    run_evict(copy.deepcopy(c), 190, 5, 1)
    run_evict(c, 100, 0, 0, record=False)


def test_evict_more_protected_than_the_budget():
    """Positions that repeat: the first protected ones stay."""
    c = C.make(33, [300], 2, 2, 128)
    c.positions[:] = 0
    run_evict(c, 40, 10, 5)


def test_evict_in_place_lengths_and_graph():
    c = spread(C.make(34, [500, 100, 130], 4, 4, 64))
    t = tensors(c)
    first = {k: t[k].clone() for k in ("cache", "weights", "positions", "seq")}

    def call():
        for k, v in first.items():
            t[k].copy_(v)
        ops.evict_paged(t["cache"], t["weights"], t["positions"], t["indices"], t["indptr"],
                        t["seq"], t["ends"], 120, 20, 4, t["seq"])
    call()
    want = {k: t[k].clone() for k in first}
    assert t["seq"].tolist() == [120, 100, 120]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call()
    for _ in range(3):
        t["cache"].zero_()
        g.replay()
        torch.cuda.synchronize()
        for k in first:
            assert torch.equal(t[k], want[k]), k
    cache, acc, pos, lens = C.evict(c, 120, 20, 4)
    assert np.array_equal(want["cache"].cpu().numpy(), cache)
