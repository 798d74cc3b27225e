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


@pytest.mark.parametrize("window", [5, 17, 24, 40, 70, 100])
def test_window_of_many_sequences(window):
    # 12 sequences of 8 kv heads: the second pass joins the statistics itself
    # up to 16 row tiles, whose number does not divide the half waves here
    lens = [3, 0, 260, 17, 129, 500, 64, 1, 90, 33, 1030, 128]
    chunks = [3, 0, 100, 1, 129, 80, 0, 1, 9, 33, 70, 128]
    run_window(C.make(900 + window, lens, 24, 8, 128), chunks, window)


def test_window_of_a_long_table():
    # a table of 8192 tokens over 32 kv heads: the first pass takes two key tiles
    # a wave; units of more than one chunk, ends inside a tile, bad pages
    c = C.make(55, [4003, 700], 32, 32, 128)
    c.indices[20], c.indices[130] = -1, c.nb
    c.indices = np.concatenate([c.indices, np.full(512 - len(c.indices), -1, np.int32)])
    run_window(c, [500, 700], 400)
    run_window(c, [33, 1], 300, signs=False)


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


@pytest.mark.parametrize("batch,hkv,hd", [(64, 1, 64), (65, 1, 64), (70, 12, 64), (3, 20, 256)])
def test_evict_many_rows_of_moves(batch, hkv, hd):
    # one, two and three rows of 64 (sequence, head group)s, the last group of
    # 4 heads; one long sequence whose rounds outnumber the others'
    lens = [(37 * b) % 90 for b in range(batch)]
    lens[batch // 2] = 3000
    run_evict(spread(C.make(batch + hkv, lens, hkv, hkv, hd)), 40, 8, 2)


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


# ------------------------------------------------------------------ together

@pytest.mark.parametrize("hq,hkv,hd,page,dtype", [(8, 2, 128, 16, "fp16"), (6, 3, 80, 32, "bf16"),
                                                  (16, 2, 256, 16, "bf16"), (8, 8, 64, 48, "fp16")])
def test_prompt_then_cut_then_decode(hq, hkv, hd, page, dtype):
    """As a server uses them: prompts written and observed, cut to the budget,
    then decode steps that write, attend and record, with a cut every few of
    them; each call against its 64-bit form from the state that it found."""
    from turboquant_amd.budget import CacheRecord
    prompt, budget, steps, every = [150, 61, 1], 64, 13, 5
    c = C.make(41, [p + steps for p in prompt], hq, hkv, hd, page=page, packed=False)
    width = len(c.indices) // 3
    table = dev(c.indices.reshape(3, width))
    c.cache[:] = 0
    cache = dev(c.cache)
    signs = dev(c.signs)
    rec = CacheRecord.beside(cache, budget, recent=9, sink=3, window=7)
    rec.weights.fill_(float("nan"))  # whatever was there before
    c.weights[:], c.positions[:] = np.nan, 0
    pd, lens, seen = c.pd, np.array(prompt, np.int32), np.array(prompt, np.int32)
    args = (hkv, hd, pd, c.scale, signs)

    def rows(n):
        return (torch.from_numpy(c.rng.standard_normal((n, hkv, hd))).to(TYPES[dtype]).to(DEV),
                torch.from_numpy(c.rng.standard_normal((n, hkv, hd))).to(TYPES[dtype]).to(DEV))

    def write(b, at, k, v):
        pg = c.indices.reshape(3, width)[b][at // page]
        ops.quantize_write_kv_cache(cache, k, v, signs, dev((pg * page + at % page)
                                                            .astype(np.int32)), hd, pd)

    def check(q, starts, window, o=None):
        c.cache, c.lens, c.ends = cache.cpu().numpy(), lens.copy(), seen.copy()
        ref_o, ref_w, ref_p = C.attend(c, q, starts, window, True, decode=o is not None)
        got = rec.weights.cpu().numpy()
        known = np.isfinite(ref_w)
        assert np.array_equal(known, np.isfinite(got))
        d = copy.copy(c)
        d.weights = np.where(np.isfinite(c.weights), c.weights, 0).astype(np.float32)
        check_weights(d, np.where(known, got, 0), np.where(known, ref_w, 0), q,
                      window * hq // hkv)
        assert np.array_equal(rec.positions.cpu().numpy(), ref_p)
        if o is not None:
            check_o(c, o, ref_o, q, dtype)
        c.weights, c.positions = got, ref_p

    def cut():
        nonlocal lens
        new = rec.evict(cache, table, dev(lens), dev(seen))
        c.lens, c.ends = lens.copy(), seen.copy()
        c.cache, c.weights, c.positions, lens = C.evict(c, budget, 9, 3)
        assert np.array_equal(new.cpu().numpy(), lens)
        assert np.array_equal(cache.cpu().numpy(), c.cache)
        assert np.array_equal(rec.weights.cpu().numpy(), c.weights, equal_nan=True)
        assert np.array_equal(rec.positions.cpu().numpy(), c.positions)

    for b, p in enumerate(prompt):
        write(b, np.arange(p), *rows(p))
    starts = np.concatenate(([0], np.cumsum(prompt))).astype(np.int32)
    q, qx = queries(c, int(starts[-1]), dtype)
    rec.observe(q, dev(starts), cache, table, dev(lens), dev(seen), *args)
    check(qx, starts, 7)
    cut()
    assert lens.tolist() == [64, 61, 1]
    for step in range(steps):
        k, v = rows(3)
        for b in range(3):
            write(b, lens[b:b + 1].copy(), k[b:b + 1], v[b:b + 1])
        lens, seen = lens + 1, seen + 1
        q, qx = queries(c, 3, dtype)
        o = torch.empty((3, hq, hd), dtype=TYPES[dtype], device=DEV)
        rec.decode(q, cache, table, dev(lens), dev(seen), *args, o)
        check(qx, np.arange(4), 1, o)
        if step % every == every - 1:
            cut()
    assert lens.max() <= budget + every


def test_two_graphs_and_a_stream_share_nothing():
    """Two captured decode calls and an eager one on a third stream, replayed
    together over caches of their own: workspaces are not shared."""
    cs = [C.make(50 + i, [400 + 30 * i, 77], 8, 2, 128) for i in range(3)]
    ts = [tensors(c) for c in cs]
    qs = [queries(c, 2, "fp16") for c in cs]
    os_ = [torch.zeros((2, 8, 128), dtype=torch.float16, device=DEV) for _ in cs]
    w0 = [t["weights"].clone() for t in ts]

    def call(i):
        c, t = cs[i], ts[i]
        t["weights"].copy_(w0[i])
        ops.decode_paged_tracked(qs[i][0], t["cache"], t["indices"], t["indptr"], t["seq"], 2, 128,
                                 128, c.scale, t["signs"], os_[i], t["weights"], t["positions"],
                                 t["ends"])
    want = []
    for i in range(3):
        call(i)
        want.append((os_[i].clone(), ts[i]["weights"].clone()))
    torch.cuda.synchronize()
    graphs = []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            call(i)
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(3)]
    for _ in range(5):
        for i in range(3):
            os_[i].zero_()
            ts[i]["weights"].zero_()
        torch.cuda.synchronize()
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                graphs[i].replay() if i < 2 else call(i)
        torch.cuda.synchronize()
        for i in range(3):
            assert torch.equal(os_[i], want[i][0]) and torch.equal(ts[i]["weights"], want[i][1])


def test_native_and_python_forms_agree():
    """The C++ form takes the ordinary call; a call that it leaves alone (an
    op's tensor subclass, here signs that are not contiguous) gives the same."""
    c = C.make(60, [300, 40], 8, 2, 128)
    nat = ops._native()
    signs2 = dev(np.stack((c.signs, c.signs), 1))[:, 0]
    assert not signs2.is_contiguous()
    got = []
    for signs in (dev(c.signs), signs2):
        t = tensors(c)
        c.rng = np.random.default_rng(1)
        q, _ = queries(c, 2, "fp16")
        o = torch.empty((2, 8, 128), dtype=torch.float16, device=DEV)
        args = (q, t["cache"], t["indices"], t["indptr"], t["seq"], 2, 128, 128, c.scale, signs, o,
                t["weights"], t["positions"], t["ends"])
        if signs is signs2:
            assert not nat.decode_tracked(*args)
        ops.decode_paged_tracked(*args)
        starts = torch.tensor([0, 1, 2], dtype=torch.int32, device=DEV)
        ops.track_window(q, starts, 1, *args[1:10], *args[11:])
        new = torch.empty(2, dtype=torch.int32, device=DEV)
        ev = (t["cache"], t["weights"], t["positions"], t["indices"], t["indptr"], t["seq"],
              t["ends"], 100, 5, 5, new)
        assert nat.evict(*ev[:6], t["ends"].long(), *ev[7:]) is False
        ops.evict_paged(*ev)
        got.append((o, t["weights"], t["positions"], t["cache"], new))
    for a, b in zip(*got):
        assert torch.equal(a, b)


def test_registered_ops_run():
    ops.register_ops()
    c = C.make(61, [90, 40], 8, 2, 64)
    t = tensors(c)
    q, qx = queries(c, 2, "fp16")
    o = torch.empty((2, 8, 64), dtype=torch.float16, device=DEV)
    v5 = torch.ops.turboquant_v5
    assert v5.decode_paged_tracked(q, t["cache"], t["indices"], t["indptr"], t["seq"], 2, 64, 64,
                                   c.scale, t["signs"], o, t["weights"], t["positions"],
                                   t["ends"]) is None
    ref_o, ref_w, _ = C.attend(c, qx, np.arange(3), 1, True, decode=True)
    check_weights(c, t["weights"].cpu().numpy(), ref_w, qx, 4)
    check_o(c, o, ref_o, qx, "fp16")
    starts = torch.tensor([0, 1, 2], dtype=torch.int32, device=DEV)
    v5.track_window(q, starts, 4, t["cache"], t["indices"], t["indptr"], t["seq"], 2, 64, 64,
                    c.scale, t["signs"], t["weights"], None, None)
    new = torch.empty(2, dtype=torch.int32, device=DEV)
    v5.evict_paged(t["cache"], t["weights"], None, t["indices"], t["indptr"], t["seq"], None, 50, 0,
                   0, new)
    assert new.tolist() == [50, 40]


def test_refused_calls_raise_from_the_library():
    c = C.make(62, [90], 8, 2, 64)
    t = tensors(c)
    new = torch.empty(1, dtype=torch.int32, device=DEV)
    args = (t["cache"], t["weights"], t["positions"], t["indices"], t["indptr"], t["seq"],
            t["ends"])
    for budget, recent, sink in ((0, 0, 0), (8, 9, 0), (8, 4, 5), (8, -1, 0)):
        with pytest.raises(RuntimeError, match="evict"):
            ops.evict_paged(*args, budget, recent, sink, new)
    with pytest.raises(RuntimeError, match="evict"):
        ops.evict_paged(t["cache"], t["weights"], None, *args[3:], 8, 2, 0, new)
    q = torch.zeros((1, 8, 64), dtype=torch.float16, device=DEV)
    starts = torch.tensor([0, 1], dtype=torch.int32, device=DEV)
    for window in (0, 257):
        with pytest.raises(RuntimeError, match="track_window"):
            ops.track_window(q, starts, window, t["cache"], t["indices"], t["indptr"], t["seq"], 2,
                             64, 64, c.scale, None, t["weights"])


# ------------------------------------------------------------ backend and harness

class _Meta:
    def __init__(self, **kw):
        self.__dict__.update(kw)


@pytest.mark.parametrize("batch,hq,hkv", [(1024, 2, 1), (2, 4096, 4096)])
def test_documented_limits(batch, hq, hkv):
    lens = [(7 * b) % 41 for b in range(batch)] if batch > 2 else [37, 20]
    run_decode(C.make(batch, lens, hq, hkv, 64))
    run_window(C.make(batch + 1, lens, hq, hkv, 64), [min(n, b % 9) for b, n in enumerate(lens)], 3)
    run_evict(spread(C.make(batch + 2, lens, hq, hkv, 64)), 12, 3, 1)


def test_offsets_beyond_32_bits():
    """Pages at the end of a cache of 8.8 GB (a slab is over 2^32 bytes) give the
    bits that the same pages in a small cache give."""
    c = spread(C.make(77, [300, 129, 40], 16, 8, 128))
    q, _ = queries(c, 3, "fp16")
    chunk, _ = queries(c, 60, "bf16")
    starts = dev(np.array([0, 40, 50, 60], np.int32))
    got = []
    for blocks in (c.nb, 430_000):
        t, at = tensors(c), blocks - c.nb
        big = {k: torch.empty(n, dtype=t[k].dtype, device=DEV) for k, n in
               (("cache", (2, blocks, 16, 8, 80)), ("weights", (blocks, 8, 16)),
                ("positions", (blocks, 8, 16)))}
        big["cache"][:, at:] = t["cache"]
        for k in ("weights", "positions"):
            big[k][at:] = t[k]
        indices, o, new = t["indices"] + at, torch.empty_like(q), torch.empty_like(t["seq"])
        tables = (indices, t["indptr"], t["seq"], 8, 128, 128, c.scale, t["signs"])
        state = (big["weights"], big["positions"], t["ends"])
        ops.track_window(chunk, starts, 7, big["cache"], *tables, *state)
        ops.decode_paged_tracked(q, big["cache"], *tables, o, *state)
        ops.evict_paged(big["cache"], big["weights"], big["positions"], indices, t["indptr"],
                        t["seq"], t["ends"], 50, 10, 4, new)
        torch.cuda.synchronize()
        got.append((o, new, big["cache"][:, at:].clone(), big["weights"][at:].clone(),
                    big["positions"][at:].clone()))
        del big
    torch.cuda.empty_cache()
    assert not torch.equal(got[0][2], tensors(c)["cache"])
    for x, y in zip(*got):
        assert torch.equal(x, y)


@pytest.mark.parametrize("hd,dtype", [(128, "fp16"), (96, "bf16")])
def test_backend_fills_its_record(hd, dtype):
    """forward with a record: a prompt batch is observed after its attention, a
    decode batch attends through the tracked op; a mixed batch too."""
    from turboquant_amd.budget import CacheRecord
    from turboquant_amd.vllm_backend_fused import TurboQuantBackend, TurboQuantFusedImpl
    hq, hkv, page, lens = 8, 2, 16, [40, 23]
    impl = TurboQuantFusedImpl(hq, hd, 1 / math.sqrt(hd), hkv, None, None, "fp8")
    plain = TurboQuantFusedImpl(hq, hd, 1 / math.sqrt(hd), hkv, None, None, "fp8")
    shape = TurboQuantBackend.get_kv_cache_shape(8, page, hkv, hd, "fp8")
    cache = torch.zeros(shape, dtype=torch.uint8, device=DEV)
    impl.record = CacheRecord.beside(cache, 64, window=5)
    table = torch.arange(8, dtype=torch.int32, device=DEV).view(2, 4)
    g = torch.Generator(device=DEV)
    g.manual_seed(3)

    def step(chunks, seq):
        n = sum(chunks)
        k, v = (torch.randn((n, hkv, hd), generator=g, device=DEV).to(TYPES[dtype])
                for _ in range(2))
        q = torch.randn((n, hq * hd), generator=g, device=DEV).to(TYPES[dtype])
        slots = torch.tensor([int(table[b, t // page]) * page + t % page
                              for b, (ql, s) in enumerate(zip(chunks, seq))
                              for t in range(s - ql, s)], dtype=torch.int32, device=DEV)
        starts = torch.tensor([0, chunks[0], n], dtype=torch.int32, device=DEV)
        meta = _Meta(max_query_len=max(chunks), num_actual_tokens=n, block_table=table,
                     seq_lens=torch.tensor(seq, dtype=torch.int32, device=DEV),
                     query_start_loc=starts, slot_mapping=slots)
        impl.do_kv_cache_update(None, k, v, cache, slots)
        a = (q, k.reshape(n, -1), v.reshape(n, -1), cache, meta)
        before = impl.record.weights.cpu().numpy()
        got, want = impl.forward(None, *a), plain.forward(None, *a)
        # two kernels of the same attention: each within the decode tolerance
        assert (got.float() - want.float()).abs().max() < 2 * (2e-3 + 1e-2 * want.abs().max())
        c = C.make(1, seq, hq, hkv, hd, page=page)
        c.cache, c.indices = cache.cpu().numpy(), table.cpu().numpy().reshape(-1)
        c.indptr, c.nb = np.array([0, 4, 8], np.int32), 8
        c.weights, c.positions = before, np.zeros_like(before, np.int32)
        c.ends, c.signs = np.array(seq, np.int32), impl._signs.cpu().numpy()
        qx = q.double().cpu().numpy().reshape(n, hq, hd)
        _, ref, _ = C.attend(c, qx, starts.cpu().numpy(), 5 if max(chunks) > 1 else 1)
        check_weights(c, impl.record.weights.cpu().numpy(), ref, qx, 5 * hq // hkv)
    step([40, 23], lens)
    step([1, 1], [41, 24])
    step([1, 7], [42, 31])


def test_harness_decodes_under_a_budget():
    """The end-to-end loop with a budget: eager and captured steps give the same
    tokens, caches stay inside it, and every layer and head keeps the first and
    the newest positions, each once."""
    from turboquant_amd import e2e
    shape = e2e.ModelShape.tiny(2)
    g = torch.Generator(device="cpu")
    g.manual_seed(7)
    prompts = torch.randint(0, shape.vocab, (3, 200), generator=g)
    rule = dict(budget=96, recent=16, sink=4, window=8, cut_every=4)
    tokens = []
    for graph in (False, True):
        r = e2e.Runner(shape, 3, 220, DEV, seed=5, **rule)
        for b in range(3):
            r.prefill(b, prompts[b, :200 - 60 * b].to(DEV))
        assert r.lens.tolist() == [96, 96, 80]
        if graph:
            r.capture(14)
            tokens.append(r.decode_graph(14).clone())
        else:
            tokens.append(r.decode_eager(14).clone())
        torch.cuda.synchronize()
        assert r.pos.tolist() == [214, 154, 94]
        assert r.lens.tolist() == [98, 98, 94]
        for impl in r.impls:
            pos = impl.record.positions.cpu().numpy()
            for b in range(3):
                n, seen = int(r.lens[b]), int(r.pos[b])
                t = np.arange(n)
                pg = r.block_table[b].cpu().numpy()[t // 16]
                for h in range(shape.kv_heads):
                    kept = set(pos[pg, h, t % 16].tolist())
                    assert len(kept) == n and kept <= set(range(seen))
                    assert set(range(4)) | set(range(seen - 16, seen)) <= kept
    assert torch.equal(tokens[0], tokens[1])


def test_harness_budget_above_every_length_changes_nothing_kept():
    """A budget that nothing exceeds: the tokens of the run without one, but for
    the rounding between two kernels of the same attention."""
    from turboquant_amd import e2e
    shape = e2e.ModelShape.tiny(2)
    g = torch.Generator(device="cpu")
    g.manual_seed(9)
    prompts = torch.randint(0, shape.vocab, (2, 100), generator=g)
    outs = []
    for rule in ({}, dict(budget=4096)):
        r = e2e.Runner(shape, 2, 110, DEV, seed=6, **rule)
        for b in range(2):
            r.prefill(b, prompts[b].to(DEV))
        r.probe = []
        r.decode_eager(1)
        outs.append([p[4].float() for p in r.probe])
        if rule:
            assert r.lens.tolist() == [101, 101]
            total = torch.stack([impl.record.weights.sum() for impl in r.impls])
            # 32 observed queries and one decode step, over two sequences, 32 heads
            assert torch.allclose(total, torch.full_like(total, 2 * 33 * 32), rtol=1e-5)
    a, b = outs[0][0], outs[1][0]  # the first layer sees the same inputs
    assert (a - b).abs().max() < 2 * (2e-3 + 1e-2 * a.abs().max())
