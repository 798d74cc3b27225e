"""Windows over keys whose norms are no numbers or infinite, and rows without a
query beside them."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import budget_cases as C
from test_gpu_budget import DEV, check_weights, dev, queries, tensors
from turboquant_amd import ops

pytestmark = pytest.mark.gpu


def set_key_norm(c, b, t, h, value):
    pg, off, _ = C.places(c, b)
    half, n = c.pd // 2, c.pd // 64
    c.cache[0, pg[t], off[t], h, half:half + 2 * n] = np.full(n, value, np.float16).view(np.uint8)


def observe(c, q, starts, window):
    t = tensors(c)
    ops.track_window(q, dev(np.asarray(starts, np.int32)), window, t["cache"], t["indices"],
                     t["indptr"], t["seq"], c.hkv, c.hd, c.pd, c.scale, t["signs"], t["weights"],
                     t["positions"], t["ends"])
    torch.cuda.synchronize()
    return t["weights"].cpu().numpy()


@pytest.mark.parametrize("hd,window,chunk", [(128, 9, 20), (64, 40, 50), (256, 3, 2), (128, 70, 300)])
def test_a_norm_that_is_no_number_stays_with_its_head(hd, window, chunk):
    """The last query sees it, so every weight of that head and sequence that the
    query adds to is no number; other heads and sequences are as without it."""
    c = C.make(401 + hd, [400, 90], 8, 2, hd)
    clean = C.make(401 + hd, [400, 90], 8, 2, hd)
    set_key_norm(c, 0, 33, 1, np.nan)
    q, qx = queries(c, chunk + 5, "fp16")
    w = observe(c, q, [0, chunk, chunk + 5], window)
    _, ref, _ = C.attend(clean, qx, np.array([0, chunk, chunk + 5]), window)
    pg, off, _ = C.places(c, 0)
    assert np.isnan(w[pg, 1, off]).all()
    w[pg, 1, off], ref[pg, 1, off] = 0, 0
    clean.weights[pg, 1, off] = 0
    check_weights(clean, w, ref, qx, window * 4)


@pytest.mark.parametrize("hd,hq", [(128, 2), (64, 2), (256, 2), (128, 8)])
def test_a_window_of_one_is_the_decode_where_norms_are_infinite(hd, hq):
    """An infinite norm's score is one of the infinities by the sign of its
    product: weight 0, or no number for the whole row; 31 or 28 rows of the tile
    have no query and add to neither."""
    c = C.make(411 + hd, [100, 70], hq, 2, hd)
    for t in (5, 60):
        for h in range(2):
            set_key_norm(c, 0, t, h, np.inf)
    some = False
    for seed in range(12):  # both signs come up
        c.rng = np.random.default_rng(seed)
        q, _ = queries(c, 2, "fp16")
        w = observe(c, q, [0, 1, 2], 1)
        t = tensors(c)
        o = torch.empty_like(q)
        ops.decode_paged_tracked(q, t["cache"], t["indices"], t["indptr"], t["seq"], 2, c.hd, c.pd,
                                 c.scale, t["signs"], o, t["weights"], t["positions"], t["ends"])
        d = t["weights"].cpu().numpy()
        assert np.array_equal(np.isnan(w), np.isnan(d))
        known = ~np.isnan(w)
        assert np.allclose(w[known], d[known], rtol=1e-4, atol=0)
        pg, off, _ = C.places(c, 0)
        some = some or not np.isnan(w[pg, :, off]).any(0).all()  # (of one head)
    assert some or hq > 2


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_missing_rows_add_nothing_to_keys_without_a_finite_norm(hd):
    """Chunks whose rows are all behind the end of q: tokens from before keep their
    weights and the chunk's get 0, whatever the norms."""
    c = C.make(421 + hd, [50, 40], 4, 2, hd)
    for t, value in ((10, np.nan), (20, np.inf), (48, np.nan)):
        set_key_norm(c, 0, t, 0, value)
    q, _ = queries(c, 4, "fp16")
    w = observe(c, q, [6, 9, 11], 4)
    want = c.weights.copy()
    for b, n, chunk in ((0, 50, 3), (1, 40, 2)):
        pg, off, _ = C.places(c, b)
        want[pg[n - chunk:], :, off[n - chunk:]] = 0
    assert np.array_equal(w, want)


@pytest.mark.parametrize("scale", [1e5, 1e9, 1e20, 1e30, 3e35])
@pytest.mark.parametrize("hq,hkv,hd", [(8, 2, 128), (16, 1, 64), (2, 2, 256)])
def test_scores_of_any_size(hq, hkv, hd, scale):
    """Scores far beyond what exp2 takes: a row's whole weight is on one key, also
    where every score is hugely negative (a sequence of one token among them)."""
    c = C.make(431 + hd, [100, 1, 47], hq, hkv, hd)
    t = tensors(c)
    q, qx = queries(c, 3 + 40, "bf16", scale)
    assert torch.isfinite(q).all()
    k0 = c.weights.copy()
    for starts, window, rows in (([0, 1, 2, 3], 1, 3), ([0, 30, 31, 40], 6, 40)):
        x, xx = q[:rows], qx[:rows]
        ref_o, ref, _ = C.attend(c, xx, np.array(starts), window, True, decode=window == 1)
        # one token a row and head: whole numbers are added (or, if new, set)
        fresh = np.zeros(k0.shape, bool)
        for b in range(3):
            pg, off, _ = C.places(c, b)
            n, chunk = int(c.lens[b]), starts[b + 1] - starts[b]
            fresh[pg[n - chunk:], :, off[n - chunk:]] = True
        added = np.rint(ref - np.where(fresh, 0, k0))
        assert np.abs(ref - np.where(fresh, 0, k0) - added).max() < 1e-9
        want = np.where(fresh, added, k0 + added).astype(np.float32)
        assert np.array_equal(observe(c, x, starts, window), want)
        if window == 1:
            o = torch.empty_like(x)
            ops.decode_paged_tracked(x, t["cache"], t["indices"], t["indptr"], t["seq"], hkv, hd,
                                     c.pd, c.scale, t["signs"], o, t["weights"], t["positions"],
                                     t["ends"])
            assert np.array_equal(t["weights"].cpu().numpy(), want)
            # one value row: its level's 8.7e-5, and the output's rounding
            err = np.abs(o.double().cpu().numpy() - ref_o)
            assert (err <= 2.0 ** -8 * np.abs(ref_o) + 2e-4 * 30).all() and np.isfinite(err).all()


def test_a_captured_window_with_other_lengths():
    """Replays after new lengths, chunks and tables have been written, with eager work
    between them: what an eager call gives."""
    c = C.make(441, [700, 90, 1], 16, 4, 128, packed=False)
    t = tensors(c)
    q, _ = queries(c, 400, "bf16")
    starts = torch.tensor([0, 300, 390, 391], dtype=torch.int32, device=DEV)
    first = {k: t[k].clone() for k in ("weights", "positions")}

    def call():
        for k, v in first.items():
            t[k].copy_(v)
        ops.track_window(q, starts, 20, t["cache"], t["indices"], t["indptr"], t["seq"], 4, 128, 128,
                         c.scale, t["signs"], t["weights"], t["positions"], t["ends"])
    call()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call()
    for lens, chunks in (([700, 90, 1], [300, 90, 1]), ([700, 2, 0], [1, 2, 0]), ([16, 90, 1], [16, 0, 1]),
                         ([650, 90, 1], [100, 90, 1])):
        t["seq"].copy_(torch.tensor(lens, dtype=torch.int32))
        starts.copy_(torch.tensor([0, *np.cumsum(chunks)], dtype=torch.int32))
        t["ends"].copy_(t["seq"] + 5)
        g.replay()
        torch.cuda.synchronize()
        got = [t[k].clone() for k in first]
        call()
        torch.cuda.synchronize()
        for a, k in zip(got, first):
            assert torch.equal(a, t[k])


@pytest.mark.parametrize("hd,hq", [(64, 32), (256, 32), (96, 96)])
def test_a_window_over_units_of_several_chunks(hd, hq):
    """32 kv heads leave few units: each walks several chunks of 128 tokens, in both
    passes; row tiles of one and of three, bad pages inside."""
    c = C.make(451 + hd, [5003, 900], hq, 32, hd)
    c.indices[20], c.indices[230] = -1, c.nb
    t = tensors(c)
    starts = np.array([0, 60, 70], np.int32)
    for window in (3, 70):
        q, qx = queries(c, 70, "fp16")
        for k in ("weights", "positions"):
            t[k].copy_(dev(getattr(c, k)))
        ops.track_window(q, dev(starts), window, t["cache"], t["indices"], t["indptr"], t["seq"], 32,
                         hd, c.pd, c.scale, t["signs"], t["weights"], t["positions"], t["ends"])
        _, ref, pos = C.attend(c, qx, starts, window)
        check_weights(c, t["weights"].cpu().numpy(), ref, qx, window * hq // 32)
        assert np.array_equal(t["positions"].cpu().numpy(), pos)
