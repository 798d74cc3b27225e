"""Windowed prefill attention and the read-back of a window on an MI355X, against
their formulas in 64 bits."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

import budget_cases as C
import window_cases as W
from turboquant_amd import ops

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
GEOMETRIES = [(32, 8, 128), (16, 4, 64), (16, 2, 256), (8, 1, 128), (12, 4, 96), (8, 8, 64),
              (32, 2, 128), (6, 3, 80), (1, 1, 40), (4, 4, 256), (20, 1, 128), (5, 5, 8)]


def make(seed, chunks, hq, hkv, hd, dtype="fp16", q_scale=1.5):
    """(q, k, v, requests) of chunks (q_len, kv_len)"""
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    pd = C.pad(hd)

    def randn(*shape):
        return torch.randn(shape, generator=g, device=DEV)
    nq, nk = sum(a for a, _ in chunks), sum(b for _, b in chunks)
    q = (randn(nq, hq, hd) * q_scale).to(TYPES[dtype])
    k, v = (torch.nn.functional.pad(randn(nk, hkv, hd).half(), (0, pd - hd)) for _ in range(2))
    reqs, qs, ks = [], 0, 0
    for a, b in chunks:
        reqs.append((qs, a, ks, b, 0))
        qs, ks = qs + a, ks + b
    return q, k, v, reqs


def check(got, q, k, v, reqs, window, sink, scale, hd):
    """u = 2^-24.  q, K and V enter as they are; a score is a chain of at most 2
    pd / 16 fp32 sums and eight roundings, relative to |q| |K| (Cauchy-Schwarz);
    a probability is off by twice that, plus its rounding to fp16 (2^-11; below
    2^-14 half a step of 2^-24 for each of the n keys in sight, where the row's
    sum is 1 or more) and fp32 sums; then the output's own rounding."""
    u = 2.0 ** -24
    half = 2.0 ** -11 if got.dtype == torch.float16 else 2.0 ** -8
    r = q.shape[1] // k.shape[1]
    ref = W.prefill(q.double(), k[..., :hd].double(), v[..., :hd].double(), reqs, r, scale, window,
                    sink)
    fin = lambda x: torch.where(torch.isfinite(x), x, 0).double()
    qk = float(fin(q).norm(dim=-1).max() * fin(k).norm(dim=-1).max()) if q.numel() else 0.0
    n = min(max((b for _, _, _, b, _ in reqs), default=0), window + sink)
    p = 2 * qk * scale * (k.shape[2] / 8 + 8) * u + 2.0 ** -11 + 64 * u + n * 2.0 ** -25
    tol = half * ref.abs() + p * (1 + half) * float(fin(v).abs().max()) + u
    err = (got.double() - ref).abs()
    assert torch.equal(torch.isnan(ref), torch.isnan(got))
    bad = ~((err <= tol) | torch.isnan(ref) | (ref == got))
    assert not bad.any(), f"off by {float(err[bad].max()):.3e}, {float((err / tol)[bad].max()):.2f} x"


def call(q, k, v, reqs, hd, window, sink, o=None, scale=None):
    o = torch.full_like(q, 7.0) if o is None else o
    return ops.prefill_attention_window(q, o, reqs, k.shape[1], hd, k.shape[2],
                                        1 / math.sqrt(hd) if scale is None else scale, window, sink,
                                        k, v)


def run(seed, chunks, hq, hkv, hd, window, sink, dtype="fp16", **kw):
    q, k, v, reqs = make(seed, chunks, hq, hkv, hd, dtype, **kw)
    o = call(q, k, v, reqs, hd, window, sink)
    check(o, q, k, v, reqs, window, sink, 1 / math.sqrt(hd), hd)


@pytest.mark.parametrize("hq,hkv,hd", GEOMETRIES)
def test_geometries(hq, hkv, hd):
    run(hq, [(37, 37), (1, 300), (200, 517), (64, 64)], hq, hkv, hd, 100, 4,
        "bf16" if hkv % 2 else "fp16")


@pytest.mark.parametrize("window", [1, 2, 31, 32, 33, 63, 64, 65, 127, 129, 200, 2 ** 31 - 1])
@pytest.mark.parametrize("sink", [0, 1, 63, 64, 65, 130, 2 ** 31 - 1])
def test_borders(window, sink):
    """Every place of both borders within a tile and a block of rows."""
    run(window % 997 + sink % 997, [(1, 1), (33, 40), (1, 257), (300, 300), (130, 391)], 2, 1, 64,
        window, sink)


@pytest.mark.parametrize("hq,hkv,hd,n,ctx,window,sink,dtype", [
    (32, 8, 128, 4096, 0, 1000, 4, "fp16"),      # 256-row blocks of eight waves
    (32, 8, 128, 2500, 900, 700, 130, "bf16"),
    (32, 8, 64, 4100, 0, 513, 1, "bf16"),        # two row blocks a wave
    (16, 4, 256, 1500, 300, 400, 70, "fp16"),
    (4, 2, 128, 100, 20000, 19000, 4, "fp16"),   # keys split over workgroups
    (2, 1, 256, 40, 9000, 2 ** 31 - 1, 0, "bf16"),
    (1, 1, 64, 21000, 0, 4000, 100, "fp16"),     # more blocks than a list holds, split
    (2, 1, 128, 21000, 0, 300, 0, "fp16"),
])
def test_shapes_of_the_kernels(hq, hkv, hd, n, ctx, window, sink, dtype):
    run(n, [(n, n + ctx)], hq, hkv, hd, window, sink, dtype)


@pytest.mark.parametrize("count,each", [(64, 300), (65, 20), (200, 7)])
def test_many_requests(count, each):
    run(count, [(each + i % 5, each + i % 11 + 40) for i in range(count)], 2, 2, 64, 50, 3)


def test_peaked_and_flat_scores():
    run(1, [(200, 900)], 4, 2, 128, 300, 4, q_scale=20.0)
    run(2, [(200, 900)], 4, 2, 128, 300, 4, q_scale=0.0)


def test_a_window_beyond_the_keys_is_full_attention():
    """Bit for bit the attention over every key."""
    for n, ctx, hq in ((4096, 0, 32), (300, 5000, 8), (700, 100, 4)):
        q, k, v, reqs = make(n, [(n, n + ctx), (17, 60)], hq, hq // 4, 128)
        o = call(q, k, v, reqs, 128, n + ctx, 5)
        full = torch.empty_like(o)
        ops.prefill_attention_batch(q, full, reqs, hq // 4, 128, 128, 1 / math.sqrt(128), k, v)
        assert torch.equal(o, full)


@pytest.mark.parametrize("hq,hkv,hd,n,ctx,window,sink", [
    (2, 1, 128, 300, 200, 100, 3), (32, 8, 128, 4096, 0, 1000, 4), (32, 8, 64, 4100, 0, 513, 1),
    (2, 1, 256, 40, 9000, 5000, 0), (1, 1, 64, 21000, 0, 4000, 100), (3, 3, 96, 150, 0, 20, 0)])
def test_nan_and_infinities_stay_with_the_rows_that_see_them(hq, hkv, hd, n, ctx, window, sink):
    """Keys and values at tile borders, ahead of and behind their rows' sight."""
    q, k, v, reqs = make(n + 1, [(n, n + ctx)], hq, hkv, hd)
    lk = n + ctx
    for x, j in ((math.nan, lk // 2), (math.inf, lk // 3 // 64 * 64), (-math.inf, lk - 1)):
        v[j, 0, 3] = x
    o = call(q, k, v, reqs, hd, window, sink)
    check(o, q, k, v, reqs, window, sink, 1 / math.sqrt(hd), hd)
    rows = torch.isnan(o[:, 0, 3])
    assert 0 < int(rows.sum()) <= 3 * window + sink and torch.isfinite(o[:, 0, 4]).all()
    # a key's row: everything of the rows that see it, and of its head
    q, k, v, reqs = make(n + 2, [(n, n + ctx)], hq, hkv, hd)
    k[lk // 2, 0, 5] = math.nan
    k[lk - 1, 0, 0] = math.inf
    o = call(q, k, v, reqs, hd, window, sink)
    pos = torch.arange(ctx, lk, device=DEV)
    sees = (pos >= lk // 2) & ((lk // 2 > pos - window) | (lk // 2 < sink))
    sees[-1] = True
    # (a score of -inf gives a finite row)
    assert torch.isnan(o[sees][:-1, 0]).all() and torch.isfinite(o[~sees]).all()
    if hkv > 1:
        assert torch.isfinite(o[:, hq // hkv:]).all()


def test_strides_sources_and_rows_of_no_request():
    q, k, v, reqs = make(5, [(130, 200), (70, 70)], 8, 2, 128, "bf16")
    want = call(q, k, v, reqs, 128, 60, 4)
    wide = torch.full((210, 3, 8, 136), 9.0, dtype=torch.bfloat16, device=DEV)
    rows = wide[5:205, 1, :, :128]
    rows.copy_(q)
    o = torch.full((210, 8, 256), 5.0, dtype=torch.bfloat16, device=DEV)
    kk = torch.full((280, 2, 2, 128), 9.0, dtype=torch.float16, device=DEV)
    kk[3:273, 1].copy_(k)
    k2, v2 = (torch.full((300, 2, 128), 9.0, dtype=torch.float16, device=DEV) for _ in range(2))
    k2[20:90], v2[20:90] = k[200:], v[200:]
    at = [(0, 130, 3, 200, 0), (130, 70, 20, 70, 1)]
    vv = torch.full((280, 2, 128), 9.0, dtype=torch.float16, device=DEV)
    vv[3:273] = v
    ops.prefill_attention_window(rows, o[2:202, :, 64:192], at, 2, 128, 128, 1 / math.sqrt(128), 60,
                                 4, kk[:, 1], vv, k2, v2)
    assert torch.equal(o[2:202, :, 64:192], want)
    o[2:202, :, 64:192] = 5.0
    assert (o == 5.0).all()
    # requests that leave rows out
    o = call(q, k, v, [reqs[0]], 128, 60, 4)
    assert torch.equal(o[:130], want[:130]) and (o[130:] == 7.0).all()
    assert (call(q, k, v, [], 128, 60, 4) == 7.0).all()
    assert (call(q, k, v, [(5, 0, 3, 9, 0)], 128, 60, 4) == 7.0).all()


def test_rows_beyond_32_bit_offsets():
    q, k, v, reqs = make(6, [(100, 300)], 8, 8, 128)
    big = [torch.empty((2_200_000, 8, 128), dtype=torch.float16, device=DEV) for _ in range(2)]
    for x, y in zip(big, (k, v)):
        x[-300:] = y
    at = [(0, 100, 2_200_000 - 300, 300, 0)]
    assert torch.equal(call(q, *big, at, 128, 60, 4), call(q, k, v, reqs, 128, 60, 4))


def test_repeated_calls_streams_and_a_graph():
    # a case whose keys are split: it has a workspace
    q, k, v, reqs = make(7, [(100, 9000), (30, 700)], 4, 2, 128)
    first = call(q, k, v, reqs, 128, 6000, 4).clone()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    outs = []
    for i in range(6):
        with torch.cuda.stream(streams[i % 2]):
            outs.append(call(q, k, v, reqs, 128, 6000, 4))
    torch.cuda.synchronize()
    assert all(torch.equal(x, first) for x in outs)
    o = torch.empty_like(q)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call(q, k, v, reqs, 128, 6000, 4, o)
    for i in range(3):
        q.copy_(torch.randn_like(q))
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, call(q, k, v, reqs, 128, 6000, 4))
        check(o, q, k, v, reqs, 6000, 4, 1 / math.sqrt(128), 128)


# ------------------------------------------------------------------ read-back

def cached(c):
    return dict(cache=torch.from_numpy(c.cache).to(DEV), signs=torch.from_numpy(c.signs).to(DEV),
                table=torch.from_numpy(c.indices.reshape(len(c.lens), -1).copy()).to(DEV))


def closed_up(c, t, reqs, sink, key, value, signs=True):
    """The same rows from a read-back of everything."""
    rows = sum(ctx + n for _, ctx, _, _, n, _ in reqs)
    ks, vs = (torch.zeros((rows, c.hkv, c.pd), dtype=torch.float16, device=DEV) for _ in range(2))
    full, at, keep = [], 0, []
    for b, ctx, first, a, n, _ in reqs:
        full.append((b, ctx, a, n, at))
        keep.append(torch.cat((torch.arange(min(sink, first)), torch.arange(first, ctx + n))) + at)
        at += ctx + n
    ops.prefill_gather(t["cache"], t["table"], key, value, full, c.hd, c.pd,
                       t["signs"] if signs else None, ks, vs)
    keep = torch.cat(keep).to(DEV)
    return ks[keep], vs[keep]


@pytest.mark.parametrize("hq,hkv,hd", GEOMETRIES[:9])
@pytest.mark.parametrize("page", [16, 48])
def test_read_back(hq, hkv, hd, page):
    """Bit for bit the rows of a read-back of everything; entries of hidden pages
    hold garbage; the rows around the output stay."""
    lens = [500, 77, 64, 1, 200, 333]
    c = C.make(hkv + page, lens, hq, hkv, hd, page=page, packed=False)
    t = cached(c)
    for window, sink, dtype in ((100, 4, "fp16"), (1, 17, "bf16"), (65, 0, "fp32"), (400, 40, "fp16"),
                                (2 ** 31 - 1, 3, "bf16")):
        fresh = [3, 0, 40, 1, 130, 0]
        key, value = (torch.randn((sum(fresh), hkv, hd), device=DEV).to(TYPES[dtype])
                      for _ in range(2))
        reqs, at, f = [], 2, 0
        for b, (n, m) in enumerate(zip(lens, fresh)):
            first = max(0, n - window + 1)
            reqs.append((b, n, first, f, m, at))
            at, f = at + min(sink, first) + n - first + m, f + m
        want = closed_up(c, t, reqs, sink, key, value)
        spoiled = dict(t, table=t["table"].clone())
        for b, n in enumerate(lens):
            see = W.sees(n, n, window, sink)
            for i in range(-(-n // page)):
                if not see[i * page:(i + 1) * page].any():
                    spoiled["table"][b, i] = 2 ** 31 - 1 - i
        out = [torch.full((at + 3, hkv, c.pd), 7.0, dtype=torch.float16, device=DEV)
               for _ in range(2)]
        ops.prefill_gather_window(t["cache"], spoiled["table"], key, value, reqs, sink, hd, c.pd,
                                  t["signs"], *out)
        for got, ref in zip(out, want):
            assert torch.equal(got[2:at], ref)
            assert (got[:2] == 7.0).all() and (got[at:] == 7.0).all()


def test_read_back_without_fresh_rows_or_signs_and_many_requests():
    lens = [(37 * i) % 90 + 1 for i in range(150)]
    c = C.make(9, lens, 2, 2, 64, packed=False)
    t = cached(c)
    reqs, at = [], 0
    for b, n in enumerate(lens):
        first = max(0, n - 20)
        reqs.append((b, n, first, 0, 0, at))
        at += min(5, first) + n - first
    empty = torch.empty((1, 2, 64), device=DEV)  # (no row of it is read)
    for signs in (True, False):
        out = [torch.empty((at, 2, 64), dtype=torch.float16, device=DEV) for _ in range(2)]
        ops.prefill_gather_window(t["cache"], t["table"], None, None, reqs, 5, 64, 64,
                                  t["signs"] if signs else None, *out)
        for got, ref in zip(out, closed_up(c, t, reqs, 5, empty, empty, signs)):
            assert torch.equal(got, ref)
    # nothing to read, nothing written
    kept = out[0].clone()
    ops.prefill_gather_window(t["cache"], t["table"], None, None, [(0, 0, 0, 0, 0, 0)], 5, 64, 64,
                              None, *out)
    ops.prefill_gather_window(t["cache"], t["table"], None, None, [(0, 50, 50, 0, 0, 0)], 0, 64, 64,
                              None, *out)
    assert torch.equal(out[0], kept)


def test_read_back_values_bad_pages_and_far_ones():
    """Against the dequantized entries in 64 bits: an fp16 row is a rounding
    (2^-11) of sums of pd levels whose fp32 chain is log2 pd + 3 long."""
    c = C.make(10, [300, 90], 8, 8, 128, packed=False)
    c.indices[2], c.indices[len(c.indices) // 2 + 4] = -1, c.nb + 5
    t = cached(c)
    far = 440_000
    big = torch.empty((2, far + c.nb, 16, 8, 80), dtype=torch.uint8, device=DEV)
    big[:, far:] = t["cache"]
    reqs = [(0, 300, 180, 0, 0, 0), (1, 90, 11, 0, 0, 160)]
    back = C.hadamard(128) * c.signs
    for cache, table in ((t["cache"], t["table"]),
                         (big, torch.where(t["table"] >= 0, t["table"] + far, -1))):
        out = [torch.empty((250, 8, 128), dtype=torch.float16, device=DEV) for _ in range(2)]
        ops.prefill_gather_window(cache, table.to(torch.int32), None, None, reqs, 40, 128, 128,
                                  t["signs"], *out)
        for slab in range(2):
            got = out[slab].double().cpu().numpy()
            for b, n, first, at in ((0, 300, 180, 0), (1, 90, 11, 160)):
                pg, off, ok = C.places(c, b)
                see = np.r_[:min(40, first), first:n]
                for h in range(8):
                    x = C.rows(c, slab, pg[see], off[see], h)
                    ref = np.where(ok[see][:, None], x @ back, 0)
                    size = np.sqrt((x ** 2).sum(-1, keepdims=True))
                    tol = 2.0 ** -11 * np.abs(ref) + size * 12 * 2.0 ** -24 + 2.0 ** -25
                    assert (np.abs(got[at:at + len(see), h] - ref) <= tol).all()


def test_read_back_then_attention_is_attention_over_everything():
    """A chunk over what the window leaves of its context, closed up, equals the
    chunk over all of it under the same window: another division into tiles, the
    same formula."""
    c = C.make(11, [3000, 70, 900], 8, 2, 128, packed=False)
    t = cached(c)
    fresh, window, sink = [200, 33, 1], 300, 4
    q, k, v, _ = make(12, [(n, n) for n in fresh], 8, 2, 128)
    part, full, gp, gf = [], [], [], []
    a = at = af = 0
    for b, (ctx, n) in enumerate(zip([3000, 70, 900], fresh)):
        first = max(0, ctx - window + 1)
        kept = min(sink, first) + ctx - first
        gp.append((b, ctx, first, a, n, at))
        gf.append((b, ctx, a, n, af))
        part.append((a, n, at, kept + n, 0))
        full.append((a, n, af, ctx + n, 0))
        a, at, af = a + n, at + kept + n, af + ctx + n
    kp, vp = (torch.empty((at, 2, 128), dtype=torch.float16, device=DEV) for _ in range(2))
    kf, vf = (torch.empty((af, 2, 128), dtype=torch.float16, device=DEV) for _ in range(2))
    ops.prefill_gather_window(t["cache"], t["table"], k, v, gp, sink, 128, 128, t["signs"], kp, vp)
    ops.prefill_gather(t["cache"], t["table"], k, v, gf, 128, 128, t["signs"], kf, vf)
    o = call(q, kp, vp, part, 128, window, sink)
    check(o, q, kp, vp, part, window, sink, 1 / math.sqrt(128), 128)
    check(o, q, kf, vf, full, window, sink, 1 / math.sqrt(128), 128)
