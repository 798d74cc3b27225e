"""Windowed attention on an MI355X where values in sight or out of it are not
finite, against the formulas in 64 bits."""
from __future__ import annotations

import copy
import math

import numpy as np
import pytest
import torch

import budget_cases as C
import test_gpu_window as D
import window_cases as W
from test_gpu_budget import queries, tensors
from test_gpu_window_prefill import call, check, make

pytestmark = pytest.mark.gpu


def scores_of_minus_infinity(q, k, keys):
    """Every query's score with the given keys: an infinite coordinate times a
    negative one."""
    q[..., 2] = -(q[..., 2].abs() + 0.1)
    k[keys, :, 2] = math.inf


@pytest.mark.parametrize("hq,hkv,hd,n,ctx,window,sink", [
    (2, 1, 128, 300, 200, 100, 1), (32, 8, 128, 4000, 100, 1000, 1),
    (32, 8, 64, 4100, 64, 513, 2), (2, 1, 256, 40, 9000, 5000, 1),    # (keys split)
    (4, 2, 128, 100, 20000, 19000, 1), (3, 3, 96, 150, 130, 20, 0), (1, 1, 64, 21000, 5, 4000, 3)])
def test_prefill_hidden_values_beside_scores_of_minus_infinity(hq, hkv, hd, n, ctx, window, sink):
    """A hidden key whose value is not finite leaves a row as it is, also where the
    first keys that the row sees, the sinks or those at the window's edge, score
    -inf and so weigh nothing."""
    q, k, v, reqs = make(n + 3, [(n, n + ctx)], hq, hkv, hd)
    lk = n + ctx
    scores_of_minus_infinity(q, k, list(range(sink)) + list(range(63, lk, 64)))
    for x, j in ((math.nan, 40), (math.inf, lk - n // 2 - 1), (math.nan, lk - n // 3)):
        v[j, 0, 3] = x
    o = call(q, k, v, reqs, hd, window, sink)
    check(o, q, k, v, reqs, window, sink, 1 / math.sqrt(hd), hd)
    assert torch.isnan(o[:, 0, 3]).any() and torch.isfinite(o[:, 0, 4]).all()


def norms(c, slab, value):
    """A copy of the case with those K or V norms: value(norms fp16 [nb, page, H])."""
    out = copy.copy(c)
    out.cache = c.cache.copy()
    at = out.cache[slab, ..., c.pd // 2:c.pd // 2 + 2 * (c.pd // 64)]
    new = value(at[..., :2].copy().view(np.float16)[..., 0]).astype(np.float16)
    at[:] = np.repeat(new[..., None], c.pd // 64, -1).view(np.uint8)
    return out


def decode_by_norms(c, q, window, sink):
    """window_cases.decode with a score as the K norm times its unit row's product,
    so that an infinite norm gives an infinite score."""
    unit, r = norms(c, 0, np.ones_like), c.hq // c.hkv
    o = np.zeros((len(c.lens), c.hq, c.pd))
    for b, n in enumerate(c.lens):
        pg, off, ok = C.places(c, b)
        see = ok & W.sees(int(n) - 1, len(pg), window, sink)
        pg, off = pg[see], off[see]
        for h in range(c.hkv):
            k = c.cache[0, pg, off, h, c.pd // 2:c.pd // 2 + 2].copy().view(np.float16)[:, 0]
            s = C.rotated(c, q[b, h * r:(h + 1) * r], True) @ C.rows(unit, 0, pg, off, h).T \
                * k.astype(np.float64) * c.scale
            p = np.exp(s - s.max(-1, keepdims=True))
            o[b, h * r:(h + 1) * r] = p / p.sum(-1, keepdims=True) @ C.rows(c, 1, pg, off, h)
    return ((o @ C.hadamard(c.pd)) * c.signs)[..., :c.hd]


@pytest.mark.parametrize("hq,hkv,hd", [(8, 2, 128), (16, 4, 64), (16, 2, 256), (16, 1, 128),
                                       (32, 2, 128), (8, 8, 256), (16, 8, 64)])
@pytest.mark.parametrize("lens,window,sink", [
    ([193, 65, 333], 300, 4), ([161, 345], 130, 1),    # one launch (up to 8 q heads a kv head)
    ([3009, 2500, 40], 2000, 4), ([193, 34, 353] * 14, 150, 0)])
@pytest.mark.parametrize("tail", [False, True])
def test_decode_scores_of_minus_infinity(hq, hkv, hd, lens, window, sink, tail):
    """Keys with an infinite norm and a negative product weigh nothing, also where a
    step, a wave's first one or a whole unit holds no others: the newest tokens
    alone (tail), or all but the newest ones."""
    c = C.make(hq + hd + len(lens), lens, hq, hkv, hd)
    q, _ = queries(c, len(lens), "fp16")
    qx = q.double().cpu().numpy()
    bad = np.zeros((c.nb, c.page), bool)
    for b, n in enumerate(c.lens):
        # one entry of each head in all the places, that whose products are furthest from 0
        pg, off, _ = C.places(c, b)
        at = slice((int(n) - 1) // 32 * 32, None) if tail else slice(0, int(n) - 3)
        bad[pg[at], off[at]] = True
        r = hq // hkv
        for h in range(hkv):
            k = C.rows(c, 0, pg, off, h)
            k /= np.linalg.norm(k, axis=-1, keepdims=True)
            x = C.rotated(c, qx[b, h * r:(h + 1) * r], True)
            dot = x / np.linalg.norm(x, axis=-1, keepdims=True) @ k.T
            best = int(np.abs(dot).min(0).argmax())
            assert np.abs(dot[:, best]).min() > 2e-3  # (far from what the kernel rounds)
            c.cache[0, pg[at], off[at], h] = c.cache[0, pg[best], off[best], h]
            q[b, h * r:(h + 1) * r] *= torch.from_numpy(-np.sign(dot[:, best]))[:, None].to(q)
    qx = q.double().cpu().numpy()
    c = norms(c, 0, lambda x: np.where(bad[..., None], np.inf, x))
    o = D.call(c, tensors(c), q, torch.full_like(q, 7.0), window, sink)
    D.check_o(norms(c, 0, lambda x: np.where(np.isfinite(x), x, 0)), o,
              decode_by_norms(c, qx, window, sink), qx, "fp16", window, sink)


@pytest.mark.parametrize("hq,hkv,hd", [(32, 8, 128), (16, 4, 64)])
@pytest.mark.parametrize("where", ["q", "k"])
def test_prefill_of_nan_scores_takes_its_usual_time(hq, hkv, hd, where):
    """Rows that their own scores make NaN are not computed a second time, one by
    one (which took 140 times as long)."""
    n, window, sink = 4096, 1024, 4
    q, k, v, reqs = make(1, [(n, n)], hq, hkv, hd)

    def time():
        start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        o = call(q, k, v, reqs, hd, window, sink)
        best = math.inf
        for _ in range(5):
            start.record()
            call(q, k, v, reqs, hd, window, sink, o)
            end.record()
            torch.cuda.synchronize()
            best = min(best, start.elapsed_time(end))
        return best, o
    usual, o = time()
    assert torch.isfinite(o).all()
    if where == "q":
        q[:] = math.nan
    else:
        k[0], v[0] = math.nan, math.nan
    spent, o = time()
    assert torch.isnan(o).all() and spent < 5 * usual


# the levels as the decode's table holds them: fp16 of 1.48098 times each, read as
# multiples of that
TABLE = (C.LEVELS * 1.4809800386428833).astype(np.float16).astype(np.float64) / 1.4809800386428833


@pytest.mark.parametrize("hq,hkv,hd", [(8, 2, 128), (16, 2, 64), (16, 2, 256), (8, 8, 128),
                                       (12, 6, 96)])
@pytest.mark.parametrize("many", [False, True])
def test_decode_of_one_token_is_its_value(monkeypatch, hq, hkv, hd, many):
    """Up to 8 q heads a kv head a probability enters as an fp16 pair and partial
    rows are fp32: a window of one token gives its V row (of the table's levels) to
    the output's rounding, 2^-11, and in front of it the pair's 2^-22 and fp32
    sums, 64 u, relative to the row, which the rotation back keeps.  One launch,
    and the split form for more workgroups than it takes (many)."""
    monkeypatch.setattr(C, "LEVELS", TABLE)
    lens = [(37 * i) % 90 + 1 for i in range(300 if many else 3)]
    c = C.make(hq + hd, lens, hq, hkv, hd)
    q, qx = queries(c, len(lens), "fp16")
    o = D.call(c, tensors(c), q, torch.full_like(q, 7.0), 1, 0).double().cpu().numpy()
    ref = W.decode(c, qx, 1, 0)
    at = [(C.places(c, b)[0][-1], C.places(c, b)[1][-1]) for b in range(len(lens))]
    size = np.stack([[np.linalg.norm(C.rows(c, 1, [pg], [off], h)) for h in range(hkv)]
                     for pg, off in at])
    tol = 2.0 ** -11 * np.abs(ref) + 2.0 ** -25 + \
        (2.0 ** -22 + 64 * 2.0 ** -24) * np.repeat(size, hq // hkv, 1)[..., None]
    err = np.abs(o - ref)
    assert (err <= tol).all(), f"off by {err.max():.3e}, {(err / tol).max():.2f} x bound"


@pytest.mark.parametrize("hq,hkv,hd", [(8, 2, 128), (16, 1, 64), (16, 2, 256)])
@pytest.mark.parametrize("lens,window", [([70, 200], 300), ([3000, 40], 2000)])
def test_rows_whose_every_score_is_minus_infinity_are_zeros(hq, hkv, hd, lens, window):
    """As the plain kernels leave them (their softmax has no value)."""
    c = C.make(5, lens, hq, hkv, hd)
    c.cache[0] = c.cache[0, :1, :1]  # (one entry a head, and so one sign of its products)
    c = norms(c, 0, lambda x: np.full_like(x, np.inf))
    unit = norms(c, 0, np.ones_like)
    q, qx = queries(c, len(lens), "fp16")
    for h in range(hkv):
        dot = C.rotated(c, qx[:, h * hq // hkv:(h + 1) * hq // hkv], True) @ \
            C.rows(unit, 0, [0], [0], h)[0]
        q[:, h * hq // hkv:(h + 1) * hq // hkv] *= torch.from_numpy(-np.sign(dot))[..., None].to(q)
    o = D.call(c, tensors(c), q, torch.full_like(q, 7.0), window, 2)
    assert (o == 0).all()
    # prefill: the first rows see the keys of the infinity alone
    q, k, v, reqs = make(3, [(lens[0], lens[0]), (3, 9000)], hq, hkv, hd)
    scores_of_minus_infinity(q, k, [0, 1, 2, *range(len(k) - 9000, len(k))])
    v[40, :, 1] = math.nan
    o = call(q, k, v, reqs, hd, window, 2)
    assert (o[:3] == 0).all() and (o[-3:] == 0).all() and torch.isfinite(o[3:40]).all()
