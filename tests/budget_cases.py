"""Shared by the cache-budget tests: random packed caches, page tables and
records, and the operators in 64 bits on the CPU (numpy, sequence by sequence).
"""
from __future__ import annotations

import math
from types import SimpleNamespace

import numpy as np

LEVELS = np.array([-2.7326368, -2.0693470, -1.6180345, -1.2562491, -0.9423684, -0.6567591,
                   -0.3880823, -0.1284154, 0.1284154, 0.3880823, 0.6567591, 0.9423684, 1.2562491,
                   1.6180345, 2.0693470, 2.7326368], np.float32).astype(np.float64)


def pad(hd):
    return max(64, 1 << (hd - 1).bit_length())


def entry(pd):
    return (pd // 2 + 2 * (pd // 64) + 15) & ~15


def hadamard(n):
    i = np.arange(n)
    x = i[:, None] & i[None, :]
    bits = np.zeros_like(x)
    while x.any():
        bits ^= x & 1
        x = x >> 1
    return (1.0 - 2.0 * bits) / math.sqrt(n)


def make(seed, lens, hq, hkv, hd, page=16, extra=3, packed=True, norm_scale=1.0):
    """A random cache with a random page permutation; pages behind a table row
    hold -1 where the rows are padded to one width (packed False)."""
    rng = np.random.default_rng(seed)
    pd = pad(hd)
    ebs = entry(pd)
    need = [-(-max(0, n) // page) for n in lens]
    nb = sum(need) + extra
    perm = rng.permutation(nb).astype(np.int32)
    cache = rng.integers(0, 256, (2, nb, page, hkv, ebs), dtype=np.uint8)
    norm = (math.sqrt(hd) * norm_scale * np.exp(0.3 * rng.standard_normal((2, nb, page, hkv)))) \
        .astype(np.float16)
    nbytes = np.repeat(norm[..., None], pd // 64, -1).view(np.uint8)
    cache[..., pd // 2:pd // 2 + 2 * (pd // 64)] = nbytes
    width = max(need) if need else 0
    if packed:
        indptr = np.concatenate(([0], np.cumsum(need))).astype(np.int32)
        indices = perm[:sum(need)].copy()
    else:
        indptr = (np.arange(len(lens) + 1) * width).astype(np.int32)
        indices = np.full(len(lens) * width, -1, np.int32)
        at = 0
        for b, n in enumerate(need):
            indices[b * width:b * width + n] = perm[at:at + n]
            at += n
    weights = rng.exponential(0.2, (nb, hkv, page)).astype(np.float32)
    positions = rng.integers(-50, 5, (nb, hkv, page)).astype(np.int32)
    ends = (np.maximum(lens, 0) + rng.integers(0, 100, len(lens))).astype(np.int32)
    signs = np.where(rng.random(pd) < 0.5, -1.0, 1.0).astype(np.float32)
    return SimpleNamespace(rng=rng, lens=np.asarray(lens, np.int32), hq=hq, hkv=hkv, hd=hd, pd=pd,
                           page=page, cache=cache, indices=indices, indptr=indptr,
                           weights=weights, positions=positions, ends=ends, signs=signs,
                           scale=1.0 / math.sqrt(hd), nb=nb)


def places(c, b):
    """(pages, offsets, there) of sequence b's tokens; there: on a page of the
    cache, reached through the table."""
    t = np.arange(max(0, int(c.lens[b])))
    e = int(c.indptr[b]) + t // c.page
    ok = (e >= 0) & (e < len(c.indices))
    pg = np.where(ok, c.indices[np.clip(e, 0, max(0, len(c.indices) - 1))]
                  if len(c.indices) else -1, -1)
    ok &= (pg >= 0) & (pg < c.nb)
    return np.where(ok, pg, 0), t % c.page, ok


def rows(c, slab, pg, off, h):
    """Dequantized entries in the rotated domain [n, pd]."""
    e = c.cache[slab, pg, off, h]
    q = e[:, :c.pd // 2]
    codes = np.stack((q >> 4, q & 15), 2).reshape(len(e), c.pd)
    norm = e[:, c.pd // 2:c.pd // 2 + 2].copy().view(np.float16).astype(np.float64)
    return LEVELS[codes] * norm / math.sqrt(c.pd)


def rotated(c, q, signs):
    x = np.zeros((*q.shape[:-1], c.pd))
    x[..., :c.hd] = q.astype(np.float64)
    return (x * c.signs) @ hadamard(c.pd) if signs else x


def attend(c, q, starts, window, signs=True, decode=False):
    """The record of the last `window` rows of each chunk; returns (o, weights,
    positions) with o None unless decode (one row per sequence)."""
    acc, pos = c.weights.astype(np.float64), c.positions.copy()
    r = c.hq // c.hkv
    o = np.zeros((len(c.lens), c.hq, c.pd))
    for b in range(len(c.lens)):
        n, chunk = int(c.lens[b]), int(starts[b + 1] - starts[b])
        w = min(chunk, window)
        if n <= 0 or w <= 0:
            continue
        pg, off, ok = places(c, b)
        t = np.arange(n)
        for h in range(c.hkv):
            k = rows(c, 0, pg, off, h)
            got = np.zeros(n)
            for i in range(w):
                qq = rotated(c, q[starts[b + 1] - w + i, h * r:(h + 1) * r], signs)
                see = ok & (t <= n - w + i)
                if not see.any():
                    continue
                with np.errstate(invalid="ignore"):
                    s = np.where(see, qq @ np.where(see[:, None], k, 0).T * c.scale, -np.inf)
                    p = np.exp(s - s.max(-1, keepdims=True))
                    p /= p.sum(-1, keepdims=True)
                got += p.sum(0)
                if decode:
                    v = rows(c, 1, pg, off, h)
                    o[b, h * r:(h + 1) * r] = p @ np.where(ok[:, None], v, 0)
            old = acc[pg, h, off]
            new = np.where(t < n - chunk, old + got, got)
            acc[pg[ok], h, off[ok]] = new[ok]
            fresh = ok & (t >= n - chunk)
            pos[pg[fresh], h, off[fresh]] = (int(c.ends[b]) - n + t)[fresh]
    if signs:
        o = (o @ hadamard(c.pd)) * c.signs
    return (o[..., :c.hd] if decode else None), acc, pos


def evict(c, budget, recent, sink):
    """(cache, weights, positions, lens) after the cut."""
    cache, acc, pos = c.cache.copy(), c.weights.copy(), c.positions.copy()
    for b in range(len(c.lens)):
        n = int(c.lens[b])
        if n <= budget:
            continue
        pg, off, ok = places(c, b)
        for h in range(c.hkv):
            w, p = acc[pg, h, off].astype(np.float64), pos[pg, h, off]
            held = (p < sink) | (p >= int(c.ends[b]) - recent)
            rank = np.where(np.isnan(w), -np.inf, w)
            order = np.lexsort((np.arange(n), -rank, np.isnan(w), ~held, ~ok))
            # protected entries among themselves by index
            hold = np.flatnonzero(held & ok)
            rest = [i for i in order if not (held[i] and ok[i])]
            keep = np.zeros(n, bool)
            keep[np.concatenate((hold, rest)).astype(int)[:budget]] = True
            to, of = np.flatnonzero(~keep[:budget]), budget + np.flatnonzero(keep[budget:])
            m = ok[to] & ok[of]
            to, of = to[m], of[m]
            acc[pg[to], h, off[to]] = acc[pg[of], h, off[of]]
            pos[pg[to], h, off[to]] = pos[pg[of], h, off[of]]
            for slab in cache:
                slab[pg[to], off[to], h] = slab[pg[of], off[of], h]
    return cache, acc, pos, np.minimum(c.lens, budget).astype(np.int32)
