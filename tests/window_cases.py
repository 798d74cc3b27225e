"""Shared by the tests of windowed attention: the operators in 64 bits on the
CPU (numpy, sequence by sequence), on the random packed caches of budget_cases.

A query at position P sees the keys j with P - window < j <= P, and j < sink."""
from __future__ import annotations

import numpy as np

import budget_cases as C


def sees(pos, n, window, sink):
    """Which of n keys a query at `pos` sees."""
    j = np.arange(n)
    return (j <= pos) & ((j > pos - window) | (j < sink))


def release(c, window, sink, garbage=(-1, 2 ** 31 - 1, -2 ** 31)):
    """Table entries of pages without a token in sight of the newest one, as a
    server that gave the pages back may leave them."""
    k = 0
    for b, n in enumerate(c.lens):
        see = sees(n - 1, max(0, int(n)), window, sink)
        for i in range(0, len(see), c.page):
            if not see[i:i + c.page].any():
                c.indices[c.indptr[b] + i // c.page] = garbage[k % len(garbage)]
                k += 1
    return c


def poison(c, window, sink):
    """Norms of hidden entries on pages that stay: NaN and infinities."""
    bad = np.array([np.nan, np.inf, -np.inf], np.float16)
    k = 0
    for b, n in enumerate(c.lens):
        pg, off, ok = C.places(c, b)
        hide = ok & ~sees(int(n) - 1, len(pg), window, sink)
        for p, o in zip(pg[hide], off[hide]):
            c.cache[:, p, o, :, c.pd // 2:c.pd // 2 + 2 * (c.pd // 64)] = \
                np.repeat(bad[k % 3:k % 3 + 1], c.pd // 64).view(np.uint8)
            k += 1
    return c


def decode(c, q, window, sink, signs=True):
    """o [B, Hq, hd] of one query per sequence, q [B, Hq, hd]."""
    r = c.hq // c.hkv
    o = np.zeros((len(c.lens), c.hq, c.pd))
    for b, n in enumerate(c.lens):
        pg, off, ok = C.places(c, b)
        see = ok & sees(int(n) - 1, len(pg), window, sink)
        pg, off = pg[see], off[see]
        if not len(pg):
            continue
        for h in range(c.hkv):
            s = C.rotated(c, q[b, h * r:(h + 1) * r], signs) @ C.rows(c, 0, pg, off, h).T * c.scale
            with np.errstate(invalid="ignore"):
                p = np.exp(s - s.max(-1, keepdims=True))
                o[b, h * r:(h + 1) * r] = p / p.sum(-1, keepdims=True) @ C.rows(c, 1, pg, off, h)
    if signs:
        o = (o @ C.hadamard(c.pd)) * c.signs
    return o[..., :c.hd]
