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


def prefill(q, k, v, requests, ratio, scale, window, sink):
    """o [T, Hq, D] (0 in rows of no request) of q [T, Hq, D] over k, v [R, Hkv,
    D], all in 64 bits; torch tensors, on their device."""
    import torch
    o = torch.zeros_like(q)
    for qs, ql, ks, kl, _ in requests:
        for at in range(0, ql, 2048):
            n = min(2048, ql - at)
            pos = torch.arange(kl - ql + at, kl - ql + at + n, device=q.device)[:, None]
            j = torch.arange(kl, device=q.device)[None]
            see = (j <= pos) & ((j > pos - window) | (j < sink))
            used = torch.nonzero(see.any(0))[:, 0]
            see = see[:, used]
            for h in range(q.shape[1]):
                kk, vv = k[ks + used, h // ratio], v[ks + used, h // ratio]
                s = (q[qs + at:qs + at + n, h] @ kk.T) * scale
                p = torch.where(see, s, -torch.inf).softmax(-1)
                # a hidden key adds nothing, whatever its value; one in sight has
                # a weight above zero
                out = p @ torch.where(torch.isfinite(vv), vv, 0.0)
                hit = lambda x: see.double() @ x.double() > 0
                up, down = hit(vv == torch.inf), hit(vv == -torch.inf)
                out = torch.where(up, torch.inf, torch.where(down, -torch.inf, out))
                out = torch.where(hit(torch.isnan(vv)) | (up & down), torch.nan, out)
                o[qs + at:qs + at + n, h] = out
    return o


def norm_rope(qkv, qw, kw, cos, sin, positions, sections, hq, hkv, hd, eps):
    """(q, k, their normed values in front of the rotation) [T, H, hd] in 64 bits
    of qkv [T, (Hq + 2 Hkv) hd]; a position outside the tables gives NaN rows."""
    import torch
    n, half = len(qkv), cos.shape[1]
    x = qkv.double().view(n, -1, hd)
    pos = positions.view(-1, n).long()
    inside = ((pos >= 0) & (pos < len(cos))).all(0)
    at, c, s = 0, [], []
    for p, m in zip(pos.clamp(0, len(cos) - 1), sections):
        c.append(cos.double()[p, at:at + m])
        s.append(sin.double()[p, at:at + m])
        at += m
    c, s = (torch.where(inside[:, None], torch.cat(t, 1), torch.nan)[:, None] for t in (c, s))
    out = []
    for y, w in ((x[:, :hq], qw), (x[:, hq:hq + hkv], kw)):
        if w is not None:
            y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps) * w.double()
        a, b = y[..., :half], y[..., half:2 * half]
        z = torch.cat((a * c - b * s, b * c + a * s, y[..., 2 * half:]), -1)
        out.append((torch.where(inside[:, None, None], z, torch.nan), y))
    return out[0][0], out[1][0], torch.cat((out[0][1], out[1][1]), 1)
