"""Outputs of the tracked decode where the value rows are small or their norms
differ widely, and most of the weight is in a long tail of small pieces: against
64 bits within the bound that every other size has to keep."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import budget_cases as C
from test_gpu_budget import DEV, check_o, check_weights, score_error, tensors
from turboquant_amd import ops

pytestmark = pytest.mark.gpu


def tail_case(seed, lens, ratio, hkv, hd, top, norm_scale=1.0):
    """Every token of a head has the same codes, so that the values add up
    instead of averaging out.  One token of each sequence scores about `top`, the
    others between 0 and top / 20 (q points along the key; norms set the rest).
    Returns the case and q fp16 [B, Hq, hd] with its exact values."""
    c = C.make(seed, lens, hkv * ratio, hkv, hd, norm_scale=norm_scale)
    half = c.pd // 2
    one = c.rng.integers(0, 256, (2, 1, 1, hkv, half), dtype=np.uint8)
    c.cache[..., :half] = one
    set_norms(c, 0, np.abs(c.rng.standard_normal((c.nb, c.page, hkv))) / 60)
    q = np.zeros((len(lens), c.hq, c.hd))
    for h in range(hkv):
        codes = np.stack((one[0, 0, 0, h] >> 4, one[0, 0, 0, h] & 15), 1).reshape(-1)
        k = C.LEVELS[codes] / np.sqrt(c.pd)
        back = ((k @ C.hadamard(c.pd)) * c.signs)[:hd]
        for i in range(ratio):  # heads differ by a few percent
            q[:, h * ratio + i] = back * top * (1 - 0.01 * i) / (c.scale * (k @ k))
    for b, n in enumerate(lens):
        pg, off, _ = C.places(c, b)
        at = n // 3
        c.cache[0, pg[at], off[at], :, half:half + 2 * (c.pd // 64)] = \
            np.full(c.pd // 64, 1.0, np.float16).view(np.uint8)
    q = torch.from_numpy(q).to(torch.float16)
    return c, q.to(DEV), q.double().numpy()


def set_norms(c, slab, norms):
    """norms [blocks, page, heads]"""
    half, n = c.pd // 2, c.pd // 64
    c.cache[slab, ..., half:half + 2 * n] = \
        np.repeat(norms.astype(np.float16)[..., None], n, -1).view(np.uint8)


def run(c, q, qx):
    t = tensors(c)
    b = len(c.lens)
    o = torch.full((b, c.hq, c.hd), 7.0, dtype=torch.float16, device=DEV)
    ops.decode_paged_tracked(q, t["cache"], t["indices"], t["indptr"], t["seq"], c.hkv, c.hd, c.pd,
                             c.scale, t["signs"], o, t["weights"], t["positions"], t["ends"])
    torch.cuda.synchronize()
    ref_o, ref_w, _ = C.attend(c, qx, np.arange(b + 1), 1, True, decode=True)
    check_weights(c, t["weights"].cpu().numpy(), ref_w, qx, c.hq // c.hkv)
    check_o(c, o, ref_o, qx, "fp16")


@pytest.mark.parametrize("norm_scale", [1.0, 1e-2, 1e-4, 1e-5])
@pytest.mark.parametrize("ratio,hkv,hd", [(4, 2, 128), (16, 1, 128), (2, 2, 64), (12, 2, 64),
                                          (4, 1, 256), (9, 1, 256)])
def test_small_values_under_a_long_tail(ratio, hkv, hd, norm_scale):
    """A tail of weight 1.1 to 3.3 beside a peak of weight 1, in pieces of e^-8 to
    e^-7.6 of the peak's: value norms down to 1e-4."""
    c, q, qx = tail_case(hd + ratio, [4000, 700], ratio, hkv, hd, 8.0, norm_scale)
    run(c, q, qx)


@pytest.mark.parametrize("ratio,hkv,hd", [(4, 2, 128), (16, 1, 128), (2, 2, 64), (4, 1, 256)])
def test_a_huge_row_that_gets_no_weight_hides_nothing(ratio, hkv, hd):
    """Value rows of norm 0.001, and one of 60000 among them whose key scores 30
    below the others' tail: its products stay far below theirs."""
    c, q, qx = tail_case(1000 + hd + ratio, [3000, 64], ratio, hkv, hd, 8.0, 1e-4)
    for b, n in enumerate((3000, 64)):
        pg, off, _ = C.places(c, b)
        at = n // 2
        for slab, norm in ((0, -4.0), (1, 60000.0)):
            c.cache[slab, pg[at], off[at], :, c.pd // 2:c.pd // 2 + 2 * (c.pd // 64)] = \
                np.full(c.pd // 64, norm, np.float16).view(np.uint8)
    t = tensors(c)
    o = torch.empty((2, c.hq, c.hd), dtype=torch.float16, device=DEV)
    ops.decode_paged_tracked(q, t["cache"], t["indices"], t["indptr"], t["seq"], c.hkv, c.hd, c.pd,
                             c.scale, t["signs"], o, t["weights"], t["positions"], t["ends"])
    ref_o, _, _ = C.attend(c, qx, np.arange(3), 1, True, decode=True)
    # check_o's bound with another largest row: what the huge one adds is below
    # e^-40 x 60000 < 1e-12 of the peak's weight, so errors go by the largest row
    # of the others (in every head and sequence).
    others = 0.0
    for b in range(2):
        pg, off, _ = C.places(c, b)
        for h in range(c.hkv):
            norms = np.sort(np.sqrt((C.rows(c, 1, pg, off, h) ** 2).sum(-1)))
            assert norms[-1] > 1e4 and norms[-2] < 0.1
            others = max(others, norms[-2])
    p = (2.0 ** -22 if ratio <= 8 else 2.0 ** -11) + 2 * score_error(c, qx) + 2.0 ** -18
    tol = 2.0 ** -11 * np.abs(ref_o) + (8.7e-5 + p) * others * (1 + 2.0 ** -11) + 2.0 ** -24
    err = np.abs(o.double().cpu().numpy() - ref_o)
    assert (err <= tol).all(), f"{(err / tol).max():.2f} x bound"


@pytest.mark.parametrize("order", ["rising", "falling", "mixed"])
@pytest.mark.parametrize("ratio,hkv,hd", [(2, 256, 128), (10, 192, 64), (1, 130, 64), (1, 128, 256)])
def test_norms_over_eight_decades(ratio, hkv, hd, order):
    """Norms from 1e-4 to 10^4 along a sequence.  With this many kv heads a wave
    takes many tiles of it, so its scale changes on the way when they rise."""
    c = C.make(hkv + hd, [1500], ratio * hkv, hkv, hd)
    pg, off, _ = C.places(c, 0)
    norms = np.zeros((c.nb, c.page, hkv))
    steps = 10.0 ** np.linspace(-4, 4, 1500)
    steps = {"rising": steps, "falling": steps[::-1], "mixed": c.rng.permutation(steps)}[order]
    norms[pg, off] = steps[:, None]
    set_norms(c, 1, norms)
    q = torch.from_numpy(c.rng.standard_normal((1, c.hq, c.hd))).to(torch.float16)
    run(c, q.to(DEV), q.double().numpy())


@pytest.mark.parametrize("top", [20.0, 34.0, 45.0, 75.0])
@pytest.mark.parametrize("ratio,hkv,hd", [(2, 256, 128), (10, 192, 64), (1, 128, 256)])
def test_tiles_of_next_to_no_weight_in_front_of_heavy_ones(ratio, hkv, hd, top):
    """Most tiles hold weights of e^-top of the heavy tokens', some 97 tokens apart,
    so that a wave meets them in any order: its scale has to change by as much."""
    c, q, qx = tail_case(hkv + hd, [1500], ratio, hkv, hd, top)
    pg, off, _ = C.places(c, 0)
    norms = np.abs(c.rng.standard_normal((c.nb, c.page, hkv))) / 60
    norms[pg[60::97], off[60::97]] = 1.0 - 0.01 * c.rng.random((len(pg[60::97]), hkv))
    set_norms(c, 0, norms)
    run(c, q, qx)
