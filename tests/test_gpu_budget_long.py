"""Long sequences under the cache-budget operators: units of many steps, plans of
extreme shape, lengths near the limits."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import budget_cases as C
from test_gpu_budget import DEV, check_o, check_weights, queries, tensors
from turboquant_amd import ops

pytestmark = pytest.mark.gpu


def test_decode_of_a_sequence_as_long_as_all_units():
    """256 sequences, one of 36 million tokens and the others of one: the plan has
    a unit for each, and the long one's is split at 62% of its tokens, a product
    beyond 2^31.  Nearly all of its pages are outside the cache, so its attention
    is that of the few tokens that are there."""
    c = C.make(201, [16 * 40 + 9] + [1] * 255, 2, 1, 128)
    entries = 36_000_000 // 16
    length = (entries - 1) * 16 + 9
    unit = -(-length // 32) * 32
    cut = min((unit * 62 // 100 + 15) & ~15, unit) // 16
    at = np.concatenate((np.arange(5), cut + np.arange(-6, 6), [entries - 1]))
    rest = np.setdiff1d(c.rng.integers(0, entries, 100), at)
    at = np.sort(np.concatenate((at, c.rng.permutation(rest)[:41 - len(at)])))
    table = np.full(entries + 255, -1, np.int32)
    table[at], table[entries:] = c.indices[:41], c.indices[41:]
    indptr = np.concatenate(([0], entries + np.arange(256))).astype(np.int32)
    t = tensors(c)
    seq = t["seq"].clone()
    seq[0] = length
    q, qx = queries(c, 256, "fp16")
    o = torch.full((256, 2, 128), 7.0, dtype=torch.float16, device=DEV)
    ops.decode_paged_tracked(q, t["cache"], torch.from_numpy(table).to(DEV),
                             torch.from_numpy(indptr).to(DEV), seq, 1, 128, 128, c.scale, t["signs"],
                             o, t["weights"], t["positions"], t["ends"])
    torch.cuda.synchronize()
    ref_o, ref_w, ref_p = C.attend(c, qx, np.arange(257), 1, True, decode=True)
    check_weights(c, t["weights"].cpu().numpy(), ref_w, qx, 2)
    check_o(c, o, ref_o, qx, "fp16")
    assert np.array_equal(t["positions"].cpu().numpy(), ref_p)


# ---------------------------------------------------- units of many steps

CHUNK = 65536


def big_cache(seed, lens, hq, hkv, hd, page=16):
    """A random case on the GPU: budget_cases.make's layout as tensors."""
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    pd = C.pad(hd)
    half, ebs = pd // 2, C.entry(pd)
    need = [-(-n // page) for n in lens]
    nb = sum(need) + 3
    cache = torch.empty((2, nb, page, hkv, ebs), dtype=torch.uint8, device=DEV)
    for slab in cache:
        slab.random_(0, 256, generator=g)
        norm = (hd ** 0.5 * (0.3 * torch.randn((nb, page, hkv), generator=g, device=DEV)).exp()).half()
        slab[..., half:half + 2 * (pd // 64)] = \
            norm[..., None].repeat(1, 1, 1, pd // 64).view(torch.uint8)
    perm = torch.randperm(nb, generator=g, device=DEV).to(torch.int32)
    indptr = np.concatenate(([0], np.cumsum(need))).astype(np.int32)
    return dict(cache=cache, indices=perm[:sum(need)].clone(), indptr=torch.from_numpy(indptr).to(DEV),
                starts=indptr, seq=torch.tensor(lens, dtype=torch.int32, device=DEV),
                weights=torch.rand((nb, hkv, page), generator=g, device=DEV),
                positions=torch.full((nb, hkv, page), -7, dtype=torch.int32, device=DEV),
                ends=torch.tensor([n + 11 * i for i, n in enumerate(lens)], dtype=torch.int32,
                                  device=DEV),
                signs=torch.where(torch.rand(pd, generator=g, device=DEV) < 0.5, -1.0, 1.0),
                lens=lens, hq=hq, hkv=hkv, hd=hd, pd=pd, page=page, nb=nb, g=g)


def rows64(c, slab, pg, off, h):
    """Dequantized entries in the rotated domain [n, pd], 64 bits."""
    e = c["cache"][slab][pg, off, h]
    half = c["pd"] // 2
    codes = torch.stack((e[:, :half] >> 4, e[:, :half] & 15), 2).reshape(len(e), c["pd"])
    norm = e[:, half:half + 2].contiguous().view(torch.float16).double()
    levels = torch.from_numpy(C.LEVELS).to(DEV)
    return levels[codes.long()] * (norm / c["pd"] ** 0.5)


def attend64(c, q):
    """(o, what each token receives, positions, weights of the rows seen, largest row
    of K and of V), the tokens of a head in chunks."""
    pd, r = c["pd"], c["hq"] // c["hkv"]
    had = torch.from_numpy(C.hadamard(pd)).to(DEV)
    o = torch.zeros((len(c["lens"]), c["hq"], pd), dtype=torch.float64, device=DEV)
    weights, positions = c["weights"].double(), c["positions"].clone()
    x = torch.zeros((*q.shape[:2], pd), dtype=torch.float64, device=DEV)
    x[..., :c["hd"]] = q.double()
    x = (x * c["signs"].double()) @ had
    top = [0.0, 0.0]
    for b, n in enumerate(c["lens"]):
        if n == 0:
            continue
        t = torch.arange(n, device=DEV)
        entry = int(c["starts"][b]) + t // c["page"]
        pg = c["indices"][entry].long()
        ok = (pg >= 0) & (pg < c["nb"])
        pg, off = torch.where(ok, pg, 0), t % c["page"]
        for h in range(c["hkv"]):
            qq = (x[b, h * r:(h + 1) * r] * c["scale"]).t().contiguous()
            s = torch.empty((n, r), dtype=torch.float64, device=DEV)
            for a in range(0, n, CHUNK):
                z = slice(a, a + CHUNK)
                k = rows64(c, 0, pg[z], off[z], h)
                s[z] = k @ qq
                top[0] = max(top[0], float(k[ok[z]].norm(dim=1).max()) if ok[z].any() else 0.0)
            s[~ok] = -torch.inf
            p = torch.softmax(s, 0) if ok.any() else torch.zeros_like(s)
            for a in range(0, n, CHUNK):
                z = slice(a, a + CHUNK)
                v = rows64(c, 1, pg[z], off[z], h)
                v[~ok[z]] = 0
                o[b, h * r:(h + 1) * r] += p[z].t().contiguous() @ v
                top[1] = max(top[1], float(v.norm(dim=1).max()))
            got = p.sum(1)
            old = weights[pg[ok], h, off[ok]]
            fresh = (t == n - 1)[ok]
            weights[pg[ok], h, off[ok]] = torch.where(fresh, 0.0, old) + got[ok]
        if ok[-1]:
            positions[pg[-1], :, off[-1]] = c["ends"][b] - 1
    return ((o @ had) * c["signs"].double())[..., :c["hd"]], weights, positions, top


def check_long(c, dtype, q_scale=4.0):
    c["scale"] = c["hd"] ** -0.5
    b = len(c["lens"])
    q = (torch.randn((b, c["hq"], c["hd"]), generator=c["g"], device=DEV) * q_scale).to(dtype)
    ref_o, ref_w, ref_p, top = attend64(c, q)
    first = c["weights"].double()
    o = torch.full(tuple(q.shape), 7.0, dtype=dtype, device=DEV)
    ops.decode_paged_tracked(q, c["cache"], c["indices"], c["indptr"], c["seq"], c["hkv"], c["hd"],
                             c["pd"], c["scale"], c["signs"], o, c["weights"], c["positions"],
                             c["ends"])
    torch.cuda.synchronize()
    u = 2.0 ** -24
    # a score's error as test_gpu_budget derives it
    score = float(q.double().norm(dim=2).max()) * top[0] * c["scale"] * (8 + c["pd"] / 8 + 8) * u
    # A normaliser's chain of roundings: up to 320 steps of a unit, two each, 512
    # parts over 64 lanes and the joins; exp2, log2 and the sum over heads
    rel = 2 * score + (2 * 320 + 8 + 64) * u
    ratio = c["hq"] // c["hkv"]
    added = ref_w - first
    err = (c["weights"].double() - ref_w).abs()
    tol = rel * torch.maximum(ref_w.abs(), added.abs().clamp_max(ratio)) + 2 * u * ref_w.abs() + 1e-37
    assert bool((err <= tol).all()), f"weights {float((err / tol).max()):.2f} x bound"
    assert torch.equal(c["positions"], ref_p)
    # Outputs: as there; sums over 320 steps and 512 parts are chains of as many
    # roundings in front of the last one
    half = torch.finfo(dtype).eps / 2
    p = (2.0 ** -22 if ratio <= 8 else 2.0 ** -11) + 2 * score + 2.0 ** -18 + 900 * u
    err = (o.double() - ref_o).abs()
    tol = half * ref_o.abs() + (8.7e-5 + p) * top[1] * (1 + half) + 2.0 ** -24
    assert bool((err <= tol).all()), f"o {float((err / tol).max()):.2f} x bound"


@pytest.mark.parametrize("hq,hkv,hd", [
    (4, 1, 128), (16, 2, 128), (8, 4, 128), (32, 8, 128), (16, 1, 128), (24, 2, 128), (36, 4, 96),
    (8, 1, 64), (4, 2, 64), (16, 4, 64), (8, 8, 64), (12, 1, 64), (32, 2, 64),
    (8, 1, 256), (4, 2, 256), (4, 4, 256), (16, 1, 200), (20, 2, 256)])
def test_decode_in_steady_state(hq, hkv, hd):
    """A sequence of 600011 tokens is a unit of over 1024 (64 tiles) for each
    workgroup: slots of the ring are used again, the tile window moves on, scores and
    weights come from the step before.  Pages outside the cache lie inside units."""
    c = big_cache(hq * 300 + hd, [600011], hq, hkv, hd)
    n = len(c["indices"])
    c["indices"][torch.arange(70, n, 977, device=DEV)] = -1
    c["indices"][n // 2] = c["nb"]
    check_long(c, torch.float16 if hkv % 2 else torch.bfloat16)


@pytest.mark.parametrize("hq,hkv,hd", [(8, 2, 128), (16, 4, 64), (8, 2, 256)])
def test_decode_of_long_and_short_sequences(hq, hkv, hd):
    """Ragged: over 64 sequences, the plan in LDS, units of many steps and of one."""
    rng = np.random.default_rng(hd)
    lens = [int(n) for n in rng.integers(0, 90, 67)]
    lens[5], lens[40], lens[66] = 400003, 150001, 33333
    check_long(big_cache(hd, lens, hq, hkv, hd, page=48 if hd == 64 else 16), torch.float16)
