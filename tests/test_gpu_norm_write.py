"""The norm-rotate-write of a fused projection on an MI355X: q and k against the
formula in 64 bits, the cache against the write of the rows it returns."""
from __future__ import annotations

import math

import pytest
import torch

import budget_cases as C
import window_cases as W
from turboquant_amd import ops

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
ROWS = 700  # of the tables


class Case:
    def __init__(self, seed, n, hq, hkv, hd, rotated=None, dtype="fp16", sections=None, norms=True,
                 slots=None, blocks=None, page=16, wide=torch.int64):
        g = torch.Generator(device=DEV)
        g.manual_seed(seed)
        self.g, self.n, self.hq, self.hkv, self.hd, self.pd = g, n, hq, hkv, hd, C.pad(hd)
        self.dt, half = TYPES[dtype], (rotated or hd) // 2
        randn = lambda *s: torch.randn(s, generator=g, device=DEV)
        self.qkv = (randn(n, hq + 2 * hkv, hd) * randn(n, hq + 2 * hkv, 1).exp()).to(self.dt) \
            .view(n, (hq + 2 * hkv) * hd)
        self.qw, self.kw = ((1 + 0.2 * randn(hd)).to(self.dt) if norms else None for _ in range(2))
        angle = torch.arange(ROWS, device=DEV).double()[:, None] \
            * 1e4 ** (-torch.arange(half, device=DEV).double() / half)
        self.cos, self.sin = angle.cos().float(), angle.sin().float()
        self.sections = sections
        axes = len(sections) if sections else 1
        pos = torch.randint(0, ROWS, (axes, n), generator=g, device=DEV)
        self.positions = (pos if sections else pos[0]).to(wide)
        nb = blocks or -(-n // page) + 2
        self.cache = torch.randint(0, 256, (2, nb, page, hkv, C.entry(self.pd)), generator=g,
                                   dtype=torch.uint8, device=DEV)
        if slots is None:
            slots = torch.randperm(nb * page, generator=g, device=DEV)[:n]
        self.slots = slots.to(torch.int32)
        self.signs = torch.where(randn(self.pd) < 0, -1.0, 1.0)
        self.eps = 1e-6

    def call(self, q=None, k=None, keep_k=True, **other):
        a = {**self.__dict__, **other}
        q = torch.full((self.n, self.hq, self.hd), 7.0, dtype=self.dt, device=DEV) \
            if q is None else q
        if k is None and keep_k:
            k = torch.full((self.n, self.hkv, self.hd), 7.0, dtype=self.dt, device=DEV)
        cache = a["cache"].clone() if "into" not in other else other["into"]
        ops.norm_rope_write(a["qkv"], a["qw"], a["kw"], a["cos"], a["sin"], a["positions"], cache,
                            a["signs"], a["slots"], self.hq, self.hd, self.pd, q, k, eps=self.eps,
                            sections=a["sections"])
        return q, k, cache

    def check(self, q, k, cache):
        """u = 2^-24.  The mean of squares is a chain of at most 32 + 3 fp32 sums,
        half of whose relative error reaches the scale; rsqrt, the products with
        scale, weight and angle and the pair's sum add at most 12 u: 32 u of both
        of a pair's values covers them; then the rounding to the rows' type."""
        if self.n == 0:
            assert torch.equal(cache, self.cache)
            return
        u = 2.0 ** -24
        half = 2.0 ** -11 if self.dt == torch.float16 else 2.0 ** -8
        rot = self.cos.shape[1]
        rq, rk, before = W.norm_rope(self.qkv, self.qw, self.kw, self.cos, self.sin, self.positions,
                                     self.sections or (rot,), self.hq, self.hkv, self.hd, self.eps)
        size = before.abs()
        pair = size[..., :rot] + size[..., rot:2 * rot]
        size = torch.cat((pair, pair, size[..., 2 * rot:]), -1)
        got = q if k is None else torch.cat((q, k), 1)
        ref = rq if k is None else torch.cat((rq, rk), 1)
        size = size[:, :got.shape[1]]
        top = torch.finfo(self.dt).max
        tol = half * ref.abs() + 32 * u * size * (1 + half) + 2.0 ** -25
        got, over = got.double(), ref.abs() > top * (1 - half)
        err = (got - ref).abs()
        assert torch.equal(torch.isnan(got), torch.isnan(ref))
        ok = (err <= tol) | torch.isnan(ref) | over
        assert ok.all(), f"off by {float(err[~ok].max()):.3e}, {float((err / tol)[~ok].max()):.2f} x"
        # the cache holds those rows as the write leaves them, everything else as it was
        want = self.cache.clone()
        v = self.qkv.view(self.n, -1, self.hd)[:, self.hq + self.hkv:]
        if k is not None:
            ops.quantize_write_kv_cache(want, k, v, self.signs, self.slots, self.hd, self.pd)
            assert torch.equal(self.plain(cache), self.plain(want))

    def plain(self, cache):
        """The bytes with every NaN norm as one NaN: which of several NaN elements
        gives the norm its sign is left open."""
        cache = cache.clone()
        at = slice(self.pd // 2, self.pd // 2 + 2 * (self.pd // 64))
        norms = cache[..., at].contiguous().view(torch.float16)
        norms = torch.where(torch.isnan(norms), torch.full_like(norms, math.nan), norms)
        cache[..., at] = norms.view(torch.uint8)
        return cache

    def run(self, **kw):
        out = self.call(**kw)
        torch.cuda.synchronize()
        self.check(*out)
        return out


@pytest.mark.parametrize("hq,hkv,hd,rotated", [
    (32, 8, 128, 128), (32, 8, 128, 64), (32, 8, 128, 96), (32, 8, 128, 16), (16, 4, 64, 64),
    (16, 4, 64, 32), (16, 4, 64, 48), (16, 2, 256, 256), (16, 2, 256, 128), (4, 4, 256, 64),
    (12, 4, 96, 96), (12, 4, 96, 48), (12, 4, 96, 64), (6, 3, 80, 80), (6, 3, 72, 64),
    (8, 1, 128, 128), (1, 1, 40, 32), (3, 3, 64, 16), (64, 8, 128, 128), (5, 5, 200, 192)])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_geometries(hq, hkv, hd, rotated, dtype):
    Case(hd + rotated, 133, hq, hkv, hd, rotated, dtype).run()


@pytest.mark.parametrize("n", [0, 1, 2, 7, 63, 64, 65, 500, 5000])
def test_tokens(n):
    Case(n, n, 8, 2, 128).run()
    Case(n, n, 3, 1, 64, dtype="bf16", norms=False).run()


@pytest.mark.parametrize("sections", [(64,), (16, 24, 24), (16, 48), (1, 62, 1), (21, 22, 21),
                                      (0, 64), (64, 0, 0, 0), (13, 17, 3, 31)])
@pytest.mark.parametrize("wide", [torch.int32, torch.int64])
def test_positions_of_several_axes(sections, wide):
    Case(len(sections), 50, 8, 2, 128, sections=sections, wide=wide).run()
    half = [s // 4 for s in sections]
    half[-1] += 16 - sum(half)  # pairs whose partner stands in another lane
    Case(9 + len(sections), 50, 8, 2, 128, rotated=32, sections=half, wide=wide,
         dtype="bf16").run()


def test_without_norms_and_without_k():
    c = Case(1, 90, 8, 2, 128, norms=False)
    c.run()
    q, k, cache = c.call()
    q2, none, cache2 = c.call(keep_k=False)
    assert none is None and torch.equal(q, q2) and torch.equal(cache, cache2)


def test_slots():
    """No slot, one beyond the cache, repeated absences; other entries stay."""
    c = Case(2, 40, 8, 2, 128)
    c.slots[::3] = -1
    c.slots[1] = c.cache.shape[1] * 16
    c.slots[2] = 2 ** 31 - 1
    c.slots[4] = -2 ** 31
    c.run()
    c.slots[:] = -1
    _, _, cache = c.run()
    assert torch.equal(cache, c.cache)


@pytest.mark.parametrize("hd,dtype", [(128, "fp16"), (128, "bf16"), (64, "fp16"), (96, "bf16"),
                                      (256, "fp16")])
def test_values_at_the_ends_of_the_types(hd, dtype):
    """Rows of zeros, of the smallest and of the largest values, NaN and infinities."""
    c = Case(3, 60, 4, 2, hd, dtype=dtype)
    x = c.qkv.view(60, 8, hd)
    top = torch.finfo(c.dt).max
    x[0], x[1], x[2] = 0.0, torch.finfo(c.dt).smallest_normal / 4, top
    x[3, :, 5], x[4, :, hd - 1], x[5, :, 0] = math.nan, math.inf, -math.inf
    x[6] *= 1e-3
    x[7, :, 1:] = 0.0
    c.run()
    c.qw = c.kw = None
    c.run()
    c.qw = c.kw = torch.ones(hd, dtype=c.dt, device=DEV)
    for c.eps in (1e-30, 2.0 ** -126):
        c.run()
    c.eps = 0.0  # (squares of small rows would be lost beside it)
    with pytest.raises(RuntimeError, match="eps"):
        c.call()


@pytest.mark.parametrize("sections", [None, (16, 24, 24)])
def test_positions_outside_the_tables_give_nan_rows(sections):
    for rotated in (128, 48):
        s = None if sections is None else [x * rotated // 128 for x in sections]
        c = Case(4, 30, 8, 2, 128, rotated=rotated, sections=s)
        p = c.positions.view(-1, 30)
        p[-1, 3], p[0, 4], p[-1, 5] = ROWS, -1, 2 ** 62
        q, k, _ = c.run()
        bad = torch.isnan(q).all(-1).all(-1)
        assert bad.nonzero()[:, 0].tolist() == [3, 4, 5]
        assert torch.isnan(k[3:6]).all()


def test_strides_and_alignment():
    c = Case(5, 70, 8, 2, 128, dtype="bf16")
    want = c.run()
    width = c.qkv.shape[1]
    for lead, extra in ((8, 24), (0, 8), (3, 5), (1, 0)):
        buf = torch.full((70, lead + width + extra), 9.0, dtype=c.dt, device=DEV)
        rows = buf[:, lead:lead + width]
        rows.copy_(c.qkv)
        got = c.call(qkv=rows)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    back = torch.empty((70, 3 * width), dtype=c.dt, device=DEV)[:, width:2 * width]
    back.copy_(c.qkv)
    wt = torch.empty(300, dtype=c.dt, device=DEV)[1:129].copy_(c.qw)
    table = torch.empty((ROWS, 130), device=DEV)
    cos, sin = table[:, 1:65].copy_(c.cos), table[:, 66:].copy_(c.sin)
    pos = torch.stack((c.positions, c.positions), 1)[:, 0]
    slots = torch.stack((c.slots, c.slots), 1)[:, 1]
    got = c.call(qkv=back, qw=wt, cos=cos, sin=sin, positions=pos, slots=slots)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_rows_and_slots_beyond_32_bit_offsets():
    c = Case(6, 3, 8, 8, 128)
    want = c.run()
    stride = 1_100_000_000  # elements
    big = torch.empty(2 * stride + c.qkv.shape[1], dtype=c.dt, device=DEV)
    rows = big.as_strided((3, c.qkv.shape[1]), (stride, 1))
    rows.copy_(c.qkv)
    assert all(torch.equal(a, b) for a, b in zip(c.call(qkv=rows), want))
    del big, rows
    far = 440_000
    cache = torch.empty((2, far + c.cache.shape[1], 16, 8, 80), dtype=torch.uint8, device=DEV)
    cache[:, far:] = c.cache
    c.call(slots=c.slots + 16 * far, into=cache)
    assert torch.equal(cache[:, far:], want[2])


def test_rows_that_overlap_are_refused():
    c = Case(7, 20, 8, 2, 128)
    flat = c.qkv.view(-1)
    for q in (flat[:20 * 8 * 128].view(20, 8, 128), flat[-20 * 8 * 128:].view(20, 8, 128)):
        with pytest.raises(RuntimeError, match="overlap"):
            c.call(q=q)
    both = torch.empty(20 * 10 * 128, dtype=c.dt, device=DEV)
    with pytest.raises(RuntimeError, match="overlap"):
        c.call(q=both[:20 * 8 * 128].view(20, 8, 128),
               k=both[20 * 7 * 128:20 * 9 * 128].view(20, 2, 128))
    c.check(*c.call(q=both[:20 * 8 * 128].view(20, 8, 128),
                    k=both[20 * 8 * 128:].view(20, 2, 128)))


def test_repeated_calls_streams_a_graph_and_the_op():
    c = Case(8, 300, 16, 4, 64, dtype="bf16")
    want = c.run()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    outs = []
    for i in range(6):
        with torch.cuda.stream(streams[i % 2]):
            outs.append(c.call())
    torch.cuda.synchronize()
    for out in outs:
        assert all(torch.equal(a, b) for a, b in zip(out, want))
    q, k, cache = torch.empty_like(want[0]), torch.empty_like(want[1]), c.cache.clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        c.call(q=q, k=k, into=cache)
    for _ in range(3):
        c.qkv.copy_(torch.randn_like(c.qkv))
        c.positions.random_(0, ROWS)
        cache.copy_(c.cache)
        g.replay()
        torch.cuda.synchronize()
        c.check(q, k, cache)
    ops.register_ops()
    into = c.cache.clone()
    torch.ops.turboquant_write.norm_rope_write(c.qkv, c.qw, c.kw, c.cos, c.sin, c.positions, into,
                                               c.signs, c.slots, 16, 64, 64, q, k, c.eps, [32])
    c.check(q, k, into)


def test_then_decode_over_the_window():
    """A few steps of a decode as a layer makes them: the new tokens' rows normed,
    rotated and written, then attended with what the window holds."""
    from test_gpu_window import check_o
    c = C.make(30, [60, 17, 200], 8, 2, 128, extra=6, packed=False)
    c.indices = c.indices.reshape(3, -1)
    table = [list(r[r >= 0]) for r in c.indices]
    free = sorted(set(range(c.nb)) - {p for t in table for p in t})
    for t in table:
        t.append(free.pop())
    c.indptr = torch.tensor([0, 5, 8], dtype=torch.int32).numpy()
    n = Case(31, 3, 8, 2, 128)
    cache = torch.from_numpy(c.cache).to(DEV)
    signs = torch.from_numpy(c.signs).to(DEV)
    c.indices = torch.tensor([p for t in table for p in t], dtype=torch.int32).numpy()
    indices, indptr = (torch.from_numpy(x).to(DEV) for x in (c.indices, c.indptr))
    for step in range(4):
        c.lens = c.lens + 1
        slots = [table[b][(m - 1) // 16] * 16 + (m - 1) % 16 for b, m in enumerate(c.lens.tolist())]
        n.qkv.copy_(torch.randn_like(n.qkv))
        n.positions = torch.from_numpy(c.lens.astype("int64") - 1).to(DEV)
        q, k, _ = n.call(slots=torch.tensor(slots, dtype=torch.int32, device=DEV), signs=signs,
                         into=cache)
        o = torch.empty_like(q)
        ops.decode_paged_window(q, cache, indices, indptr, torch.from_numpy(c.lens).to(DEV), 2, 128,
                                128, c.scale, signs, o, 50, 4)
        c.cache = cache.cpu().numpy()
        qx = q.double().cpu().numpy()
        check_o(c, o, W.decode(c, qx, 50, 4), qx, "fp16", 50, 4)
