"""The windowed layers' operators on an MI355X at the sizes where another variant
takes over: read-backs of four vectors a thread, norm-rotate-writes of several
launches."""
from __future__ import annotations

import pytest
import torch

import budget_cases as C
from test_gpu_norm_write import Case
from test_gpu_window_prefill import DEV, cached, closed_up
from turboquant_amd import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hkv,hd", [(8, 128), (7, 128), (8, 256), (3, 200), (16, 64)])
@pytest.mark.parametrize("page", [16, 48])
@pytest.mark.parametrize("more", [0, 1])
def test_read_back_where_four_vectors_a_thread_take_over(hkv, hd, page, more):
    """Bit for bit the rows of a read-back of everything: uneven requests with and
    without a gap and fresh rows, together of 2^24 dims (one vector a thread at
    padded sizes 128 and 256) and one token more (four)."""
    sink = 5
    total = 2 ** 24 // (hkv * C.pad(hd)) + more  # tokens that stay
    # (cached, first in sight): no gap, a gap inside a page, one token, nothing cached
    # but sinks, a long gap
    shapes = [(1000, 0), (1333, 77), (1, 0), (64, 64), (0, 0), (900, 640)]
    left = total - sum(min(sink, f) + n - f for n, f in shapes)
    shapes.append((left - sink + 3000, 3000))
    lens, fresh = [n for n, _ in shapes], [3, 0, 40, 1, 2, 0, 130]
    c = C.make(hkv + page, lens, hkv, hkv, hd, page=page, packed=False)
    t = cached(c)
    g = torch.Generator(device=DEV)
    g.manual_seed(hd)
    key, value = (torch.randn((sum(fresh), hkv, hd), generator=g, device=DEV).half()
                  for _ in range(2))
    reqs, at, f = [], 2, 0
    for b, ((n, first), m) in enumerate(zip(shapes, fresh)):
        reqs.append((b, n, first, f, m, at))
        at, f = at + min(sink, first) + n - first + m, f + m
    assert at - 2 - sum(fresh) == total
    want = closed_up(c, t, reqs, sink, key, value)
    out = [torch.full((at + 3, hkv, c.pd), 7.0, dtype=torch.float16, device=DEV) for _ in range(2)]
    ops.prefill_gather_window(t["cache"], t["table"], key, value, reqs, sink, hd, c.pd, t["signs"],
                              *out)
    for got, ref in zip(out, want):
        assert torch.equal(got[2:at], ref)
        assert (got[:2] == 7.0).all() and (got[at:] == 7.0).all()


@pytest.mark.parametrize("hq,hkv,hd,rotated,n,sections", [
    (1024, 3, 16, 16, 2051, None),        # launches of 2048 tokens
    (1024, 1, 64, 32, 2048, (5, 11)),
    (2, 1024, 16, 16, 4100, None),
    (4096, 2, 16, 16, 300, (3, 5))])      # of 128
def test_norm_write_of_several_launches(monkeypatch, hq, hkv, hd, rotated, n, sections):
    write = ops.quantize_write_kv_cache

    def in_slices(cache, key, value, signs, slots, *geometry):
        # (the plain write, which the cache is compared with, takes no 4100 x 1024 vectors)
        for a in range(0, n, 1000):
            write(cache, *(x[a:a + 1000] for x in (key, value)), signs, slots[a:a + 1000],
                  *geometry)
    monkeypatch.setattr(ops, "quantize_write_kv_cache", in_slices)
    c = Case(n, n, hq, hkv, hd, rotated, "bf16", sections=sections)
    c.run()
