"""The windowed operators as a layer uses them: the vLLM-facing backend with a
sliding window, and the end-to-end loop with windowed layers."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

import budget_cases as C
import window_cases as W
from test_gpu_window import check_o
from turboquant_amd import e2e
from turboquant_amd.vllm_backend_fused import TurboQuantBackend, TurboQuantFusedImpl

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def as_case(impl, cache, table, lens):
    """A decode case over the backend's cache, for the 64-bit forms."""
    c = C.make(0, [0], impl.num_heads, impl.num_kv_heads, impl.head_size, page=cache.shape[2])
    c.cache, c.nb = cache.cpu().numpy(), cache.shape[1]
    c.indices = table.cpu().numpy().reshape(-1).astype(np.int32)
    c.indptr = (np.arange(len(lens) + 1) * table.shape[1]).astype(np.int32)
    c.lens = np.asarray(lens, np.int32)
    c.signs, c.scale = impl._signs.cpu().numpy(), impl.scale
    return c


def context(c, b, n, first, sink):
    """K and V rows [kept, H, hd] that a chunk behind n cached tokens sees."""
    pg, off, _ = C.places(c, b)
    see = np.r_[:min(sink, first), first:n]
    back = C.hadamard(c.pd) * c.signs
    out = [np.stack([C.rows(c, slab, pg[see], off[see], h) @ back for h in range(c.hkv)], 1)
           for slab in range(2)]
    return [torch.from_numpy(x[..., :c.hd]).to(DEV) for x in out]


@pytest.mark.parametrize("hq,hkv,hd,dtype,window,sink", [
    (32, 8, 128, "fp16", 100, 4), (8, 2, 64, "bf16", 37, 0), (16, 2, 256, "fp16", 64, 1),
    (16, 2, 96, "bf16", 200, 16), (4, 2, 128, "fp32", 1, 0), (6, 2, 84, "fp16", 90, 3),
    (8, 1, 64, "fp16", 2 ** 31 - 1, 0)])
@pytest.mark.parametrize("cpu_copies", [False, True])
def test_mixed_batch(hq, hkv, hd, dtype, window, sink, cpu_copies):
    """A fresh prompt, two chunks behind cached tokens and two decode rows apart
    from each other, in two steps of one cache; then a decode batch.  Pages that
    no later query sees are given back (their table entries overwritten) in
    between."""
    g = torch.Generator(device=DEV)
    g.manual_seed(hd)
    randn = lambda *s: torch.randn(s, generator=g, device=DEV).to(TYPES[dtype])
    impl = TurboQuantFusedImpl(hq, hd, 1 / math.sqrt(hd), hkv, None, window, "fp8")
    impl.sink = sink
    first_lens, chunks = [0, 300, 60, 500, 45], [20, 37, 1, 130, 1]
    nb = 90
    cache = torch.zeros(TurboQuantBackend.get_kv_cache_shape(nb, 16, hkv, hd, "fp8"),
                        dtype=torch.uint8, device=DEV)
    perm = torch.randperm(nb, generator=g, device=DEV).to(torch.int32)
    table = torch.full((5, 42), -1, dtype=torch.int32, device=DEV)
    at = 0
    for b, (x, n) in enumerate(zip(first_lens, chunks)):
        m = -(-(x + n + 3) // 16)
        table[b, :m] = perm[at:at + m]
        at += m

    def slots(b, t):
        return table[b, t // 16].long() * 16 + t % 16
    # what earlier steps left
    for b, x in enumerate(first_lens):
        if x:
            t = torch.arange(x, device=DEV)
            impl.do_kv_cache_update(None, randn(x, hkv, hd), randn(x, hkv, hd), cache,
                                    slots(b, t).to(torch.int32))
    lens = [x + n for x, n in zip(first_lens, chunks)]
    full = table.clone()
    for b, (x, n) in enumerate(zip(first_lens, lens)):
        see = W.sees(x, x + 1, window, sink)
        for i in range(-(-x // 16)):
            if not see[16 * i:16 * i + 16].any():
                table[b, i] = 10 ** 6
    total = sum(chunks)
    q, k, v = randn(total, hq, hd), randn(total, hkv, hd), randn(total, hkv, hd)
    t = [torch.arange(x, x + n, device=DEV) for x, n in zip(first_lens, chunks)]
    sm = torch.cat([slots(b, tt) for b, tt in enumerate(t)]).to(torch.int32)
    impl.do_kv_cache_update(None, k, v, cache, sm)
    starts = np.concatenate([[0], np.cumsum(chunks)]).astype(np.int32)
    meta = e2e.Meta(max(chunks), total, table, torch.tensor(lens, dtype=torch.int32, device=DEV),
                    torch.from_numpy(starts).to(DEV), sm)
    if cpu_copies:
        meta.query_start_loc_cpu = torch.from_numpy(starts)
        meta.seq_lens_cpu = torch.tensor(lens)
    out = torch.full((total, hq, hd), 7.0, dtype=TYPES[dtype], device=DEV)
    impl.forward(None, q.view(total, -1), k.view(total, -1), v.view(total, -1), cache, meta,
                 output=out.view(total, -1))
    c = as_case(impl, cache, full, lens)
    qx = q.half() if dtype == "fp32" else q  # (as the kernels take it)
    odt = "fp16" if dtype == "fp32" else dtype
    # decode rows: their 64-bit form over the cache
    rows = [starts[2], starts[4]]
    d = as_case(impl, cache, full[[2, 4]], [lens[2], lens[4]])
    qd = qx[rows].double().cpu().numpy()
    check_o(d, out[rows], W.decode(d, qd, window, sink), qd, odt, window, sink)
    # chunks: the rows in sight, then their own in the type that the kernel takes
    for b in (0, 1, 3):
        x, n, a = first_lens[b], chunks[b], starts[b]
        first = max(0, x - window + 1)
        ctx = context(c, b, x, first, sink) if x else [torch.zeros((0, hkv, hd), device=DEV)] * 2
        kk, vv = (torch.cat((y.double(), f[a:a + n].half().double()))
                  for y, f in zip(ctx, (k, v)))
        ref = W.prefill(qx[a:a + n].double(), kk, vv, [(0, n, 0, len(kk), 0)], hq // hkv,
                        impl.scale, window, sink)
        # the read-back rounds the context to fp16: 2^-11 of K and V, to a score
        # 2^-11 |q| |K| scale; the rest as the prefill tests have it
        half = 2.0 ** -8 if odt == "bf16" else 2.0 ** -11
        s = float(qx[a:a + n].double().norm(dim=-1).max() * kk.norm(dim=-1).max()) * impl.scale
        p = 2 * s * (2.0 ** -11 + 40 * 2.0 ** -24) + 2 * 2.0 ** -11 + len(kk) * 2.0 ** -25
        tol = half * ref.abs() + p * (1 + half) * float(vv.abs().max()) + 2.0 ** -24
        assert ((out[a:a + n].double() - ref).abs() <= tol).all(), b
    # one more token each, as a decode batch
    lens = [n + 1 for n in lens]
    kd, vd, q = randn(5, hkv, hd), randn(5, hkv, hd), randn(5, hq, hd)
    sm = torch.cat([slots(b, torch.tensor([n - 1], device=DEV)) for b, n in enumerate(lens)])
    impl.do_kv_cache_update(None, kd, vd, cache, sm.to(torch.int32))
    meta = e2e.Meta(1, 5, table, torch.tensor(lens, dtype=torch.int32, device=DEV),
                    torch.arange(6, dtype=torch.int32, device=DEV), None)
    out = impl.forward(None, q.view(5, -1), None, None, cache, meta).view(5, hq, hd)
    c = as_case(impl, cache, full, lens)
    qd = (q.half() if dtype == "fp32" else q).double().cpu().numpy()
    check_o(c, out, W.decode(c, qd, window, sink), qd, odt, window, sink)


def test_prefill_without_a_cache_and_in_passes(monkeypatch):
    """A profiling step has no cache; a step whose rows exceed the bound of a pass
    goes in several."""
    from turboquant_amd import vllm_backend_fused as B
    impl = TurboQuantFusedImpl(8, 128, 0.09, 2, None, 50, "fp8")
    g = torch.Generator(device=DEV)
    g.manual_seed(4)
    q, k, v = (torch.randn((260, h, 128), generator=g, device=DEV).bfloat16() for h in (8, 2, 2))
    starts = torch.tensor([0, 200, 201, 260], dtype=torch.int32, device=DEV)
    meta = e2e.Meta(200, 260, None, None, starts, None)
    run = lambda: impl.forward(None, q.view(260, -1), k.view(260, -1), v.view(260, -1), None, meta)
    out = run()
    ref = W.prefill(q.double(), k.double(), v.double(),
                    [(0, 200, 0, 200, 0), (200, 1, 200, 1, 0), (201, 59, 201, 59, 0)], 4, 0.09, 50, 0)
    # (bf16 K and V in fp16's normal range are exact in it but for their smallest values)
    err = (out.view(260, 8, 128).double() - ref).abs()
    assert (err <= 2.0 ** -8 * ref.abs() + 2.0 ** -9 * float(v.abs().max())).all()
    monkeypatch.setattr(B, "GATHER_BYTES", 100 * 4 * 2 * 128)
    assert torch.equal(run(), out)


def test_more_decode_rows_than_a_plan_takes():
    impl = TurboQuantFusedImpl(4, 64, 0.125, 2, None, 20, "fp8")
    c = C.make(6, [(7 * i) % 60 + 1 for i in range(1500)], 4, 2, 64, packed=False)
    cache = torch.from_numpy(c.cache).to(DEV)
    table = torch.from_numpy(c.indices.reshape(1500, -1)).to(DEV)
    q = torch.randn((1500, 4, 64), device=DEV).half()
    meta = e2e.Meta(1, 1500, table, torch.from_numpy(c.lens).to(DEV),
                    torch.arange(1501, dtype=torch.int32, device=DEV), None)
    out = impl.forward(None, q.view(1500, -1), None, None, cache, meta).view(1500, 4, 64)
    c.signs = impl._signs.cpu().numpy()
    qx = q.double().cpu().numpy()
    check_o(c, out, W.decode(c, qx, 20, 0), qx, "fp16", 20, 0)


def test_page_starts_of_a_capture_are_its_own():
    """The first decode of a table's shape inside a capture, an eager one of the
    same shape in front of any replay, and both on several streams."""
    impl = TurboQuantFusedImpl(8, 128, 0.09, 2, None, 60, "fp8")
    c = C.make(9, [300, 40, 111], 8, 2, 128, packed=False)
    cache = torch.from_numpy(c.cache).to(DEV)
    table = torch.from_numpy(c.indices.reshape(3, -1)).to(DEV)
    lens = torch.from_numpy(c.lens).to(DEV)
    q = torch.randn((3, 8 * 128), device=DEV).half()

    def call(n, pad):
        tab = torch.nn.functional.pad(table[:n], (0, pad), value=-1)
        meta = e2e.Meta(1, n, tab, lens[:n], torch.arange(n + 1, dtype=torch.int32, device=DEV), None)
        return impl.forward(None, q[:n], None, None, cache, meta)

    call(2, 1)  # (what a first call sets up)
    c.scale, c.signs = 0.09, impl._signs.cpu().numpy()
    qx = q.view(3, 8, 128).double().cpu().numpy()
    ref = W.decode(c, qx, 60, 0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            held = call(3, 0)
        eager = call(3, 0)
    other = call(3, 0)
    torch.cuda.synchronize()
    check_o(c, eager.view(3, 8, 128), ref, qx, "fp16", 60, 0)
    assert torch.equal(other, eager)
    for _ in range(3):
        held.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held, eager)
        assert torch.equal(call(3, 0), eager)


def test_without_a_window_nothing_changes():
    """sliding_window None: the calls that the backend made before."""
    impl = TurboQuantFusedImpl(8, 128, 0.09, 2, None, None, "fp8")
    assert impl.window == 0
    c = C.make(7, [300, 40], 8, 2, 128, packed=False)
    cache = torch.from_numpy(c.cache).to(DEV)
    meta = e2e.Meta(1, 2, torch.from_numpy(c.indices.reshape(2, -1)).to(DEV),
                    torch.from_numpy(c.lens).to(DEV),
                    torch.arange(3, dtype=torch.int32, device=DEV), None)
    q = torch.randn((2, 8 * 128), device=DEV).half()
    out = impl.forward(None, q, None, None, cache, meta)
    wide = TurboQuantFusedImpl(8, 128, 0.09, 2, None, 1000, "fp8")
    # (a window beyond the sequences: the same sum in another order)
    qx = q.view(2, 8, 128).double().cpu().numpy()
    c.scale, c.signs = 0.09, impl._signs.cpu().numpy()
    ref = W.decode(c, qx, 1000, 0)
    for x in (out, wide.forward(None, q, None, None, cache, meta)):
        check_o(c, x.view(2, 8, 128), ref, qx, "fp16", 1000, 0)


def test_project_and_update():
    """The fused form gives do_kv_cache_update's cache over its own k and v."""
    impl = TurboQuantFusedImpl(8, 128, 0.09, 2, None, 64, "fp8")
    qkv = torch.randn((40, 12 * 128), device=DEV).half()
    w = torch.ones(128, dtype=torch.float16, device=DEV)
    cos, sin = e2e.rope_angles(100, 128, 1e6, DEV)
    caches = [torch.zeros((2, 4, 16, 2, 80), dtype=torch.uint8, device=DEV) for _ in range(2)]
    slots = torch.arange(40, device=DEV)
    pos = torch.arange(40, device=DEV) + 7
    q, k, v = impl.project_and_update(qkv, w, w, cos, sin, pos, caches[0], slots)
    impl.do_kv_cache_update(None, k, v, caches[1], slots)
    assert torch.equal(caches[0], caches[1])
    shape = e2e.ModelShape(heads=8, kv_heads=2, head_dim=128)
    q2, k2 = e2e.qk_norm_rope(qkv, shape, w, w, *e2e.rope_tables(100, 128, 1e6, DEV), pos)
    # the harness's glue rounds the normed values and both tables as well: three
    # times 2^-11, and its angles are fp32 (up to 107 turns of 2^-24), of both values
    # of a pair, and each side's own rounding
    for a, b in ((q, q2), (k, k2)):
        top = 2 * float(torch.maximum(a.abs(), b.abs()).max())
        assert (a.float() - b.float()).abs().max() <= (4 * 2.0 ** -11 + 107 * 2.0 ** -24) * top


# ------------------------------------------------------------------ end to end

def runner(**kw):
    shape = e2e.ModelShape.tiny(3)
    r = e2e.Runner(shape, 3, 220, DEV, seed=5, **kw)
    g = torch.Generator(device="cpu")
    g.manual_seed(7)
    for b in range(3):
        r.prefill(b, torch.randint(0, shape.vocab, (200 - 30 * b,), generator=g).to(DEV))
    return r


def test_e2e_windowed_layers():
    """Every layer's decode attention against its 64-bit form: windowed layers
    over the window, the third over everything; replays of the captured step give
    the eager steps' tokens."""
    r = runner(attention_window=48, attention_sink=4, full_every=3)
    assert [i.window for i in r.impls] == [48, 48, 0]
    saved = (r.pos.clone(), r.tok.clone())
    r.probe = []
    r.decode_eager(1)
    probe, r.probe = r.probe, None
    for li, q, _, _, o in probe:
        c = as_case(r.impls[li], r.caches[li], r.block_table, r.seq_lens.tolist())
        window = r.impls[li].window or 10 ** 6
        qx = q.double().cpu().numpy()
        check_o(c, o.view(q.shape), W.decode(c, qx, window, 4), qx, "fp16", window, 4)
    r.pos.copy_(saved[0])
    r.tok.copy_(saved[1])
    eager = r.decode_eager(9).clone()
    r.pos.copy_(saved[0])
    r.tok.copy_(saved[1])
    r.capture(9)
    for _ in range(2):
        r.pos.copy_(saved[0])
        r.tok.copy_(saved[1])
        assert torch.equal(r.decode_graph(9), eager)


def test_e2e_run_with_a_window():
    res = e2e.run(e2e.ModelShape.tiny(2), 2, 300, 12, attention_window=64, attention_sink=4)
    assert res["attention_window"] == 64 and res["output_tok_s"] > 0
    a = e2e.run(e2e.ModelShape.tiny(2), 2, 300, 12, attention_window=64, attention_sink=4)
    assert a["first_tokens"] == res["first_tokens"]
