"""The operators of windowed layers without a GPU: refusals of the ops and the C
ABI, the ops' schemas, and the 64-bit forms that the GPU tests compare with."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

import budget_cases as C
import window_cases as W
from turboquant_amd import _lib, ops


def _decode_args(**bad):
    """A call's tensors on the meta device, all well formed but those given."""
    def t(shape, dtype):
        return torch.empty(shape, dtype=dtype, device="meta")
    a = dict(q=t((2, 8, 128), torch.float16), cache=t((2, 9, 16, 2, 80), torch.uint8),
             indices=t((8,), torch.int32), indptr=t((3,), torch.int32),
             seq=t((2,), torch.int32), hkv=2, hd=128, pd=128, signs=None,
             o=t((2, 8, 128), torch.float16), window=4, sink=0)
    a.update(bad)
    return a


def _decode(a):
    return ops.decode_paged_window(a["q"], a["cache"], a["indices"], a["indptr"], a["seq"], a["hkv"],
                                   a["hd"], a["pd"], 0.1, a["signs"], a["o"], a["window"], a["sink"])


def _meta(shape, dtype):
    return torch.empty(shape, dtype=dtype, device="meta")


def test_cpu_tensors_are_refused():
    a = {k: torch.zeros(v.shape, dtype=v.dtype) if isinstance(v, torch.Tensor) else v
         for k, v in _decode_args().items()}
    with pytest.raises(RuntimeError, match="GPU only"):
        _decode(a)


@pytest.mark.parametrize("bad,match", [
    (dict(q=_meta((2, 8, 64), torch.float16)), "q must be"),
    (dict(q=_meta((2, 8, 128), torch.float32)), "q must be"),
    (dict(q=_meta((2, 7, 128), torch.float16)), "q heads"),
    (dict(cache=_meta((2, 9, 16, 4, 80), torch.uint8)), "kv heads"),
    (dict(cache=_meta((1, 9, 16, 2, 80), torch.uint8)), "kv_cache must be"),
    (dict(indices=_meta((8,), torch.int64)), "indices must be"),
    (dict(indptr=_meta((1,), torch.int32)), "indptr must be"),
    (dict(seq=_meta((1,), torch.int32)), "seq_lens must be"),
    (dict(o=_meta((2, 8, 128), torch.float32)), "o must be"),
    (dict(o=_meta((2, 8, 64), torch.float16)), "o must be"),
    (dict(signs=_meta((64,), torch.float32)), "signs must be"),
    (dict(window=0), "must be positive"),
    (dict(window=-3), "must be positive"),
    (dict(sink=-1), "not negative"),
    (dict(window=2 ** 31), "out of range"),
    (dict(sink=2 ** 32 + 1), "out of range"),
    (dict(pd=2 ** 32 + 128), "out of range"),
])
def test_decode_refusals(monkeypatch, bad, match):
    monkeypatch.setattr(ops, "_require_gpu", lambda *t: None)
    with pytest.raises(RuntimeError, match=match):
        _decode(_decode_args(**bad))


def _buffer():
    buf = (ctypes.c_char * 8192)()
    p = ctypes.addressof(buf)
    return buf, p + -p % 256


@pytest.mark.parametrize("bad,match", [
    (dict(window=0), b"window"), (dict(sink=-1), b"sink"), (dict(hd=0), b"head_dim"),
    (dict(hd=129), b"head_dim"), (dict(hd=100), b"multiple of 8"), (dict(qt=0), b"fp16 or bf16"),
    (dict(ot=3), b"fp16 or bf16"), (dict(n=-1), b"num_indices"), (dict(o=None), b"null"),
    (dict(ws=None), b"null"), (dict(pd=96, hd=96), b"padded_dim"), (dict(hq=7), b"integer"),
    (dict(hq=34), b"integer"), (dict(hkv=0), b"integer"), (dict(bs=8), b"block_size"),
    (dict(bs=0), b"block_size"), (dict(ebs=96), b"ebs"), (dict(batch=-1), b"batch"),
    (dict(q=None), b"null"), (dict(k=None), b"null"), (dict(sh=64), b"q_stride_h"),
    (dict(sb=1001), b"strides"),
])
def test_abi_refuses_bad_decode_arguments(bad, match):
    """Addresses that are never read: every case is refused before a launch."""
    lib = _lib.load()
    buf, p = _buffer()
    a = dict(q=p, sb=1024, sh=128, qt=1, k=p, n=8, batch=2, hq=8, hkv=2, hd=128, pd=128, bs=16,
             ebs=80, nb=9, window=4, sink=0, o=p, ot=1, ws=p, wsb=1 << 40)
    a.update(bad)

    def call():
        return lib.tq_decode_paged_window(
            a["q"], a["sb"], a["sh"], a["qt"], a["k"], a["k"], p, a["n"], p, p, a["batch"], a["hq"],
            a["hkv"], a["hd"], a["pd"], a["bs"], a["ebs"], a["nb"], 0.1, None, a["window"],
            a["sink"], a["o"], a["ot"], a["ws"], a["wsb"], None)
    assert call() == -22 and match in lib.tq_last_error(), lib.tq_last_error()
    for key, off in (("q", 2), ("k", 8), ("o", 4), ("ws", 8)):
        a.update(q=p, sb=1024, sh=128, qt=1, k=p, n=8, batch=2, hq=8, hkv=2, hd=128, pd=128, bs=16,
                 ebs=80, nb=9, window=4, sink=0, o=p, ot=1, ws=p, wsb=1 << 40)
        a[key] = p + off
        assert call() == -22 and b"aligned" in lib.tq_last_error()
    a.update(q=p, k=p, o=p, ws=p, batch=0)
    assert call() == 0


def test_schemas_declare_the_writes():
    ops.register_ops()
    written = {"turboquant_v5.decode_paged_window": {"o"},
               "turboquant_write.norm_rope_write": {"kv_cache", "q", "k"}}
    for name, want in written.items():
        space, name = name.split(".")
        schema = getattr(getattr(torch.ops, space), name).default._schema
        got = {a.name for a in schema.arguments if a.alias_info and a.alias_info.is_write}
        assert got == want and not schema.returns


# ---------------------------------------------------- the 64-bit forms themselves

def test_reference_decode():
    """A window over everything is the oracle's attention; a shorter one is that
    of a sequence holding the tokens in sight alone."""
    import oracle
    c = C.make(4, [61, 40], 8, 2, 128)
    q = c.rng.standard_normal((2, 8, 128)).astype(np.float16)
    ref = oracle.decode(q, c.cache, c.indices, c.indptr, c.lens, 2, 128, c.scale, c.signs)
    o = W.decode(c, q.astype(np.float64), 61, 0)
    # (the oracle works in fp32: 128 products and 61 tokens)
    assert np.abs(o - ref).max() < 1e-4
    o = W.decode(c, q.astype(np.float64), 9, 16)
    seen = c.indices[[0, 3]]  # the sinks' page and the last: 61 - 9 = 52 = 3 * 16 + 4
    cut = c.cache.copy()
    cut[:, seen[1], :9] = c.cache[:, seen[1], 4:13]
    ref = oracle.decode(q[:1], cut, seen, np.array([0, 2], np.int32), np.array([25], np.int32), 2,
                        128, c.scale, c.signs)
    assert np.abs(o[:1] - ref).max() < 1e-4
    assert W.sees(9, 12, 3, 2).tolist() == [True] * 2 + [False] * 5 + [True] * 3 + [False] * 2


# ---------------------------------------------------- prefill and read-back

def _prefill(monkeypatch=None, **bad):
    a = dict(q=_meta((40, 8, 128), torch.float16), o=_meta((40, 8, 128), torch.float16),
             reqs=[(0, 30, 0, 50, 0)], hkv=2, hd=128, pd=128, scale=0.1, window=4, sink=0,
             k=_meta((60, 2, 128), torch.float16), v=_meta((60, 2, 128), torch.float16), k2=None,
             v2=None)
    a.update(bad)
    return ops.prefill_attention_window(a["q"], a["o"], a["reqs"], a["hkv"], a["hd"], a["pd"],
                                        a["scale"], a["window"], a["sink"], a["k"], a["v"], a["k2"],
                                        a["v2"])


@pytest.mark.parametrize("bad,match", [
    (dict(window=0), "must be positive"), (dict(sink=-1), "not negative"),
    (dict(window=2 ** 31), "out of range"), (dict(sink=2 ** 40), "out of range"),
    (dict(scale=0.0), "sm_scale"), (dict(scale=-0.1), "sm_scale"),
    (dict(scale=float("nan")), "sm_scale"), (dict(scale=float("inf")), "sm_scale"),
    (dict(q=_meta((40, 8, 128), torch.float32)), "fp16 or bf16"),
    (dict(o=_meta((41, 8, 128), torch.float16)), "q / o must be"),
    (dict(k=_meta((60, 2, 128), torch.bfloat16)), "k / v must be"),
    (dict(k=_meta((60, 4, 128), torch.float16)), "k / v must be"),
    (dict(v=None), "go together"), (dict(v=_meta((61, 2, 128), torch.float16)), "go together"),
    (dict(reqs=[(20, 30, 0, 50, 0)]), "out of range"),
    (dict(reqs=[(0, 30, 20, 50, 0)]), "out of range"),
    (dict(reqs=[(0, 30, 0, 29, 0)]), "out of range"),
    (dict(reqs=[(0, 30, 0, 50, 1)]), "out of range"),
    (dict(reqs=[(-1, 30, 0, 50, 0)]), "out of range"),
])
def test_prefill_refusals(monkeypatch, bad, match):
    monkeypatch.setattr(ops, "_require_gpu", lambda *t: None)
    with pytest.raises(RuntimeError, match=f"prefill_attention_window: .*{match}"):
        _prefill(**bad)


def _gather(**bad):
    half = lambda *s: torch.zeros(s, dtype=torch.float16)
    a = dict(cache=torch.zeros((2, 9, 16, 2, 80), dtype=torch.uint8),
             table=torch.zeros((2, 3), dtype=torch.int32), key=half(20, 2, 128),
             value=half(20, 2, 128), reqs=[(0, 40, 30, 0, 5, 0)], sink=4, hd=128, pd=128, signs=None,
             k=half(19, 2, 128), v=half(19, 2, 128))
    a.update(bad)
    return ops.prefill_gather_window(a["cache"], a["table"], a["key"], a["value"], a["reqs"],
                                     a["sink"], a["hd"], a["pd"], a["signs"], a["k"], a["v"])


@pytest.mark.parametrize("bad,match", [
    (dict(sink=-1), "negative"), (dict(sink=2 ** 31), "out of range"),
    (dict(key=None), "go together"), (dict(key=None, value=None), "out of range"),
    (dict(key=_meta((20, 2, 128), torch.float64)), "float dtype"),
    (dict(key=_meta((20, 2, 96), torch.float16)), "key/value must be"),
    (dict(k=_meta((19, 2, 64), torch.float16)), "out_k / out_v"),
    (dict(k=_meta((19, 2, 128), torch.bfloat16)), "out_k / out_v"),
    (dict(k=_meta((18, 2, 128), torch.float16)), "out of range"),
    (dict(cache=_meta((2, 9, 16, 4, 80), torch.uint8)), "kv heads"),
    (dict(cache=None), "needs the cache"), (dict(table=None), "needs the cache"),
    (dict(table=_meta((2, 3), torch.int64)), "block_table"),
    (dict(reqs=[(2, 40, 30, 0, 5, 0)]), "table row"),
    (dict(reqs=[(0, 49, 39, 0, 5, 0)]), "pages do not cover"),
    (dict(reqs=[(0, 40, 41, 0, 5, 0)]), "out of range"),
    (dict(reqs=[(0, 40, -1, 0, 5, 0)]), "out of range"),
    (dict(reqs=[(0, -1, -1, 0, 5, 0)]), "out of range"),
    (dict(reqs=[(0, 40, 29, 0, 5, 0)]), "out of range"),
    (dict(reqs=[(0, 40, 30, 16, 5, 0)]), "out of range"),
    (dict(reqs=[(0, 40, 30, 0, 5, 1)]), "out of range"),
    (dict(reqs=[(0, 40, 30, 0, 5, -1)]), "out of range"),
    (dict(signs=_meta((64,), torch.float32)), "signs"),
])
def test_gather_refusals(monkeypatch, bad, match):
    monkeypatch.setattr(ops, "_require_gpu", lambda *t: None)
    with pytest.raises(RuntimeError, match=match):
        _gather(**bad)


def test_prefill_and_gather_refuse_cpu_tensors():
    half = lambda *s: torch.zeros(s, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="GPU only"):
        _prefill(q=half(40, 8, 128), o=half(40, 8, 128), k=half(60, 2, 128), v=half(60, 2, 128))
    with pytest.raises(RuntimeError, match="GPU only"):
        _gather()


def _ints(*x):
    return (ctypes.c_int32 * max(1, len(x)))(*x)


@pytest.mark.parametrize("bad,match", [
    (dict(window=0), b"window"), (dict(sink=-1), b"sink"), (dict(scale=0.0), b"sm_scale"),
    (dict(scale=float("nan")), b"sm_scale"), (dict(pd=96), b"padded_dim"),
    (dict(hq=7), b"multiple"), (dict(hkv=0), b"multiple"), (dict(hd=100), b"multiple of 8"),
    (dict(hd=136), b"multiple of 8"), (dict(qt=0), b"fp16 or bf16"), (dict(ql=(50,)), b"q_len"),
    (dict(ql=(-1,)), b"q_len"), (dict(qs=(-1,)), b"bad request"), (dict(ks=(-1,)), b"bad request"),
    (dict(q=None), b"null"), (dict(k=None), b"null"), (dict(src=(1,)), b"null"),
    (dict(st=1001), b"strides"), (dict(kst=64), b"strides"), (dict(off=8), b"aligned"),
    (dict(n=-1), b"bad sizes"),
])
def test_abi_refuses_bad_prefill_arguments(bad, match):
    lib = _lib.load()
    buf, p = _buffer()
    a = dict(q=p, st=1024, qt=1, k=p, kst=256, qs=(0,), ql=(20,), ks=(0,), kl=(40,), src=(0,), n=1,
             hq=8, hkv=2, hd=128, pd=128, scale=0.1, window=4, sink=0, off=0)
    a.update(bad)
    q = a["q"] and a["q"] + a["off"]
    rc = lib.tq_prefill_attention_window(
        q, a["st"], 128, a["qt"], a["k"], a["kst"], 128, a["k"], a["kst"], 128, None, None, 0, 0, p,
        1024, 128, 1, _ints(*a["qs"]), _ints(*a["ql"]), _ints(*a["ks"]), _ints(*a["kl"]),
        _ints(*a["src"]), a["n"], a["hq"], a["hkv"], a["hd"], a["pd"], a["scale"], a["window"],
        a["sink"], p, 1 << 40, None)
    assert rc == -22 and match in lib.tq_last_error(), lib.tq_last_error()


def test_prefill_workspace_follows_the_window():
    """(without a GPU the plan is that of 256 CUs)  A short chunk's keys are split
    where its window is long, and need no workspace where it is short."""
    lib = _lib.load()
    size = lambda w, s=0: lib.tq_prefill_window_workspace_bytes(_ints(100), _ints(20000), 1, 4, 128,
                                                                w, s)
    assert size(0) == 0 and size(5, -1) == 0 and size(200) == 0
    assert size(19000) > 0 and size(2 ** 31 - 1, 2 ** 31 - 1) == \
        lib.tq_prefill_batch_workspace_bytes(_ints(100), _ints(20000), 1, 4, 128)


def test_abi_names_the_workspace_that_is_too_small():
    """(refused in front of the launch; the addresses are never read)"""
    lib = _lib.load()
    buf, p = _buffer()
    size = lib.tq_prefill_window_workspace_bytes(_ints(100), _ints(20000), 1, 4, 128, 19000, 0)
    assert size > 0
    rc = lib.tq_prefill_attention_window(
        p, 512, 128, 1, p, 256, 128, p, 256, 128, None, None, 0, 0, p, 512, 128, 1, _ints(0),
        _ints(100), _ints(0), _ints(20000), _ints(0), 1, 4, 2, 128, 128, 0.1, 19000, 0, p, size - 1,
        None)
    assert rc == -22 and b"tq_prefill_window_workspace_bytes" in lib.tq_last_error()


@pytest.mark.parametrize("bad,match", [
    (dict(sink=-1), b"negative"), (dict(first=None), b"null"), (dict(first=(41,)), b"bad request"),
    (dict(first=(-1,)), b"bad request"), (dict(ctx=(-1,), first=(-1,)), b"bad request"),
    (dict(fresh=(-1,)), b"bad request"), (dict(out=(-1,)), b"bad request"),
    (dict(row=(-1,)), b"bad request"), (dict(key=None), b"null"), (dict(k=None), b"null"),
    (dict(pd=96), b"padded_dim"), (dict(ebs=81), b"ebs"), (dict(dt=5), b"dtype"),
    (dict(n=-1), b"bad sizes"), (dict(o=8), b"aligned"),
])
def test_abi_refuses_bad_gather_arguments(bad, match):
    lib = _lib.load()
    buf, p = _buffer()
    a = dict(k=p, key=p, dt=1, row=(0,), ctx=(40,), first=(30,), fs=(0,), fresh=(5,), out=(0,), n=1,
             sink=4, hd=128, pd=128, bs=16, ebs=80, o=0)
    a.update(bad)
    rc = lib.tq_prefill_gather_window(
        a["k"], a["k"], p, 3, 2, a["hd"], a["pd"], a["bs"], a["ebs"], 9, None, a["key"], a["key"],
        a["dt"], 256, 128, 256, 128, _ints(*a["row"]), _ints(*a["ctx"]),
        None if a["first"] is None else _ints(*a["first"]), _ints(*a["fs"]), _ints(*a["fresh"]),
        _ints(*a["out"]), a["n"], a["sink"], p + a["o"], p, None)
    assert rc == -22 and match in lib.tq_last_error(), lib.tq_last_error()


def test_reference_prefill():
    """In 64 bits: a window over everything is causal attention; rows of a window
    of one token and no sinks are their own value; values out of sight do not
    count."""
    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn((n, h, 8), generator=g, dtype=torch.float64)
               for n, h in ((5, 4), (9, 2), (9, 2)))
    o = W.prefill(q, k, v, [(0, 5, 0, 9, 0)], 2, 0.3, 9, 0)
    for i in range(5):
        for h in range(4):
            p = (k[:5 + i, h // 2] @ q[i, h] * 0.3).softmax(0)
            assert torch.allclose(o[i, h], p @ v[:5 + i, h // 2])
    o = W.prefill(q, k, v, [(0, 5, 0, 9, 0)], 2, 0.3, 1, 0)
    assert torch.allclose(o, v[4:].repeat_interleave(2, 1))
    v[2], v[8] = torch.nan, torch.inf
    o = W.prefill(q, k, v, [(0, 5, 0, 9, 0)], 2, 0.3, 3, 1)
    assert torch.isnan(o[0]).all() and torch.isfinite(o[1:4]).all() and (o[4] == torch.inf).all()


# ---------------------------------------------------- norm, rotation and write

def _norm_write(**bad):
    t = lambda s, d: torch.zeros(s, dtype=d)
    half = torch.float16
    a = dict(qkv=t((5, 12 * 128), half), qw=t((128,), half), kw=t((128,), half),
             cos=t((30, 64), torch.float32), sin=t((30, 64), torch.float32),
             pos=t((5,), torch.int64), cache=t((2, 4, 16, 2, 80), torch.uint8),
             signs=t((128,), torch.float32), slots=t((5,), torch.int32), hq=8, hd=128, pd=128,
             q=t((5, 8, 128), half), k=t((5, 2, 128), half), eps=1e-6, sections=None)
    a.update(bad)
    ops.norm_rope_write(a["qkv"], a["qw"], a["kw"], a["cos"], a["sin"], a["pos"], a["cache"],
                        a["signs"], a["slots"], a["hq"], a["hd"], a["pd"], a["q"], a["k"], a["eps"],
                        a["sections"])


@pytest.mark.parametrize("bad,match", [
    (dict(qkv=_meta((5, 12 * 128), torch.float32)), "qkv must be"),
    (dict(qkv=_meta((5, 11 * 128), torch.float16)), "qkv must be"),
    (dict(hq=9), "qkv must be"), (dict(hq=0), "q heads"), (dict(hq=2 ** 33), "out of range"),
    (dict(qw=None), "both weights"), (dict(qw=_meta((128,), torch.bfloat16)), "q_weight"),
    (dict(kw=_meta((64,), torch.float16)), "k_weight"),
    (dict(cos=_meta((30, 64), torch.float16)), "cos and sin"),
    (dict(sin=_meta((30, 32), torch.float32)), "cos and sin"),
    (dict(pos=_meta((4,), torch.int64)), "positions"),
    (dict(pos=_meta((5,), torch.int16)), "positions"),
    (dict(pos=_meta((3, 5), torch.int64)), "sections"),
    (dict(pos=_meta((3, 5), torch.int64), sections=(32, 32)), "sections"),
    (dict(pos=_meta((3, 5), torch.int64), sections=(32, 32, 1)), "sections"),
    (dict(pos=_meta((3, 5), torch.int64), sections=(65, -2, 1)), "sections"),
    (dict(pos=_meta((5, 5), torch.int64), sections=(60, 1, 1, 1, 1)), "sections"),
    (dict(slots=_meta((5,), torch.int64)), "slot_mapping"),
    (dict(slots=_meta((4,), torch.int32)), "slot_mapping"),
    (dict(q=_meta((5, 8, 128), torch.bfloat16)), "q must be"),
    (dict(q=_meta((4, 8, 128), torch.float16)), "q must be"),
    (dict(k=_meta((5, 8, 128), torch.float16)), "k must be"),
    (dict(cache=_meta((1, 4, 16, 2, 80), torch.uint8)), "kv_cache"),
    (dict(cache=_meta((4, 16, 2, 80), torch.uint8)), "kv_cache"),
    (dict(signs=_meta((64,), torch.float32)), "signs"),
])
def test_norm_write_refusals(monkeypatch, bad, match):
    monkeypatch.setattr(ops, "_require_gpu", lambda *t: None)
    with pytest.raises(RuntimeError, match=f"norm_rope_write: .*{match}"):
        _norm_write(**bad)


def test_norm_write_refuses_cpu_tensors():
    with pytest.raises(RuntimeError, match="GPU only"):
        _norm_write()


@pytest.mark.parametrize("bad,match", [
    (dict(pd=96), b"padded_dim"), (dict(hd=100), b"head_dim"), (dict(hd=64), b"head_dim"),
    (dict(hd=0), b"head_dim"), (dict(rot=0), b"rotated"), (dict(rot=24), b"rotated"),
    (dict(rot=144), b"rotated"), (dict(dt=0), b"fp16 or bf16"), (dict(ebs=82), b"ebs"),
    (dict(hq=0), b"bad sizes"), (dict(hkv=5000), b"bad sizes"), (dict(bs=0), b"bad sizes"),
    (dict(n=-1), b"bad sizes"), (dict(rows=-1), b"bad sizes"), (dict(pb=2), b"positions"),
    (dict(axes=0), b"positions"), (dict(axes=5), b"positions"), (dict(sec=(63,)), b"sections"),
    (dict(sec=(65, -1), axes=2), b"sections"), (dict(kw=None), b"both weights"),
    (dict(eps=0.0), b"eps"), (dict(eps=-1.0), b"eps"), (dict(eps=float("nan")), b"eps"),
    (dict(eps=float("inf")), b"eps"), (dict(qkv=None), b"null"), (dict(cos=None), b"null"),
    (dict(slots=None), b"null"), (dict(cache=None), b"null"), (dict(q=None), b"null"),
    (dict(signs=None), b"null"), (dict(rows=0), b"empty"), (dict(st=1528), b"stride"),
    (dict(st=1540), b"stride"), (dict(off=8), b"aligned"), (dict(q=0x1000), b"overlap"),
    (dict(k=0x1000), b"overlap"),
])
def test_abi_refuses_bad_norm_write_arguments(bad, match):
    lib = _lib.load()
    at = lambda i: 0x1000 + (i << 24)  # addresses that are never read
    a = dict(qkv=at(0), st=1536, dt=1, qw=at(1), kw=at(1), eps=1e-6, cos=at(2), rows=30, rot=128,
             pos=at(3), pb=8, sec=(64,), axes=1, cache=at(4), signs=at(5), slots=at(6), n=5, hq=8,
             hkv=2, hd=128, pd=128, bs=16, ebs=80, q=at(7), k=at(8), off=0)
    a.update(bad)
    qkv = a["qkv"] and a["qkv"] + a["off"]

    def call():
        return lib.tq_norm_rope_write(
            qkv, a["st"], a["dt"], a["qw"], a["kw"], a["eps"], a["cos"], a["cos"], a["rows"],
            a["rot"], a["pos"], a["pb"], 5, _ints(*a["sec"]), a["axes"], a["cache"], a["cache"],
            a["signs"], a["slots"], a["n"], a["hq"], a["hkv"], a["hd"], a["pd"], a["bs"], a["ebs"],
            9, a["q"], a["k"], None)
    assert call() == -22 and match in lib.tq_last_error(), lib.tq_last_error()


def test_norm_write_of_no_tokens_does_nothing():
    lib = _lib.load()
    assert lib.tq_norm_rope_write(None, 0, 1, None, None, 1e-6, None, None, 0, 128, None, 8, 0,
                                  _ints(64), 1, None, None, None, None, 0, 8, 2, 128, 128, 16, 80, 9,
                                  None, None, None) == 0


def test_reference_norm_and_rotation():
    """A rotation keeps a pair's length and turns it by its position's angle; the
    norm makes the mean square 1."""
    g = torch.Generator().manual_seed(2)
    qkv = torch.randn((4, 3 * 8), generator=g, dtype=torch.float64)
    ones = torch.ones(8)
    angle = torch.arange(10)[:, None] * torch.tensor([[1.0, 0.1, 0.01]])
    pos = torch.tensor([[0, 3, 9, 10], [5, 3, 2, 1]])
    q, k, before = W.norm_rope(qkv, ones, ones, angle.cos(), angle.sin(), pos, (2, 1), 1, 1, 8,
                               1e-12)
    assert torch.allclose((before ** 2).mean(-1), torch.ones((4, 2), dtype=torch.float64))
    assert torch.isnan(q[3]).all() and torch.isnan(k[3]).all()
    z0 = torch.complex(before[:, 0, :3], before[:, 0, 3:6])[:3]
    z1 = torch.complex(q[:, 0, :3], q[:, 0, 3:6])[:3]
    turn = torch.stack((angle[pos[0, :3], 0], angle[pos[0, :3], 1], angle[pos[1, :3], 2]), 1)
    assert torch.allclose(z1, z0 * torch.polar(torch.ones(3, 3), turn).to(z0.dtype), atol=1e-6)
    assert torch.equal(q[:3, 0, 6:], before[:3, 0, 6:])


# ---------------------------------------------------- backend and end-to-end loop

def test_backend_windows():
    from turboquant_amd.vllm_backend_fused import TurboQuantFusedImpl
    make = lambda w: TurboQuantFusedImpl(4, 64, 0.125, 2, None, w, "fp8")
    assert make(None).window == 0 and make(128).window == 128 and make(128).sink == 0
    for bad in (0, -1):
        with pytest.raises(ValueError, match="sliding_window"):
            make(bad)


@pytest.mark.parametrize("window", [None, 0, -1, 128, (127, 0)])
@pytest.mark.parametrize("dtype", ["auto", "bfloat16"])
def test_windows_of_an_unpacked_cache_are_the_parents(window, dtype):
    """Such a layer takes whatever its parent takes; the window of the packed
    cache's calls is not looked at."""
    from turboquant_amd.vllm_backend_fused import TurboQuantFusedImpl
    impl = TurboQuantFusedImpl(4, 64, 0.125, 2, None, window, dtype)
    assert impl.window == 0 and impl.sliding_window == window


def test_starts_of_a_traced_call_are_not_kept():
    """A call over fake tensors leaves nothing that a later call would get."""
    from torch._subclasses.fake_tensor import FakeTensor, FakeTensorMode
    from turboquant_amd.vllm_backend_fused import TurboQuantFusedImpl
    impl = TurboQuantFusedImpl(4, 64, 0.125, 2, None, 8, "fp8")
    with FakeTensorMode():
        fake = impl._window_starts(torch.empty((3, 7), dtype=torch.int32))
    assert isinstance(fake, FakeTensor) and fake.shape == (4,)
    starts = impl._window_starts(torch.empty((3, 7), dtype=torch.int32))
    assert type(starts) is torch.Tensor and starts.tolist() == [0, 7, 14, 21]
    with FakeTensorMode():  # nor does it get theirs
        assert isinstance(impl._window_starts(torch.empty((3, 7), dtype=torch.int32)), FakeTensor)


def test_starts_are_made_on_the_host_whatever_the_default_device():
    """(a default device of "cuda" would make them on the current stream, which
    another stream's first call does not wait for; "meta" shows it without a GPU)"""
    from turboquant_amd.vllm_backend_fused import TurboQuantFusedImpl
    impl = TurboQuantFusedImpl(4, 64, 0.125, 2, None, 8, "fp8")
    table = torch.empty((3, 7), dtype=torch.int32)
    with torch.device("meta"):
        starts = impl._window_starts(table)
    assert starts.device == table.device and starts.tolist() == [0, 7, 14, 21]


def test_a_record_does_not_go_with_a_window():
    from turboquant_amd import e2e
    from turboquant_amd.budget import CacheRecord
    from turboquant_amd.vllm_backend_fused import TurboQuantFusedImpl
    impl = TurboQuantFusedImpl(4, 64, 0.125, 2, None, 8, "fp8")
    cache = torch.zeros((2, 5, 16, 2, 48), dtype=torch.uint8)
    impl.record = CacheRecord.beside(cache, 8)
    meta = e2e.Meta(1, 1, torch.zeros((1, 2), dtype=torch.int32),
                    torch.ones(1, dtype=torch.int32), torch.tensor([0, 1]), None)
    with pytest.raises(RuntimeError, match="sliding window"):
        impl.forward(None, torch.zeros((1, 256)), None, None, cache, meta)
    with pytest.raises(RuntimeError, match="packed"):
        TurboQuantFusedImpl(4, 64, 0.125, 2, None, 8, "auto").project_and_update(
            None, None, None, None, None, None, None, None)


def test_e2e_refuses_a_window_beside_a_budget():
    from turboquant_amd import e2e
    for kw in (dict(budget=64), dict(keep_fp16_kv=True)):
        with pytest.raises(ValueError, match="attention window"):
            e2e.Runner(e2e.ModelShape.tiny(1), 1, 32, torch.device("cpu"), attention_window=8, **kw)
    with pytest.raises(ValueError, match="attention window"):
        e2e.run(e2e.ModelShape.tiny(1), 1, 16, 4, compare_steps=2, device="cpu", attention_window=8)
