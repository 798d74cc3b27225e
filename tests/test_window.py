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
    written = {"decode_paged_window": {"o"}}
    for name, want in written.items():
        schema = getattr(torch.ops.turboquant_v5, name).default._schema
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
