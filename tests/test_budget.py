"""The cache budget without a GPU: refusals of the ops, the record and the C
ABI, the ops' schemas, and the 64-bit forms that the GPU tests compare with."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

import budget_cases as C
from turboquant_amd import _lib, ops
from turboquant_amd.budget import CacheRecord


def _args(**bad):
    """A call's tensors on the meta device, all well formed but those given."""
    def t(shape, dtype):
        return torch.empty(shape, dtype=dtype, device="meta")
    a = dict(q=t((2, 8, 128), torch.float16), cache=t((2, 9, 16, 2, 80), torch.uint8),
             indices=t((8,), torch.int32), indptr=t((3,), torch.int32),
             seq=t((2,), torch.int32), o=t((2, 8, 128), torch.float16),
             weights=t((9, 2, 16), torch.float32), positions=t((9, 2, 16), torch.int32),
             ends=t((2,), torch.int32), starts=t((3,), torch.int32),
             new=t((2,), torch.int32), signs=None)
    a.update(bad)
    return a


def _decode(a):
    return ops.decode_paged_tracked(a["q"], a["cache"], a["indices"], a["indptr"], a["seq"], 2, 128,
                                    128, 0.1, a["signs"], a["o"], a["weights"], a["positions"],
                                    a["ends"])


def _window(a, window=4):
    return ops.track_window(a["q"], a["starts"], window, a["cache"], a["indices"], a["indptr"],
                            a["seq"], 2, 128, 128, 0.1, a["signs"], a["weights"], a["positions"],
                            a["ends"])


def _evict(a, budget=8, recent=0, sink=0):
    return ops.evict_paged(a["cache"], a["weights"], a["positions"], a["indices"], a["indptr"],
                           a["seq"], a["ends"], budget, recent, sink, a["new"])


def test_cpu_tensors_are_refused():
    a = {k: (v if v is None else torch.zeros(v.shape, dtype=v.dtype)) for k, v in _args().items()}
    for call in (_decode, _window, _evict):
        with pytest.raises(RuntimeError, match="GPU only"):
            call(a)


@pytest.mark.parametrize("call,key,shape,dtype,match", [
    (_decode, "q", (2, 8, 64), torch.float16, "q must be"),
    (_decode, "q", (2, 8, 128), torch.float32, "q must be"),
    (_decode, "q", (2, 7, 128), torch.float16, "q heads"),
    (_decode, "cache", (2, 9, 16, 4, 80), torch.uint8, "kv heads"),
    (_decode, "cache", (1, 9, 16, 2, 80), torch.uint8, "kv_cache must be"),
    (_decode, "indices", (8,), torch.int64, "indices must be"),
    (_decode, "indptr", (1,), torch.int32, "indptr must be"),
    (_decode, "seq", (1,), torch.int32, "seq_lens must be"),
    (_decode, "o", (2, 8, 128), torch.float32, "o must be"),
    (_decode, "o", (2, 8, 64), torch.float16, "o must be"),
    (_decode, "weights", (9, 16, 2), torch.float32, "weights must be"),
    (_decode, "weights", (9, 2, 16), torch.float16, "weights must be"),
    (_decode, "positions", (9, 2, 16), torch.int64, "positions must be"),
    (_decode, "positions", (8, 2, 16), torch.int32, "positions must be"),
    (_decode, "ends", (1,), torch.int32, "ends must be"),
    (_window, "starts", (0,), torch.int32, "batch \\+ 1"),
    (_window, "starts", (3,), torch.int64, "query_start_loc must be"),
    (_window, "q", (2, 8, 128), torch.float64, "q must be"),
    (_window, "weights", (9, 2, 17), torch.float32, "weights must be"),
    (_evict, "new", (1,), torch.int32, "new_lens must be"),
    (_evict, "new", (2,), torch.int64, "new_lens must be"),
    (_evict, "cache", (2, 9, 16, 2, 96), torch.uint8, "entries of 96 bytes"),
    (_evict, "positions", (9, 2, 16), torch.float32, "positions must be"),
])
def test_refusals(monkeypatch, call, key, shape, dtype, match):
    monkeypatch.setattr(ops, "_require_gpu", lambda *t: None)
    bad = torch.empty(shape, dtype=dtype, device="meta")
    with pytest.raises(RuntimeError, match=match):
        call(_args(**{key: bad}))


def test_integers_that_32_bits_would_wrap_are_refused(monkeypatch):
    monkeypatch.setattr(ops, "_require_gpu", lambda *t: None)
    a, wrap = _args(), 2 ** 32
    for call in (lambda: _window(a, window=wrap + 4), lambda: _evict(a, budget=wrap + 8),
                 lambda: _evict(a, recent=wrap), lambda: _evict(a, sink=-wrap),
                 lambda: ops.decode_paged_tracked(
                     a["q"], a["cache"], a["indices"], a["indptr"], a["seq"], 2, 128, wrap + 128,
                     0.1, None, a["o"], a["weights"], a["positions"], a["ends"])):
        with pytest.raises(RuntimeError, match="out of range"):
            call()


def test_positions_need_ends(monkeypatch):
    monkeypatch.setattr(ops, "_require_gpu", lambda *t: None)
    for call in (_decode, _window, _evict):
        with pytest.raises(RuntimeError, match="positions need ends"):
            call(_args(ends=None))


def test_record_refuses_a_rule_that_cannot_hold():
    for rule in (dict(budget=0), dict(budget=8, recent=5, sink=4), dict(budget=8, recent=-1),
                 dict(budget=8, window=0)):
        with pytest.raises(ValueError):
            CacheRecord(4, 16, 2, device="cpu", **rule)
    r = CacheRecord.beside(torch.zeros((2, 5, 32, 3, 48), dtype=torch.uint8), 8, recent=4, sink=4)
    assert r.weights.shape == r.positions.shape == (5, 3, 32)
    table = torch.arange(6, dtype=torch.int64).view(2, 3)
    indices, indptr = r._tables(table)
    assert indices.dtype == torch.int32 and indptr.tolist() == [0, 3, 6]
    assert r._tables(table)[1] is indptr


def _abi():
    """The three calls of the C ABI with addresses that are never read: every
    case below is refused before a launch."""
    lib = _lib.load()
    buf = (ctypes.c_char * 4096)()
    p = ctypes.addressof(buf)
    p += -p % 256

    def decode(q=p, qt=1, k=p, n=8, batch=2, hq=8, hkv=2, hd=128, pd=128, bs=16, ebs=80, nb=9, o=p,
               ot=1, w=p, pos=p, ends=p, ws=p, wsb=1 << 40):
        return lib.tq_decode_paged_tracked(q, 1024, 128, qt, k, k, p, n, p, p, batch, hq, hkv, hd,
                                           pd, bs, ebs, nb, 0.1, None, o, ot, w, pos, ends, ws,
                                           wsb, None)

    def window(q=p, rows=2, qt=1, starts=p, window=4, k=p, n=8, batch=2, hq=8, hkv=2, hd=128,
               pd=128, bs=16, ebs=80, nb=9, w=p, pos=p, ends=p, ws=p, wsb=1 << 40):
        return lib.tq_track_window(q, rows, 1024, 128, qt, starts, window, k, p, n, p, p, batch, hq,
                                   hkv, hd, pd, bs, ebs, nb, 0.1, None, w, pos, ends, ws, wsb, None)

    def evict(k=p, w=p, pos=p, n=8, ends=p, batch=2, hkv=2, pd=128, bs=16, ebs=80, nb=9, budget=8,
              recent=2, sink=2, new=p, ws=p, wsb=1 << 40):
        return lib.tq_evict_paged(k, k, w, pos, p, n, p, p, ends, batch, hkv, pd, bs, ebs, nb,
                                  budget, recent, sink, new, ws, wsb, None)
    return lib, dict(decode=decode, window=window, evict=evict, buf=buf, p=p)


BAD = [("decode", dict(pd=96)), ("decode", dict(hq=7)), ("decode", dict(hq=34)),
       ("decode", dict(hkv=0)), ("decode", dict(bs=8)), ("decode", dict(bs=0)),
       ("decode", dict(batch=-1)), ("decode", dict(batch=1025)), ("decode", dict(n=-1)),
       ("decode", dict(n=1 << 31)), ("decode", dict(hd=0)), ("decode", dict(hd=129)),
       ("decode", dict(qt=0)), ("decode", dict(q=None)), ("decode", dict(ebs=48)),
       ("decode", dict(nb=0)), ("decode", dict(nb=1 << 31)), ("decode", dict(nb=1 << 27)),
       ("decode", dict(k=None)), ("decode", dict(w=None)), ("decode", dict(ends=None)),
       ("decode", dict(o=None)), ("decode", dict(ot=0)), ("decode", dict(hkv=8192, hq=8192)),
       ("window", dict(window=0)), ("window", dict(window=257)), ("window", dict(starts=None)),
       ("window", dict(rows=-1)), ("window", dict(pd=32)), ("window", dict(batch=1025)),
       ("window", dict(w=None)), ("window", dict(ends=None)), ("window", dict(qt=3)),
       ("evict", dict(budget=0)), ("evict", dict(recent=-1)), ("evict", dict(sink=-1)),
       ("evict", dict(recent=5, sink=4)), ("evict", dict(pos=None)), ("evict", dict(ends=None)),
       ("evict", dict(new=None)), ("evict", dict(pd=100)), ("evict", dict(ebs=81)),
       ("evict", dict(bs=20)), ("evict", dict(nb=0)), ("evict", dict(batch=70000)),
       ("evict", dict(ws=None)), ("evict", dict(wsb=16)), ("evict", dict(n=1 << 28))]


@pytest.mark.parametrize("call,bad", BAD)
def test_abi_refuses_bad_arguments(call, bad):
    lib, calls = _abi()
    assert calls[call](**bad) == -22, bad
    assert lib.tq_last_error()


def test_abi_refuses_unaligned_state():
    lib, calls = _abi()
    p = calls["p"]
    for call in ("decode", "evict"):
        assert calls[call](w=p + 4) == -22 and b"aligned" in lib.tq_last_error()
        assert calls[call](k=p + 8) == -22 and b"aligned" in lib.tq_last_error()
    assert calls["evict"](pos=p + 4) == -22


def test_empty_batches_do_nothing():
    _, calls = _abi()
    for call in ("decode", "window", "evict"):
        assert calls[call](batch=0) == 0


def test_evict_workspace_holds_the_lists():
    lib = _lib.load()
    for b, h, n, bs, budget in ((1, 1, 1, 16, 5), (8, 8, 2048, 16, 8192), (3, 2, 5, 48, 10 ** 9)):
        got = lib.tq_evict_workspace_bytes(b, h, n, bs, budget)
        room = n * bs
        assert got >= b * h * (2 * 4 * min(budget, room) + 4) + (room * h * 4 if room > 32768 else 0)
    assert lib.tq_evict_workspace_bytes(1, 1, 1, 16, 0) == -22
    assert lib.tq_track_window_workspace_bytes(1, 300, 8, 2, 128) == -22
    assert lib.tq_decode_tracked_workspace_bytes(1, 1, 8, 2, 100, 16) == -22


def test_schemas_declare_the_writes():
    ops.register_ops()
    written = {"decode_paged_tracked": {"o", "weights", "positions"},
               "track_window": {"weights", "positions"},
               "evict_paged": {"kv_cache", "weights", "positions", "new_lens"}}
    for name, want in written.items():
        schema = getattr(torch.ops.turboquant_v5, name).default._schema
        got = {a.name for a in schema.arguments if a.alias_info and a.alias_info.is_write}
        assert got == want and not schema.returns


# ---------------------------------------------------- the 64-bit forms themselves

def test_reference_attention_is_a_softmax():
    """A decode's weights sum to the q heads per kv head; a window's to as many
    per query; a window of one is the decode."""
    c = C.make(3, [37, 5], 8, 2, 64)
    q = c.rng.standard_normal((2, 8, 64))
    o, w, p = C.attend(c, q, np.arange(3), 1, decode=True)
    c.weights[:] = 0
    _, w, p = C.attend(c, q, np.arange(3), 1)
    for b in range(2):
        pg, off, _ = C.places(c, b)
        assert np.allclose(w[pg, :, off].sum(0), 4)
        assert p[pg[-1], 0, off[-1]] == c.ends[b] - 1
    q = c.rng.standard_normal((12, 8, 64))
    _, w, p = C.attend(c, q, np.array([0, 7, 12]), 3)
    for b in range(2):
        pg, off, _ = C.places(c, b)
        assert np.allclose(w[pg, :, off].sum(0), 12)
    assert np.isfinite(o).all()


def test_reference_attention_is_the_oracle():
    import oracle
    c = C.make(4, [61, 40], 8, 2, 128)
    q = c.rng.standard_normal((2, 8, 128)).astype(np.float16)
    o, _, _ = C.attend(c, q.astype(np.float64), np.arange(3), 1, decode=True)
    ref = oracle.decode(q, c.cache, c.indices, c.indptr, c.lens, 2, 128, c.scale, c.signs)
    # (the oracle works in fp32: 128 products and 61 tokens)
    assert np.abs(o - ref).max() < 1e-4


def test_reference_eviction_keeps_the_largest():
    c = C.make(5, [50, 8], 2, 2, 64)
    for b in range(2):
        pg, off, _ = C.places(c, b)
        c.positions[pg, :, off] = np.arange(len(pg))[:, None]
    cache, w, p, lens = C.evict(c, 20, 6, 3)
    assert lens.tolist() == [20, 8]
    pg, off, _ = C.places(c, 0)
    for h in range(2):
        kept = set(p[pg[:20], h, off[:20]].tolist())
        assert len(kept) == 20
        end = int(c.ends[0])
        old = c.weights[pg, h, off]
        must = {i for i in range(50) if i < 3 or i >= end - 6}
        assert must <= kept
        rest = sorted((i for i in range(50) if i not in must), key=lambda i: -old[i])
        assert kept == must | set(rest[:20 - len(must)])
        for i in range(20):  # entries went with their weights
            at = p[pg[i], h, off[i]]
            assert w[pg[i], h, off[i]] == old[at]
            assert (cache[:, pg[i], off[i], h] == c.cache[:, pg[at], off[at], h]).all()
