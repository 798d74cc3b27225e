"""The operators of layers that attend over a sliding window with a few first
tokens that stay visible, from the fused projection to the attention's output,
as cases to be timed and compared.

A query at position P sees the keys j with P - window < j <= P, and those with
j < sink.  Four kinds of call:

* ``decode`` -- ``ops.decode_paged_window``: one new token per sequence attends
  over the packed paged cache;
* ``prefill`` -- ``ops.prefill_attention_window``: the chunks of a step attend
  over fp16 rows, the tokens that a chunk still sees followed by its own;
* ``readback`` -- ``ops.prefill_gather_window``: those rows from the packed
  cache, followed by the chunk's fresh ones;
* ``write`` -- ``ops.norm_rope_write``: the fused projection's rows normed per
  head, rotated (positions with one or three axes) and, for K and V, quantised
  into the cache; the written entries are read back as the values they stand for.

The cache is uint8 [2, blocks, page, kv heads, entry bytes]: 4-bit codes (dim
2k in the high nibble of byte k), then the fp16 norm.  Pages that no later query
sees are given back, as a server does: their table entries are -1.  Cases are
plain dicts; lengths come from the case itself, so that ``work`` needs no GPU.
"""
from __future__ import annotations

import math
import random
from types import SimpleNamespace

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
# Lloyd-Max levels of N(0, 1) at 4 bits and the boundaries between them
LEVELS = (-2.7326368, -2.0693470, -1.6180345, -1.2562491, -0.9423684, -0.6567591, -0.3880823,
          -0.1284154, 0.1284154, 0.3880823, 0.6567591, 0.9423684, 1.2562491, 1.6180345, 2.0693470,
          2.7326368)
UPPER = (0.2582488430577470, 0.5224207238480534, 0.7995637494657970, 1.0993087223329937,
         1.4371417912897455, 1.8436907609368955, 2.4009919259139040)
# (q heads, kv heads, head size): the Qwen3-8B geometry and the head-size
# 64 / 256 geometries of the ragged configuration, more q heads per kv head,
# a tensor-parallel shard with one kv head, a padded head size, one q head per
# kv head, and 16 q heads per kv head
GEOMETRIES = [(32, 8, 128), (16, 4, 64), (16, 2, 256), (64, 8, 128), (8, 1, 128), (12, 4, 96),
              (8, 8, 64), (32, 2, 128)]
EPS = 1e-6
THETA = 1e6
TABLE = 40960  # rows of the rotation tables
BLOCK = 512    # query rows that the plain prefill takes together


def listed():
    return [
        # one interactive user behind a long conversation: latency
        dict(name="decode_single", kind="decode", batch=1, lo=9001, hi=9001, window=1024, sink=4,
             len_seed=1, geometry=0, page=16, dtype="fp16"),
        # a full server at the headline geometry, every sequence beyond its window
        dict(name="decode_batch_4k", kind="decode", batch=64, lo=32768, hi=32768, window=4096,
             sink=4, len_seed=2, geometry=0, page=16, dtype="fp16"),
        # ragged lengths, some inside the window, an odd window, head size 64
        dict(name="decode_ragged_hd64", kind="decode", batch=48, lo=5, hi=16384, window=1000,
             sink=0, len_seed=3, geometry=1, page=16, dtype="bf16"),
        # short prompts prefilled together
        dict(name="prefill_prompts", kind="prefill", batch=4, chunk_lo=37, chunk_hi=1500, ctx_lo=0,
             ctx_hi=0, window=512, sink=4, len_seed=11, geometry=0, dtype="fp16"),
        # one long prompt
        dict(name="prefill_prompt_32k", kind="prefill", batch=1, chunk_lo=32768, chunk_hi=32768,
             ctx_lo=0, ctx_hi=0, window=4096, sink=4, len_seed=12, geometry=0, dtype="fp16"),
        # later chunks of three prompts, head size 64
        dict(name="prefill_chunks_hd64", kind="prefill", batch=3, chunk_lo=700, chunk_hi=2048,
             ctx_lo=4000, ctx_hi=16000, window=1000, sink=0, len_seed=13, geometry=1, dtype="bf16"),
        # what those chunks of a step read in front of the attention
        dict(name="readback_chunks", kind="readback", batch=3, chunk_lo=700, chunk_hi=2048,
             ctx_lo=4000, ctx_hi=16000, window=1024, sink=4, len_seed=21, geometry=0, page=16,
             dtype="bf16"),
        # sixteen sequences taken up again with a few new tokens each
        dict(name="readback_batch_4k", kind="readback", batch=16, chunk_lo=1, chunk_hi=64,
             ctx_lo=8192, ctx_hi=32000, window=4096, sink=4, len_seed=22, geometry=0, page=16,
             dtype="fp16"),
        # a decode step of eight sequences: latency
        dict(name="write_step", kind="write", batch=8, chunk_lo=1, chunk_hi=1, ctx_lo=1000,
             ctx_hi=30000, len_seed=31, geometry=0, page=16, dtype="fp16", axes=1, rotated=128,
             norms=True),
        # a prompt's chunk, positions of images and video (time, height, width)
        dict(name="write_chunk_axes", kind="write", batch=1, chunk_lo=8192, chunk_hi=8192, ctx_lo=0,
             ctx_hi=0, len_seed=32, geometry=0, page=16, dtype="bf16", axes=3, rotated=128,
             norms=True),
        # four prompts of odd lengths, half of each head of 64 rotated, no norms
        dict(name="write_half_hd64", kind="write", batch=4, chunk_lo=37, chunk_hi=1500, ctx_lo=0,
             ctx_hi=500, len_seed=33, geometry=1, page=16, dtype="bf16", axes=1, rotated=32,
             norms=False),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    kind = rng.choice(["decode", "prefill", "readback", "write"])
    geometry, page = rng.randrange(len(GEOMETRIES)), rng.choice([16, 16, 16, 32, 48])
    hq, hkv, hd = GEOMETRIES[geometry]
    case = dict(kind=kind, len_seed=rng.randrange(1 << 30), geometry=geometry,
                dtype=rng.choice(["fp16", "bf16"]))
    window = _log_int(rng, 1, 4096)
    sink = rng.choice([0, 1, 4, 4, rng.randint(0, 100)])
    if kind == "decode":
        batch = _log_int(rng, 1, 64)
        hi = _log_int(rng, 1, 32768)
        return dict(case, batch=batch, lo=rng.choice([0, 1, hi // 2, hi]), hi=hi, window=window,
                    sink=sink, page=page)
    if kind == "write":
        batch = _log_int(rng, 1, 32)
        most = 8192 * 48 * 128 // ((hq + 2 * hkv) * hd)
        hi = _log_int(rng, 1, min(8192, most // batch))
        ctx_hi = rng.choice([0, _log_int(rng, 1, 30000)])
        return dict(case, batch=batch, chunk_lo=max(1, hi // rng.choice([1, 3])), chunk_hi=hi,
                    ctx_lo=ctx_hi // 2, ctx_hi=ctx_hi, page=page, axes=rng.choice([1, 1, 3]),
                    rotated=rng.choice([hd, hd, hd // 2 // 16 * 16]), norms=rng.random() < 0.7)
    batch = rng.randrange(1, 9)
    hi = _log_int(rng, 1, 16384 // batch)
    ctx_hi = _log_int(rng, 1, 16384) if kind == "readback" or rng.random() < 0.5 else 0
    case.update(batch=batch, chunk_lo=max(1, hi // rng.choice([1, 3])), chunk_hi=hi,
                ctx_lo=ctx_hi // rng.choice([1, 4]), ctx_hi=ctx_hi, window=window, sink=sink)
    return dict(case, page=page) if kind == "readback" else case


# ------------------------------------------------------------------ geometry

def _pad(head):
    return max(64, 1 << (head - 1).bit_length())


def _entry_bytes(pd):
    return (pd // 2 + 2 * (pd // 64) + 15) & ~15


def _lengths(case):
    """(chunk, cached before it) of each sequence; a decode step's chunk is its
    newest token, already in the cache (none: an empty row of the batch)."""
    r = random.Random(case["len_seed"])
    if case["kind"] == "decode":
        n = [r.randint(case["lo"], case["hi"]) for _ in range(case["batch"])]
        return [(min(1, x), max(0, x - 1)) for x in n]
    return [(r.randint(case["chunk_lo"], case["chunk_hi"]), r.randint(case["ctx_lo"], case["ctx_hi"]))
            for _ in range(case["batch"])]


def _kept(case, ctx):
    """(first, rows): of ctx cached tokens the first query behind them sees the
    sinks and those from `first` on, `rows` in all."""
    first = max(0, ctx - case["window"] + 1)
    return first, min(case["sink"], first) + ctx - first


def _sections(case):
    """Rotated pairs of each axis of the positions: the later two take three quarters."""
    half = case["rotated"] // 2
    if case["axes"] == 1:
        return (half,)
    rest = (half - half // 4) // 2
    return (half - 2 * rest, rest, rest)


def work(case):
    hq, hkv, hd = GEOMETRIES[case["geometry"]]
    pd = _pad(hd)
    code = pd // 2 + 2  # bytes of one cached vector that carry information
    lens = _lengths(case)
    fresh = sum(c for c, _ in lens)
    if case["kind"] == "decode":
        seen = sum(c + _kept(case, x)[1] for c, x in lens)
        return {"bytes": seen * (hkv * 2 * code + 4 / case["page"]) + len(lens) * (4 * hq * hd + 8),
                "flops": 4.0 * seen * hq * hd}
    if case["kind"] == "prefill":
        rows = sum(c + _kept(case, x)[1] for c, x in lens)
        pairs = 0
        for c, x in lens:
            # position P sees min(P + 1, window) keys and the sinks before them
            w, s = case["window"], case["sink"]
            def upto(n):  # over P < n
                full = max(0, n - w)
                out = min(n, w) * (min(n, w) + 1) // 2 + full * w
                m = min(full, s)
                return out + m * (m + 1) // 2 + (full - m) * s
            pairs += upto(c + x) - upto(x)
        return {"bytes": 4 * fresh * hq * hd + 4 * rows * hkv * hd, "flops": 4.0 * pairs * hq * hd}
    if case["kind"] == "readback":
        kept = sum(_kept(case, x)[1] for _, x in lens)
        return {"bytes": kept * hkv * (2 * code + 4 * pd) + fresh * hkv * (4 * hd + 4 * pd),
                "flops": 2.0 * kept * hkv * pd * math.log2(pd)}
    table = 4 * case["rotated"] * min(fresh, TABLE)
    # the write, and the written entries read back as fp16 rows
    return {"bytes": fresh * (2 * (hq + 2 * hkv) * hd + 2 * (hq + hkv) * hd + hkv * 2 * code
                              + 8 * case["axes"] + 4) + table + fresh * hkv * (2 * code + 4 * pd),
            "flops": fresh * ((hq + hkv) * 8.0 * hd + hkv * 4.0 * pd * math.log2(pd))}


# ------------------------------------------------------------------ inputs

def prepare(case, seed):
    dev = torch.device("cuda:0")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    hq, hkv, hd = GEOMETRIES[case["geometry"]]
    pd = _pad(hd)
    kind, lens, dt = case["kind"], _lengths(case), DTYPES[case["dtype"]]
    batch = len(lens)

    def randn(*shape):
        return torch.randn(shape, generator=g, device=dev)

    levels = torch.tensor(LEVELS, device=dev)
    st = SimpleNamespace(kind=kind, hq=hq, hkv=hkv, hd=hd, pd=pd, scale=1.0 / math.sqrt(hd),
                         lens=lens, levels=levels, dt=dt, window=case.get("window"),
                         sink=case.get("sink"), signs=torch.where(randn(pd) < 0, -1.0, 1.0))
    total = sum(c for c, _ in lens)
    starts = [sum(c for c, _ in lens[:b]) for b in range(batch)]
    if kind == "prefill":
        kv = [c + _kept(case, x)[1] for c, x in lens]
        st.requests = [(starts[b], lens[b][0], sum(kv[:b]), kv[b], 0) for b in range(batch)]
        st.q = (randn(total, hq, hd) * 2.0).to(dt)
        # keys with a few strong coordinates, as real ones have
        gain = torch.where(randn(hkv, hd) > 2.0, 4.0, 1.0)
        st.k = torch.nn.functional.pad((randn(sum(kv), hkv, hd) * gain).half(), (0, pd - hd))
        st.v = torch.nn.functional.pad(randn(sum(kv), hkv, hd).half(), (0, pd - hd))
        st.o = torch.empty_like(st.q)
        return st

    # the cache: pages of the tokens that a query still sees, in random places
    bs = st.bs = case["page"]
    ebs = _entry_bytes(pd)
    have = [c + x if kind != "readback" else x for c, x in lens]
    width = max(1, -(-max(have) // bs))
    pages = torch.arange(width, device=dev)
    table = torch.full((batch, width), -1, dtype=torch.int32, device=dev)
    need, held = 0, []
    for (c, x), n in zip(lens, have):
        first, sink = (_kept(case, x)[0], case["sink"]) if kind != "write" else (x, 0)
        on = (pages * bs < n) & ((pages * bs < min(sink, n)) | ((pages + 1) * bs > first))
        held.append(on)
        need += int(on.sum())
    nb = need + 3
    perm = torch.randperm(nb, generator=g, device=dev).to(torch.int32)
    at = 0
    for b, on in enumerate(held):
        n = int(on.sum())
        table[b, on] = perm[at:at + n]
        at += n
    bounds = (levels[1:] + levels[:-1]) / 2
    st.cache = torch.zeros((2, nb, bs, hkv, ebs), dtype=torch.uint8, device=dev)
    for slab in range(2):
        for a in range(0, nb, 4096):
            n = min(4096, nb - a)
            codes = torch.bucketize(randn(n, bs, hkv, pd), bounds).to(torch.uint8)
            st.cache[slab, a:a + n, ..., :pd // 2] = (codes[..., 0::2] << 4) | codes[..., 1::2]
            norm = (math.sqrt(hd) * (0.25 * randn(n, bs, hkv)).exp()).to(torch.float16)
            st.cache[slab, a:a + n, ..., pd // 2:pd // 2 + 2 * (pd // 64)] = \
                norm[..., None].repeat(1, 1, 1, pd // 64).view(torch.uint8)
    st.table = table
    if kind == "decode":
        st.seq = torch.tensor(have, dtype=torch.int32, device=dev)
        st.indices = table.reshape(-1)
        st.indptr = torch.arange(batch + 1, dtype=torch.int32, device=dev) * width
        st.q = (randn(batch, hq, hd) * 2.0).to(dt)
        st.o = torch.empty_like(st.q)
        return st
    if kind == "readback":
        st.key, st.value = (randn(total, hkv, hd).to(dt) for _ in range(2))
        st.requests, rows = [], 0
        for b, (c, x) in enumerate(lens):
            first, kept = _kept(case, x)
            st.requests.append((b, x, first, starts[b], c, rows))
            rows += kept + c
    else:
        # the rows of the fused projection, then their cache slots; a padded
        # step's last row has no slot
        st.qkv = (randn(total, hq + 2 * hkv, hd) * (0.5 * randn(total, hq + 2 * hkv, 1)).exp()) \
            .to(dt).view(total, -1)
        st.norms, st.eps = case["norms"], EPS
        st.qw, st.kw = ((1.0 + 0.1 * randn(hd)).to(dt) if case["norms"] else None for _ in range(2))
        half = case["rotated"] // 2
        freq = THETA ** (-torch.arange(half, dtype=torch.float64, device=dev) / half)
        angle = torch.arange(TABLE, dtype=torch.float64, device=dev)[:, None] * freq
        st.cos, st.sin = angle.cos().float(), angle.sin().float()
        t = torch.cat([torch.arange(x, x + c, device=dev) for c, x in lens])
        st.sections = _sections(case)
        # time runs on, the two places in a picture of 24 columns repeat
        st.positions = t if case["axes"] == 1 else torch.stack((t // 4, t // 24 % 32, t % 24))
        seq = torch.repeat_interleave(torch.arange(batch, device=dev),
                                      torch.tensor([c for c, _ in lens], device=dev))
        st.slots = (table[seq, t // bs].long() * bs + t % bs).to(torch.int32)
        if total > 1:
            st.slots[-1] = -1
        st.q = torch.empty((total, hq, hd), dtype=dt, device=dev)
        st.k = torch.empty((total, hkv, hd), dtype=dt, device=dev)
        st.requests = [(b, x + c, x, 0, 0, starts[b]) for b, (c, x) in enumerate(lens)]
        st.sink, rows = 0, total
    st.out_k, st.out_v = (torch.empty((rows, hkv, pd), dtype=torch.float16, device=dev)
                          for _ in range(2))
    return st


# ------------------------------------------------------------------ calls

def run(st):
    if own:
        from turboquant_amd import ops
        if st.kind == "decode":
            ops.decode_paged_window(st.q, st.cache, st.indices, st.indptr, st.seq, st.hkv, st.hd,
                                    st.pd, st.scale, st.signs, st.o, st.window, st.sink)
            return {"o": st.o}
        if st.kind == "prefill":
            ops.prefill_attention_window(st.q, st.o, st.requests, st.hkv, st.hd, st.pd, st.scale,
                                         st.window, st.sink, st.k, st.v)
            return {"o": st.o}
        if st.kind == "readback":
            ops.prefill_gather_window(st.cache, st.table, st.key, st.value, st.requests, st.sink,
                                      st.hd, st.pd, st.signs, st.out_k, st.out_v)
            return {"k": st.out_k, "v": st.out_v}
        ops.norm_rope_write(st.qkv, st.qw, st.kw, st.cos, st.sin, st.positions, st.cache, st.signs,
                            st.slots, st.hq, st.hd, st.pd, st.q, st.k, eps=st.eps,
                            sections=st.sections)
        ops.prefill_gather_window(st.cache, st.table, None, None, st.requests, 0, st.hd, st.pd,
                                  st.signs, st.out_k, st.out_v)
        return {"q": st.q, "k": st.k, "cached_k": st.out_k, "cached_v": st.out_v}
    if st.kind == "decode":
        return {"o": _plain_decode(st)}
    if st.kind == "prefill":
        return {"o": _plain_prefill(st)}
    if st.kind == "readback":
        return {"k": _plain_readback(st, 0, st.key), "v": _plain_readback(st, 1, st.value)}
    return _plain_write(st)


# ------------------------------------------------------------------ plain forms

def _hadamard(n, device, dtype=torch.float32):
    """H[i, j] = (-1)^popcount(i & j) / sqrt(n), symmetric and its own inverse."""
    i = torch.arange(n, device=device)
    x = i[:, None] & i[None, :]
    for s in (8, 4, 2, 1):
        x = x ^ (x >> s)
    return (1 - 2 * (x & 1)).to(dtype) / math.sqrt(n)


def _read(st, slab, slot):
    """Cached rows [*slot.shape, H, pd] fp32 in the rotated domain."""
    e = st.cache[slab].reshape(-1, st.hkv, st.cache.shape[-1])[slot]
    codes = e[..., :st.pd // 2]
    codes = torch.stack((codes >> 4, codes & 15), dim=-1).flatten(-2)
    norm = e[..., st.pd // 2:st.pd // 2 + 2].contiguous().view(torch.float16).float()
    return st.levels[codes.int()] * (norm / math.sqrt(st.pd))


def _plain_decode(st):
    b, r, dev = st.seq.numel(), st.hq // st.hkv, st.q.device
    seq = st.seq.long()[:, None]
    # the sinks, then the window's places up to the newest token
    i = torch.arange(st.sink + st.window, device=dev)[None, :]
    low = (seq - st.window).clamp_min(0)
    t = torch.where(i < st.sink, i, low + i - st.sink)
    seen = torch.where(i < st.sink, t < low.clamp_max(st.sink), t < seq)
    t = torch.where(seen, t, 0)
    slot = torch.where(seen, st.table.gather(1, t // st.bs).long() * st.bs + t % st.bs, 0)
    q = torch.nn.functional.pad(st.q.float(), (0, st.pd - st.hd)) * st.signs
    q = (q @ _hadamard(st.pd, dev)).view(b, st.hkv, r, st.pd)
    k = _read(st, 0, slot).permute(0, 2, 3, 1).contiguous()
    s = torch.where(seen[:, None, None], (q * st.scale) @ k, -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(torch.isinf(top), 0.0, top))
    p = p / p.sum(-1, keepdim=True).clamp_min(1e-30)
    v = torch.where(seen[..., None, None], _read(st, 1, slot), 0.0)
    o = (p @ v.transpose(1, 2).contiguous()).reshape(b, st.hq, st.pd)
    return ((o @ _hadamard(st.pd, dev)) * st.signs)[..., :st.hd].to(st.q.dtype)


def _plain_prefill(st):
    """Blocks of query rows over the keys that any row of the block sees: the
    sinks, then the window's places in front of the block's last row."""
    dev, r = st.q.device, st.hq // st.hkv
    spans = torch.tensor([(a, ql, k0, kl) for a, ql, k0, kl, _ in st.requests], device=dev)
    blocks = -(-spans[:, 1] // BLOCK)
    req = torch.repeat_interleave(torch.arange(len(st.requests), device=dev), blocks)
    nth = torch.arange(req.numel(), device=dev) - (blocks.cumsum(0) - blocks)[req]
    a, ql, k0, kl = (x[:, None] for x in spans[req].unbind(1))
    i = nth[:, None] * BLOCK + torch.arange(BLOCK, device=dev)  # rows of the request
    there = i < ql
    pos = kl - ql + i  # their places among the request's keys
    n = st.window + BLOCK - 1
    j = torch.arange(st.sink + n, device=dev)[None, :]
    last = kl - ql + nth[:, None] * BLOCK + BLOCK - 1
    key = torch.where(j < st.sink, j, last - n + 1 + j - st.sink)
    ok = (key >= 0) & (key < kl)
    seen = (ok & (j < st.sink))[:, None, :] & (key[:, None, :] <= pos[..., None] - st.window) | \
        (ok & (j >= st.sink))[:, None, :] & (key[:, None, :] <= pos[..., None]) \
        & (key[:, None, :] > pos[..., None] - st.window)
    row = torch.where(there, a + i, 0)
    at = torch.where(ok, k0 + key, 0)
    q = torch.nn.functional.pad(st.q[row].float(), (0, st.pd - st.hd))
    q = q.view(-1, BLOCK, st.hkv, r, st.pd).permute(0, 2, 3, 1, 4) \
        .reshape(-1, st.hkv, r * BLOCK, st.pd)
    k = st.k[at].float().permute(0, 2, 3, 1).contiguous()
    s = ((q * st.scale) @ k).view(-1, st.hkv, r, BLOCK, j.numel())
    s.masked_fill_(~seen[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    p = s.sub_(torch.where(torch.isinf(top), 0.0, top)).exp_()
    p = p.div_(p.sum(-1, keepdim=True).clamp_min(1e-30)).view(-1, st.hkv, r * BLOCK, j.numel())
    o = p @ st.v[at].float().permute(0, 2, 1, 3).contiguous()
    o = o.view(-1, st.hkv, r, BLOCK, st.pd).permute(0, 3, 1, 2, 4).reshape(-1, BLOCK, st.hq, st.pd)
    out = torch.empty_like(st.q)
    out[row[there]] = o[there][..., :st.hd].to(st.q.dtype)
    return out


def _plain_rows(st):
    """Of every output row its request, its place among the request's tokens
    (cached, then fresh), and which rows are cached."""
    dev = st.table.device
    spans = torch.tensor([(b, x, f, a, n) for b, x, f, a, n, _ in st.requests], device=dev)
    kept = spans[:, 2].clamp_max(st.sink) + spans[:, 1] - spans[:, 2]
    rows = kept + spans[:, 4]
    req = torch.repeat_interleave(torch.arange(len(st.requests), device=dev), rows)
    i = torch.arange(req.numel(), device=dev) - (rows.cumsum(0) - rows)[req]
    b, ctx, first, fresh, _ = spans[req].unbind(1)
    sinks = first.clamp_max(st.sink)
    t = torch.where(i < sinks, i, first + i - sinks)
    return b, t, t < ctx, fresh + t - ctx


def _plain_cached(st, slab, b, t):
    page = st.table[b, t // st.bs].long()
    rows = _read(st, slab, page.clamp_min(0) * st.bs + t % st.bs)
    rows = (rows @ _hadamard(st.pd, rows.device)) * st.signs
    rows = rows * (torch.arange(st.pd, device=rows.device) < st.hd)
    return torch.where((page >= 0)[:, None, None], rows, 0.0)


def _plain_readback(st, slab, fresh):
    b, t, cached, f = _plain_rows(st)
    old = _plain_cached(st, slab, b, torch.where(cached, t, 0)).half()
    new = torch.nn.functional.pad(fresh[torch.where(cached, 0, f)].half(), (0, st.pd - st.hd))
    return torch.where(cached[:, None, None], old, new)


def _plain_write(st):
    n = st.qkv.shape[0]
    x = st.qkv.view(n, -1, st.hd).float()
    qk = x[:, :st.hq + st.hkv]
    if st.norms:
        w = torch.cat((st.qw.expand(st.hq, -1), st.kw.expand(st.hkv, -1))).float()
        qk = qk * torch.rsqrt(qk.square().mean(-1, keepdim=True) + st.eps) * w
    half = st.cos.shape[1]
    axis = torch.repeat_interleave(torch.arange(len(st.sections), device=x.device),
                                   torch.tensor(st.sections, device=x.device))
    pos = st.positions.view(-1, n)[axis]  # [half, tokens]
    pair = torch.arange(half, device=x.device)[:, None]
    cos, sin = (y[pos, pair].T[:, None] for y in (st.cos, st.sin))
    a, b = qk[..., :half], qk[..., half:2 * half]
    qk = torch.cat((a * cos - b * sin, b * cos + a * sin, qk[..., 2 * half:]), -1).to(st.dt)
    k, v = qk[:, st.hq:], st.qkv.view(n, -1, st.hd)[:, st.hq + st.hkv:]
    # the borders between codes in 64 bits
    spin = _hadamard(st.pd, x.device, torch.float64)
    upper = torch.tensor(UPPER, dtype=torch.float32, device=x.device).double()
    bounds = torch.cat((-upper.flip(0), upper.new_zeros(1), upper))
    cache = st.cache.view(2, -1, st.hkv, st.cache.shape[-1])
    into = st.slots >= 0
    at = st.slots[into].long()
    for slab, rows in enumerate((k, v)):
        y = torch.nn.functional.pad(rows[into].double(), (0, st.pd - st.hd)) * st.signs
        norm = y.norm(dim=-1, keepdim=True)
        y = (y / norm.clamp_min(1e-30)) @ spin * math.sqrt(st.pd)
        codes = torch.bucketize(y, bounds, right=True).to(torch.uint8)
        cache[slab, at, :, :st.pd // 2] = (codes[..., 0::2] << 4) | codes[..., 1::2]
        cache[slab, at, :, st.pd // 2:st.pd // 2 + 2 * (st.pd // 64)] = \
            norm.half().repeat(1, 1, st.pd // 64).view(torch.uint8)
    b, t, _, _ = _plain_rows(st)
    return {"q": qk[:, :st.hq].contiguous(), "k": k.contiguous(),
            "cached_k": _plain_cached(st, 0, b, t).half(),
            "cached_v": _plain_cached(st, 1, b, t).half()}


# ------------------------------------------------------------------ in 64 bits

def _exact_entries(cache, levels, pd, back, page, place):
    """Entries [n, H, pd] of a slab in the original domain."""
    e = cache[page, place]
    hi, lo = e[..., :pd // 2] // 16, e[..., :pd // 2] % 16
    x = torch.stack((levels[hi.int()], levels[lo.int()]), -1).flatten(-2)
    norm = e[..., pd // 2:pd // 2 + 2].contiguous().view(torch.float16).double()
    return (x * norm / math.sqrt(pd)) @ back


def exact(case, seed):
    """The definition, sequence by sequence in 64 bits; keys and values in the
    original domain."""
    st = prepare(case, seed)
    dev = st.signs.device
    w, sink, r, hd, pd = st.window, st.sink, st.hq // st.hkv, st.hd, st.pd
    # rows of the inverse rotation: c -> (c H) * signs
    back = _hadamard(pd, dev, torch.float64) * st.signs.double()
    levels = torch.tensor(LEVELS, dtype=torch.float32, device=dev).double()
    if st.kind == "prefill":
        o = torch.zeros(st.q.shape, dtype=torch.float64, device=dev)
        for a, ql, k0, kl, _ in st.requests:
            for h in range(st.hq):
                k = st.k[k0:k0 + kl, h // r, :hd].double()
                v = st.v[k0:k0 + kl, h // r, :hd].double()
                for i in range(0, ql, 4096):
                    n = min(4096, ql - i)
                    p = torch.arange(kl - ql + i, kl - ql + i + n, device=dev)[:, None]
                    lo, up = max(0, kl - ql + i - w + 1), kl - ql + i + n
                    j = torch.cat((torch.arange(min(sink, lo), device=dev),
                                   torch.arange(lo, up, device=dev)))
                    s = (st.q[a + i:a + i + n, h].double() @ k[j].T) * st.scale
                    hid = (j > p) | ((j <= p - w) & (j >= sink))
                    o[a + i:a + i + n, h] = s.masked_fill_(hid, -math.inf).softmax(-1) @ v[j]
        return {"o": o}
    if st.kind == "decode":
        o = torch.zeros(st.q.shape, dtype=torch.float64, device=dev)
        for b, n in enumerate(st.seq.tolist()):
            if n == 0:
                continue
            t = torch.arange(n, device=dev)
            t = t[(t < sink) | (t > n - 1 - w)]
            page, place = st.table[b, t // st.bs].long(), t % st.bs
            k, v = (_exact_entries(x, levels, pd, back, page, place)[..., :hd] for x in st.cache)
            for h in range(st.hq):
                s = (k[:, h // r] @ st.q[b, h].double()) * st.scale
                o[b, h] = s.softmax(0) @ v[:, h // r]
        return {"o": o}
    if st.kind == "readback":
        out = [torch.zeros(st.out_k.shape, dtype=torch.float64, device=dev) for _ in range(2)]
        for b, ctx, first, a, n, row in st.requests:
            t = torch.arange(ctx, device=dev)
            t = t[(t < sink) | (t >= first)]
            page, place = st.table[b, t // st.bs].long(), t % st.bs
            for x, y, fresh in zip(out, st.cache, (st.key, st.value)):
                x[row:row + len(t), :, :hd] = \
                    _exact_entries(y, levels, pd, back, page, place)[..., :hd]
                x[row + len(t):row + len(t) + n, :, :hd] = fresh[a:a + n].double()
        return {"k": out[0], "v": out[1]}
    # write: each rotated pair as a complex number turned by its angle
    n, half = st.qkv.shape[0], st.cos.shape[1]
    x = st.qkv.view(n, -1, hd).double()
    q, k, v = x[:, :st.hq], x[:, st.hq:st.hq + st.hkv], x[:, st.hq + st.hkv:]
    at = 0
    turn = torch.empty((n, half), dtype=torch.complex128, device=dev)
    for axis, m in enumerate(st.sections):
        p = st.positions.view(-1, n)[axis]
        turn[:, at:at + m] = torch.complex(st.cos[p, at:at + m].double(),
                                           st.sin[p, at:at + m].double())
        at += m

    def done(y, weight):
        if weight is not None:
            y = y / ((y * y).sum(-1, keepdim=True) / hd + st.eps).sqrt() * weight.double()
        z = torch.complex(y[..., :half], y[..., half:2 * half]) * turn[:, None]
        return torch.cat((z.real, z.imag, y[..., 2 * half:]), -1)

    q, k = done(q, st.qw), done(k, st.kw)
    out = {"q": q, "k": k}
    upper = torch.tensor(UPPER, dtype=torch.float32, device=dev).double()
    bounds = torch.cat((-upper.flip(0), upper.new_zeros(1), upper))
    # the cache takes a key as its row's type holds it
    for name, y, slab in (("cached_k", k.to(st.dt).double(), 0), ("cached_v", v, 1)):
        norm = y.square().sum(-1, keepdim=True).sqrt()
        z = torch.nn.functional.pad(y / norm.clamp_min(1e-30), (0, pd - hd)) @ back.T * math.sqrt(pd)
        z = levels[torch.bucketize(z, bounds, right=True)] * norm.half().double() / math.sqrt(pd)
        z = (z @ back)[..., :hd]
        if int(st.slots[-1]) < 0:  # the row without a slot: what the cache held there
            b, ctx = len(st.lens) - 1, sum(st.lens[-1])
            t = torch.tensor([ctx - 1], device=dev)
            z[-1:] = _exact_entries(st.cache[slab], levels, pd, back,
                                    st.table[b, t // st.bs].long(), t % st.bs)[..., :hd]
        out[name] = torch.nn.functional.pad(z, (0, pd - hd))
    return out
