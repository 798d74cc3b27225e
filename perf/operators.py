"""The operators that keep a sequence inside a cache budget, as cases to be
timed and compared: attention that records what each cached token receives,
and the eviction that goes by that record.

Three kinds of call:

* ``decode`` -- ``ops.decode_paged_tracked``: one new token per sequence
  attends over the packed paged cache, and the weight that each cached entry
  receives is added to its accumulator;
* ``window`` -- ``ops.track_window``: the weights that the last queries of a
  prompt chunk give to the cached tokens, added up over those queries;
* ``evict`` -- ``ops.evict_paged``: per sequence and kv head the entries with
  the largest accumulated weight are kept and moved to the front.

The cache is uint8 [2, blocks, page, kv heads, entry bytes]: 4-bit codes (dim
2k in the high nibble of byte k), then the fp16 norm.  Beside it stand the
accumulators, fp32 [blocks, kv heads, page], and the positions of the entries,
int32 of that shape.  Cases are plain dicts; lengths come from the case itself,
so that ``work`` needs no GPU.
"""
from __future__ import annotations

import math
import random
from types import SimpleNamespace

import numpy as np
import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
# Lloyd-Max levels of N(0, 1) at 4 bits
LEVELS = (-2.7326368, -2.0693470, -1.6180345, -1.2562491, -0.9423684, -0.6567591, -0.3880823,
          -0.1284154, 0.1284154, 0.3880823, 0.6567591, 0.9423684, 1.2562491, 1.6180345, 2.0693470,
          2.7326368)
# (q heads, kv heads, head size): the Qwen3-8B geometry and the head-size
# 64 / 256 geometries of the ragged configuration, more q heads per kv head,
# a tensor-parallel shard with one kv head, a padded head size, one q head per
# kv head, and 16 q heads per kv head
GEOMETRIES = [(32, 8, 128), (16, 4, 64), (16, 2, 256), (64, 8, 128), (8, 1, 128), (12, 4, 96),
              (8, 8, 64), (32, 2, 128)]


def listed():
    return [
        # one interactive user, about a thousand cached tokens: latency
        dict(name="track_single_1k", kind="decode", batch=1, lo=1021, hi=1021, len_seed=1,
             geometry=0, page=16, dtype="fp16"),
        # the headline configuration: 8 sequences of 32768 tokens
        dict(name="track_batch_32k", kind="decode", batch=8, lo=32768, hi=32768, len_seed=3,
             geometry=0, page=16, dtype="fp16"),
        # a busy bf16 server with ragged lengths, head size 64
        dict(name="track_ragged_hd64", kind="decode", batch=48, lo=512, hi=16384, len_seed=4,
             geometry=1, page=16, dtype="bf16"),
        # the same at head size 256, larger pages
        dict(name="track_ragged_hd256", kind="decode", batch=24, lo=1024, hi=16384, len_seed=5,
             geometry=2, page=32, dtype="bf16"),
        # short prompts of odd lengths prefilled together, 32 observed queries each
        dict(name="window_prompts", kind="window", batch=4, chunk_lo=37, chunk_hi=1500, ctx_lo=0,
             ctx_hi=0, window=32, len_seed=11, geometry=0, page=16, dtype="fp16"),
        # one long prompt, 64 observed queries
        dict(name="window_prompt_32k", kind="window", batch=1, chunk_lo=32768, chunk_hi=32768,
             ctx_lo=0, ctx_hi=0, window=64, len_seed=12, geometry=0, page=16, dtype="fp16"),
        # the second chunks of three prompts at head size 64, eight queries
        dict(name="window_chunks_hd64", kind="window", batch=3, chunk_lo=700, chunk_hi=2048,
             ctx_lo=4000, ctx_hi=16000, window=8, len_seed=13, geometry=1, page=16, dtype="bf16"),
        # a server whose sequences are cut back every 16 steps: latency
        dict(name="evict_steps", kind="evict", batch=32, lo=2048, hi=2064, budget=2048, recent=256,
             sink=4, len_seed=21, geometry=0, page=16),
        # prompts of 32768 tokens cut to a quarter right after the prefill
        dict(name="evict_prompts_32k", kind="evict", batch=8, lo=32768, hi=32768, budget=8192,
             recent=1024, sink=4, len_seed=22, geometry=0, page=16),
        # a ragged batch cut to half of its longest, head size 64: some are under the budget
        dict(name="evict_ragged_hd64", kind="evict", batch=48, lo=512, hi=16384, budget=7001,
             recent=500, sink=0, len_seed=23, geometry=1, page=16),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    kind = rng.choice(["decode", "decode", "window", "evict"])
    geometry, page = rng.randrange(len(GEOMETRIES)), rng.choice([16, 16, 16, 32, 48])
    if kind == "window":
        batch = rng.randrange(1, 5)
        window = _log_int(rng, 1, 64)
        hi = _log_int(rng, 1, 16384 // batch)
        ctx = rng.random() < 0.5
        ctx_hi = _log_int(rng, 1, 16384 // batch) if ctx else 0
        return dict(kind=kind, batch=batch, chunk_lo=max(1, hi // rng.choice([1, 3])), chunk_hi=hi,
                    ctx_lo=ctx_hi // rng.choice([1, 4]), ctx_hi=ctx_hi, window=window,
                    len_seed=rng.randrange(1 << 30), geometry=geometry, page=page,
                    dtype=rng.choice(["fp16", "bf16"]))
    batch = _log_int(rng, 1, 48)
    # cached values of all sequences and heads: at most those of the largest listed case
    most = 8 * 32768 * 8 * 128 // (GEOMETRIES[geometry][1] * _pad(GEOMETRIES[geometry][2]))
    hi = _log_int(rng, 1, min(32768, most // (2 * batch)))
    lo = max(1, rng.choice([1, hi // 16, hi // 2, hi]))
    case = dict(kind=kind, batch=batch, lo=lo, hi=hi, len_seed=rng.randrange(1 << 30),
                geometry=geometry, page=page)
    if kind == "decode":
        return dict(case, dtype=rng.choice(["fp16", "bf16"]))
    budget = max(1, int(hi * rng.uniform(0.1, 0.95)))
    sink = min(rng.choice([0, 1, 4]), budget)
    return dict(case, budget=budget, sink=sink, recent=rng.randint(0, (budget - sink) // 2))


# ------------------------------------------------------------------ geometry

def _pad(head):
    return max(64, 1 << (head - 1).bit_length())


def _entry_bytes(pd):
    return (pd // 2 + 2 * (pd // 64) + 15) & ~15


def _lengths(case):
    """(chunk, cached before it) of each sequence; a decode step is a chunk of one token."""
    r = random.Random(case["len_seed"])
    if case["kind"] == "window":
        return [(r.randint(case["chunk_lo"], case["chunk_hi"]),
                 r.randint(case["ctx_lo"], case["ctx_hi"])) for _ in range(case["batch"])]
    return [(1, r.randint(case["lo"], case["hi"]) - 1) for _ in range(case["batch"])]


def work(case):
    hq, hkv, hd = GEOMETRIES[case["geometry"]]
    pd = _pad(hd)
    code = pd // 2 + 2  # bytes of one cached vector that carry information
    lens = _lengths(case)
    total = sum(c + x for c, x in lens)
    pages = sum(-(-(c + x) // case["page"]) for c, x in lens)
    if case["kind"] == "decode":
        known = sum(x for _, x in lens)
        return {"bytes": total * hkv * (2 * code + 4) + known * hkv * 4
                + case["batch"] * (2 * hq * hd * 2 + 4 * hkv + 12) + 4 * pages,
                "flops": 4.0 * total * hq * hd}
    if case["kind"] == "window":
        rows = sum(min(c, case["window"]) for c, _ in lens)
        pairs = sum(min(c, case["window"]) * (c + x) - min(c, case["window"]) *
                    (min(c, case["window"]) - 1) // 2 for c, x in lens)
        known, fresh = sum(x for _, x in lens), sum(c for c, _ in lens)
        return {"bytes": total * hkv * code + known * hkv * 8 + fresh * hkv * 8
                + rows * hq * hd * 2 + 16 * case["batch"] + 4 * pages,
                "flops": 2.0 * pairs * hq * hd}
    over = [c + x for c, x in lens if c + x > case["budget"]]
    moved = 0.0  # kept entries behind the budget: the recent ones, and their share of the others
    for n in over:
        tail = n - case["budget"]
        recent = min(case["recent"], tail)
        free = case["budget"] - case["recent"] - case["sink"]
        others = max(1, n - case["recent"] - case["sink"])
        moved += recent + max(0, tail - recent) * free / others
    return {"bytes": hkv * (8.0 * sum(over) + moved * 2 * (2 * code + 8)) + 16 * case["batch"]
            + 4 * pages, "flops": 8.0 * hkv * sum(over)}


# ------------------------------------------------------------------ inputs

def prepare(case, seed):
    dev = torch.device("cuda:0")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    hq, hkv, hd = GEOMETRIES[case["geometry"]]
    pd, bs = _pad(hd), case["page"]
    ebs = _entry_bytes(pd)
    lens = _lengths(case)
    batch = len(lens)
    longest = max(c + x for c, x in lens)
    width = -(-longest // bs)
    need = [-(-(c + x) // bs) for c, x in lens]
    nb = sum(need) + 3

    def randn(*shape):
        return torch.randn(shape, generator=g, device=dev)

    # a random page permutation; table rows are as wide as the longest sequence
    perm = torch.randperm(nb, generator=g, device=dev).to(torch.int32)
    table = torch.full((batch, width), -1, dtype=torch.int32, device=dev)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = perm[at:at + n]
        at += n
    # codes of Gaussian coordinates, norms of rows of hd coordinates whose
    # scale varies from token to token
    levels = torch.tensor(LEVELS, device=dev)
    bounds = (levels[1:] + levels[:-1]) / 2
    cache = torch.zeros((2, nb, bs, hkv, ebs), dtype=torch.uint8, device=dev)
    for slab in range(2):
        for a in range(0, nb, 4096):
            n = min(4096, nb - a)
            codes = torch.bucketize(randn(n, bs, hkv, pd), bounds).to(torch.uint8)
            cache[slab, a:a + n, ..., :pd // 2] = (codes[..., 0::2] << 4) | codes[..., 1::2]
            norm = (math.sqrt(hd) * (0.25 * randn(n, bs, hkv)).exp()).to(torch.float16)
            cache[slab, a:a + n, ..., pd // 2:pd // 2 + 2 * (pd // 64)] = \
                norm[..., None].repeat(1, 1, 1, pd // 64).view(torch.uint8)
    signs = torch.where(randn(pd) < 0, -1.0, 1.0)
    seq = torch.tensor([c + x for c, x in lens], dtype=torch.int32, device=dev)
    # what earlier steps left: accumulated weight with a few heavy tokens
    acc = randn(nb, hkv, bs).square() * 0.05 + (randn(nb, hkv, bs) > 3.0) * 4.0
    ends = seq + torch.randint(0, 500, (batch,), generator=g, device=dev, dtype=torch.int32)
    pos = torch.full((nb, hkv, bs), -5, dtype=torch.int32, device=dev)
    st = SimpleNamespace(
        kind=case["kind"], cache=cache, weights=acc, positions=pos, table=table,
        indices=table.reshape(-1),
        indptr=torch.arange(batch + 1, dtype=torch.int32, device=dev) * width, seq=seq, ends=ends,
        hq=hq, hkv=hkv, hd=hd, pd=pd, bs=bs, signs=signs, scale=1.0 / math.sqrt(hd),
        levels=levels, lens=lens)
    # sequences that have been cut before: the entries' positions rise with the
    # index, with gaps, up to the newest one
    for b, n in enumerate(need):
        length, end = lens[b][0] + lens[b][1], int(ends[b])
        up = torch.arange(n * bs, device=dev)
        p = torch.where(up < length // 2, up, up + end - length).to(torch.int32)
        pos[table[b, :n].long()] = p.view(n, 1, bs).expand(n, hkv, bs)
    if case["kind"] == "evict":
        # a tenth of the entries never received anything (ties)
        st.weights = torch.where(randn(nb, hkv, bs) < -1.28, torch.zeros_like(acc), acc)
        st.first_weights, st.first_positions = st.weights.clone(), st.positions.clone()
        st.budget, st.recent, st.sink = case["budget"], case["recent"], case["sink"]
        st.new_lens = torch.zeros(batch, dtype=torch.int32, device=dev)
    else:
        rows = [1] * batch if case["kind"] == "decode" else [c for c, _ in lens]
        st.q = (randn(sum(rows), hq, hd) * 2.0).to(DTYPES[case["dtype"]])
        st.starts = torch.tensor([0] + rows, dtype=torch.int32, device=dev).cumsum(0).to(torch.int32)
        st.window = case.get("window", 1)
        st.o = torch.zeros_like(st.q) if case["kind"] == "decode" else None
    return st


# ------------------------------------------------------------------ calls

def run(st):
    if st.kind == "evict":
        # every pass cuts the same sequences: the record starts over
        st.weights.copy_(st.first_weights)
        st.positions.copy_(st.first_positions)
    if own:
        from turboquant_amd import ops
        if st.kind == "decode":
            ops.decode_paged_tracked(st.q, st.cache, st.indices, st.indptr, st.seq, st.hkv, st.hd,
                                     st.pd, st.scale, st.signs, st.o, st.weights, st.positions,
                                     st.ends)
            return {"o": st.o, "weights": st.weights, "positions": st.positions}
        if st.kind == "window":
            ops.track_window(st.q, st.starts, st.window, st.cache, st.indices, st.indptr, st.seq,
                             st.hkv, st.hd, st.pd, st.scale, st.signs, st.weights, st.positions,
                             st.ends)
            return {"weights": st.weights, "positions": st.positions}
        ops.evict_paged(st.cache, st.weights, st.positions, st.indices, st.indptr, st.seq, st.ends,
                        st.budget, st.recent, st.sink, st.new_lens)
        return {"cache": st.cache, "weights": st.weights, "positions": st.positions,
                "lens": st.new_lens}
    if st.kind == "decode":
        o = _plain_decode(st)
        return {"o": o, "weights": st.weights, "positions": st.positions}
    if st.kind == "window":
        _plain_window(st)
        return {"weights": st.weights, "positions": st.positions}
    _plain_evict(st)
    return {"cache": st.cache, "weights": st.weights, "positions": st.positions,
            "lens": st.new_lens}


# ------------------------------------------------------------------ plain forms

def _hadamard(n, device, dtype=torch.float32):
    """H[i, j] = (-1)^popcount(i & j) / sqrt(n), symmetric and its own inverse."""
    i = torch.arange(n, device=device)
    x = i[:, None] & i[None, :]
    for s in (8, 4, 2, 1):
        x = x ^ (x >> s)
    return (1 - 2 * (x & 1)).to(dtype) / math.sqrt(n)


def _slots(st):
    """Entry (page * page size + place) of every token [B, T], and which exist."""
    t = torch.arange(st.table.shape[1] * st.bs, device=st.table.device)
    slot = st.table.long().clamp_min(0)[:, t // st.bs] * st.bs + t % st.bs
    return slot, t[None, :] < st.seq[:, None]


def _read(st, slab, slot):
    """Cached rows [B, H, T, pd] fp32 in the rotated domain."""
    e = st.cache[slab].reshape(-1, st.hkv, st.cache.shape[-1])[slot]
    codes = e[..., :st.pd // 2]
    codes = torch.stack((codes >> 4, codes & 15), dim=-1).flatten(-2)
    norm = e[..., st.pd // 2:st.pd // 2 + 2].contiguous().view(torch.float16).float()
    rows = st.levels[codes.int()] * (norm / math.sqrt(st.pd))
    return rows.permute(0, 2, 1, 3).contiguous()


def _rotate(st, x):
    """x [..., hd] in the rotated domain, fp32 [..., pd]."""
    x = torch.nn.functional.pad(x.float(), (0, st.pd - st.hd))
    return (x * st.signs) @ _hadamard(st.pd, x.device)


def _weights(st, q, mask):
    """Softmax weights fp32 [B, H, R, T] of rows q [B, H, R, pd] over the cached
    keys, mask [B, 1 or R, T] true where a row sees a token; a row that sees
    nothing has zero weights."""
    slot, _ = _slots(st)
    s = (q * st.scale) @ _read(st, 0, slot).transpose(2, 3).contiguous()
    s = torch.where(mask[:, None], s, -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(torch.isinf(top), 0.0, top))
    return p / p.sum(-1, keepdim=True).clamp_min(1e-30)


def _record(st, received, fresh):
    """Adds received [B, H, T] to the accumulators; the last fresh [B] tokens are new."""
    slot, there = _slots(st)
    t = torch.arange(slot.shape[1], device=slot.device)
    new = t[None, :] >= (st.seq - fresh)[:, None]
    head = torch.arange(st.hkv, device=slot.device)[None, :, None]
    where = ((slot // st.bs)[:, None] * st.hkv + head) * st.bs + (slot % st.bs)[:, None]
    there, new = there[:, None].expand(where.shape), new[:, None].expand(where.shape)
    acc, pos = st.weights.view(-1), st.positions.view(-1)
    at = where[there]
    acc[at] = torch.where(new[there], 0.0, acc[at]) + received[there]
    born = (st.ends - st.seq)[:, None, None] + t[None, None, :]
    pos[at] = torch.where(new, born, -1)[there].to(torch.int32) * new[there] \
        + pos[at] * ~new[there]


def _plain_decode(st):
    slot, there = _slots(st)
    b, r = st.seq.numel(), st.hq // st.hkv
    q = _rotate(st, st.q).view(b, st.hkv, r, st.pd)
    p = _weights(st, q, there[:, None])
    o = (p @ _read(st, 1, slot)).reshape(b, st.hq, st.pd)
    o = (o @ _hadamard(st.pd, o.device)) * st.signs
    _record(st, p.sum(2), torch.ones_like(st.seq))
    return o[..., :st.hd].to(st.q.dtype)


def _plain_window(st):
    b, r, w = st.seq.numel(), st.hq // st.hkv, st.window
    fresh = st.starts[1:] - st.starts[:-1]
    i = torch.arange(w, device=st.q.device)
    row = st.starts[1:, None] - w + i  # the last w rows of each chunk
    valid = i[None, :] >= (w - fresh)[:, None]
    q = _rotate(st, st.q[row.clamp_min(0)]).view(b, w, st.hkv, r, st.pd).transpose(1, 2)
    t = torch.arange(st.table.shape[1] * st.bs, device=st.q.device)
    mask = (t[None, None, :] <= (st.seq[:, None] - w + i)[:, :, None]) & valid[:, :, None]
    p = _weights(st, q.reshape(b, st.hkv, w * r, st.pd), mask.repeat_interleave(r, dim=1))
    _record(st, p.sum(2), fresh)


def _plain_evict(st):
    slot, there = _slots(st)
    t = torch.arange(slot.shape[1], device=slot.device)
    head = torch.arange(st.hkv, device=slot.device)[None, :, None]
    where = ((slot // st.bs)[:, None] * st.hkv + head) * st.bs + (slot % st.bs)[:, None]
    acc, pos = st.weights.view(-1), st.positions.view(-1)
    w, p = acc[where], pos[where]
    held = (p < st.sink) | (p >= (st.ends - st.recent)[:, None, None])
    key = torch.where(held, math.inf, w)
    key = torch.where(there[:, None], key, -math.inf)
    order = key.argsort(dim=-1, descending=True, stable=True)
    keep = torch.zeros_like(there[:, None].expand(key.shape)).scatter(
        -1, order, (t < st.budget).expand(order.shape)) & there[:, None]
    full = (st.seq > st.budget)[:, None, None]
    hole = ~keep & (t < st.budget) & full
    more = keep & (t >= st.budget) & full
    # masks list their places in the order of the index, and hold as many each
    # in every row: i-th to i-th
    to, of = where[hole], where[more]
    acc[to], pos[to] = acc[of], pos[of]
    e = st.cache.view(2, -1, st.hkv, st.cache.shape[-1])
    h = head.expand(where.shape)
    s = slot[:, None].expand(where.shape)
    e[:, s[hole], h[hole]] = e[:, s[more], h[more]]
    st.new_lens.copy_(st.seq.clamp_max(st.budget))


# ------------------------------------------------------------------ in 64 bits

def exact(case, seed):
    """The definition, sequence by sequence in 64 bits; keys and values in the
    original domain."""
    st = prepare(case, seed)
    lens = [c + x for c, x in st.lens]
    acc = st.weights.double()
    pos = st.positions.clone()
    if case["kind"] == "evict":
        return _exact_evict(st, lens)
    # rows of the inverse rotation: c -> (c H) * signs
    back = _hadamard(st.pd, st.q.device, torch.float64) * st.signs.double()
    levels = torch.tensor(LEVELS, dtype=torch.float32, device=st.q.device).double()
    r = st.hq // st.hkv
    out = []
    for b, n in enumerate(lens):
        pages = st.table[b, :-(-n // st.bs)].long()
        c = st.lens[b][0]
        w = min(c, st.window)
        end = int(st.starts[b + 1])
        o = torch.zeros((st.hq, st.pd), dtype=torch.float64, device=st.q.device)
        for h in range(st.hkv):
            def rows(slab):
                e = st.cache[slab, pages, :, h].reshape(-1, st.cache.shape[-1])[:n]
                hi, lo = e[:, :st.pd // 2] // 16, e[:, :st.pd // 2] % 16
                x = torch.stack((levels[hi.int()], levels[lo.int()]), 2).view(n, st.pd)
                norm = e[:, st.pd // 2:st.pd // 2 + 2].contiguous().view(torch.float16).double()
                return (x * norm / math.sqrt(st.pd)) @ back
            k = rows(0)[:, :st.hd].contiguous()
            q = st.q[end - w:end, h * r:(h + 1) * r].double().reshape(w * r, st.hd)
            s = (q @ k.T) * st.scale
            if w > 1:
                i = torch.arange(w, device=s.device).repeat_interleave(r)
                t = torch.arange(n, device=s.device)
                s = s.masked_fill(t[None, :] > (n - w + i)[:, None], -math.inf)
            p = s.softmax(-1)
            got = torch.zeros(len(pages) * st.bs, dtype=torch.float64, device=s.device)
            got[:n] = p.sum(0)
            old = acc[pages, h].reshape(-1)
            t = torch.arange(len(old), device=s.device)
            acc[pages, h] = torch.where(t < n - c, old + got, torch.where(t < n, got, old)) \
                .view(len(pages), st.bs)
            was = pos[pages, h].reshape(-1)
            born = (t + int(st.ends[b]) - n).to(torch.int32)
            pos[pages, h] = torch.where((t >= n - c) & (t < n), born, was).view(len(pages), st.bs)
            if case["kind"] == "decode":
                o[h * r:(h + 1) * r] = p @ rows(1)
        out.append(o[:, :st.hd])
    if case["kind"] == "decode":
        return {"o": torch.stack(out), "weights": acc, "positions": pos}
    return {"weights": acc, "positions": pos}


def _exact_evict(st, lens):
    cache = st.cache.cpu().numpy().copy()
    acc, pos = st.weights.cpu().numpy().astype(np.float64), st.positions.cpu().numpy().copy()
    table, ends = st.table.cpu().numpy(), st.ends.cpu().numpy()
    new = []
    for b, n in enumerate(lens):
        new.append(min(n, st.budget))
        if n <= st.budget:
            continue
        t = np.arange(n)
        page, place = table[b, t // st.bs], t % st.bs
        for h in range(st.hkv):
            w, p = acc[page, h, place], pos[page, h, place]
            held = (p < st.sink) | (p >= ends[b] - st.recent)
            keep = np.zeros(n, bool)
            keep[np.lexsort((t, -w, ~held))[:st.budget]] = True
            to, of = np.flatnonzero(~keep[:st.budget]), st.budget + np.flatnonzero(keep[st.budget:])
            acc[page[to], h, place[to]] = acc[page[of], h, place[of]]
            pos[page[to], h, place[to]] = pos[page[of], h, place[of]]
            for slab in cache:
                slab[page[to], place[to], h] = slab[page[of], place[of], h]
    return {"cache": cache, "weights": acc, "positions": pos, "lens": np.array(new, np.int32)}
