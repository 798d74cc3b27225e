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
