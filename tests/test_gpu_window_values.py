"""Windowed attention on an MI355X where values in sight or out of it are not
finite, against the formulas in 64 bits."""
from __future__ import annotations

import math

import pytest
import torch

from test_gpu_window_prefill import DEV, call, check, make

pytestmark = pytest.mark.gpu


def scores_of_minus_infinity(q, k, keys):
    """Every query's score with the given keys: an infinite coordinate times a
    negative one."""
    q[..., 2] = -(q[..., 2].abs() + 0.1)
    k[keys, :, 2] = math.inf


@pytest.mark.parametrize("hq,hkv,hd,n,ctx,window,sink", [
    (2, 1, 128, 300, 200, 100, 1), (32, 8, 128, 4000, 100, 1000, 1),
    (32, 8, 64, 4100, 64, 513, 2), (2, 1, 256, 40, 9000, 5000, 1),    # (keys split)
    (4, 2, 128, 100, 20000, 19000, 1), (3, 3, 96, 150, 130, 20, 0), (1, 1, 64, 21000, 5, 4000, 3)])
def test_prefill_hidden_values_beside_scores_of_minus_infinity(hq, hkv, hd, n, ctx, window, sink):
    """A hidden key whose value is not finite leaves a row as it is, also where the
    first keys that the row sees, the sinks or those at the window's edge, score
    -inf and so weigh nothing."""
    q, k, v, reqs = make(n + 3, [(n, n + ctx)], hq, hkv, hd)
    lk = n + ctx
    scores_of_minus_infinity(q, k, list(range(sink)) + list(range(63, lk, 64)))
    for x, j in ((math.nan, 40), (math.inf, lk - n // 2 - 1), (math.nan, lk - n // 3)):
        v[j, 0, 3] = x
    o = call(q, k, v, reqs, hd, window, sink)
    check(o, q, k, v, reqs, window, sink, 1 / math.sqrt(hd), hd)
    assert torch.isnan(o[:, 0, 3]).any() and torch.isfinite(o[:, 0, 4]).all()
