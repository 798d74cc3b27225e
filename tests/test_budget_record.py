"""CacheRecord's page-table starts: complete for any stream, and not growing."""
from __future__ import annotations

import pytest
import torch

from turboquant_amd import budget
from turboquant_amd.budget import CacheRecord


def record(device="cpu"):
    return CacheRecord(4, 16, 2, budget=8, device=device)


def held(r):
    """Elements of the tensors that a record keeps beside its state."""
    seen, todo = {}, [v for k, v in vars(r).items() if k not in ("weights", "positions")]
    while todo:
        x = todo.pop()
        if isinstance(x, torch.Tensor):
            st = x.untyped_storage()
            seen[st.data_ptr()] = st.nbytes()
        elif isinstance(x, dict):
            todo += list(x.values())
        elif isinstance(x, (tuple, list)):
            todo += list(x)
    return sum(seen.values())


def test_starts_are_the_rows_of_the_table():
    r = record()
    for b, width in ((2, 3), (1, 3), (5, 3), (5, 7), (0, 4), (3, 0), (2000, 2), (2, 3)):
        table = torch.arange(b * width, dtype=torch.int32).view(b, width)
        indices, indptr = r._tables(table)
        assert torch.equal(indices, table.reshape(-1)) and indptr.dtype == torch.int32
        assert indptr.tolist() == [i * width for i in range(b + 1)]


def test_starts_do_not_grow_with_the_shapes():
    r = record()
    for b in range(1, 1024, 3):
        r._tables(torch.zeros((b, 5), dtype=torch.int32))
    one = held(r)
    assert one <= 4 * 1025
    for width in range(1, 500):
        indptr = r._tables(torch.zeros((3, width), dtype=torch.int32))[1]
        assert indptr.tolist() == [0, width, 2 * width, 3 * width]
    assert held(r) <= budget.STARTS_KEPT * 4 * 1025


@pytest.mark.gpu
def test_starts_are_there_for_another_stream():
    """The first call runs on a stream with much work in front of it; what a second
    stream gets at once is complete."""
    dev = torch.device("cuda:0")
    busy = torch.randn((4096, 4096), device=dev)
    table = torch.zeros((500, 77), dtype=torch.int32, device=dev)
    want = torch.arange(501, dtype=torch.int32, device=dev) * 77
    first, second = torch.cuda.Stream(), torch.cuda.Stream()
    r = record(dev)
    torch.cuda.synchronize()
    with torch.cuda.stream(first):
        for _ in range(50):
            busy = busy @ busy * 1e-2
        r._tables(table)
    with torch.cuda.stream(second):
        got = r._tables(table)[1].clone()
    second.synchronize()
    assert torch.equal(got, want)
    torch.cuda.synchronize()


@pytest.mark.gpu
def test_starts_inside_a_capture_belong_to_it():
    """A width first met inside a capture leaves nothing behind; a known one is used
    as it is."""
    dev = torch.device("cuda:0")
    r = record(dev)
    known, fresh = (torch.zeros((4, w), dtype=torch.int32, device=dev) for w in (6, 9))
    r._tables(known)
    before = held(r)
    out = torch.zeros((2, 5), dtype=torch.int32, device=dev)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out[0].copy_(r._tables(known)[1])
        out[1].copy_(r._tables(fresh)[1])
    assert held(r) == before
    for _ in range(3):
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert out.tolist() == [[0, 6, 12, 18, 24], [0, 9, 18, 27, 36]]
    assert r._tables(fresh)[1].tolist() == [0, 9, 18, 27, 36]


class _Meta:
    def __init__(self, **kw):
        self.__dict__.update(kw)


@pytest.mark.parametrize("most", [1, 5])
@pytest.mark.parametrize("missing", ["kv_cache", "seq_lens", "packed"])
def test_a_batch_that_cannot_be_recorded_is_refused(missing, most):
    from turboquant_amd.vllm_backend_fused import TurboQuantFusedImpl
    impl = TurboQuantFusedImpl(4, 64, 0.125, 2, None, None,
                               "auto" if missing == "packed" else "fp8")
    cache = torch.zeros((2, 4, 16, 2, 48), dtype=torch.uint8)
    impl.record = CacheRecord.beside(cache, 8)
    n = 2 * most
    q, kv = torch.zeros((n, 256)), torch.zeros((n, 128))
    meta = _Meta(max_query_len=most, num_actual_tokens=n,
                 block_table=torch.zeros((2, 2), dtype=torch.int32),
                 seq_lens=None if missing == "seq_lens" else torch.full((2,), most, dtype=torch.int32),
                 query_start_loc=torch.tensor([0, most, n], dtype=torch.int32), slot_mapping=None)
    with pytest.raises(RuntimeError, match="cache record needs"):
        impl.forward(None, q, kv, kv, None if missing == "kv_cache" else cache, meta)
    # without metadata nothing is cached (a profiling pass): nothing to record
    assert torch.equal(impl.forward(None, q, kv, kv, None, None), torch.zeros_like(q))


def test_starts_of_a_traced_call_are_not_kept():
    """A call over fake tensors leaves nothing that a later call would get, and gets
    nothing of an earlier one."""
    from torch._subclasses.fake_tensor import FakeTensor, FakeTensorMode
    r, table = record(), torch.zeros((3, 7), dtype=torch.int32)
    for _ in range(2):
        with FakeTensorMode():
            fake = r._tables(torch.empty((3, 7), dtype=torch.int32))[1]
        assert isinstance(fake, FakeTensor) and fake.shape == (4,)
        starts = r._tables(table)[1]
        assert type(starts) is torch.Tensor and starts.tolist() == [0, 7, 14, 21]


def test_starts_are_made_on_the_host_whatever_the_default_device():
    """(a default device of "cuda" would make them on the current stream, which
    another stream's first call does not wait for; "meta" shows it without a GPU)"""
    r, table = record(), torch.zeros((3, 7), dtype=torch.int32)
    with torch.device("meta"):
        starts = r._tables(table)[1]
    assert starts.device == table.device and starts.tolist() == [0, 7, 14, 21]
