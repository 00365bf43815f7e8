"""The paged cache's calls and PyTorch's modes: what a call under a dispatch mode, in a capture or in inference mode
leaves behind does not reach the calls after it."""

import warnings

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from tests.kv_q4_ref import State
from tests.test_kv_cache_gpu import rope_table
from torchnative_b200 import _native as N
from torchnative_b200 import kv_cache as kv

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


def calls(st, q, qkv, rope):
    """Every call that allocates, on copies of what it changes."""
    table, lengths = st.table.clone(), st.lengths.clone()
    pages = st.pool.shape[0]  # the table's ids are of these
    free, count, status = (torch.arange(pages, dtype=torch.int32, device=q.device), torch.full_like(lengths[:1], 9),
                           torch.zeros_like(lengths[:1]))
    attend = kv.sdpa_q4_cache(q, st.pool, st.table, st.lengths)
    step = kv.sdpa_q4_decode_step(qkv, rope, st.pool.clone(), st.table, st.lengths, q.shape[1])
    return (*attend, step, *kv.kv_pages_resize(table, lengths, free, count, status, 16, 5, grow=1))


@pytest.mark.parametrize("heads, kv_heads, dim", [(6, 2, 64), (5, 1, 128)])
def test_fake_tensors_are_refused_and_forgotten(cuda_device, heads, kv_heads, dim):
    st = State([33, 7, 90], kv_heads, dim, 16, cuda_device, seed=heads)
    q, qkv = st.randn(3, heads, dim, dtype=BF), st.randn(3, (heads + 2 * kv_heads) * dim, dtype=BF)
    rope = rope_table(99, dim, cuda_device)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # a stream without scratch of its own yet
        mode = FakeTensorMode()
        fake = [mode.from_tensor(x) for x in (q, st.pool, st.table, st.lengths, qkv, rope)]
        i32 = dict(dtype=torch.int32, device=cuda_device)
        with warnings.catch_warnings():
            warnings.simplefilter("ignore")  # torch's own about data_ptr() of fake tensors
            with mode:
                with pytest.raises(RuntimeError):
                    kv.sdpa_q4_cache(*fake[:4])
                with pytest.raises(RuntimeError):
                    kv.sdpa_q4_decode_step(fake[4], fake[5], *fake[1:4], heads)
                with pytest.raises(RuntimeError):
                    kv.kv_pages_resize(fake[2], fake[3], torch.empty(9, **i32), torch.empty(1, **i32), torch.empty(1, **i32),
                                       16, 5, grow=1)
            with pytest.raises(RuntimeError, match="granted"):
                kv.sdpa_q4_decode_step(qkv, rope, st.pool, st.table, st.lengths, heads, granted=fake[3])
        got = calls(st, q, qkv, rope)
        assert all(type(x) is torch.Tensor and x.data_ptr() for x in got)
    torch.cuda.synchronize()
    want = calls(st, q, qkv, rope)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    N.device_status()


def test_a_first_call_in_a_capture_or_in_inference_mode(cuda_device):
    """Shapes that are met there first: the graph's memory is the graph's alone, and later results are ordinary tensors."""
    st = State([33, 7, 90, 5], 3, 64, 16, cuda_device)
    q, qkv = st.randn(4, 21, 64, dtype=BF), st.randn(4, 27 * 64, dtype=BF)
    rope = rope_table(99, 64, cuda_device)
    with torch.inference_mode():
        calls(st, q, qkv, rope)
    out = kv.sdpa_q4_cache(q, st.pool, st.table, st.lengths)
    assert not any(x.is_inference() for x in out)
    torch.cuda.synchronize()
    q = st.randn(4, 15, 64, dtype=BF)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        kv.sdpa_q4_cache(st.randn(4, 3, 64, dtype=BF), st.pool, st.table, st.lengths)
    torch.cuda.synchronize()
    before = torch.cuda.memory_stats()["reserved_bytes.all.current"]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        captured = kv.sdpa_q4_cache(q, st.pool, st.table, st.lengths)
    graph.replay()
    got = [x.clone() for x in captured]
    want = kv.sdpa_q4_cache(q, st.pool, st.table, st.lengths)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    del captured
    graph.reset()
    del graph
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    assert torch.cuda.memory_stats()["reserved_bytes.all.current"] <= before  # no block of the graph's pool is held
    N.device_status()
