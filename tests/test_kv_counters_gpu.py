"""Launch counters of attention over the paged cache: a call counts once, under the kernel that it took."""

import pytest
import torch

from tests.kv_q4_ref import State
from tests.test_kv_cache_gpu import rope_table, starts
from torchnative_b200 import _native as N
from torchnative_b200 import kv_cache as kv

pytestmark = pytest.mark.gpu


def test_a_call_counts_as_the_kernel_that_it_took(cuda_device):
    st = State([900], 4, 128, 64, cuda_device)
    q = st.randn(800, 32, 128, dtype=torch.bfloat16)
    start = starts([800], cuda_device)
    qkv, rope = st.randn(1, 40 * 128, dtype=torch.bfloat16), rope_table(900, 128, cuda_device)
    for call, tiles in ((lambda: kv.sdpa_q4_cache(q, st.pool, st.table, st.lengths, query_start=start), 1),
                        (lambda: kv.sdpa_q4_cache(q[:1], st.pool, st.table, st.lengths), 0),
                        (lambda: kv.sdpa_q4_decode_step(qkv, rope, st.pool, st.table, st.lengths, 32), 0)):
        before = N.counters()
        call()
        after = N.counters()
        got = [after[k] - before[k] for k in ("sdpa_calls", "sdpa_prefill_launches", "sdpa_decode_launches")]
        assert got == [1, tiles, 1 - tiles]
