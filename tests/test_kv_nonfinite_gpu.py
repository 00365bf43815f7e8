"""Attention over the paged 4-bit cache where value scales are infinite or NaN at tokens that some rows of a tile see and
others, in the same tile, do not: those rows' results are what they are without, in either kernel."""

import pytest
import torch

from tests.kv_q4_ref import State, attention, dense_request
from tests.test_kv_cache_gpu import starts
from torchnative_b200 import _native as N
from torchnative_b200 import kv_cache as kv

pytestmark = pytest.mark.gpu

BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize("most, dtype", [(None, BF), (1, BF), (1, F16), (1, F32)])
@pytest.mark.parametrize("heads, kv_heads, dim, page_size, new, lengths", [
    (32, 4, 128, 64, [800], [900]), (9, 3, 64, 16, [1000, 0, 700], [1300, 5, 690]), (16, 16, 128, 128, [129, 700], [129, 1001])])
def test_values_that_are_not_finite_reach_only_rows_that_see_them(cuda_device, heads, kv_heads, dim, page_size, new, lengths,
                                                                  most, dtype):
    st = State(lengths, kv_heads, dim, page_size, cuda_device, seed=dim)
    q = st.randn(sum(new), heads, dim, dtype=dtype)
    start = starts(new, cuda_device)
    b = max(range(len(new)), key=lambda i: new[i])
    n, length = new[b], lengths[b]
    # one inside the first tiles that rows differ in, one at a tile's end, two close to the last token; three kinds: every
    # element's float16 scale overflows; one infinite element; a scale that is NaN
    at = sorted({max(length - n, 0) + 5, max(length - n, 0) // 64 * 64 + 127, length - 70, length - 2})
    before = st.pool.clone()
    for i, pos in enumerate(at):
        slot = st.table[b, pos // page_size].long() * page_size + pos % page_size
        k = torch.zeros((1, kv_heads, dim), device=cuda_device)
        v = torch.zeros((1, kv_heads, dim), device=cuda_device)
        block = slice(32 * (i % (dim // 32)), 32 * (i % (dim // 32)) + 32)
        kv.kv_q4_append(k, v, before, slot[None])
        v[:, :, block] = 6e5 * torch.tensor([1.0, -1.0] * 16, device=cuda_device)
        if i == 1:
            v[:, 0, block] = 1.0
            v[:, 0, block.start + 3] = -float("inf")
        kv.kv_q4_append(k, v, st.pool, slot[None])
        if i == 2:
            scale = 17 * dim + (pos % 16 * (dim // 32) + block.start // 32) * 2
            st.pool[st.table[b, pos // page_size].long(), -1, pos % page_size // 16, scale:scale + 2] = torch.tensor(
                [0x01, 0x7e], dtype=torch.uint8, device=cuda_device)
    got, lse = kv.sdpa_q4_cache(q, st.pool, st.table, st.lengths, query_start=start, max_tokens=most)
    N.device_status()
    tiles = most is None
    # `before` has zeros where they are: what every result is without them
    want, want_lse, bound, lse_bound = attention(q, before, st.table, st.lengths, page_size, start, tiles=tiles)
    got, lse = got.double().cpu(), lse.double().cpu()
    rows = ~want_lse.isnan().any(-1)
    assert ((lse - want_lse).abs() <= lse_bound)[rows].all()
    # what the tokens that a row sees add: an infinity of its sign, or NaN, in the elements of their blocks
    v = dense_request(st.pool, st.table[b], length, page_size)[1].cpu().repeat_interleave(heads // kv_heads, 0)
    first = int(start[b])
    add = torch.zeros_like(want)
    for pos in at:
        odd = torch.where(torch.isfinite(v[:, pos]), 0.0, v[:, pos])  # [heads, D]
        seen = first + max(0, pos - (length - n))
        add[seen:first + n] += odd
    hit = ~torch.isfinite(add) & rows[:, None, None]
    assert hit.any() and ((got - want).abs() <= bound)[rows[:, None, None] & ~hit].all()
    if dtype == BF:
        assert torch.equal(got[hit].nan_to_num(3.0, 1.0, -1.0), add[hit].nan_to_num(3.0, 1.0, -1.0))
    else:
        assert not torch.isfinite(got[hit]).any()  # a probability's two terms: an infinity less itself
