"""The paged 4-bit KV cache on a B200: each operator against plain 64-bit arithmetic, a run of them together, graphs,
streams, and device data that is out of range."""

import random

import pytest
import torch

from tests.kv_q4_ref import State, attention, check_attention, resize
from torchnative_b200 import _native as N
from torchnative_b200 import kv_cache as kv
from torchnative_b200 import quant

pytestmark = pytest.mark.gpu

BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def starts(new, device):
    return torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], dtype=torch.int32, device=device)


# ---- pages


def as_lists(cache):
    return (cache.page_table.tolist(), cache.lengths.tolist(), cache.free_pages.tolist(), cache.free_count.item())


@pytest.mark.parametrize("requests, page_size, seed", [(1, 16, 0), (3, 64, 1), (33, 32, 2), (700, 16, 3), (1025, 128, 4),
                                                       (2600, 16, 5), (5000, 32, 6)])
def test_resize_matches_plain(cuda_device, requests, page_size, seed):
    rng = random.Random(seed)
    width = 5
    cache = kv.PagedQ4Cache(1, 1, 64, requests * 3 + 2, requests, width, page_size, cuda_device)
    for turn in range(6):
        old = as_lists(cache)
        if turn == 4:
            grow = rng.randint(1, 3)
            new = [n + grow if n else 0 for n in old[1]]
            new = [min(n, width * page_size) for n in new]
            if any(n + grow > width * page_size for n in old[1]):
                grow = 0
                new = list(old[1])
        else:
            new = [rng.choice([0, o, min(o + rng.randint(0, 2 * page_size), width * page_size),
                               rng.randint(0, 2 * page_size + 1)]) for o in old[1]]
        tokens = sum(max(0, n - o) for o, n in zip(old[1], new)) + turn
        if turn == 4:
            got = cache.resize(tokens, grow=grow)
        else:
            got = cache.resize(tokens, new_lengths=torch.tensor(new, dtype=torch.int32, device=cuda_device))
        want = resize(*old, new, page_size, tokens)
        assert as_lists(cache) == (want[0], want[1], want[2], want[3])
        assert tuple(x.tolist() for x in got) == (want[4], want[5], want[6])
        assert cache.status.item() == want[7]
        cache.status.zero_()


def test_resize_rolls_back(cuda_device):
    cache = kv.PagedQ4Cache(1, 1, 64, 40, 4, 12, 16, cuda_device)
    first = torch.tensor([5, 0, 64, 17], dtype=torch.int32, device=cuda_device)
    cache.resize(100, new_lengths=first)
    before = as_lists(cache)[:2], cache.free_pages[:cache.free_count.item()].tolist()
    cache.resize(200, new_lengths=torch.tensor([50, 33, 64, 100], dtype=torch.int32, device=cuda_device))
    cache.resize(0, new_lengths=first)
    assert (as_lists(cache)[:2], cache.free_pages[:cache.free_count.item()].tolist()) == before
    cache.check()


@pytest.mark.parametrize("new, tokens, code", [([200, 5, 0], 400, 1), ([-1, 0, 0], 10, 2), ([16 * 20 + 1, 0, 0], 400, 2),
                                               ([30, 30, 0], 59 - 20, 3)])
def test_resize_that_cannot_be_met_changes_nothing(cuda_device, new, tokens, code):
    cache = kv.PagedQ4Cache(1, 1, 64, 9, 3, 20, 16, cuda_device)
    cache.resize(64, new_lengths=torch.tensor([20, 0, 16], dtype=torch.int32, device=cuda_device))
    before = as_lists(cache)
    slots, positions, start = cache.resize(tokens, new_lengths=torch.tensor(new, dtype=torch.int32, device=cuda_device))
    assert as_lists(cache) == before
    assert (slots == -1).all() and (positions == -1).all() and (start == 0).all()
    with pytest.raises(RuntimeError, match="kv_pages_resize"):
        cache.check()
    assert cache.status.item() == 0
    cache.resize(64, grow=1)  # and the next one goes on
    assert cache.lengths.tolist() == [21, 0, 17]
    cache.check()


@pytest.mark.parametrize("requests, width", [(3, 6000), (40, 500), (700, 24)])
def test_resize_of_wide_tables(cuda_device, requests, width):
    """Tables in which more pages may move than one CTA moves: long prompts in, some out, one that is refused, back."""
    rng = random.Random(requests)
    cache = kv.PagedQ4Cache(1, 1, 64, requests * width // 2, requests, width, 16, cuda_device)
    lengths = [rng.randint(0, width * 12) for _ in range(requests)]
    if requests == 3:
        lengths = [width * 15 + 3, 17, width * 7]
    for new, code in ((lengths, 0), ([0 if i % 3 == 0 else n // (1 + i % 2) for i, n in enumerate(lengths)], 0),
                      ([width * 16] * requests, 1), ([width * 16 + 1] * requests, 2), (lengths, 0), ([0] * requests, 0)):
        old = as_lists(cache)
        tokens = sum(max(0, n - o) for o, n in zip(old[1], new)) + 5
        got = cache.resize(tokens, new_lengths=torch.tensor(new, dtype=torch.int32, device=cuda_device))
        want = resize(*old, new, 16, tokens)
        assert want[7] == code
        assert as_lists(cache) == (want[0], want[1], want[2], want[3])
        assert tuple(x.tolist() for x in got) == (want[4], want[5], want[6])
        assert cache.status.item() == code
        cache.status.zero_()


def test_resize_refuses_a_corrupt_stack(cuda_device):
    cache = kv.PagedQ4Cache(1, 1, 64, 4, 2, 4, 16, cuda_device)
    cache.resize(32, new_lengths=torch.tensor([16, 16], dtype=torch.int32, device=cuda_device))
    cache.free_count.fill_(4)
    cache.resize(0, new_lengths=torch.tensor([0, 0], dtype=torch.int32, device=cuda_device))
    assert cache.status.item() == 4 and cache.lengths.tolist() == [16, 16]


# ---- append


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("tokens, heads, dim, page_size", [(1, 1, 64, 16), (1, 8, 128, 64), (37, 3, 64, 32),
                                                           (200, 2, 128, 16), (1003, 3, 128, 1024)])
def test_append_is_the_q4_0_quantiser(cuda_device, dtype, tokens, heads, dim, page_size):
    st = State([0], heads, dim, page_size, cuda_device, spare=-(-2 * tokens // page_size) + 1)
    pool = torch.randint(0, 256, st.pool.shape, generator=st.g, dtype=torch.uint8).to(cuda_device)
    before = pool.clone()
    x = [st.randn(tokens, heads, dim, dtype=dtype) for _ in range(2)]
    for t in x:  # ties of magnitude, an all-zero block, a block of one sign, large and tiny blocks
        t[0, 0, :32] = 0
        t[-1, -1, 32:64] = torch.tensor([1.5, -1.5] * 16, dtype=dtype)
        t[tokens // 2, 0, 32:64] = t[tokens // 2, 0, 32:64].abs() * 1000
        t[tokens // 3, -1, :32] *= 2.0**-12
    slots = torch.randperm(pool.shape[0] * page_size, generator=st.g)[:tokens].to(cuda_device)
    skipped = torch.arange(tokens, device=cuda_device) % 5 == 4
    kv.kv_q4_append(x[0], x[1], pool, torch.where(skipped, -1, slots))
    N.device_status()
    for got, want in zip(kv.kv_q4_dense(pool), x):
        want = quant._dequantize(quant._quantize(want.float().reshape(-1, dim))).view(tokens, heads, dim)
        got = got.transpose(1, 2).reshape(-1, heads, dim)[slots]
        assert torch.equal(got[~skipped], want[~skipped])
    # every other slot's bytes are as they were
    live = slots[~skipped]
    again = pool.clone()
    for p, g in {(int(s) // page_size, int(s) % page_size // 16) for s in live}:
        again[p, :, g] = before[p, :, g]
    assert torch.equal(again, before)
    old, new = (torch.stack(kv.kv_q4_dense(p)).transpose(2, 3).reshape(2, -1, heads, dim) for p in (before, pool))
    others = torch.ones(old.shape[1], dtype=torch.bool, device=cuda_device)
    others[live] = False
    assert torch.equal(old[:, others].nan_to_num(7.0), new[:, others].nan_to_num(7.0))


def test_append_reads_strided_rows(cuda_device):
    """Keys and values as slices of a projection's rows, and rows that the kernel cannot read in place."""
    st = State([0], 2, 64, 16, cuda_device, spare=4)
    rows = st.randn(9, 8 * 64, dtype=BF).unflatten(1, (8, 64))
    odd = st.randn(9, 2, 65, dtype=BF)[..., 1:]
    turned = st.randn(9, 64, 2, dtype=BF).transpose(1, 2)
    slots = torch.arange(9, device=cuda_device) * 3
    for k, v in ((rows[:, 4:6], rows[:, 6:8]), (odd, turned)):
        a, b = st.pool.clone(), st.pool.clone()
        kv.kv_q4_append(k, v, a, slots)
        kv.kv_q4_append(k.contiguous(), v.contiguous(), b, slots)
        assert torch.equal(a, b)


def test_append_of_specials_is_the_codec(cuda_device):
    st = State([0], 1, 64, 16, cuda_device, spare=1)
    x = st.randn(6, 1, 64)
    x[0, 0, 3], x[1, 0, 40], x[2, 0, 0], x[3, 0, 31] = float("inf"), float("-inf"), float("nan"), 3e38
    x[4] = 1e-42
    x[5, 0, :32] = float("nan")
    kv.kv_q4_append(x, x, st.pool, torch.arange(6, device=cuda_device))
    want = quant._dequantize(quant._quantize(x.reshape(6, 64)))
    for got in kv.kv_q4_dense(st.pool):
        assert torch.equal(got[0, 0, :6].nan_to_num(5.0), want.nan_to_num(5.0))


def test_append_skips_slots_outside_the_pool(cuda_device):
    st = State([0], 2, 64, 16, cuda_device, spare=2)
    before = st.pool.clone()
    x = st.randn(3, 2, 64)
    kv.kv_q4_append(x, x, st.pool, torch.tensor([32, 1 << 40, -(1 << 40)], device=cuda_device))
    with pytest.raises(RuntimeError, match="slot"):
        N.device_status()
    assert torch.equal(st.pool, before)
    N.device_status()


# ---- attention


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("heads, kv_heads, dim", [(4, 4, 64), (9, 3, 64), (8, 2, 128), (16, 2, 128), (7, 1, 128),
                                                  (12, 1, 64), (20, 1, 128)])
@pytest.mark.parametrize("page_size", [16, 64])
def test_decode_attention(cuda_device, dtype, heads, kv_heads, dim, page_size):
    lengths = [1, 0, 15, 16, 17, 63, 64, 65, 200, 1000]
    st = State(lengths, kv_heads, dim, page_size, cuda_device, seed=heads)
    q = st.randn(len(lengths), heads, dim, dtype=dtype)
    got = kv.sdpa_q4_cache(q, st.pool, st.table, st.lengths)
    N.device_status()
    check_attention(got, q, st.pool, st.table, st.lengths, page_size)
    assert (got[0][1] == 0).all() and (got[1][1] == 0).all()


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("batch, length, heads, kv_heads, dim", [(1, 2048, 8, 2, 128), (1, 20000, 4, 1, 128),
                                                                 (2, 5000, 6, 2, 64), (1, 131, 32, 8, 128),
                                                                 (3, 4097, 9, 3, 64)])
def test_long_decode_attention(cuda_device, dtype, batch, length, heads, kv_heads, dim):
    lengths = [length - 7 * i for i in range(batch)]
    st = State(lengths, kv_heads, dim, 64, cuda_device, seed=length)
    q = st.randn(batch, heads, dim, dtype=dtype)
    got = kv.sdpa_q4_cache(q, st.pool, st.table, st.lengths, scale=0.3)
    N.device_status()
    check_attention(got, q, st.pool, st.table, st.lengths, 64, scale=0.3)


@pytest.mark.parametrize("dim", [64, 128])
def test_float32_sums_over_many_keys(cuda_device, dim):
    """The error of float32 results on the whole, where a warp sums some hundred groups of keys. A probability is off by
    2^-21 (its score, exponential and two terms, each 2^-22 or less and random from key to key), which is as much of the
    result; a group's sum by two roundings, the sum over a hundred groups by sqrt(100) 2^-25, the join of twelve warps by
    2^-23: 2^-20 together."""
    st = State([20000], 2, dim, 64, cuda_device, seed=dim)
    q = st.randn(128, 8, dim)
    start = starts([128], cuda_device)
    out, lse = (x.double().cpu() for x in kv.sdpa_q4_cache(q, st.pool, st.table, st.lengths, query_start=start, max_tokens=128))
    want, want_lse, _, _ = attention(q, st.pool, st.table, st.lengths, 64, start)
    assert ((out - want).norm() / want.norm()).item() <= 2.0**-20
    assert ((lse - want_lse).norm() / want_lse.norm()).item() <= 2.0**-20


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("heads, kv_heads, dim, page_size", [(8, 2, 128, 64), (3, 3, 64, 16), (7, 1, 128, 32),
                                                             (16, 2, 64, 128)])
@pytest.mark.parametrize("new, lengths", [
    ([2, 1, 5, 0, 3], [2, 40, 5, 9, 130]),
    ([17, 1, 64, 33], [100, 1, 64, 999]),
    ([300, 129, 0, 2], [300, 700, 50, 2]),
])
def test_many_token_attention(cuda_device, dtype, heads, kv_heads, dim, page_size, new, lengths):
    st = State(lengths, kv_heads, dim, page_size, cuda_device, seed=sum(new))
    q = st.randn(sum(new), heads, dim, dtype=dtype)
    start = starts(new, cuda_device)
    got = kv.sdpa_q4_cache(q, st.pool, st.table, st.lengths, query_start=start, max_tokens=max(new))
    N.device_status()
    check_attention(got, q, st.pool, st.table, st.lengths, page_size, start)
    # the bound on one request's tokens chooses a kernel, never a result out of its bounds
    for most in (None, 1, 10**6):
        got = kv.sdpa_q4_cache(q, st.pool, st.table, st.lengths, query_start=start, max_tokens=most)
        check_attention(got, q, st.pool, st.table, st.lengths, page_size, start)


@pytest.mark.parametrize("heads, kv_heads, dim, page_size, new, lengths", [
    (32, 4, 128, 64, [800], [900]), (8, 2, 128, 16, [3300, 1, 700], [3300, 7, 5000]),
    (9, 3, 64, 32, [1000, 0, 2000], [3000, 5, 2100]), (64, 8, 64, 128, [400, 3], [390, 100]),
    (16, 16, 128, 1024, [129, 130, 700, 900], [129, 1000, 701, 0]), (30, 2, 64, 16, [513, 400], [600, 405])])
def test_attention_of_whole_tiles(cuda_device, heads, kv_heads, dim, page_size, new, lengths):
    """Enough bf16 rows for the tensor-core tiles; the same call with a small bound on a request's tokens, or in float16,
    takes the other kernel. More tokens than keys among them: zeros."""
    st = State(lengths, kv_heads, dim, page_size, cuda_device, seed=sum(new), magnitude=2.0)
    q = st.randn(sum(new), heads, dim, dtype=BF)
    start = starts(new, cuda_device)
    for most, x, tiles in ((max(new), q, 1), (1, q, 0), (max(new), q.to(F16), 0)):
        before = N.counters()["sdpa_prefill_launches"]
        got = kv.sdpa_q4_cache(x, st.pool, st.table, st.lengths, query_start=start, max_tokens=most)
        N.device_status()
        assert N.counters()["sdpa_prefill_launches"] - before == tiles
        check_attention(got, x, st.pool, st.table, st.lengths, page_size, start, tiles=bool(tiles))


def test_tiles_with_odd_contents(cuda_device):
    """Scales over their range in keys and values, queries of any magnitude, missing pages and garbage behind the last
    token, in the tensor-core tiles."""
    new, lengths = [500, 400], [530, 1001]
    st = State(lengths, 2, 64, 64, cuda_device)
    slots = torch.arange(st.pool.shape[0] * 64, device=cuda_device)
    k, v = st.randn(len(slots), 2, 64), st.randn(len(slots), 2, 64)
    v[0::4] *= 2.0**13
    v[1::4, :, :32] *= 2.0**-12
    v[2::4] = 0
    k[3::5] *= 2.0**-9
    kv.kv_q4_append(k, v, st.pool, slots)
    q = st.randn(900, 32, 64)
    q[::3] *= 2.0**-60
    q[1::3] *= 4
    q[2] = 0
    q = q.to(BF)
    start = starts(new, cuda_device)
    want = kv.sdpa_q4_cache(q, st.pool, st.table, st.lengths, query_start=start)
    N.device_status()
    check_attention(want, q, st.pool, st.table, st.lengths, 64, start, tiles=True)
    bad = torch.full((64, 2, 64), float("nan"), device=cuda_device)
    bad[::2] = float("inf")
    behind = torch.cat([st.table[0, 8] * 64 + torch.arange(18, 64, device=cuda_device),
                        st.table[1, 15] * 64 + torch.arange(41, 64, device=cuda_device)]).long()
    kv.kv_q4_append(bad.repeat(2, 1, 1)[:len(behind)], bad.repeat(2, 1, 1)[:len(behind)], st.pool, behind)
    got = kv.sdpa_q4_cache(q, st.pool, st.table, st.lengths, query_start=start)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    st.table[0, 1], st.table[0, 3] = 1 << 30, -1
    got = kv.sdpa_q4_cache(q, st.pool, st.table, st.lengths, query_start=start)
    with pytest.raises(RuntimeError, match="page id"):
        N.device_status()
    assert torch.equal(got[0][500:], want[0][500:]) and torch.isfinite(got[0]).all()
    # the keys of the missing pages are left out: as if the request had only the others
    kept = st.table[:1, [0, 2, 4, 5, 6, 7, 8]].contiguous()
    last = torch.tensor([530 - 128], dtype=torch.int32, device=cuda_device)
    check_attention((got[0][400:500], got[1][400:500]), q[400:500], st.pool, kept, last, 64, starts([100], cuda_device),
                    tiles=True)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("dim", [64, 128])
def test_more_tokens_than_keys(cuda_device, dtype, dim):
    """Tokens before a request's first key see none: zeros and logsumexp 0."""
    new, lengths = [5, 40, 200, 3], [2, 17, 100, 0]
    st = State(lengths, 2, dim, 16, cuda_device)
    q = st.randn(sum(new), 4, dim, dtype=dtype)
    start = starts(new, cuda_device)
    for most in (1, 8, 200):
        got = kv.sdpa_q4_cache(q, st.pool, st.table, st.lengths, query_start=start, max_tokens=most)
        check_attention(got, q, st.pool, st.table, st.lengths, 16, start)
        assert (got[0][:3] == 0).all() and (got[1][:3] == 0).all()
        assert (got[0][45:145] == 0).all() and (got[1][245:] == 0).all()


def test_rows_behind_the_last_request_are_left(cuda_device):
    """In C, with output buffers of the caller's: a padded batch."""
    import ctypes

    for most, new in ((1, [1, 1, 1]), (70, [70, 0, 3])):
        st = State([90, 3, 40], 2, 128, 64, cuda_device)
        t = sum(new) + 9
        q = st.randn(t, 8, 128, dtype=BF)
        start = starts(new, cuda_device)
        out = torch.full((t, 8, 128), 7.0, dtype=BF, device=cuda_device)
        lse = torch.full((t, 8), 7.0, device=cuda_device)
        lib = N.lib()
        ws = torch.empty(lib.tn_sdpa_q4_workspace_bytes(t, 8, 2, 128, most), dtype=torch.uint8, device=cuda_device)
        N.check(lib.tn_sdpa_q4_cache(
            q.data_ptr(), N.TN_BF16, (ctypes.c_int64 * 2)(1024, 128), t, 8, st.pool.data_ptr(), st.pool.shape[0], 2, 128,
            64, st.table.data_ptr(), st.table.shape[1], st.table.shape[1], st.lengths.data_ptr(), 3, start.data_ptr(),
            most, out.data_ptr(), lse.data_ptr(), 0.0, ws.data_ptr(), ws.numel(),
            torch.cuda.current_stream().cuda_stream))
        N.device_status()
        check_attention((out, lse), q, st.pool, st.table, st.lengths, 64, start)
        assert (out[sum(new):] == 7).all() and (lse[sum(new):] == 7).all()


@pytest.mark.parametrize("dtype", [BF, F16, F32])
def test_query_magnitudes(cuda_device, dtype):
    """Queries far above and below float16's range, elements far apart in one row, and a peaked softmax."""
    lengths = [300, 77, 1200, 5]
    st = State(lengths, 2, 128, 64, cuda_device)
    q = st.randn(4, 8, 128, dtype=torch.float32)
    big = 2.0**15 if dtype == F16 else 2.0**100
    for row, factor in ((0, big), (1, 1 / big), (2, 30.0)):
        q[row] *= factor
    q[3, :, ::2] *= 2.0**-12
    q = q.clamp(-60000, 60000).to(dtype) if dtype == F16 else q.to(dtype)
    for scale in (2.0**-100 if dtype != F16 else 2.0**-15, 1.0):
        rows = [0, 2] if scale < 1 else [1, 2, 3]
        got = kv.sdpa_q4_cache(q, st.pool, st.table, st.lengths, scale=scale)
        N.device_status()
        table, some = st.table[rows], st.lengths[rows]
        check_attention((got[0][rows], got[1][rows]), q[rows], st.pool, table, some, 64, scale=scale)


def test_value_scales_over_their_whole_range(cuda_device):
    """Blocks of values whose scales are float16's largest, its smallest and zero, next to each other."""
    st = State([400, 33], 1, 64, 16, cuda_device)
    k, v = st.randn(st.pool.shape[0] * 16, 1, 64), st.randn(st.pool.shape[0] * 16, 1, 64)
    v[0::4] *= 2.0**17
    v[1::4, :, :32] *= 2.0**-20
    v[2::4] = 0
    kv.kv_q4_append(k, v.clamp(-5e5, 5e5), st.pool, torch.arange(len(k), device=cuda_device))
    for dtype in (F32, BF):
        q = st.randn(2, 4, 64, dtype=dtype) * 3
        got = kv.sdpa_q4_cache(q, st.pool, st.table, st.lengths)
        N.device_status()
        check_attention(got, q, st.pool, st.table, st.lengths, 16)
    one = State([16, 16], 1, 64, 16, cuda_device)  # nothing but zero and tiny values
    v = torch.zeros(16, 1, 64, device=cuda_device)
    slots = one.table[0, 0].long() * 16 + torch.arange(16, device=cuda_device)
    kv.kv_q4_append(st.randn(16, 1, 64) * 20, v, one.pool, slots)
    v[:, :, 32:] = 2.0**-21
    kv.kv_q4_append(st.randn(16, 1, 64) * 20, v, one.pool, one.table[1, 0].long() * 16 + slots % 16)
    q = st.randn(2, 4, 64)
    got = kv.sdpa_q4_cache(q, one.pool, one.table, one.lengths)
    check_attention(got, q, one.pool, one.table, one.lengths, 16)
    assert (got[0][0] == 0).all()


def test_unread_places_may_hold_anything(cuda_device):
    """NaN and infinite scales behind a request's last token, in its last group and page, reach no result."""
    for new in ([1, 1], [90, 3]):
        st = State([101, 3], 2, 128, 64, cuda_device)
        q = st.randn(sum(new), 4, 128, dtype=BF)
        start = starts(new, cuda_device)
        want = kv.sdpa_q4_cache(q, st.pool, st.table, st.lengths, query_start=start, max_tokens=max(new))
        bad = torch.full((64, 2, 128), float("nan"), device=cuda_device)
        bad[::2] = float("inf")
        slots = torch.cat([st.table[0, 1] * 64 + torch.arange(37, 64, device=cuda_device),
                           st.table[1, 0] * 64 + torch.arange(3, 64, device=cuda_device)]).long()
        kv.kv_q4_append(bad.repeat(2, 1, 1)[:len(slots)], bad.repeat(2, 1, 1)[:len(slots)], st.pool, slots)
        got = kv.sdpa_q4_cache(q, st.pool, st.table, st.lengths, query_start=start, max_tokens=max(new))
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_strided_queries(cuda_device):
    st = State([70, 9], 2, 64, 16, cuda_device)
    rows = st.randn(2, 8 * 64, dtype=BF).unflatten(1, (8, 64))
    for q in (rows[:, 2:6], st.randn(4, 2, 64, dtype=F16).transpose(0, 1), st.randn(2, 4, 65)[..., 1:]):
        a = kv.sdpa_q4_cache(q, st.pool, st.table, st.lengths)
        b = kv.sdpa_q4_cache(q.contiguous(), st.pool, st.table, st.lengths)
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_bad_pages_and_lengths_are_reported_and_not_followed(cuda_device):
    for new in (1, 70):
        st = State([100, 50, 20], 2, 64, 16, cuda_device)
        q = st.randn(3 * new, 4, 64)
        start = starts([new] * 3, cuda_device)
        want = kv.sdpa_q4_cache(q, st.pool, st.table, st.lengths, query_start=start, max_tokens=new)
        st.table[0, 2], st.table[1, 1] = 1 << 30, -5
        got = kv.sdpa_q4_cache(q, st.pool, st.table, st.lengths, query_start=start, max_tokens=new)
        with pytest.raises(RuntimeError, match="page id"):
            N.device_status()
        assert torch.equal(got[0][2 * new:], want[0][2 * new:]) and torch.isfinite(got[0]).all()
        st = State([100, 50, 20], 2, 64, 16, cuda_device)
        st.lengths.copy_(torch.tensor([2**31 - 1, -7, 20]))
        got = kv.sdpa_q4_cache(q, st.pool, st.table[:, :2].contiguous(), st.lengths, query_start=start, max_tokens=new)
        N.device_status()
        check_attention(got, q, st.pool, st.table[:, :2], st.lengths.clamp(0, 32), 16, start)


def test_attention_is_the_same_every_time_and_in_any_order(cuda_device):
    """Bits do not depend on scheduling; two states in turn do not disturb each other."""
    a, b = State([4000, 77, 1, 900], 2, 128, 64, cuda_device), State([50, 3000], 2, 128, 64, cuda_device, seed=5)
    qa, qb = a.randn(4, 16, 128, dtype=BF), b.randn(2, 16, 128, dtype=BF)
    want = kv.sdpa_q4_cache(qa, a.pool, a.table, a.lengths)
    for _ in range(20):
        kv.sdpa_q4_cache(qb, b.pool, b.table, b.lengths)
        got = kv.sdpa_q4_cache(qa, a.pool, a.table, a.lengths)
        assert all(torch.equal(x, y) for x, y in zip(got, want))


# ---- the decode step


def rotate(x, cos, sin):
    a, b = x.float().chunk(2, -1)
    return torch.cat((a * cos - b * sin, b * cos + a * sin), -1).to(x.dtype)


def rope_table(rows, dim, device):
    angle = torch.arange(rows, dtype=torch.float64)[:, None] / 10000.0 ** (torch.arange(0, dim, 2) / dim)
    return torch.cat((angle.cos(), angle.sin()), 1).bfloat16().to(device)


@pytest.mark.parametrize("heads, kv_heads, dim, page_size", [(8, 2, 128, 64), (9, 3, 64, 16), (16, 2, 128, 32),
                                                             (1, 1, 64, 128), (7, 1, 128, 16)])
@pytest.mark.parametrize("lengths", [[1], [1, 0, 16, 17, 64, 65, 500, 33], [3000, 1], [0, 0]])
def test_step_is_rope_append_attend(cuda_device, heads, kv_heads, dim, page_size, lengths):
    st = State(lengths, kv_heads, dim, page_size, cuda_device, seed=len(lengths))
    b = len(lengths)
    qkv = st.randn(b, (heads + 2 * kv_heads) * dim, dtype=BF)
    rope = rope_table(max(lengths) + 1, dim, cuda_device)
    q, k, v = qkv.unflatten(1, (-1, dim)).split([heads, kv_heads, kv_heads], 1)
    at = st.lengths.long() - 1
    cos, sin = rope[at.clamp(min=0)].float()[:, None].chunk(2, -1)
    q, k = rotate(q, cos, sin), rotate(k, cos, sin)
    slots = st.table.gather(1, (at.clamp(min=0) // page_size)[:, None])[:, 0].long() * page_size + at % page_size
    pool = st.pool.clone()
    kv.kv_q4_append(k, v, pool, torch.where(at >= 0, slots, -1))
    nb = heads * dim // 32
    q8 = (torch.empty((b, heads * dim), dtype=torch.int8, device=cuda_device),
          torch.empty((b, nb), device=cuda_device), torch.empty((b, nb), device=cuda_device))
    out = kv.sdpa_q4_decode_step(qkv, rope, st.pool, st.table, st.lengths, heads, q8=q8)
    N.device_status()
    assert torch.equal(st.pool, pool)
    lse = kv.sdpa_q4_cache(q, pool, st.table, st.lengths)[1]
    check_attention((out, lse), q, pool, st.table, st.lengths, page_size)
    want = tuple(torch.empty_like(t) for t in q8)
    N.check(N.lib().tn_q8_0_quantize_planar(out.data_ptr(), N.TN_BF16, heads * dim, want[0].data_ptr(), heads * dim,
                                            want[1].data_ptr(), want[2].data_ptr(), b, heads * dim,
                                            torch.cuda.current_stream().cuda_stream))
    assert all(torch.equal(x, y) for x, y in zip(q8, want))
    again = kv.sdpa_q4_decode_step(qkv, rope, st.pool, st.table, st.lengths, heads)
    assert torch.equal(again, out) and torch.equal(st.pool, pool)


def test_step_beyond_the_rotary_table_or_its_pages(cuda_device):
    st = State([40, 20, 30], 2, 64, 16, cuda_device)
    qkv = st.randn(3, 8 * 64, dtype=BF)
    before = st.pool.clone()
    want = kv.sdpa_q4_decode_step(qkv, rope_table(50, 64, cuda_device), st.pool.clone(), st.table, st.lengths, 4)
    out = kv.sdpa_q4_decode_step(qkv, rope_table(35, 64, cuda_device), st.pool, st.table, st.lengths, 4)
    with pytest.raises(RuntimeError, match="position"):
        N.device_status()
    assert torch.equal(out[1:], want[1:])
    assert torch.equal(st.pool[st.table[0, 2]], before[st.table[0, 2]])  # nothing was appended at position 39
    page = st.table[1, 1].item()
    st.table[1, 1] = 99
    out = kv.sdpa_q4_decode_step(qkv, rope_table(50, 64, cuda_device), st.pool, st.table, st.lengths, 4)
    with pytest.raises(RuntimeError, match="page id"):
        N.device_status()
    assert torch.equal(out[2], want[2]) and torch.isfinite(out).all()
    assert page != 99


# ---- together


def test_a_conversation_in_pages(cuda_device):
    """Prompts of differing lengths come in, are attended in chunks, decode token by token, one ends and another takes
    its pages -- all against dense caches of the quantised rows."""
    heads, kv_heads, dim, page = 8, 2, 128, 16
    g = torch.Generator().manual_seed(1)
    cache = kv.PagedQ4Cache(2, kv_heads, dim, 24, 3, 10, page, cuda_device)
    dense = [[[], []] for _ in range(3)]  # a request's rows of keys and values

    def put(slots, positions, start, layer):
        t = slots.shape[0]
        k, v = (torch.randn((t, kv_heads, dim), generator=g).to(BF).to(cuda_device) for _ in range(2))
        cache.append(layer, k, v, slots)
        if layer == 1:
            s = start.tolist()
            for b in range(3):
                for rows, x in zip(dense[b], (k, v)):
                    y = x[s[b]:s[b + 1]].float().reshape(-1, dim)
                    if len(y):
                        rows.append(quant._dequantize(quant._quantize(y)).view(-1, kv_heads, dim).double().cpu())

    def attend(start, most):
        s = start.tolist()
        q = torch.randn((s[-1] + 2, heads, dim), generator=g).to(BF).to(cuda_device)
        out, lse = cache.attend(1, q, query_start=start, max_tokens=most)
        for b in range(3):
            n = s[b + 1] - s[b]
            if n == 0:
                continue
            k, v = (torch.cat(x).transpose(0, 1).repeat_interleave(heads // kv_heads, 0) for x in dense[b])
            sc = q[s[b]:s[b + 1]].double().cpu().transpose(0, 1) @ k.transpose(1, 2) / dim**0.5
            hide = torch.arange(k.shape[1])[None] > (k.shape[1] - n + torch.arange(n))[:, None]
            sc = sc.masked_fill(hide, -float("inf"))
            want = (torch.softmax(sc, -1) @ v).transpose(0, 1)
            err = (out[s[b]:s[b + 1]].double().cpu() - want).abs().max()
            assert err <= 2.0**-7 * max(1.0, want.abs().max()), err
            assert (lse[s[b]:s[b + 1]].double().cpu() - torch.logsumexp(sc, -1).T).abs().max() < 1e-4

    def turn(tokens, most, **to):
        slots, positions, start = cache.resize(tokens, **to)
        for layer in range(2):
            put(slots, positions, start, layer)
        attend(start, most)

    i32 = dict(dtype=torch.int32, device=cuda_device)
    turn(150, 100, new_lengths=torch.tensor([40, 0, 100], **i32))
    turn(90, 60, new_lengths=torch.tensor([100, 9, 120], **i32))
    for _ in range(20):
        turn(3, 1, grow=1)
    dense[0] = [[], []]  # request 0 ends
    cache.resize(0, new_lengths=torch.tensor([0, 29, 140], **i32))
    turn(140, 130, new_lengths=torch.tensor([130, 29, 141], **i32))
    for _ in range(3):
        turn(6, 2, grow=2)
    assert cache.lengths.tolist() == [136, 35, 147]
    cache.check()


def test_captured_steps_replay_while_lengths_grow(cuda_device):
    """One graph of resize + step serves every token; two graphs replayed in turn and an eager call between them keep
    apart; the pools equal those of eager steps."""
    heads, kv_heads, dim, page = 8, 2, 128, 16
    rope = rope_table(200, dim, cuda_device)
    g = torch.Generator().manual_seed(3)
    rows = [torch.randn((3, (heads + 2 * kv_heads) * dim), generator=g).to(BF).to(cuda_device) for _ in range(12)]

    def fresh():
        c = kv.PagedQ4Cache(1, kv_heads, dim, 40, 3, 12, page, cuda_device)
        c.resize(200, new_lengths=torch.tensor([7, 0, 150], dtype=torch.int32, device=cuda_device))
        c.pools[0].copy_(fill)
        return c

    fill = torch.zeros((40, kv_heads, 1, 18 * dim), dtype=torch.uint8, device=cuda_device)
    x = torch.randn((640, kv_heads, dim), generator=g).to(cuda_device)
    kv.kv_q4_append(x, x.flip(0), fill, torch.arange(640, device=cuda_device))
    eager, outs = fresh(), []
    for r in rows:
        eager.resize(3, grow=1)
        outs.append(eager.decode_step(0, r, rope, heads))
    captured = []
    for _ in range(2):
        c, qkv = fresh(), rows[0].clone()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            c.resize(3, grow=1)
            c.decode_step(0, qkv, rope, heads)
        side.synchronize()
        c.resize(0, new_lengths=torch.tensor([7, 0, 150], dtype=torch.int32, device=cuda_device))
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            c.resize(3, grow=1)
            out = c.decode_step(0, qkv, rope, heads)
        captured.append((c, qkv, graph, out))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for r, want in zip(rows, outs):
        torch.cuda.synchronize()
        for c, qkv, graph, out in captured:
            qkv.copy_(r)
        torch.cuda.synchronize()
        for s, (c, qkv, graph, out) in zip(streams, captured):
            with torch.cuda.stream(s):
                graph.replay()
        eager.decode_step(0, rows[-1], rope, heads)
        torch.cuda.synchronize()
        for c, qkv, graph, out in captured:
            assert torch.equal(out, want)
    for c, *_ in captured:
        assert torch.equal(c.pools[0], eager.pools[0]) and torch.equal(c.lengths, eager.lengths)
        c.check()


def test_two_graphs_of_split_attention_at_the_same_time(cuda_device):
    """Contexts that many CTAs share and join: two graphs captured on one stream, replayed on two, an eager call beside."""
    states = [State([9000, 3000], 2, 128, 64, cuda_device, seed=i) for i in range(3)]
    queries = [s.randn(2, 8, 128, dtype=BF) for s in states]
    want = [kv.sdpa_q4_cache(q, s.pool, s.table, s.lengths) for q, s in zip(queries, states)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs = []
    for q, s in zip(queries[:2], states):
        with torch.cuda.stream(side):
            kv.sdpa_q4_cache(q, s.pool, s.table, s.lengths)
        side.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            outs = [kv.sdpa_q4_cache(q, s.pool, s.table, s.lengths) for _ in range(8)]
        graphs.append((g, outs))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(20):
        torch.cuda.synchronize()
        for stream, (g, _) in zip(streams, graphs):
            with torch.cuda.stream(stream):
                g.replay()
        mine = kv.sdpa_q4_cache(queries[2], states[2].pool, states[2].table, states[2].lengths)
        torch.cuda.synchronize()
        for (_, outs), w in zip(graphs, want):
            assert all(torch.equal(a, b) for o in outs for a, b in zip(o, w))
        assert all(torch.equal(a, b) for a, b in zip(mine, want[2]))
    N.device_status()


def test_another_stream(cuda_device):
    st = State([900, 33], 2, 128, 64, cuda_device)
    q = st.randn(2, 8, 128, dtype=BF)
    want = kv.sdpa_q4_cache(q, st.pool, st.table, st.lengths)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = [kv.sdpa_q4_cache(q, st.pool, st.table, st.lengths) for _ in range(3)]
    other = [kv.sdpa_q4_cache(q, st.pool, st.table, st.lengths) for _ in range(3)]
    torch.cuda.synchronize()
    for g in got + other:
        assert all(torch.equal(a, b) for a, b in zip(g, want))


def test_a_pool_beyond_32_bit_offsets(cuda_device):
    """5 GB of pages; the requests' lie at its end, and across byte 2^32."""
    heads, dim, page = 8, 128, 64
    num = 5 * 2**30 // (heads * page // 16 * 18 * dim)
    pool = kv.kv_q4_pool(num, heads, dim, page, cuda_device)
    st = State([130, 200], heads, dim, page, cuda_device)
    at = 2**32 // (heads * page // 16 * 18 * dim)
    pages = torch.tensor([num - 1, at, num - 3, at + 1, 0, num - 2, at - 1], dtype=torch.int32, device=cuda_device)
    k, v = st.randn(330, heads, dim), st.randn(330, heads, dim)
    table = torch.full((2, 4), -1, dtype=torch.int32, device=cuda_device)
    table[0, :3], table[1, :4] = pages[:3], pages[3:]
    pos = torch.cat([torch.arange(130), torch.arange(200)]).to(cuda_device)
    row = torch.cat([torch.zeros(130), torch.ones(200)]).long().to(cuda_device)
    slots = table[row, pos // page].long() * page + pos % page
    assert slots.max() * heads * dim > 2**32 // 2
    kv.kv_q4_append(k, v, pool, slots)
    small = kv.kv_q4_pool(7, heads, dim, page, cuda_device)
    small.copy_(pool[pages.long()])
    same = torch.where(table >= 0, torch.arange(7, dtype=torch.int32, device=cuda_device)[
        (table[..., None] == pages).long().argmax(-1)], -1).to(torch.int32)
    q = st.randn(330, 16, dim, dtype=BF)
    start = starts([130, 200], cuda_device)
    for most, x, begin in ((1, q[:2], None), (8, q, start), (200, q, start)):
        a = kv.sdpa_q4_cache(x, pool, table, st.lengths, query_start=begin, max_tokens=most)
        b = kv.sdpa_q4_cache(x, small, same, st.lengths, query_start=begin, max_tokens=most)
        assert all(torch.equal(i, j) for i, j in zip(a, b))
        check_attention(b, x, small, same, st.lengths, page, begin, tiles=most == 200)
    N.device_status()


def test_an_empty_pool_and_no_rows(cuda_device):
    pool = kv.kv_q4_pool(0, 2, 64, 16, cuda_device)
    table = torch.zeros((2, 3), dtype=torch.int32, device=cuda_device)
    lengths = torch.tensor([0, 20], dtype=torch.int32, device=cuda_device)
    out, lse = kv.sdpa_q4_cache(torch.ones(2, 4, 64, device=cuda_device), pool, table, lengths)
    with pytest.raises(RuntimeError, match="page id"):
        N.device_status()
    assert (out == 0).all() and (lse == 0).all()
    x = torch.ones(1, 2, 64, device=cuda_device)
    kv.kv_q4_append(x, x, pool, torch.zeros(1, dtype=torch.int64, device=cuda_device))
    with pytest.raises(RuntimeError, match="slot"):
        N.device_status()
    kv.kv_q4_append(x[:0], x[:0], pool, torch.zeros(0, dtype=torch.int64, device=cuda_device))
    start = torch.zeros(3, dtype=torch.int32, device=cuda_device)
    out, lse = kv.sdpa_q4_cache(torch.ones(0, 4, 64, device=cuda_device), pool, table, lengths, query_start=start)
    assert out.shape == (0, 4, 64) and lse.shape == (0, 4)
    none = kv.sdpa_q4_cache(torch.ones(3, 4, 64, device=cuda_device), pool, table, lengths, query_start=start)
    assert none[0].shape == (3, 4, 64)  # rows of no request: not written
    N.device_status()


def test_refusals(cuda_device):
    st = State([20, 9], 2, 64, 16, cuda_device)
    q = st.randn(2, 4, 64)
    with pytest.raises(NotImplementedError, match="float32, float16 or bfloat16"):
        kv.sdpa_q4_cache(q.double(), st.pool, st.table, st.lengths)
    with pytest.raises(RuntimeError, match="tokens, heads"):
        kv.sdpa_q4_cache(q[..., :32], st.pool, st.table, st.lengths)
    with pytest.raises(RuntimeError, match="one query token"):
        kv.sdpa_q4_cache(q[:1], st.pool, st.table, st.lengths)
    with pytest.raises(RuntimeError, match="query_start"):
        kv.sdpa_q4_cache(q, st.pool, st.table, st.lengths, query_start=st.lengths)
    with pytest.raises(RuntimeError, match="multiple of"):
        kv.sdpa_q4_cache(q[:, :3], st.pool, st.table, st.lengths)
    with pytest.raises(NotImplementedError, match="lengths"):
        kv.sdpa_q4_cache(q, st.pool, st.table, st.lengths.long())
    with pytest.raises(RuntimeError, match="same requests"):
        kv.sdpa_q4_cache(q, st.pool, st.table, st.lengths[:1])
    with pytest.raises(RuntimeError, match="same device"):
        kv.sdpa_q4_cache(q, st.pool, st.table, st.lengths.cpu())
    with pytest.raises(RuntimeError, match="contiguous"):
        kv.sdpa_q4_cache(q, st.pool, st.table[:, :1], st.lengths)
    with pytest.raises(RuntimeError, match="do not fit"):
        kv.kv_q4_append(q, q, st.pool, torch.zeros(2, dtype=torch.int64, device=cuda_device))
    with pytest.raises(NotImplementedError, match="slots"):
        kv.kv_q4_append(q[:, :2], q[:, :2], st.pool, st.lengths)
    with pytest.raises(NotImplementedError, match="key and value"):
        kv.kv_q4_append(q[:, :2], q[:, :2].half(), st.pool, torch.zeros(2, dtype=torch.int64, device=cuda_device))
    with pytest.raises(RuntimeError, match="not both"):
        kv.kv_pages_resize(st.table, st.lengths, st.lengths, st.lengths[:1], st.lengths[:1], 16, 0, new_lengths=st.lengths,
                           grow=1)
    rope = rope_table(30, 64, cuda_device)
    with pytest.raises(RuntimeError, match="qkv"):
        kv.sdpa_q4_decode_step(q.reshape(2, -1).to(BF), rope, st.pool, st.table, st.lengths, 4)
    with pytest.raises(RuntimeError, match="rope"):
        kv.sdpa_q4_decode_step(st.randn(2, 512, dtype=BF), rope[:, :32].contiguous(), st.pool, st.table, st.lengths, 4)
    with pytest.raises(NotImplementedError, match="at most 8"):
        kv.sdpa_q4_decode_step(st.randn(2, 22 * 64, dtype=BF), rope, st.pool, st.table, st.lengths, 18)
    N.device_status()
