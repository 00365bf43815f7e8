"""The paged 4-bit cache where something runs out: pages, a request's table, the engine's capacity. What cannot be met
leaves pools, lengths and tokens as they were, and the next call that can be goes on from there."""

import pytest
import torch

from tests.kv_q4_ref import State
from tests.test_decode_paged_gpu import small, tokens
from tests.test_kv_cache_gpu import rope_table
from torchnative_b200 import _native as N
from torchnative_b200 import kv_cache as kv

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


def i32(values, device):
    return torch.tensor(values, dtype=torch.int32, device=device)


@pytest.mark.parametrize("batch, replay", [(2, False), (2, True), (6, False), (6, True)])
def test_a_full_sequence_leaves_the_others_alone(cuda_device, batch, replay):
    """One sequence at its capacity: the step changes nothing; without it the others go on as if it had never been."""
    dec = small(batch, cuda_device)
    rest = [20 + 3 * i for i in range(1, batch)]
    dec.fill_prompt_cache([0] + rest)
    dec.start(tokens(batch, cuda_device))
    want = []
    for _ in range(6):
        dec.step()
        want.append(dec.tokens[1:].tolist())
    graph = dec.capture() if replay else None
    step = graph.replay if replay else dec.step
    dec.fill_prompt_cache([79] + rest)
    dec.paged.check()
    dec.start(tokens(batch, cuda_device))
    step()  # the first sequence's last place
    got = [dec.tokens[1:].tolist()]
    before = [p.clone() for p in dec.paged.pools], dec.tokens.clone(), dec.h.clone(), dec.paged.lengths.tolist()
    for _ in range(3):
        step()
        assert all(torch.equal(a, b) for a, b in zip(dec.paged.pools, before[0]))
        assert torch.equal(dec.tokens, before[1]) and torch.equal(dec.h, before[2])
        assert dec.paged.lengths.tolist() == before[3]
    with pytest.raises(RuntimeError, match="length"):
        dec.paged.check()
    dec.paged.resize(0, new_lengths=i32([0] + before[3][1:], cuda_device))
    for _ in range(5):
        step()
        got.append(dec.tokens[1:].tolist())
    dec.paged.check()
    assert got == want


@pytest.mark.parametrize("heads, kv_heads, dim", [(8, 2, 128), (3, 3, 64)])
def test_a_step_behind_a_refused_resize_appends_nothing(cuda_device, heads, kv_heads, dim):
    """Pages run out: the step gives zeros and leaves the pool, byte for byte; with pages again it is an ordinary one."""
    cache = kv.PagedQ4Cache(1, kv_heads, dim, 3, 2, 4, 16, cuda_device)
    g = torch.Generator().manual_seed(dim)
    x = torch.randn((33, kv_heads, dim), generator=g).to(cuda_device)
    slots, _, _ = cache.resize(33, new_lengths=i32([32, 1], cuda_device))
    assert cache.granted.tolist() == [32, 1]
    cache.append(0, x, x.flip(0), slots)
    qkv = torch.randn((2, (heads + 2 * kv_heads) * dim), generator=g).to(BF).to(cuda_device)
    rope = rope_table(64, dim, cuda_device)
    nb = heads * dim // 32
    q8 = (torch.ones((2, heads * dim), dtype=torch.int8, device=cuda_device), torch.ones((2, nb), device=cuda_device),
          torch.ones((2, nb), device=cuda_device))
    before = cache.pools[0].clone()
    cache.resize(2, grow=1)
    out = cache.decode_step(0, qkv, rope, heads, q8=q8)
    assert cache.granted.tolist() == [0, 0]
    assert (out == 0).all() and (q8[0] == 0).all() and (q8[1] == 0).all()
    assert torch.equal(cache.pools[0], before)
    with pytest.raises(RuntimeError, match="pages"):
        cache.check()
    cache.resize(0, new_lengths=i32([32, 0], cuda_device))  # the second request ends
    cache.resize(1, grow=1)
    assert cache.granted.tolist() == [1, 0]
    out = cache.decode_step(0, qkv, rope, heads)
    cache.check()
    other = before.clone()
    want = kv.sdpa_q4_decode_step(qkv, rope, other, cache.page_table, cache.lengths, heads)
    assert torch.equal(out, want) and torch.equal(cache.pools[0], other) and (out[0] != 0).any()


def test_rows_without_a_grant_keep_their_token(cuda_device):
    g = torch.Generator().manual_seed(4)
    logits = torch.randn((4, 999), generator=g).to(BF).to(cuda_device)
    embed = torch.randn((999, 64), generator=g).to(BF).to(cuda_device)
    had, granted = i32([7, 8, 9, 10], cuda_device), i32([1, 0, 3, -1], cuda_device)
    h = torch.zeros((4, 64), dtype=BF, device=cuda_device)
    for given in (granted, None):
        got = had.clone()
        N.check(N.lib().tn_llama_argmax_embed_granted(
            logits.data_ptr(), 4, 999, got.data_ptr(), embed.data_ptr(), 64, h.data_ptr(), None,
            None if given is None else given.data_ptr(), torch.cuda.current_stream().cuda_stream))
        best = logits.float().argmax(-1).to(torch.int32)
        want = best if given is None else torch.where(given > 0, best, had)
        assert torch.equal(got, want) and torch.equal(h, embed[want.long()])


def test_granted_is_checked(cuda_device):
    cache = kv.PagedQ4Cache(1, 1, 64, 4, 2, 2, 16, cuda_device)
    args = (cache.page_table, cache.lengths, cache.free_pages, cache.free_count, cache.status, 16, 2)
    qkv, rope = torch.zeros((2, 192), dtype=BF, device=cuda_device), rope_table(9, 64, cuda_device)
    step = (qkv, rope, cache.pools[0], cache.page_table, cache.lengths, 1)
    for bad, error, match in ((i32([0], cuda_device), RuntimeError, "granted"), (i32([0, 0], "cpu"), RuntimeError, "device"),
                              (torch.zeros(2, device=cuda_device), NotImplementedError, "granted"),
                              (i32([0, 0, 0, 0], cuda_device)[::2], RuntimeError, "contiguous")):
        with pytest.raises(error, match=match):
            kv.kv_pages_resize(*args, grow=1, granted=bad)
        with pytest.raises(error, match=match):
            kv.sdpa_q4_decode_step(*step, granted=bad)


@pytest.mark.parametrize("what", ["rope", "table"])
def test_a_token_without_a_place_is_left_out(cuda_device, what):
    """Lengths beyond the rotary table, or beyond what the page table can name: nothing is appended, nothing that lies at
    the place is read, and it is reported; the other requests are as they are without."""
    st = State([40, 20, 48], 2, 64, 16, cuda_device)
    qkv = st.randn(3, 8 * 64, dtype=BF)
    rope = rope_table(50, 64, cuda_device)
    table, lengths = st.table, st.lengths.clone()
    if what == "rope":
        rope, lost = rope[:39].contiguous(), [0, 2]  # positions 39 and 47
    else:
        lengths[0], lengths[2], lost = 49, 2**31 - 1, [0, 2]
    own = st.pool.clone()
    want = kv.sdpa_q4_decode_step(qkv[1:2].contiguous(), rope, own, table[1:2], lengths[1:2], 4)
    for fill in (None, 0xff):  # an unwritten place may hold anything: NaN scales among it
        pool = st.pool.clone()
        if fill is not None:
            pool[table[0].long(), :, 0] = fill
            pool[table[2].long(), :, 0] = fill
        before = pool.clone()
        out = kv.sdpa_q4_decode_step(qkv, rope, pool, table, lengths, 4)
        with pytest.raises(RuntimeError, match="position"):
            N.device_status()
        assert (out[lost] == 0).all() and torch.equal(out[1:2], want)
        for b in (0, 2):
            pages = table[b].long()
            assert torch.equal(pool[pages], before[pages])
        assert torch.equal(pool[table[1, 1]], own[table[1, 1]])


@pytest.mark.parametrize("batch", [2, 6])
def test_a_capacity_that_ends_inside_a_page(cuda_device, batch):
    """The last page's places beyond the capacity are places like others: tokens there are those of a larger engine."""
    from torchnative_b200.llama_decode import LlamaShape, Q4LlamaDecoder

    shape = LlamaShape(hidden=512, inter=1024, heads=8, kv_heads=2, head_dim=64, vocab=2048, layers=2, rope_theta=10000.0)
    runs = []
    for capacity in (70, 80):
        dec = Q4LlamaDecoder(shape, batch=batch, capacity=capacity, device=cuda_device, seed=12, kv_cache="q4_0", page_size=16)
        dec.fill_prompt_cache([66] + [9] * (batch - 1))
        dec.start(tokens(batch, cuda_device))
        runs.append([])
        for _ in range(14):
            dec.step()
            runs[-1].append(dec.tokens.tolist())
        dec.paged.check()
        assert dec.paged.lengths.tolist() == [80] + [23] * (batch - 1)
        runs[-1].append([p.cpu() for p in dec.paged.pools])
        dec.step()  # the page's end
        with pytest.raises(RuntimeError, match="length"):
            dec.paged.check()
    assert runs[0][:-1] == runs[1][:-1]
    assert all(torch.equal(a, b) for a, b in zip(runs[0][-1], runs[1][-1]))


def bad_slot(device):
    pool = kv.kv_q4_pool(1, 1, 64, 16, device)
    x = torch.ones((1, 1, 64), device=device)
    kv.kv_q4_append(x, x, pool, torch.tensor([16], device=device))


def test_a_bad_slot_stops_no_other_kernel(cuda_device):
    """The persistent decode kernel, whose waits end early once one has given up, beside a reported slot."""
    from torchnative_b200.llama_decode import LLAMA3_8B, Q4LlamaDecoder

    dec = Q4LlamaDecoder(LLAMA3_8B, batch=1, capacity=64, device=cuda_device, seed=3, layers=1, mega=True)
    runs = []
    for bad in (False, True):
        dec.fill_prompt_cache(40)
        dec.start(torch.tensor([17], device=cuda_device))
        if bad:
            bad_slot(cuda_device)
        runs.append([])
        for _ in range(3):
            dec.step()
            runs[-1].append((dec.tokens.item(), dec.logits.clone()))
    with pytest.raises(RuntimeError, match="slot"):
        N.device_status()
    N.device_status()
    dec.close()
    assert all(a[0] == b[0] and torch.equal(a[1], b[1]) for a, b in zip(*runs))


def test_a_bad_slot_hides_no_timeout(cuda_device):
    """A gather whose peer never signals, its wait cut to about 1 ms, behind a slot that was reported: both are told, the
    timeout by its status, and both are cleared."""
    import ctypes

    lib = N.lib()
    N.device_status()
    regions = []
    for _ in range(2):
        base, handle = ctypes.c_void_p(), (ctypes.c_uint8 * 64)()
        N.check(lib.tn_tp_region_alloc(1 << 16, ctypes.byref(base), handle))
        regions.append(base)
    bases = (ctypes.c_void_p * 2)(*[r.value for r in regions])
    local = torch.ones((1, 64), dtype=BF, device=cuda_device)
    prev = N.set_wait_budget(2_000_000)
    try:
        bad_slot(cuda_device)
        N.check(lib.tn_tp_allgather(bases, 0, 2, local.data_ptr(), 64, 1, 64, 0, 128, 0,
                                    torch.cuda.current_stream().cuda_stream))
        cache = kv.PagedQ4Cache(1, 1, 64, 1, 1, 1, 16, cuda_device)
        cache.resize(0, new_lengths=i32([17], cuda_device))
        with pytest.raises(TimeoutError, match="length.*gave up.*slot"):
            cache.check()
        cache.check()
    finally:
        N.set_wait_budget(prev)
        torch.cuda.synchronize()
        for base in regions:
            lib.tn_tp_region_free(base)


def test_caches_of_many_and_of_very_many_requests_at_the_same_time(cuda_device):
    """Two host threads, whose calls need different amounts of shared memory; and a graph of the larger one that is made
    before and replayed after a smaller call."""
    import threading

    caches = [kv.PagedQ4Cache(1, 1, 64, n, n, 1, 16, cuda_device) for n in (8192, 2600)]
    new = [torch.ones_like(c.lengths) for c in caches]
    gate, failed = threading.Barrier(2), []

    def work(c, one):
        try:
            with torch.cuda.device(cuda_device), torch.cuda.stream(torch.cuda.Stream(cuda_device)):
                zero = torch.zeros_like(one)
                gate.wait(timeout=60)
                for _ in range(300):
                    c.resize(0, new_lengths=zero)
                    c.resize(len(one), new_lengths=one)
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # noqa: BLE001 -- shown below
            failed.append(e)

    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=x) for x in zip(caches, new)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed
    for c in caches:
        c.check()
        assert (c.lengths == 1).all() and c.free_count.item() == 0
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        caches[0].resize(8192, grow=1)
    caches[1].resize(2600, grow=1)
    graph.instantiate()
    graph.replay()
    torch.cuda.synchronize()
    assert (caches[0].lengths == 2).all() and (caches[1].lengths == 2).all()
    caches[0].check()


def test_the_most_new_tokens_that_a_call_takes(cuda_device):
    """2^31 - 1 of them (26 GB of slots and positions), into longer buffers whose ends stay as they were."""
    most, tail = 2**31 - 1, 5
    cache = kv.PagedQ4Cache(1, 1, 64, 8, 2, 4, 16, cuda_device)
    slots = torch.full((most + tail,), 7, dtype=torch.int64, device=cuda_device)
    positions = torch.full((most + tail,), 7, dtype=torch.int32, device=cuda_device)
    start = torch.empty(3, dtype=torch.int32, device=cuda_device)
    new = i32([33, 5], cuda_device)
    for shift in (0, 1):  # in 16-byte vectors, and not
        ahead = slots[:shift].clone(), positions[:shift].clone()
        N.check(N.lib().tn_kv_pages_resize(
            cache.page_table.data_ptr(), 4, 4, cache.lengths.data_ptr(), new.data_ptr(), 0, 2, cache.free_pages.data_ptr(),
            cache.free_count.data_ptr(), 8, 16, slots.data_ptr() + 8 * shift, positions.data_ptr() + 4 * shift, most,
            start.data_ptr(), cache.status.data_ptr(), torch.cuda.current_stream().cuda_stream))
        cache.check()
        first, last = (x[shift:shift + 38].tolist() for x in (slots, positions))
        rows = cache.page_table.tolist()
        at = [(b, p) for b, n in enumerate([33, 5]) for p in range(n)]
        assert first == [rows[b][p // 16] * 16 + p % 16 for b, p in at] and last == [p for _, p in at]
        for x, y in zip((slots, positions), ahead):
            assert (x[shift + 38:shift + 1000] == -1).all() and (x[most + shift - 5:most + shift] == -1).all()
            assert (x[most + shift:] == 7).all() and torch.equal(x[:shift], y)
        cache.resize(0, new_lengths=i32([0, 0], cuda_device))


@pytest.mark.parametrize("tokens", [40, 5000])
@pytest.mark.parametrize("bad", [-1, -7, 8, 1 << 30])
def test_new_tokens_in_pages_that_are_none_are_reported(cuda_device, tokens, bad):
    """A page id on the stack, or in the table, that is not one of the pool's: its tokens get no slot; the others theirs."""
    for where in ("stack", "table"):
        cache = kv.PagedQ4Cache(1, 1, 64, 8, 2, 4, 16, cuda_device)
        cache.resize(40, new_lengths=i32([0, 20], cuda_device))
        if where == "stack":
            cache.free_pages[5] = bad  # the page that the first request takes
        else:
            cache.page_table[1, 1] = bad
        slots, positions, _ = cache.resize(tokens, new_lengths=i32([5, 23], cuda_device))
        first = [2 * 16 + i for i in range(5)] if where == "table" else [-1] * 5
        second = [16 + i for i in range(4, 7)] if where == "stack" else [-1] * 3
        assert slots[:8].tolist() == first + second
        assert positions[:8].tolist() == [0, 1, 2, 3, 4, 20, 21, 22]
        assert (slots[8:] == -1).all()
        with pytest.raises(RuntimeError, match="page id"):
            cache.check()
        cache.check()


def test_a_pool_without_heads_is_refused(cuda_device):
    pool = torch.zeros((4, 0, 1, 18 * 64), dtype=torch.uint8, device=cuda_device)
    table, lengths = i32([[0], [1]], cuda_device), i32([3, 4], cuda_device)
    with pytest.raises(RuntimeError, match="multiple of"):
        kv.sdpa_q4_cache(torch.zeros((2, 4, 64), device=cuda_device), pool, table, lengths)
    with pytest.raises(RuntimeError, match="multiple of"):
        kv.sdpa_q4_decode_step(torch.zeros((2, 256), dtype=BF, device=cuda_device), rope_table(9, 64, cuda_device), pool, table,
                               lengths, 4)
    x = torch.zeros((2, 0, 64), device=cuda_device)
    with pytest.raises(RuntimeError, match="head count"):
        kv.kv_q4_append(x, x, pool, torch.zeros(2, dtype=torch.int64, device=cuda_device))


def test_grants_outlast_resizes_of_other_requests(cuda_device):
    """A request that grew steps although another one ended or came in since; one that ended, or did not grow, does not."""
    cache = kv.PagedQ4Cache(1, 2, 64, 12, 3, 4, 16, cuda_device)
    g = torch.Generator().manual_seed(9)
    x = torch.randn((50, 2, 64), generator=g).to(cuda_device)
    slots, _, _ = cache.resize(50, new_lengths=i32([20, 30, 0], cuda_device))
    cache.append(0, x, x.flip(0), slots)
    qkv = torch.randn((3, 8 * 64), generator=g).to(BF).to(cuda_device)
    rope = rope_table(64, 64, cuda_device)
    cache.resize(2, grow=1)
    cache.resize(0, new_lengths=i32([21, 0, 0], cuda_device))
    assert cache.granted.tolist() == [1, 0, 0]
    want_pool = cache.pools[0].clone()
    want = kv.sdpa_q4_decode_step(qkv, rope, want_pool, cache.page_table, cache.lengths, 4)
    out = cache.decode_step(0, qkv, rope, 4)
    assert torch.equal(out, want) and torch.equal(cache.pools[0], want_pool) and (out[0] != 0).any()
    assert (out[1:] == 0).all()
    cache.resize(40, new_lengths=i32([21, 0, 40], cuda_device))
    assert cache.granted.tolist() == [1, 0, 40]
    cache.resize(400, new_lengths=i32([21, 0, 400], cuda_device))
    assert cache.granted.tolist() == [0, 0, 0]
    with pytest.raises(RuntimeError, match="length"):
        cache.check()
    cache.resize(0, new_lengths=i32([20, 0, 40], cuda_device))
    assert cache.granted.tolist() == [0, 0, 0]
    cache.check()


@pytest.mark.parametrize("requests, width", [(3, 5), (40, 500), (2600, 8)])
def test_grants_follow_the_last_change_of_a_length(cuda_device, requests, width):
    """In one CTA and in a cluster, up and down, with calls that cannot be met between."""
    import random

    rng = random.Random(requests)
    cache = kv.PagedQ4Cache(1, 1, 64, requests * width, requests, width, 16, cuda_device)
    want = [0] * requests
    for turn in range(8):
        old = cache.lengths.tolist()
        new = [rng.choice([n, n, 0, min(n + 1, 16 * width), rng.randint(0, 16 * width)]) for n in old]
        if turn in (3, 6):
            new[rng.randrange(requests)] = 16 * width + 1
            want = [0] * requests
        else:
            want = [w if n == o else max(0, n - o) for w, n, o in zip(want, new, old)]
        cache.resize(requests * width * 16, new_lengths=i32(new, cuda_device))
        assert cache.granted.tolist() == want
        assert cache.status.item() == (2 if turn in (3, 6) else 0)
        cache.status.zero_()
