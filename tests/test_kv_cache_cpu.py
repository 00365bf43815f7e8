"""The paged 4-bit KV cache without a GPU: what the calls refuse, page sizes in bytes, the layout's plain reading."""

import ctypes

import pytest
import torch

from torchnative_b200 import _native as N
from torchnative_b200 import build, kv_cache as kv

I64x2 = ctypes.c_int64 * 2
A = 1 << 20  # stands for an aligned device address: every call here is refused before one is used


@pytest.fixture(scope="module")
def lib():
    build.build()
    return N.lib()


def test_page_bytes(lib):
    assert lib.tn_kv_q4_page_bytes(8, 128, 64) == 8 * 64 * 128 * 2 * 18 // 32
    assert lib.tn_kv_q4_page_bytes(3, 64, 16) == 3 * 16 * 64 * 2 * 18 // 32
    for heads, dim, page in ((8, 128, 48), (8, 128, 8), (8, 128, 2048), (8, 96, 64), (0, 128, 64), (8, 128, 0)):
        assert lib.tn_kv_q4_page_bytes(heads, dim, page) == -1, (heads, dim, page)


RESIZE = dict(table=A, stride=4, max_pages=4, lengths=A, new=None, grow=1, requests=2, free=A, count=A, num_pages=8,
              page=64, slots=A, positions=A, max_tokens=2, start=A, status=A)


@pytest.mark.parametrize("change, status", [
    (dict(page=24), N.TN_ERR_NOT_IMPLEMENTED), (dict(requests=8193), N.TN_ERR_NOT_IMPLEMENTED),
    (dict(requests=-1), N.TN_ERR_SHAPE), (dict(stride=3), N.TN_ERR_SHAPE), (dict(grow=-1), N.TN_ERR_SHAPE),
    (dict(num_pages=-1), N.TN_ERR_SHAPE), (dict(max_tokens=1 << 31), N.TN_ERR_SHAPE),
    (dict(max_pages=1 << 26, stride=1 << 26), N.TN_ERR_SHAPE),
    (dict(count=None), N.TN_ERR_INVALID), (dict(lengths=None), N.TN_ERR_INVALID), (dict(table=None), N.TN_ERR_INVALID),
    (dict(slots=None), N.TN_ERR_INVALID), (dict(start=None), N.TN_ERR_INVALID), (dict(status=None), N.TN_ERR_INVALID),
    (dict(free=None), N.TN_ERR_INVALID), (dict(new=A), N.TN_ERR_INVALID)])
def test_resize_refusals(lib, change, status):
    assert lib.tn_kv_pages_resize(*{**RESIZE, **change}.values(), None) == status
    assert "tn_kv_pages_resize" in N.last_error()


APPEND = dict(k=A, v=A, dtype=N.TN_BF16, ks=I64x2(1024, 128), vs=I64x2(1024, 128), tokens=3, slots=A, pool=A, pages=4,
              heads=8, dim=128, page=64)


@pytest.mark.parametrize("change, status", [
    (dict(dtype=N.TN_F64), N.TN_ERR_NOT_IMPLEMENTED), (dict(dim=96), N.TN_ERR_NOT_IMPLEMENTED),
    (dict(page=40), N.TN_ERR_NOT_IMPLEMENTED), (dict(tokens=-1), N.TN_ERR_SHAPE), (dict(heads=0), N.TN_ERR_SHAPE),
    (dict(k=None), N.TN_ERR_INVALID), (dict(slots=None), N.TN_ERR_INVALID), (dict(pool=None), N.TN_ERR_INVALID),
    (dict(pool=A + 8), N.TN_ERR_INVALID), (dict(k=A + 2), N.TN_ERR_INVALID), (dict(ks=I64x2(1023, 128)), N.TN_ERR_INVALID),
    (dict(vs=I64x2(1024, 12)), N.TN_ERR_INVALID)])
def test_append_refusals(lib, change, status):
    assert lib.tn_kv_q4_append(*{**APPEND, **change}.values(), None) == status
    assert "tn_kv_q4_append" in N.last_error()


ATTEND = dict(q=A, dtype=N.TN_BF16, qs=I64x2(4096, 128), tokens=2, heads=32, pool=A, pages=4, kv_heads=8, dim=128,
              page=64, table=A, stride=4, max_pages=4, lengths=A, requests=2, start=None, most=1, out=A, lse=A, scale=0.0,
              ws=A, ws_bytes=1 << 40)


@pytest.mark.parametrize("change, status", [
    (dict(dtype=N.TN_F64), N.TN_ERR_NOT_IMPLEMENTED), (dict(dim=80), N.TN_ERR_NOT_IMPLEMENTED),
    (dict(page=65), N.TN_ERR_NOT_IMPLEMENTED), (dict(heads=12), N.TN_ERR_SHAPE), (dict(tokens=3), N.TN_ERR_SHAPE),
    (dict(stride=2), N.TN_ERR_SHAPE), (dict(requests=65536), N.TN_ERR_SHAPE), (dict(q=None), N.TN_ERR_INVALID),
    (dict(out=None), N.TN_ERR_INVALID), (dict(lengths=None), N.TN_ERR_INVALID), (dict(table=None), N.TN_ERR_INVALID),
    (dict(q=A + 4), N.TN_ERR_INVALID), (dict(qs=I64x2(4096, 129)), N.TN_ERR_INVALID), (dict(ws=None), N.TN_ERR_SHAPE),
    (dict(ws_bytes=16), N.TN_ERR_SHAPE)])
def test_attend_refusals(lib, change, status):
    assert lib.tn_sdpa_q4_cache(*{**ATTEND, **change}.values(), None) == status
    assert "tn_sdpa_q4_cache" in N.last_error()


STEP = dict(qkv=A, rope=A, rows=100, pool=A, pages=4, heads=32, kv_heads=8, dim=128, page=64, table=A, stride=4,
            max_pages=4, lengths=A, requests=2, out=A, lse=None, codes=None, scales=None, offsets=None, scale=0.0, ws=A,
            ws_bytes=1 << 40)


@pytest.mark.parametrize("change, status", [
    (dict(heads=72), N.TN_ERR_NOT_IMPLEMENTED), (dict(dim=256), N.TN_ERR_NOT_IMPLEMENTED), (dict(rows=0), N.TN_ERR_SHAPE),
    (dict(heads=33), N.TN_ERR_SHAPE), (dict(qkv=None), N.TN_ERR_INVALID), (dict(qkv=A + 8), N.TN_ERR_INVALID),
    (dict(codes=A), N.TN_ERR_INVALID), (dict(ws_bytes=0), N.TN_ERR_SHAPE)])
def test_step_refusals(lib, change, status):
    assert lib.tn_sdpa_q4_decode_step(*{**STEP, **change}.values(), None) == status
    assert "tn_sdpa_q4_decode_step" in N.last_error()


def test_empty_calls_are_no_ops(lib):
    assert lib.tn_kv_q4_append(*{**APPEND, "tokens": 0}.values(), None) == N.TN_OK
    assert lib.tn_sdpa_q4_cache(*{**ATTEND, "tokens": 0, "requests": 0}.values(), None) == N.TN_OK
    assert lib.tn_sdpa_q4_decode_step(*{**STEP, "requests": 0}.values(), None) == N.TN_OK


def test_cpu_tensors_are_refused_by_name(lib):
    i32 = torch.zeros(2, dtype=torch.int32)
    table, pool = torch.zeros((2, 3), dtype=torch.int32), torch.zeros((4, 2, 1, 18 * 64), dtype=torch.uint8)
    with pytest.raises(NotImplementedError, match="kv_pages_resize"):
        kv.kv_pages_resize(table, i32, i32, i32[:1], i32[:1], 16, 4)
    with pytest.raises(NotImplementedError, match="kv_q4_append"):
        kv.kv_q4_append(torch.zeros(1, 2, 64), torch.zeros(1, 2, 64), pool, torch.zeros(1, dtype=torch.int64))
    with pytest.raises(NotImplementedError, match="sdpa_q4_cache"):
        kv.sdpa_q4_cache(torch.zeros(2, 4, 64), pool, table, i32)
    with pytest.raises(NotImplementedError, match="sdpa_q4_decode_step"):
        kv.sdpa_q4_decode_step(torch.zeros(2, 512).bfloat16(), torch.zeros(9, 64).bfloat16(), pool, table, i32, 4)
    with pytest.raises(NotImplementedError, match="PagedQ4Cache"):
        kv.PagedQ4Cache(1, 2, 64, 4, 2, 3, device="cpu")
    with pytest.raises(NotImplementedError, match="head dimensions"):
        kv.kv_q4_pool(1, 1, 96, 16, "cpu")


@pytest.mark.parametrize("dim", [64, 128])
def test_layout(lib, dim):
    """Every code and scale of a group lies where the header says (kv_q4.cuh), by writing one at a time."""
    nb = dim // 32
    for key in range(16):
        for e in range(0, dim, 5):
            block, i = e // 32, e % 32
            pool = torch.full((1, 1, 1, 18 * dim), 0x88, dtype=torch.uint8)  # every code 8: value 0
            for base in (8 * dim, 17 * dim):
                pool[..., base:base + dim] = torch.full((16 * nb,), 0.5, dtype=torch.float16).view(torch.uint8)
            t, j = i // 8, i % 8
            nib = j // 2 + 4 * (j % 2)
            at = key * (dim // 2) + (t * nb + block) * 4 + nib // 2
            pool[..., at] = 0x80 | 0x0A if nib % 2 == 0 else 0xA0 | 0x08
            g, n = i // 4, i % 4
            at = 9 * dim + (key // 8) * 4 * dim + ((g * 4 + key % 8 // 2) * nb + block) * 4 + (key % 2) * 2 + n // 2
            pool[..., at] = 0x80 | 0x03 if n % 2 == 0 else 0x30 | 0x08
            k, v = kv.kv_q4_dense(pool)
            assert k[0, 0, key, e] == 1.0 and k.count_nonzero() == 1, (key, e)
            assert v[0, 0, key, e] == -2.5 and v.count_nonzero() == 1, (key, e)
