"""A paged KV cache in 4 bits, and the operators that keep and read it.

The reference's cache is dense (PreallocatedCache, torchnative/python/torchnative/
kernels/kv_cache.py:51-185: one [B, Hkv, capacity, D] buffer a layer). Here keys
and values are GGML Q4_0 blocks (4.5 bits an element, the weights' format) in
pages of `page_size` tokens, which requests take and give back as they grow and
end:

- `kv_pages_resize`: block tables and slot maps from request lengths
- `kv_q4_append`: keys and values quantised into their slots
- `sdpa_q4_cache`: attention over the cached pages, one or many tokens a request
- `sdpa_q4_decode_step`: one decode token's rotary embedding, append and
  attention
- `PagedQ4Cache`: the pools, tables and lengths of a model's layers

The compute is the C ABI's (include/torchnative_b200.h). No CPU path: a CPU
tensor is refused by name.
"""

from __future__ import annotations

import ctypes

import torch

from . import _native as N

GROUP = 16  # tokens of one head that lie together
_U8, _I32, _I64, _F32, _BF16 = torch.uint8, torch.int32, torch.int64, torch.float32, torch.bfloat16
_current_device = getattr(torch._C, "_cuda_getDevice", None)
_current_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
_capturing = getattr(torch._C, "_cuda_isCurrentStreamCapturing", None)
_TwoStrides = ctypes.c_int64 * 2
_CODE = {torch.float32: N.TN_F32, torch.bfloat16: N.TN_BF16, torch.float16: N.TN_F16}
_STATUS = {1: "not enough free pages", 2: "a request's length is outside [0, max_pages * page_size]",
           3: "more new tokens than max_tokens", 4: "more free pages than the pool has"}


def _require(op: str, device: torch.device, name: str, t: torch.Tensor, dtype: torch.dtype) -> None:
    """t on `device`, contiguous, of its dtype."""
    if t.dtype is not dtype:
        raise NotImplementedError(f"{op}: {name} must be {dtype}, got {t.dtype}")
    if t.device != device:
        raise RuntimeError(f"{op}: Expected all tensors to be on the same device, but found at least two devices, "
                           f"{device} and {t.device} ({name})")
    if not t.is_contiguous():
        raise RuntimeError(f"{op}: {name} must be contiguous")


def _require_cuda(op: str, device: torch.device) -> None:
    if device.type != "cuda":
        raise NotImplementedError(f"{op}: this is the CUDA arm (sm_100a); a {device.type} tensor belongs to "
                                  "torchnative's CPU path")


def _call(index: int, name: str, *args) -> None:
    """One library call on device `index`'s current stream; the library takes
    the current device, which may be another one."""
    fn = getattr(N.lib(), name)
    if index == _current_device():
        status = fn(*args, _current_stream(index))
    else:
        with torch.cuda.device(index):
            status = fn(*args, _current_stream(index))
    if status:
        N.check(status)


_empty_like, _contiguous = torch.empty_like, torch.contiguous_format
_empty_strided = torch.empty_strided  # on the host half of torch.empty's time


_scratch: dict = {}


def _workspace(device: torch.device, index: int, rows: int, dim: int, *shape: int) -> torch.Tensor:
    """The attention calls' scratch: one a stream, since calls on a stream run
    one after the other; a captured call gets memory of its graph's own, since
    graphs captured on one stream may be replayed on several. What a dispatch
    mode gives instead of memory (a fake tensor) is not kept."""
    key = (index, _current_stream(index), rows > 8, dim)
    ws = _scratch.get(key)
    if index == _current_device():
        capturing = _capturing()
    else:
        with torch.cuda.device(index):
            capturing = _capturing()
    if ws is None or capturing:
        tokens, heads, kv_heads, most = shape
        ws = torch.empty(N.lib().tn_sdpa_q4_workspace_bytes(tokens, heads, kv_heads, dim, most), dtype=_U8, device=device)
        if not capturing and type(ws) is torch.Tensor:
            _scratch[key] = ws
    return ws


def _table_shape(op: str, page_table: torch.Tensor, lengths: torch.Tensor):
    if page_table.dim() != 2 or lengths.shape != page_table.shape[:1]:
        raise RuntimeError(f"{op}: page_table {list(page_table.shape)} and lengths {list(lengths.shape)} do not "
                           "describe the same requests ([requests, max_pages] and [requests])")
    return page_table.shape


def _granted(op: str, device: torch.device, granted: torch.Tensor, lengths: torch.Tensor) -> int:
    _require(op, device, "granted", granted, _I32)
    if granted.shape != lengths.shape:
        raise RuntimeError(f"{op}: granted {list(granted.shape)} does not fit lengths {list(lengths.shape)}")
    address = granted.data_ptr()
    if not address and granted.numel():
        raise RuntimeError(f"{op}: granted has no memory (a fake tensor)")
    return address


def _pool_shape(op: str, pool: torch.Tensor):
    """(pages, KV heads, page size, head dimension) of a pool [pages, heads, page_size / 16, 18 D]."""
    shape = pool.shape
    if len(shape) != 4 or shape[3] % 18:
        raise RuntimeError(f"{op}: a pool is [pages, kv_heads, page_size / {GROUP}, 18 * head_dim], got "
                           f"{list(shape)}")
    pages, heads, groups, row = shape
    return pages, heads, groups * GROUP, row // 18


def kv_q4_pool(num_pages: int, kv_heads: int, head_dim: int, page_size: int, device="cuda") -> torch.Tensor:
    """A zeroed pool: `num_pages` pages of `page_size` tokens of every KV head."""
    if N.lib().tn_kv_q4_page_bytes(kv_heads, head_dim, page_size) < 0:
        raise NotImplementedError(N.last_error())
    return torch.zeros((num_pages, kv_heads, page_size // GROUP, 18 * head_dim), dtype=torch.uint8, device=device)


def kv_pages_resize(page_table: torch.Tensor, lengths: torch.Tensor, free_pages: torch.Tensor,
                    free_count: torch.Tensor, status: torch.Tensor, page_size: int, max_tokens: int, *,
                    new_lengths: torch.Tensor | None = None, grow: int = 0, granted: torch.Tensor | None = None):
    """Take every request from its length to `new_lengths`, or, without them,
    grow every request that has tokens by `grow`; returns (slots int64 and
    positions int32 [max_tokens], query_start int32 [requests + 1]) of the new
    tokens, packed request by request, -1 behind the last. Pages come from and
    go back to the stack free_pages[:free_count]; page_table, lengths,
    free_pages and free_count are updated in place. Nothing waits for the GPU:
    a call that cannot be met changes nothing, gives no token a slot and sets
    `status` (see `PagedQ4Cache.check`). `granted` (int32 [requests], zeroed
    once) keeps each request's new tokens of the last call that changed its
    length, and 0 for all after one that could not be met: what a decode step
    needs to leave the cache alone then."""
    op = "kv_pages_resize"
    device, index = page_table.device, page_table.get_device()
    if not (index >= 0 and page_table.dtype is lengths.dtype is free_pages.dtype is free_count.dtype is status.dtype is _I32
            and index == lengths.get_device() == free_pages.get_device() == free_count.get_device() == status.get_device()
            and page_table.is_contiguous() and lengths.is_contiguous() and free_pages.is_contiguous()):
        _require_cuda(op, device)
        for name, t in (("page_table", page_table), ("lengths", lengths), ("free_pages", free_pages),
                        ("free_count", free_count), ("status", status)):
            _require(op, device, name, t, _I32)
    requests, max_pages = _table_shape(op, page_table, lengths)
    if free_pages.dim() != 1 or free_count.numel() != 1 or status.numel() != 1:
        raise RuntimeError(f"{op}: free_pages is [pages], free_count and status one number each")
    if max_tokens < 0:
        raise RuntimeError(f"{op}: max_tokens must not be negative, got {max_tokens}")
    new = None
    if new_lengths is not None:
        if grow:
            raise RuntimeError(f"{op}: new_lengths or grow, not both")
        if not (new_lengths.dtype is _I32 and new_lengths.get_device() == index and new_lengths.is_contiguous()
                and new_lengths.shape == lengths.shape):
            _require(op, device, "new_lengths", new_lengths, _I32)
            raise RuntimeError(f"{op}: new_lengths {list(new_lengths.shape)} do not fit lengths {list(lengths.shape)}")
        new = new_lengths.data_ptr()
    if granted is not None:
        granted = _granted(op, device, granted, lengths)
    slots = _empty_strided((max_tokens,), (1,), dtype=_I64, device=device)
    positions = _empty_strided((max_tokens,), (1,), dtype=_I32, device=device)
    query_start = _empty_strided((requests + 1,), (1,), dtype=_I32, device=device)
    _call(index, "tn_kv_pages_resize_granted", page_table.data_ptr(), max_pages, max_pages, lengths.data_ptr(), new,
          int(grow), requests, free_pages.data_ptr(), free_count.data_ptr(), free_pages.shape[0], page_size,
          slots.data_ptr(), positions.data_ptr(), max_tokens, query_start.data_ptr(), status.data_ptr(),
          granted)
    return slots, positions, query_start


def _rows(t: torch.Tensor) -> torch.Tensor:
    """t [tokens, heads, D] with the unit inner stride and 16-byte aligned rows the kernels read, copied if need be."""
    if t.data_ptr() % 16 == 0:
        if t.is_contiguous():  # whole rows of 64 or 128
            return t
        es = t.element_size()
        if (t.stride(2) == 1 and (t.shape[0] == 1 or t.stride(0) * es % 16 == 0)
                and (t.shape[1] == 1 or t.stride(1) * es % 16 == 0)):
            return t
    return t.clone(memory_format=torch.contiguous_format)


_contiguous_rows: dict = {}


def _row_strides(t: torch.Tensor):
    """Element strides of token and head; a size-1 dimension is never stepped through."""
    if t.is_contiguous():
        key = t.shape[1:]
        strides = _contiguous_rows.get(key)
        if strides is None:
            strides = _contiguous_rows[key] = _TwoStrides(key[0] * key[1], key[1])
        return strides
    token, head, _ = t.stride()
    return _TwoStrides(token if t.shape[0] > 1 else 0, head if t.shape[1] > 1 else 0)


def kv_q4_append(key: torch.Tensor, value: torch.Tensor, pool: torch.Tensor, slots: torch.Tensor) -> None:
    """Quantise key and value [tokens, kv_heads, D] (float32, float16 or
    bfloat16) into the pool at `slots` (int64 [tokens], all different; a
    negative one skips its token), in place. Codes and scales are those of
    `torch._C._quantize(..., "q4_0")`."""
    op = "kv_q4_append"
    index = pool.get_device()
    code = _CODE.get(key.dtype)
    if not (index >= 0 and pool.dtype is _U8 and slots.dtype is _I64 and code is not None and value.dtype is key.dtype
            and index == key.get_device() == value.get_device() == slots.get_device() and pool.is_contiguous()
            and slots.is_contiguous()):
        device = pool.device
        _require_cuda(op, device)
        _require(op, device, "pool", pool, _U8)
        _require(op, device, "slots", slots, _I64)
        if code is None or value.dtype != key.dtype:
            raise NotImplementedError(f"{op}: key and value must both be float32, float16 or bfloat16, got {key.dtype} "
                                      f"and {value.dtype}")
        raise RuntimeError(f"{op}: Expected all tensors to be on the same device, but found {device}, {key.device} (key) "
                           f"and {value.device} (value)")
    pages, heads, page_size, dim = _pool_shape(op, pool)
    tokens = slots.shape[0] if slots.dim() == 1 else -1
    if key.shape != (tokens, heads, dim) or key.shape != value.shape:
        raise RuntimeError(f"{op}: key {list(key.shape)}, value {list(value.shape)} and slots {list(slots.shape)} do "
                           f"not fit a pool of {heads} heads of {dim}")
    key, value = _rows(key), _rows(value)
    _call(index, "tn_kv_q4_append", key.data_ptr(), value.data_ptr(), code, _row_strides(key),
          _row_strides(value), tokens, slots.data_ptr(), pool.data_ptr(), pages, heads, dim, page_size)


def sdpa_q4_cache(query: torch.Tensor, pool: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor, *,
                  query_start: torch.Tensor | None = None, max_tokens: int | None = None, scale: float | None = None):
    """(out, logsumexp) of attention over the cache. query [tokens, heads, D]
    holds the requests' query tokens packed, those of request b in rows
    query_start[b] to query_start[b + 1] (None: one each); they are the last of
    its lengths[b] cached tokens, and each sees the tokens up to its own. A
    token that sees none gives zeros and logsumexp 0; rows behind the last
    request's are not written. `max_tokens`, a bound on one request's query
    tokens, chooses the kernel (None: all of them). A `scale` of 0 or less, as
    none, is 1 / sqrt(D), as in the dense operator; gradients do not pass."""
    op = "sdpa_q4_cache"
    device, index = query.device, query.get_device()
    code = _CODE.get(query.dtype)
    if not (index >= 0 and code is not None and pool.dtype is _U8 and page_table.dtype is lengths.dtype is _I32
            and index == pool.get_device() == page_table.get_device() == lengths.get_device() and pool.is_contiguous()
            and page_table.is_contiguous() and lengths.is_contiguous()):
        _require_cuda(op, device)
        if code is None:
            raise NotImplementedError(f"{op}: the query must be float32, float16 or bfloat16, got {query.dtype}")
        _require(op, device, "pool", pool, _U8)
        _require(op, device, "page_table", page_table, _I32)
        _require(op, device, "lengths", lengths, _I32)
    pages, kv_heads, page_size, dim = _pool_shape(op, pool)
    requests, max_pages = _table_shape(op, page_table, lengths)
    if query.dim() != 3 or query.shape[2] != dim:
        raise RuntimeError(f"{op}: query {list(query.shape)} must be [tokens, heads, {dim}]")
    tokens, heads, _ = query.shape
    if heads == 0 or kv_heads == 0 or heads % kv_heads:
        raise RuntimeError(f"{op}: query heads ({heads}) must be a multiple of the cache's heads ({kv_heads})")
    start, most = None, 1
    if query_start is not None:
        if not (query_start.dtype is _I32 and query_start.get_device() == index and query_start.is_contiguous()
                and query_start.numel() == requests + 1):
            _require(op, device, "query_start", query_start, _I32)
            raise RuntimeError(f"{op}: query_start must have requests + 1 = {requests + 1} entries, got "
                               f"{query_start.numel()}")
        start = query_start.data_ptr()
        most = tokens if max_tokens is None else max(1, min(max_tokens, tokens))
    query = _rows(query)
    out = _empty_like(query, memory_format=_contiguous)
    lse = _empty_strided((tokens, heads), (heads, 1), dtype=_F32, device=device)
    ws = _workspace(device, index, heads // kv_heads * most, dim, tokens, heads, kv_heads, most)
    _call(index, "tn_sdpa_q4_cache", query.data_ptr(), code, _row_strides(query), tokens, heads, pool.data_ptr(),
          pages, kv_heads, dim, page_size, page_table.data_ptr(), max_pages, max_pages, lengths.data_ptr(), requests,
          start, most, out.data_ptr(), lse.data_ptr(), 0.0 if scale is None else float(scale), ws.data_ptr(), ws.numel())
    return out, lse


def sdpa_q4_decode_step(qkv: torch.Tensor, rope: torch.Tensor, pool: torch.Tensor, page_table: torch.Tensor,
                        lengths: torch.Tensor, heads: int, *, scale: float | None = None, q8=None,
                        granted: torch.Tensor | None = None) -> torch.Tensor:
    """One decode token's attention block of every request, bf16: from the
    projection rows qkv [requests, (heads + 2 kv_heads) D], rotate q and k at
    position lengths - 1 (rows of `rope` [positions, D]: cosines, then sines),
    append k and v there in 4 bits, attend. Returns [requests, heads, D]; q8 =
    (codes int8 [requests, heads D], scales and offsets float32 [requests,
    heads D / 32]) also receives its planar Q8_0, the next linear's
    activations. A request of length 0 appends nothing and gives zeros, and so
    does one with granted[b] <= 0: pass what the resize before granted. Without
    it every length counts a new token, and a step behind a resize that could
    not be met writes over the last cached ones. A position outside the page
    table or `rope` is reported (`PagedQ4Cache.check`); its request appends
    nothing and gives zeros."""
    op = "sdpa_q4_decode_step"
    device, index = qkv.device, qkv.get_device()
    if not (index >= 0 and qkv.dtype is rope.dtype is _BF16 and pool.dtype is _U8
            and page_table.dtype is lengths.dtype is _I32 and index == rope.get_device() == pool.get_device()
            == page_table.get_device() == lengths.get_device() and qkv.is_contiguous() and rope.is_contiguous()
            and pool.is_contiguous() and page_table.is_contiguous() and lengths.is_contiguous()):
        _require_cuda(op, device)
        _require(op, device, "qkv", qkv, _BF16)
        _require(op, device, "rope", rope, _BF16)
        _require(op, device, "pool", pool, _U8)
        _require(op, device, "page_table", page_table, _I32)
        _require(op, device, "lengths", lengths, _I32)
    pages, kv_heads, page_size, dim = _pool_shape(op, pool)
    requests, max_pages = _table_shape(op, page_table, lengths)
    if heads <= 0 or kv_heads == 0 or heads % kv_heads:
        raise RuntimeError(f"{op}: query heads ({heads}) must be a multiple of the cache's heads ({kv_heads})")
    if qkv.shape != (requests, (heads + 2 * kv_heads) * dim):
        raise RuntimeError(f"{op}: qkv {list(qkv.shape)} must be [{requests}, {(heads + 2 * kv_heads) * dim}]")
    if rope.dim() != 2 or rope.shape[1] != dim:
        raise RuntimeError(f"{op}: rope {list(rope.shape)} must be [positions, {dim}]")
    codes = scales = offsets = None
    if q8 is not None:
        codes, scales, offsets = q8
        _require(op, device, "codes", codes, torch.int8)
        _require(op, device, "scales", scales, _F32)
        _require(op, device, "offsets", offsets, _F32)
        if codes.numel() != requests * heads * dim or not scales.numel() == offsets.numel() == codes.numel() // 32:
            raise RuntimeError(f"{op}: q8 must be codes [{requests}, {heads * dim}], scales and offsets "
                               f"[{requests}, {heads * dim // 32}]")
        codes, scales, offsets = codes.data_ptr(), scales.data_ptr(), offsets.data_ptr()
    if granted is not None:
        granted = _granted(op, device, granted, lengths)
    out = _empty_strided((requests, heads, dim), (heads * dim, dim, 1), dtype=_BF16, device=device)
    ws = _workspace(device, index, heads // kv_heads, dim, requests, heads, kv_heads, 1)
    _call(index, "tn_sdpa_q4_decode_step_granted", qkv.data_ptr(), rope.data_ptr(), rope.shape[0], pool.data_ptr(), pages,
          heads, kv_heads, dim, page_size, page_table.data_ptr(), max_pages, max_pages, lengths.data_ptr(), requests,
          out.data_ptr(), None, codes, scales, offsets, 0.0 if scale is None else float(scale), ws.data_ptr(),
          ws.numel(), granted)
    return out


def kv_q4_dense(pool: torch.Tensor):
    """(keys, values) of a pool as float32 [pages, kv_heads, page_size, D]: the
    values its codes stand for, by plain torch operations on any device. For
    looking into a cache; attention reads the pool itself."""
    op = "kv_q4_dense"
    pages, heads, page_size, dim = _pool_shape(op, pool)
    nb = dim // 32
    kc, ks, vc, vs = pool.split([8 * dim, dim, 8 * dim, dim], -1)

    def nibbles(u):
        return torch.stack((u & 15, u >> 4), -1).flatten(-2)

    k = nibbles(kc.unflatten(-1, (16, 4, nb, 4)))[..., [0, 4, 1, 5, 2, 6, 3, 7]]  # token, t, block, element 8t + i
    k = k.transpose(-3, -2).flatten(-2)
    v = nibbles(vc.unflatten(-1, (2, 8, 4, nb, 2, 2)))  # h, g, t, block, p, element 4g + n
    v = v.permute(0, 1, 2, 3, 5, 7, 6, 4, 8).flatten(3, 5).flatten(-2)
    return tuple(((c.float() - 8.0) * s.contiguous().view(torch.float16).unflatten(-1, (16, nb)).float()[..., None])
                 .reshape(pages, heads, page_size, dim) for c, s in ((k, ks), (v, vs)))


class PagedQ4Cache:
    """The 4-bit KV cache of a model: one pool a layer, and the block table,
    lengths and free pages that all layers share. `num_pages` pages of
    `page_size` tokens serve up to `max_requests` requests of up to
    `max_pages` pages each."""

    def __init__(self, layers: int, kv_heads: int, head_dim: int, num_pages: int, max_requests: int, max_pages: int,
                 page_size: int = 64, device="cuda"):
        device = torch.device(device)
        _require_cuda("PagedQ4Cache", device)
        self.page_size = page_size
        self.pools = [kv_q4_pool(num_pages, kv_heads, head_dim, page_size, device) for _ in range(layers)]
        i32 = dict(dtype=torch.int32, device=device)
        self.page_table = torch.full((max_requests, max_pages), -1, **i32)
        self.lengths = torch.zeros(max_requests, **i32)
        # the top of the stack is its end: page 0 is taken first
        self.free_pages = torch.arange(num_pages - 1, -1, -1, **i32)
        self.free_count = torch.full((1,), num_pages, **i32)
        self.status = torch.zeros(1, **i32)
        # the new tokens that resizes gave each request, 0 behind one that was refused: for the decode steps
        self.granted = torch.zeros(max_requests, **i32)

    def nbytes(self) -> int:
        return sum(p.numel() for p in self.pools)

    def resize(self, max_tokens: int, *, new_lengths: torch.Tensor | None = None, grow: int = 0):
        """`kv_pages_resize` of this cache: (slots, positions, query_start)."""
        return kv_pages_resize(self.page_table, self.lengths, self.free_pages, self.free_count, self.status,
                               self.page_size, max_tokens, new_lengths=new_lengths, grow=grow, granted=self.granted)

    def append(self, layer: int, key: torch.Tensor, value: torch.Tensor, slots: torch.Tensor) -> None:
        kv_q4_append(key, value, self.pools[layer], slots)

    def attend(self, layer: int, query: torch.Tensor, *, query_start=None, max_tokens=None, scale=None):
        return sdpa_q4_cache(query, self.pools[layer], self.page_table, self.lengths, query_start=query_start,
                             max_tokens=max_tokens, scale=scale)

    def decode_step(self, layer: int, qkv: torch.Tensor, rope: torch.Tensor, heads: int, *, scale=None, q8=None):
        """`sdpa_q4_decode_step` of the tokens that `resize` granted; a request
        that has none, and every one behind a `resize` that could not be met,
        keeps its cache and gives zeros."""
        return sdpa_q4_decode_step(qkv, rope, self.pools[layer], self.page_table, self.lengths, heads, scale=scale,
                                   q8=q8, granted=self.granted)

    def check(self) -> None:
        """Wait for the cache's GPU and raise for a resize that could not be met
        since the last check, a page, slot or position outside its range, or a
        wait that gave up; all of it is read and cleared before one is raised."""
        with torch.cuda.device(self.status.device):
            met = None
            try:
                N.device_status()
            except (RuntimeError, TimeoutError) as e:
                met = e
            code = int(self.status.item())
            self.status.zero_()
        refused = f"kv_pages_resize: {_STATUS.get(code, code)}; that call changed nothing"
        if met is not None:
            raise type(met)(f"{refused}; {met}" if code else str(met))
        if code:
            raise RuntimeError(refused)
