"""Plain 64-bit reference of the paged 4-bit KV cache's operators, and the error bounds their tests hold them to."""

import math

import torch

from torchnative_b200 import kv_cache as kv

HALF_STEP = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}
# half the spacing of a type's subnormals: float16 values below 2^-14 are multiples of 2^-24, float32's and bfloat16's
# lie below what any result here is compared at
HALF_SUBNORMAL = {torch.bfloat16: 2.0**-134, torch.float16: 2.0**-25, torch.float32: 2.0**-150}


class State:
    """A cache with every page's contents random, and requests whose pages lie in no order."""

    def __init__(self, lengths, kv_heads, dim, page_size, device, seed=0, spare=3, width=None, magnitude=1.0):
        g = torch.Generator().manual_seed(seed)
        self.g, self.page_size, self.dim, self.kv_heads, self.device = g, page_size, dim, kv_heads, device
        need = [-(-max(n, 0) // page_size) for n in lengths]
        num = sum(need) + spare
        self.pool = kv.kv_q4_pool(num, kv_heads, dim, page_size, device)
        k = torch.randn((num * page_size, kv_heads, dim), generator=g) * magnitude
        v = torch.randn((num * page_size, kv_heads, dim), generator=g) * magnitude
        kv.kv_q4_append(k.to(device), v.to(device), self.pool, torch.arange(num * page_size, device=device))
        order = torch.randperm(num, generator=g).to(torch.int32)
        width = max(max(need, default=0), 1) if width is None else width
        table = torch.full((len(lengths), width), -1, dtype=torch.int32)
        at = 0
        for b, n in enumerate(need):
            table[b, :n] = order[at:at + n]
            at += n
        self.table = table.to(device)
        self.lengths = torch.tensor(lengths, dtype=torch.int32, device=device)

    def randn(self, *shape, dtype=torch.float32):
        return torch.randn(shape, generator=self.g).to(dtype).to(self.device)


def dense_request(pool, table_row, length, page_size):
    """(keys, values) [heads, length, D] float64 of one request."""
    pages = table_row[:-(-length // page_size)].long()
    return tuple(x[pages].transpose(0, 1).flatten(1, 2)[:, :length].double() for x in kv.kv_q4_dense(pool))


def attention(q, pool, table, lengths, page_size, query_start=None, scale=None, tiles=False):
    """(out, lse, bound, lse_bound), all float64; rows that belong to no request are NaN.

    The bounds, first order, for kernels that multiply exact 4-bit codes with queries and probabilities carried in
    11-bit (22-bit for float32) significands, sums in float32 of at most half a step 2^-24 an addition:
      a score sums D products in any order and meets at most 8 further roundings, and a query element far below its
      row's largest may be off by 2^-24 of that largest: ds = scale * ((D + 8) 2^-24 sum|q k| + 2^-24 max|q| sum|k|);
      the exponential, its argument and the running maximum add 2^-20 and 2^-23 |s| (arguments in float32 units of
      log 2 are subtracted once the product is rounded), so a probability is off by e = 2 max(ds + 2^-22 |s|) + 2^-20
      relative (numerator and denominator);
      a probability times a value's scale is rounded to the carrier, half a step of it; for bfloat16 results the
      probability is rounded to it before as well, 2 * 2^-11 in all, an eighth of the step of the result;
      sums over n keys in at most n / 16 + 64 additions of partial sums: (n / 16 + 64) 2^-24;
      below float16's normal numbers those roundings are half a subnormal step, 2^-25, where the row's largest
      probability, times a scale of the larger of 1 and twice the largest scale d, stands for 2^10 at least: at most
      2 * 2^-35 max(1, 2 d), times a code of at most 8, for every key that the row sees;
      in the tcgen05 tiles (`tiles`) keys and values are float16 themselves, a group of 16 tokens taken to a largest
      scale below 1 by a power of two, at most twice its largest scale: a scale 2^-14 or less of that is rounded to
      subnormals, half a step 2^-25, times a code of at most 8: 2^-22 of the power, 2^-21 of the largest scale, in
      every element of a key (times its query element) and of a value (times its probability);
      the result is rounded to its type: half a step of its value, or half the spacing of the subnormals."""
    h = {torch.float32: 2.0**-22, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-10}[q.dtype]
    step = HALF_STEP[q.dtype]
    t, hq, dim = q.shape
    scale = 1 / math.sqrt(dim) if scale is None else scale
    out = torch.full((t, hq, dim), math.nan, dtype=torch.float64)
    lse = torch.full((t, hq), math.nan, dtype=torch.float64)
    bound, lse_bound = torch.zeros_like(out), torch.zeros_like(lse)
    starts = list(range(t + 1)) if query_start is None else query_start.tolist()
    for b, length in enumerate(lengths.tolist()):
        n = starts[b + 1] - starts[b]
        if n <= 0:
            continue
        length = max(0, min(length, table.shape[1] * page_size))
        rows = slice(starts[b], starts[b] + n)
        out[rows], lse[rows] = 0.0, 0.0
        if length == 0:
            continue
        k, v = (x.cpu().repeat_interleave(hq // x.shape[0], 0) for x in dense_request(pool, table[b], length, page_size))
        x = q[rows].double().cpu().transpose(0, 1)  # [heads, n, D]
        s = x @ k.transpose(1, 2) * scale
        ds = scale * 2.0**-24 * ((dim + 8) * (x.abs() @ k.abs().transpose(1, 2))
                                 + x.abs().amax(-1, keepdim=True) * k.abs().sum(-1)[:, None])
        sees = torch.arange(length)[None] < (length - n + 1 + torch.arange(n))[:, None]
        dmax = [(x.abs().amax() / 8).item() for x in (k, v)]  # a block's largest element has code 0: eight scales
        if tiles:
            ds = ds + scale * 2.0**-21 * dmax[0] * x.abs().sum(-1, keepdim=True)
        s = s.masked_fill(~sees, -math.inf)
        some = sees.any(-1)
        e = torch.logsumexp(s, -1)
        p = torch.where(some[:, None], (s - e[..., None]).exp(), 0.0)
        ds = torch.where(sees, ds + 2.0**-22 * torch.where(sees, s, 0.0).abs(), 0.0).amax(-1)
        rel = 2 * ds + 2.0**-20 + (length / 16 + 64) * 2.0**-24
        o = p @ v
        out[rows] = o.transpose(0, 1)
        lse[rows] = torch.where(some, e, 0.0).transpose(0, 1)
        floor = sees.sum(-1)[:, None] * 16 * 2.0**-35 * max(1.0, 2 * dmax[1]) + (2.0**-21 * dmax[1] if tiles else 0.0)
        bound[rows] = ((rel + h)[..., None] * (p @ v.abs()) + floor + (step * o.abs()).clamp(min=HALF_SUBNORMAL[q.dtype]) + 1e-30).transpose(0, 1)
        lse_bound[rows] = (rel + 2.0**-22 * e.abs()).transpose(0, 1)
    return out, lse, bound, lse_bound


def check_attention(got, q, pool, table, lengths, page_size, query_start=None, scale=None, tiles=False):
    out, lse = (x.double().cpu() for x in got)
    want, want_lse, bound, lse_bound = attention(q, pool, table, lengths, page_size, query_start, scale, tiles)
    rows = ~want_lse.isnan().any(-1)
    assert torch.isfinite(out[rows]).all()
    over = ((out - want).abs() - bound)[rows]
    assert (over <= 0).all(), f"out: {over.max().item()} over the bound {bound[rows].flatten()[over.argmax()].item()}"
    over = ((lse - want_lse).abs() - lse_bound)[rows]
    assert (over <= 0).all(), f"lse: {over.max().item()} over the bound"


def resize(table, lengths, free, count, new, page_size, max_tokens):
    """kv_pages_resize in plain Python on lists; returns (table, lengths, free, count, slots, positions, start, code)."""
    b, width = len(lengths), len(table[0]) if table else 0
    table, free = [list(r) for r in table], list(free)
    pages = lambda n: -(-n // page_size)  # noqa: E731
    nothing = (table, list(lengths), free, count, [-1] * max_tokens, [-1] * max_tokens, [0] * (b + 1))
    if any(not 0 <= n <= width * page_size for n in list(new) + list(lengths)):
        return (*nothing, 2)
    gives = sum(max(0, pages(o) - pages(n)) for o, n in zip(lengths, new))
    takes = sum(max(0, pages(n) - pages(o)) for o, n in zip(lengths, new))
    if count < 0 or count + gives > len(free):
        return (*nothing, 4)
    if takes > count + gives:
        return (*nothing, 1)
    if sum(max(0, n - o) for o, n in zip(lengths, new)) > max_tokens:
        return (*nothing, 3)
    given = []
    for i in range(b):
        for j in range(pages(new[i]), pages(lengths[i])):
            given.append(table[i][j])
            table[i][j] = -1
    for page in reversed(given):
        free[count] = page
        count += 1
    slots, positions, start = [], [], [0]
    for i in range(b):
        for j in range(pages(lengths[i]), pages(new[i])):
            count -= 1
            table[i][j] = free[count]
        for pos in range(lengths[i], new[i]):
            slots.append(table[i][pos // page_size] * page_size + pos % page_size)
            positions.append(pos)
        start.append(len(slots))
    pad = [-1] * (max_tokens - len(slots))
    return table, list(new), free, count, slots + pad, positions + pad, start, 0
