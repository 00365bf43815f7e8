"""The paged 4-bit KV cache's operators, measured: block tables and slot maps from request lengths, the quantising
append, attention over the cached pages, and one decode token's attention block.

`listed()` and `draw()` give the cases, `prepare()` a user's data, `run()` one pass: the framework's calls where `own`
is true, plain torch operations otherwise. `work()` counts what a pass cannot do without; `exact()` is the same in 64
bits, written apart.

A page holds `page` tokens of every KV head as groups of 16 tokens; a group of one head is 18 * D bytes:
  K codes  [16 tokens][4 t][D/32 blocks][4 bytes]  word (t, block): nibble n < 4 is element 8t + 2n of the block's 32,
                                                   nibble 4 + n is element 8t + 2n + 1
  K scales [16 tokens][D/32] f16
  V codes  [2 h][8 g][4 t][D/32][2 tokens][2 bytes]  token 8h + 2t + (0 or 1); nibble n is element 4g + n
  V scales [16 tokens][D/32] f16
Codes and scales are GGML Q4_0's (32 elements to a block): d = m / -8 for the element m of largest magnitude,
code = min(15, trunc(x / d + 8.5)), value = (code - 8) * d, all in float32 and d kept in float16.
"""
import math

import torch

own = False

DEV = "cuda" if torch.cuda.is_available() else "cpu"
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BYTES = {"bf16": 2, "f16": 2, "f32": 4}


def listed():
    return [
        # one decode token of one conversation over a short context: the latency that a chat turn feels
        dict(name="attend_b1_s2048", op="attend", type="bf16", batch=1, heads=32, kv_heads=8, dim=128, longest=2048,
             ragged=False, tokens=1, page=64),
        # a serving batch in mid-flight: every request at another length, some slots empty, a large model's heads
        dict(name="attend_b32_ragged_s8192", op="attend", type="bf16", batch=32, heads=64, kv_heads=8, dim=128,
             longest=8192, ragged=True, tokens=1, page=64),
        # two long documents, a small model's odd heads, half precision, an odd length
        dict(name="attend_b2_s131071_f16", op="attend", type="f16", batch=2, heads=9, kv_heads=3, dim=64,
             longest=131071, ragged=False, tokens=1, page=128),
        # drafted tokens checked in one pass, in float32, small pages
        dict(name="attend_b16_draft5_f32", op="attend", type="f32", batch=16, heads=32, kv_heads=8, dim=128,
             longest=2055, ragged=True, tokens=5, page=16),
        # the next piece of two long prompts, read against everything cached before it
        dict(name="attend_b2_chunk1536", op="attend", type="bf16", batch=2, heads=32, kv_heads=8, dim=128,
             longest=9728, ragged=False, tokens=1536, page=64),
        # the keys and values of one decode step
        dict(name="append_b32", op="append", type="bf16", tokens=32, kv_heads=8, dim=128, page=64),
        # a prompt of 8192 tokens
        dict(name="append_prompt8192", op="append", type="bf16", tokens=8192, kv_heads=8, dim=128, page=64),
        # an odd number of tokens, float32, a small model's heads
        dict(name="append_1003_f32", op="append", type="f32", tokens=1003, kv_heads=3, dim=64, page=32),
        # a decode step's pages: every live request grows by a token, then the step is rolled back
        dict(name="pages_step_b32", op="pages", batch=32, longest=8192, grow=1, page=64),
        # prompts admitted to a large batch while others end, then taken back
        dict(name="pages_admit_b512", op="pages", batch=512, longest=4096, grow=0, page=16),
        # a decode token's whole attention block: rotary embedding, append, attention
        dict(name="step_b1_s2048", op="step", batch=1, heads=32, kv_heads=8, dim=128, longest=2048, ragged=False,
             page=64),
        dict(name="step_b32_ragged_s8192", op="step", batch=32, heads=32, kv_heads=8, dim=128, longest=8192,
             ragged=True, page=64),
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["attend", "attend", "attend", "append", "pages", "step"])
    page = rng.choice([16, 32, 64, 128])
    if op == "pages":
        grow = rng.choice([0, 0, 1, rng.randint(2, 9)])
        return dict(op=op, batch=log(1, 700), longest=log(16, 8000), grow=grow, page=page)
    dim = rng.choice([64, 128])
    if op == "append":
        return dict(op=op, type=rng.choice(list(TYPES)), tokens=log(1, 8000), kv_heads=rng.choice([1, 2, 3, 8]),
                    dim=dim, page=page)
    kv, rep = rng.choice([(8, 4), (8, 8), (3, 3), (1, 7), (4, 1), (2, 2)])
    c = dict(op=op, batch=log(1, 64), heads=kv * rep, kv_heads=kv, dim=dim, longest=log(1, 100000),
             ragged=rng.random() < 0.6, page=page)
    if op == "attend":
        c["type"] = rng.choice(list(TYPES))
        c["tokens"] = rng.choice([1, rng.randint(2, 16), log(17, 1500)])
        c["longest"] = max(c["longest"], c["tokens"] + rng.randint(0, 300))
    n = c.get("tokens", 1)
    # the padded scores and caches of the plain form stay below those of the largest listed cases
    while c["batch"] > 1 and (c["batch"] * c["heads"] * n * c["longest"] > 9 * 10**8
                              or c["batch"] * kv * dim * c["longest"] > 2.6 * 10**8):
        c["batch"] = c["batch"] // 2
    if c["heads"] * n * c["longest"] > 9 * 10**8:
        c["longest"] = 9 * 10**8 // (c["heads"] * n)
    return c


# ---- sizes


def _lengths(case):
    """The cached tokens of each request, those of this pass included; of a ragged batch every eighth slot is empty."""
    b, longest = case["batch"], case["longest"]
    if not case.get("ragged"):
        return [longest] * b
    n = case.get("tokens", 1)
    spread = [max(n, longest * (1 + i * 29 % b) // b - i % 3) for i in range(b)]
    return [0 if i % 8 == 7 else s for i, s in enumerate(spread)]


def _new_tokens(case):
    """Query tokens of each request: one for every slot in decode, none for an empty one otherwise; ragged batches
    draft or read differing numbers."""
    n = case.get("tokens", 1)
    if n == 1:
        return [1] * case["batch"]
    if not case["ragged"]:
        return [n] * case["batch"]
    return [0 if s == 0 else 1 + (n - 1) * (1 + i % 4) // 4 for i, s in enumerate(_lengths(case))]


def _pages_lengths(case):
    """(before, after) of the page bookkeeping: a decode step grows every live request by `grow`; otherwise prompts
    come in where slots are empty, some requests go on and some end."""
    b, longest = case["batch"], case["longest"]
    before = [0 if i % 5 == 3 else 1 + (longest - 1) * (1 + i * 29 % b) // b for i in range(b)]
    if case["grow"]:
        return before, [s + case["grow"] if s else 0 for s in before]
    return before, [longest * (1 + i % 7) // 8 if s == 0 else 0 if i % 9 == 4 else s + i % 4
                    for i, s in enumerate(before)]


def _ceil(a, b):
    return -(-a // b)


# ---- the page layout and the quantiser in plain torch

_K_ORDER = [0, 4, 1, 5, 2, 6, 3, 7]  # element 8t + i of a block is nibble _K_ORDER[i] of word t


def _nibbles(u):
    return torch.stack((u & 15, u >> 4), -1).flatten(-2)


def _bytes(n):
    n = n.unflatten(-1, (-1, 2))
    return n[..., 0] | (n[..., 1] << 4)


def _quantize(x):
    """[..., D] float32 -> (codes uint8 [..., D/32, 32], scales f16 [..., D/32])."""
    x = x.unflatten(-1, (-1, 32))
    at = x.abs().argmax(-1, keepdim=True)
    d = x.gather(-1, at) / -8.0
    inv = torch.where(d != 0, 1.0 / d, torch.zeros_like(d))
    codes = (x * inv + 8.5).clamp(0.0, 15.0).to(torch.uint8)
    return codes, d.squeeze(-1).to(torch.float16)


def _k_bytes(codes):
    """codes [..., D/32, 32] of one token -> its bytes [..., D/2] in word order (t, block)."""
    n = codes.unflatten(-1, (4, 8))
    inverse = [_K_ORDER.index(i) for i in range(8)]
    return _bytes(n[..., inverse]).transpose(-3, -2).flatten(-3)


def _v_bytes(codes):
    """codes [..., D/32, 32] of one token -> its bytes [..., 8 g, D/32, 2]."""
    return _bytes(codes.unflatten(-1, (8, 4))).transpose(-3, -2)


def _unpack(groups, dim):
    """groups [..., 18 D] uint8 -> keys and values [..., 16, D] float32."""
    nb = dim // 32
    kc, ks, vc, vs = groups.split([8 * dim, dim, 8 * dim, dim], -1)
    k = _nibbles(kc.unflatten(-1, (16, 4, nb, 4)))[..., _K_ORDER].transpose(-3, -2).flatten(-2)
    v = _nibbles(vc.unflatten(-1, (2, 8, 4, nb, 2, 2)))  # h, g, t, block, token, n
    v = v.permute(*range(v.dim() - 6), -6, -4, -2, -3, -5, -1).flatten(-6, -4).flatten(-2)
    out = []
    for codes, scales in ((k, ks), (v, vs)):
        d = scales.contiguous().view(torch.float16).unflatten(-1, (16, nb)).float()
        out.append(((codes.float() - 8.0) * d[..., None]).flatten(-2))
    return out


def _pack(k, v):
    """keys and values [..., 16, D] float32 -> groups [..., 18 D] uint8."""
    (kc, ks), (vc, vs) = _quantize(k), _quantize(v)
    vb = _v_bytes(vc).unflatten(-4, (2, 4, 2))  # h, t, token, g, block, byte
    vb = vb.permute(*range(vb.dim() - 6), -6, -3, -5, -2, -4, -1).flatten(-6)
    return torch.cat((_k_bytes(kc).flatten(-2), ks.flatten(-2).view(torch.uint8), vb, vs.flatten(-2).view(torch.uint8)),
                     -1)


# ---- a user's data


def _normal(shape, gen, dtype=torch.float32):
    return torch.randn(shape, device=DEV, generator=gen).to(dtype)


def _cache(case, lengths, gen, spare=3):
    """A pool whose pages hold quantised N(0, 1) keys (some channels larger, as trained keys have) and values, and a
    block table that takes them in no order."""
    page, hkv, dim = case["page"], case["kv_heads"], case["dim"]
    need = [_ceil(s, page) for s in lengths]
    width, total = max(max(need), 1) + 1, sum(need)
    num = total + spare
    channel = torch.where(torch.rand((hkv, 1, 1, dim), device=DEV, generator=gen) < 0.05, 4.0, 1.0)
    pool = _pack(_normal((num, hkv, page // 16, 16, dim), gen) * channel, _normal((num, hkv, page // 16, 16, dim), gen))
    order = torch.randperm(num, device=DEV, generator=gen).to(torch.int32)
    table = torch.full((len(lengths), width), -1, dtype=torch.int32)
    at, rows = 0, []
    for b, n in enumerate(need):
        rows.append((b, n, at))
        at += n
    table = table.to(DEV)
    for b, n, at in rows:
        table[b, :n] = order[at:at + n]
    return pool, table, torch.tensor(lengths, dtype=torch.int32, device=DEV)


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    op, page = case["op"], case["page"]
    s = dict(case=case, op=op)
    if op == "pages":
        before, after = _pages_lengths(case)
        b = case["batch"]
        have = [_ceil(x, page) for x in before]
        most = [_ceil(max(x, y), page) for x, y in zip(before, after)]
        num = sum(most) + 5
        order = torch.randperm(num, device=DEV, generator=gen).to(torch.int32)
        counts = torch.tensor(have, device=DEV)
        start = counts.cumsum(0) - counts
        j = torch.arange(max(most) + 1, device=DEV)[None]
        inside = j < counts[:, None]
        s["table"] = torch.where(inside, order[(start[:, None] + j).clamp(max=num - 1)], -1).to(torch.int32)
        used = sum(have)
        s["free"] = torch.zeros(num, dtype=torch.int32, device=DEV)
        s["free"][:num - used] = order[used:]
        s["count"] = torch.tensor([num - used], dtype=torch.int32, device=DEV)
        s["status"] = torch.zeros(1, dtype=torch.int32, device=DEV)
        s["lengths"] = torch.tensor(before, dtype=torch.int32, device=DEV)
        s["before"] = s["lengths"].clone()
        s["after"] = torch.tensor(after, dtype=torch.int32, device=DEV)
        s["tokens"] = sum(max(0, y - x) for x, y in zip(before, after)) + 2
        s["tokens_back"] = sum(max(0, x - y) for x, y in zip(before, after))
        return s
    if op == "append":
        n, hkv, dim = case["tokens"], case["kv_heads"], case["dim"]
        pages = _ceil(n, page) + 2
        s["pool"], _, _ = _cache(case, [pages * page], gen)
        order = torch.randperm(s["pool"].shape[0], device=DEV, generator=gen)
        tok = torch.arange(n, device=DEV) + page // 3  # a request that had a part of a page before
        s["slots"] = order[tok // page] * page + tok % page
        s["key"] = _normal((n, hkv, dim), gen, TYPES[case["type"]])
        s["value"] = _normal((n, hkv, dim), gen, TYPES[case["type"]])
        return s
    lengths = _lengths(case)
    s["pool"], s["table"], s["lengths"] = _cache(case, lengths, gen)
    hq, hkv, dim = case["heads"], case["kv_heads"], case["dim"]
    if op == "step":
        s["qkv"] = _normal((case["batch"], (hq + 2 * hkv) * dim), gen, torch.bfloat16)
        angle = torch.arange(case["longest"] + 1, device=DEV, dtype=torch.float64)[:, None] / (
            500000.0 ** (torch.arange(0, dim, 2, device=DEV, dtype=torch.float64) / dim))
        s["rope"] = torch.cat((angle.cos(), angle.sin()), 1).to(torch.bfloat16)
        return s
    new = _new_tokens(case)
    s["query"] = _normal((sum(new), hq, dim), gen, TYPES[case["type"]])
    s["most"] = max(new)
    s["start"] = None
    if case["tokens"] > 1:
        s["start"] = torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], dtype=torch.int32, device=DEV)
    return s


# ---- one pass


def run(s):
    return {"attend": _attend, "append": _append, "pages": _pages, "step": _step}[s["op"]](s)


def _attend(s):
    if own:
        from torchnative_b200 import kv_cache

        return kv_cache.sdpa_q4_cache(s["query"], s["pool"], s["table"], s["lengths"], query_start=s["start"],
                                      max_tokens=s["most"])
    return _plain_attend(s["query"], s["pool"], s["table"], s["lengths"], s["start"], s["most"])


def _plain_attend(query, pool, table, lengths, start, most):
    """Query token i of n of a request of length S attends its keys 0 .. S - n + i; one that sees none gives zeros."""
    t, hq, dim = query.shape
    hkv, page = pool.shape[1], pool.shape[2] * 16
    batch, width = table.shape
    k, v = _unpack(pool[table.clamp(min=0).long()], dim)  # [B, pages, Hkv, groups, 16, D]
    k = k.transpose(1, 2).reshape(batch, hkv, width * page, dim)
    v = v.transpose(1, 2).reshape(batch, hkv, width * page, dim)
    if start is None:
        start = torch.arange(batch + 1, device=query.device)
    first, n = start[:-1, None].long(), (start[1:] - start[:-1])[:, None]
    i = torch.arange(most, device=query.device)[None]
    row = (first + i).clamp(max=t - 1)  # [B, most]; rows past a request's n are dropped again below
    q = query[row].float().unflatten(2, (hkv, hq // hkv)).permute(0, 2, 3, 1, 4).flatten(2, 3)  # [B, Hkv, rep most, D]
    scores = (q @ k.transpose(-1, -2)).unflatten(2, (-1, most)) / math.sqrt(dim)
    sees = torch.arange(width * page, device=query.device) < (lengths[:, None] - n + i + 1)[..., None]  # [B, most, S]
    scores.masked_fill_(~sees[:, None, None], -math.inf)
    m = scores.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, 0.0, m)
    p = scores.sub_(m).exp_()
    total = p.sum(-1)
    o = (p.flatten(2, 3) @ v).unflatten(2, (-1, most)) / torch.where(total == 0, 1.0, total)[..., None]
    lse = torch.where(total == 0, 0.0, total.log() + m[..., 0])
    # token r of the packed rows is token r - start of its request
    r = torch.arange(t, device=query.device)
    b = torch.searchsorted(start[1:].contiguous(), r.to(start.dtype), right=True)
    at = r - start[b]
    o = o.flatten(1, 2)[b, :, at]
    return o.to(query.dtype), lse.flatten(1, 2)[b, :, at]


def _append(s):
    if own:
        from torchnative_b200 import kv_cache

        kv_cache.kv_q4_append(s["key"], s["value"], s["pool"], s["slots"])
    else:
        _plain_append(s["key"], s["value"], s["pool"], s["slots"])
    return s["pool"]


def _plain_append(key, value, pool, slots):
    dim, page = key.shape[-1], pool.shape[2] * 16
    nb = dim // 32
    where = (slots // page, slots % page // 16, slots % 16)
    p, g, k = (w[:, None] for w in where)
    h = torch.arange(pool.shape[1], device=pool.device)[None]
    (kc, ks), (vc, vs) = _quantize(key.float()), _quantize(value.float())
    kb, ksb, vb, vsb = pool.split([8 * dim, dim, 8 * dim, dim], -1)
    kb.unflatten(-1, (16, 8 * dim // 16))[p, h, g, k] = _k_bytes(kc)
    ksb.unflatten(-1, (16, 2 * nb))[p, h, g, k] = ks.view(torch.uint8)
    vb.unflatten(-1, (2, 8, 4, nb, 2, 2))[p, h, g, k // 8, :, k % 8 // 2, :, k % 2] = _v_bytes(vc)
    vsb.unflatten(-1, (16, 2 * nb))[p, h, g, k] = vs.view(torch.uint8)


def _pages(s):
    page, grow = s["case"]["page"], s["case"]["grow"]
    args = (s["table"], s["lengths"], s["free"], s["count"], s["status"], page)
    if own:
        from torchnative_b200 import kv_cache

        to = dict(grow=grow) if grow else dict(new_lengths=s["after"])
        there = kv_cache.kv_pages_resize(*args, s["tokens"], **to)
        back = kv_cache.kv_pages_resize(*args, s["tokens_back"], new_lengths=s["before"])
    else:
        after = torch.where(s["lengths"] > 0, s["lengths"] + grow, 0) if grow else s["after"]
        there = _plain_resize(*args, s["tokens"], after)
        back = _plain_resize(*args, s["tokens_back"], s["before"])
    return there, back, s["table"], s["lengths"], s["free"], s["count"], s["status"]


def _plain_resize(table, lengths, free, count, status, page, tokens, new):
    """Requests that shrink give their last pages back, requests that grow take pages from the top of the free stack
    (request 0's first page first); what was given back last is what was taken first. A call that cannot be met leaves
    everything and sets the status."""
    old = lengths.long()
    new = new.long()
    have, want = (old + page - 1) // page, (new + page - 1) // page
    give, take = (have - want).clamp(min=0), (want - have).clamp(min=0)
    give_at, take_at = give.cumsum(0) - give, take.cumsum(0) - take
    gives, takes = give.sum(), take.sum()
    grown = (new - old).clamp(min=0)
    start = torch.cat((grown.new_zeros(1), grown.cumsum(0)))
    top = count[0].long() + gives  # of the stack, what is given back on it
    bad = torch.where(((new < 0) | (want > table.shape[1])).any(), 2,
                      torch.where(takes > top, 1, torch.where(start[-1] > tokens, 3, 0)))
    ok = bad == 0
    j = torch.arange(table.shape[1], device=table.device)[None]
    leaves = ok & (j >= want[:, None]) & (j < have[:, None])
    enters = ok & (j >= have[:, None]) & (j < want[:, None])
    # the stack with one place more, for what is not written
    place = torch.where(leaves, top - 1 - (give_at[:, None] + j - want[:, None]), free.numel())
    stack = torch.cat((free, free.new_zeros(1))).scatter_(0, place.flatten(), table.flatten())
    free.copy_(stack[:-1])
    source = torch.where(enters, top - 1 - (take_at[:, None] + j - have[:, None]), 0)
    table.copy_(torch.where(enters, stack[source], torch.where(leaves, -1, table)))
    count.copy_(torch.where(ok, top - takes, count[0].long()).reshape(1))
    status.copy_(torch.where(status == 0, bad.to(torch.int32), status))
    start = torch.where(ok, start, 0)
    lengths.copy_(torch.where(ok, new, old))
    r = torch.arange(tokens, device=table.device)
    b = torch.searchsorted(start[1:].contiguous(), r, right=True)
    live = b < table.shape[0]
    b = b.clamp(max=table.shape[0] - 1)
    position = old[b] + r - start[b]
    slot = table[b, (position // page).clamp(0, table.shape[1] - 1)].long() * page + position % page
    return (torch.where(live, slot, -1), torch.where(live, position, -1).to(torch.int32), start.to(torch.int32))


def _step(s):
    c = s["case"]
    if own:
        from torchnative_b200 import kv_cache

        out = kv_cache.sdpa_q4_decode_step(s["qkv"], s["rope"], s["pool"], s["table"], s["lengths"], c["heads"])
        return out, s["pool"]
    hq, hkv, dim = c["heads"], c["kv_heads"], c["dim"]
    q, k, v = s["qkv"].unflatten(1, (-1, dim)).split([hq, hkv, hkv], 1)
    position = (s["lengths"].long() - 1)
    cos, sin = s["rope"][position.clamp(min=0)].float()[:, None].chunk(2, -1)
    q, k = _rotate(q, cos, sin), _rotate(k, cos, sin)
    page = c["page"]
    slot = s["table"].gather(1, (position.clamp(min=0) // page)[:, None])[:, 0].long() * page + position % page
    # an empty request has no slot: what would be its token goes where the first live one's goes, and is the same
    live = position >= 0
    one = live.to(torch.int32).argmax()
    slot = torch.where(live, slot, slot[one])
    k = torch.where(live[:, None, None], k, k[one])
    v = torch.where(live[:, None, None], v, v[one])
    _plain_append(k, v, s["pool"], slot)
    out, _ = _plain_attend(q, s["pool"], s["table"], s["lengths"], None, 1)
    return out, s["pool"]


def _rotate(x, cos, sin):
    """The rotary embedding (halves rotated against each other), rounded once, to the model's bf16."""
    a, b = x.float().chunk(2, -1)
    return torch.cat((a * cos - b * sin, b * cos + a * sin), -1).to(x.dtype)


# ---- what a pass cannot do without


def work(case):
    op = case["op"]
    if op == "pages":
        before, after = _pages_lengths(case)
        moved = sum(abs(_ceil(y, case["page"]) - _ceil(x, case["page"])) for x, y in zip(before, after))
        tokens = sum(max(0, y - x) for x, y in zip(before, after))
        back = sum(max(0, x - y) for x, y in zip(before, after))
        # there and back: lengths read and written, a page id read and written, a token's slot and position written
        return {"bytes": 2 * (3 * 4 * case["batch"] + 8 * moved) + 12 * (tokens + back), "flops": 2 * (moved + tokens + back)}
    dim, hkv = case["dim"], case["kv_heads"]
    row = 9 * dim // 8  # a token of one head, K and V: 4 bits an element and 16 bits a block of 32
    if op == "append":
        n = case["tokens"] * hkv
        return {"bytes": n * (2 * dim * BYTES[case["type"]] + row) + 8 * case["tokens"], "flops": 6 * n * 2 * dim}
    hq, lengths = case["heads"], _lengths(case)
    if op == "step":
        b = case["batch"]
        return {"bytes": sum(lengths) * hkv * row + b * dim * (2 * (2 * hq + 2 * hkv) + 2),
                "flops": 4 * hq * dim * sum(lengths)}
    new = _new_tokens(case)
    pairs = sum(sum(max(0, s - n + i + 1) for i in range(n)) for s, n in zip(lengths, new))
    return {"bytes": sum(lengths) * hkv * row + sum(new) * hq * (2 * dim * BYTES[case["type"]] + 4),
            "flops": 4 * hq * dim * pairs}


# ---- the same in 64 bits, request by request


def exact(case, seed):
    if case["op"] in ("pages", "append"):
        return None  # whole numbers and the codes of a 4-bit format: nothing that is rounded
    s = prepare(case, seed)
    query, lengths, new = s.get("query"), _lengths(case), _new_tokens(case)
    if case["op"] == "step":
        query = _exact_step(s, case, lengths)
    out, lse = [], []
    at = 0
    for b, (length, n) in enumerate(zip(lengths, new)):
        o, e = _exact_request(query[at:at + n].double(), s["pool"], s["table"][b], length, case)
        out.append(o)
        lse.append(e)
        at += n
    if case["op"] == "step":
        return torch.cat(out), None
    return torch.cat(out), torch.cat(lse)


def _exact_step(s, case, lengths):
    """Rotates and appends with complex numbers; the model's tensors between two operators are bf16."""
    dim, hq, hkv = case["dim"], case["heads"], case["kv_heads"]
    rows = s["qkv"].double().view(len(lengths), hq + 2 * hkv, dim)
    at = torch.tensor([max(x - 1, 0) for x in lengths], device=rows.device)
    turn = torch.complex(s["rope"][at, :dim // 2].double(), s["rope"][at, dim // 2:].double())[:, None]
    z = torch.complex(rows[..., :dim // 2], rows[..., dim // 2:])[:, :hq + hkv] * turn
    turned = torch.cat((z.real, z.imag), -1).to(torch.bfloat16)
    for b, length in enumerate(lengths):
        if length:
            position = length - 1
            slot = int(s["table"][b, position // case["page"]]) * case["page"] + position % case["page"]
            _plain_append(turned[b:b + 1, hq:], s["qkv"].view(len(lengths), -1, dim)[b:b + 1, hq + hkv:], s["pool"],
                          torch.tensor([slot], device=rows.device))
    return turned[:, :hq]


def _exact_request(q, pool, table, length, case):
    n, hq, dim = q.shape
    hkv, page, nb = case["kv_heads"], case["page"], dim // 32
    out, lse = torch.zeros_like(q), torch.zeros((n, hq), dtype=torch.float64, device=q.device)
    if length == 0 or n == 0:
        return out, lse
    groups = pool[table[:_ceil(length, page)].long()].transpose(0, 1).reshape(hkv, -1, 18 * dim)
    kw = groups[..., :8 * dim].contiguous().view(torch.int32).view(hkv, -1, 16, 4, nb)
    vw = groups[..., 9 * dim:17 * dim].contiguous().view(torch.int32).view(hkv, -1, 2, 8, 4, nb)
    kd = groups[..., 8 * dim:9 * dim].contiguous().view(torch.float16).view(hkv, -1, nb).double()
    vd = groups[..., 17 * dim:].contiguous().view(torch.float16).view(hkv, -1, nb).double()
    count = groups.shape[1] * 16
    k = torch.empty((hkv, groups.shape[1], 16, nb, 4, 8), dtype=torch.float64, device=q.device)
    v = torch.empty((hkv, groups.shape[1], 2, 4, 2, nb, 8, 4), dtype=torch.float64, device=q.device)
    for i in range(8):
        code = ((kw >> (4 * i)) & 15).double() - 8
        k[..., 2 * (i % 4) + i // 4] = code.transpose(-1, -2)
        code = ((vw >> (4 * i)) & 15).double() - 8  # h, g, t, block
        v[:, :, :, :, i // 4, :, :, i % 4] = code.permute(0, 1, 2, 4, 5, 3)
    k = (k.view(hkv, count, nb, 32) * kd[..., None]).view(hkv, count, dim)[:, :length]
    v = (v.view(hkv, count, nb, 32) * vd[..., None]).view(hkv, count, dim)[:, :length]
    last = torch.arange(n, device=q.device)[:, None] + length - n  # the last key that a token sees
    hidden = torch.arange(length, device=q.device)[None] > last
    for h in range(hq):
        x = (q[:, h] @ k[h * hkv // hq].T) / math.sqrt(dim)
        x = x.masked_fill(hidden, -math.inf)
        e = torch.logsumexp(x, -1)
        sees = last[:, 0] >= 0
        w = torch.where(sees[:, None], (x - torch.where(sees, e, 0.0)[:, None]).exp(), 0.0)
        out[:, h] = w @ v[h * hkv // hq]
        lse[:, h] = torch.where(sees, e, 0.0)
    return out, lse
