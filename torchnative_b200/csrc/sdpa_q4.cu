// sdpa_q4.cu -- attention over the paged 4-bit KV cache.
//
// Token i of the n query tokens of a request whose cache holds S tokens (its
// own included) attends keys 0 .. S - n + i:
//   s_j = scale * q . (d_j * (code_j - 8)),  out = sum_j e^(s_j - m) v_j / l,
//   lse = m + log l;
// a token that sees no key gives zeros and lse 0, as the dense operator does.
#include <algorithm>
#include <atomic>
#include <chrono>

#include "sdpa_q4.cuh"

namespace tn {
namespace {

// ---- the kernel
//
// One unit of work is 32 tokens of one (request, row tile, KV head); a row tile
// is 8 NT of the request's query rows (tokens times the heads that share the KV
// head), and an item is all units of one of them. The items of a call stand in
// one line, each as long as its units plus what an item costs besides, and CTA c
// of G takes the c-th part of the line: every CTA gets as much whatever the
// lengths, which only the device knows.
//
// A CTA is W consumer warps and four producer warps, one CTA an SM. Unit i of a
// CTA goes to warp i mod W, through stage i / W of a ring that the copy warps'
// bulk copies fill (three of them, in a decode step two: one's copies were issued
// too slowly for twelve consumers; the third then brings the new tokens); a stage
// is filled again when every warp is through with it, so that the warps stay
// together: without that bound the SM's scheduler let some run ahead, and the
// last ones ended alone (127 us for 82 at 2 x 100,000 tokens of 8 heads, then).
// The first producer warp prepares each item's queries.
//
// What bounds it: the consumers' own latencies. A unit (bf16, D 128) is ~580
// instructions, 26 us of issue at one a cycle for 2 x 100,000 tokens of 8 heads of
// 128, which take 55 us (4.2 TB/s, 65% of a copy's rate): a scheduler issues in
// 54% of the cycles, and its three consumer warps wait for their chain of scores,
// vote, exponents and products, for the tensor and conversion pipes, and at an
// item's end for one another. Of shorter lines start and join take more: issue in
// 46% of the cycles for 32 ragged requests, 34% for drafts of 5 in float32; one
// request of 2048 takes 10.4 us, ~3 us to the first products, ~4 us for the join.
//
// Per 16 tokens a warp computes, with m16n8k16 tensor instructions,
//   S^T[16 tokens, 8 rows] = sum over blocks b of d_k[token, b] * (codes_b . q_b)
//   O^T[D, 8 rows] += sum over blocks: codes_b^T . (p[token, row] * d_v[token, b])
// so that the 4-bit codes enter the products as the small integers they are
// (exact in f16), the tall side of both products is the cache's, and a tile of 8
// rows wastes nothing. A code costs about one instruction to unpack: masks put
// the nibble below a float16 exponent (1024 + c, or 64 + c for a nibble at bit
// 4), and 1032 or 72 goes off again, for a part of K in the accumulators' start.
// The scores' fragment is turned into the second product's operand by a register
// transpose (movmatrix).
//
// p is 2^(s - ref) times 2^10, f16, where ref follows the row's maximum by more
// than 2^5 only (a vote per unit; out = O / l holds for any ref), and goes down
// when the value scales are above 1, so that p * d_v stays in f16's range. For a
// bf16 result p is one f16 term, and rounded again after its value's scale: each
// time by 2^-11 at most, random from key to key, where the result's own rounding
// is 2^-8. That shows as other neighbours of a result near the middle between two
// (9e-4 of its norm), not as error: 0.0017 of it against 64 bits, as with float32
// probabilities rounded once. For f16 and float32 results p * d_v has two terms.
// The sums l and the products' accumulators are float32.
constexpr int kMaxGrid = 148;  // CTAs whose parts a workspace holds
constexpr int kUnitGroups = 2, kUnit = kUnitGroups * kKvGroup;
constexpr float kBias = 10.0f, kSlack = 5.0f;
// What an item costs besides its units (queries, the warps' results joined), in units: with 8, 12, 16, 20 the ragged
// batch of 32 up to 8192 tokens (heads of 128, 8 of them) takes 47.4, 43.5, 41.8, 41.8 us, one request of 8192 12.7,
// 12.9, 12.4, 12.9.
constexpr int kItemCost = 16;
// A CTA has 2^kMinPlaces places of the line before another one is used: with 8, 16, 32 of them one request of 2048
// takes 10.1, 10.4, 11.6 us, of 8192 tokens 13.3, 12.4, 13.0.
constexpr int kMinPlaces = 4;

// What the producer tells the consumers of an item.
struct Item {
    int end;             // no item: the work is done
    int g0, g1;          // this CTA's units of it
    int i0;              // the CTA's units before
    int whole, c0, c1;   // all of its units; otherwise the CTAs that have some
    int h, S;
    int new_unit;        // decode step: the unit of the new token, -1 where this CTA has it not
    int single;          // the request has one query token
    int rows, row0;      // query rows of the tile, of the request before it
    int first, all_see;  // the request's first packed token; keys that every row of the tile sees
};

// A token's bytes in its group: K words, V pieces by element, scales.
template <int D>
struct NewToken {
    uint32_t k[D / 8];
    uint16_t v[D / 4];
    __half ks[D / 32], vs[D / 32];
    int key;  // its place in the group, -1: none
};

template <typename T, int D, int NT>
struct Shape {
    static constexpr bool F32 = sizeof(T) == 4, BF = std::is_same<T, __nv_bfloat16>::value;
    static constexpr int NQ = F32 ? 2 : 1;  // f16 terms of a query element
    static constexpr int NP = BF ? 1 : 2;   // f16 terms of a probability
    static constexpr int NB = D / 32;
    // Consumer warps, and the registers of a thread: what the four producer warps do not need goes to them (one CTA has
    // the 65,536 of its SM).
    static constexpr int W = NT == 2 ? 8 : 12;
    static constexpr int CONSUMER_REGS = NT == 2 ? 208 : 152, PRODUCER_REGS = NT == 2 ? 88 : 56;
    static_assert(W * 32 * CONSUMER_REGS + 128 * PRODUCER_REGS <= (NT == 2 ? 384 * 168 : 512 * 128), "what the CTA is launched with");
    static constexpr int STAGES = D == 64 ? 4 : 3;
    static constexpr int UNIT = kUnitGroups * KvQ4<D>::GROUP_BYTES;
    static constexpr int RING = W * STAGES * UNIT;
    static constexpr int ROW = D + 4;  // floats of a row of the merge buffer: rows 2t of a fragment differ in their banks
    static constexpr int MERGE = W * 8 * ROW * 4;
    // an item's queries, a lane's data as it takes them
    struct Slot {
        uint4 q[NT][NB][NQ][32];
        float2 start[NT][NB][32];  // what a score's accumulator starts from, for the columns 2t, 2t + 1
        float2 to_log2[NT][32];
        int2 limit[NT][32];  // keys that the columns' rows see
        Item item;
        NewToken<D> added;  // decode step: the token that the item's last unit gets
    };
    static constexpr int SMEM = RING + MERGE + 2 * (int)sizeof(Slot);
    static_assert(kMaxGrid * 8 * 8 <= MERGE, "the weights of an item's parts fit");
    static_assert(SMEM <= 226 * 1024, "shared memory of one SM");
};

struct Split {
    Attend a;
    float *part_o;        // [kMaxGrid][2][8 NT][D]
    float *part_ml;       // [kMaxGrid][2][8 NT][2]
    unsigned long long *flags;  // [kMaxGrid][2]
    unsigned long long nonce;
    uint32_t f16_1024, f16_64;  // 1024 and 64 as half2: here so that the compiler keeps them in registers
    // decode step
    const __nv_bfloat16 *qkv, *rope;
    int places;  // positions that a new token may have: the table's, and the rotary table's
    int8_t *codes;
    float *scales, *offsets;
    const int *granted;  // [requests] new tokens that the resize gave, or NULL: one to each
    // The tokens of request b, its new one among them: none where the resize gave none, so that nothing is appended
    // over what the cache holds, and none where the new one has no place, so that what lies there is not read.
    __device__ __forceinline__ int step_length(int b) const {
        const int n = a.c.lengths[b], new_tokens = granted ? granted[b] : 1;
        return new_tokens > 0 && (unsigned)n <= (unsigned)places ? n : 0;
    }
};

__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1, const float (&c)[4]) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}

// A place in the line of units: group g of item (b, tile u, head h), whose
// groups this CTA has from `from` to `upto`. `rel` is the place of the item's
// group 0 against the first of the CTA's `len` places.
template <int RT, bool STEP>
struct Cursor {
    int b, u, h, G, rel;
    int S, n, first, tiles;

    __device__ __forceinline__ void load_request(const Split &s) {
        const Attend &p = s.a;
        S = STEP ? s.step_length(b) : p.c.length(b);
        n = p.query_tokens(b, &first);
        tiles = (n * p.rep + RT - 1) / RT;
    }
    // units that the tile's last row sees; 1 where it sees none, so that someone writes its zeros
    __device__ __forceinline__ int tile_units(const Attend &p, int tile) const {
        const int last = n == 1 ? 0 : min(n - 1, (tile * RT + RT - 1) / p.rep);
        return max(1, (S - n + last + kUnit) / kUnit);
    }
    __device__ __forceinline__ long long request_places(const Attend &p) const {
        long long places = 0;
#pragma unroll 1
        for (int t = 0; t < tiles; ++t) places += tile_units(p, t) + kItemCost;
        return places * p.c.kv_heads;
    }
    __device__ __forceinline__ int from() const { return max(0, -rel); }
    __device__ __forceinline__ int upto(int len) const { return min(G, len - rel); }
    // The next item; past the last one rel is beyond every len.
    __device__ __forceinline__ void next_item(const Split &s) {
        const Attend &p = s.a;
        rel += G + kItemCost;
        if (++h < p.c.kv_heads) return;
        h = 0;
        if (++u >= tiles) {
            u = 0;
#pragma unroll 1
            do {
                if (++b >= p.c.requests) {
                    rel = INT32_MAX / 2;
                    G = 1;
                    return;
                }
                load_request(s);
            } while (tiles == 0);
        }
        G = tile_units(p, u);
    }
};

// The rotary embedding of the lane's elements (32 b + 8 t .. + 7 of every block
// b) of a row: halves rotated against each other, rounded once, to bf16.
template <int D>
__device__ __forceinline__ void rotate(const __nv_bfloat16 *rope, int t, float (&x)[D / 32][8]) {
    constexpr int H = D / 64;
#pragma unroll
    for (int b = 0; b < H; ++b) {
        float c[8], s[8];
        load8<__nv_bfloat16>(rope + b * 32 + t * 8, c);
        load8<__nv_bfloat16>(rope + D / 2 + b * 32 + t * 8, s);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float x1 = x[b][i], x2 = x[b + H][i];
            x[b][i] = round_bf16(x1 * c[i] - x2 * s[i]);
            x[b + H][i] = round_bf16(x2 * c[i] + x1 * s[i]);
        }
    }
}

// One warp: the new token's key (rotated) and value of head h at position pos,
// in 4 bits, into the cache and into `added`, from where the warp that has its
// unit puts it into its copy.
template <int D>
__device__ __forceinline__ void append_new(const Split &p, int b, int h, int pos, NewToken<D> &added) {
    using Q = KvQ4<D>;
    constexpr int NB = Q::NB, H = D / 64;
    const Attend &a = p.a;
    const int lane = threadIdx.x & 31, t = lane & 3, block = (lane >> 2) % NB, is_v = (lane >> 2) / NB % 2;
    uint8_t *group = nullptr;
    if (pos >= 0) {
        group = a.c.group<D>(b, h, pos >> 4);
    } else if (a.c.lengths[b] > p.places && (!p.granted || p.granted[b] > 0)) {
        record_bad_page(a.c.err);
    }
    if (lane == 0) added.key = group ? pos & 15 : -1;
    if (!group) return;
    const __nv_bfloat16 *row = p.qkv + ((int64_t)b * (a.heads + 2 * a.c.kv_heads) + a.heads + (is_v ? a.c.kv_heads : 0) + h) * D;
    float x[8];
    load8<__nv_bfloat16>(row + block * 32 + t * 8, x);
    if (!is_v) {
        const int first = block % H;
        float y[8], c[8], s[8];
        load8<__nv_bfloat16>(row + (block + H) % NB * 32 + t * 8, y);
        load8<__nv_bfloat16>(p.rope + (int64_t)pos * D + first * 32 + t * 8, c);
        load8<__nv_bfloat16>(p.rope + (int64_t)pos * D + D / 2 + first * 32 + t * 8, s);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = round_bf16(block < H ? x[i] * c[i] - y[i] * s[i] : x[i] * c[i] + y[i] * s[i]);
    }
    const float d = q4_0_scale(q4_0_extreme(x)), inv = q4_0_inverse(d);
    if (lane >= 8 * NB) return;
    const int key = pos & 15;
    const __half d16 = __float2half_rn(d);
    if (is_v) {
        const uint32_t w = q4_0_v_halves(x, inv);
        *reinterpret_cast<uint16_t *>(group + Q::v_half(key, 2 * t, block)) = added.v[block * 8 + 2 * t] = (uint16_t)w;
        *reinterpret_cast<uint16_t *>(group + Q::v_half(key, 2 * t + 1, block)) = added.v[block * 8 + 2 * t + 1] = (uint16_t)(w >> 16);
        if (t == 0) *reinterpret_cast<__half *>(group + Q::v_scale(key, block)) = added.vs[block] = d16;
    } else {
        *reinterpret_cast<uint32_t *>(group + Q::k_word(key, t, block)) = added.k[t * NB + block] = q4_0_k_word(x, inv);
        if (t == 0) *reinterpret_cast<__half *>(group + Q::k_scale(key, block)) = added.ks[block] = d16;
    }
}

// One warp: the new token into its group's copy in shared memory.
template <int D>
__device__ __forceinline__ void patch_new(const NewToken<D> &added, uint8_t *buf) {
    using Q = KvQ4<D>;
    const int lane = threadIdx.x & 31, key = added.key;
    if (lane < D / 8) *reinterpret_cast<uint32_t *>(buf + Q::K_CODES + key * (D / 2) + lane * 4) = added.k[lane];
    if (lane < D / 4) *reinterpret_cast<uint16_t *>(buf + Q::v_half(key, lane & 7, lane >> 3)) = added.v[lane];
    if (lane < D / 32) {
        *reinterpret_cast<__half *>(buf + Q::k_scale(key, lane)) = added.ks[lane];
        *reinterpret_cast<__half *>(buf + Q::v_scale(key, lane)) = added.vs[lane];
    }
    fence_proxy_async_smem();  // before the bulk copy that the stage gets next
    __syncwarp();
}

template <typename T>
__device__ __forceinline__ void store4(void *out, int64_t at, const float (&v)[4]) {
    if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<float4 *>(static_cast<float *>(out) + at) = make_float4(v[0], v[1], v[2], v[3]);
    } else {
        T e[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (std::is_same<T, __half>::value)
                e[i] = __float2half_rn(v[i]);
            else
                e[i] = __float2bfloat16_rn(v[i]);
        }
        uint2 w;
        memcpy(&w, e, 8);
        *reinterpret_cast<uint2 *>(static_cast<T *>(out) + at) = w;
    }
}

// Four finished values of one row (d .. d + 3 of query head hq of packed token r).
template <typename T, int D, bool STEP>
__device__ __forceinline__ void finish4(const Split &p, int r, int hq, int d, const float (&v)[4]) {
    const int64_t at = ((int64_t)r * p.a.heads + hq) * D + d;
    store4<T>(p.a.out, at, v);
    if constexpr (STEP) {
        if (p.codes) {
            // planar Q8_0 (k_quants.rs:676-706) of the bf16 output: 8 neighbouring lanes hold a block of 32
            const unsigned gm = 0xffu << (threadIdx.x & 24);
            float q[4], amax = 0.0f;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                q[e] = __bfloat162float(__float2bfloat16_rn(v[e]));
                amax = fmaxf(amax, fabsf(q[e]));
            }
#pragma unroll
            for (int off = 1; off < 8; off <<= 1) amax = fmaxf(amax, __shfl_xor_sync(gm, amax, off));
            const float dq = __fdiv_rn(amax, 127.0f), id = (dq != 0.0f) ? __fdiv_rn(1.0f, dq) : 0.0f;
            uint32_t word = 0;
            int sum = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float t = roundf(__fmul_rn(q[e], id));
                const int c = !(t == t) ? 0 : (t <= -128.0f ? -128 : (t >= 127.0f ? 127 : __float2int_rz(t)));
                sum += c;
                word |= (uint32_t)(c & 0xff) << (8 * e);
            }
#pragma unroll
            for (int off = 1; off < 8; off <<= 1) sum += __shfl_xor_sync(gm, sum, off);
            *reinterpret_cast<uint32_t *>(p.codes + at) = word;
            if ((threadIdx.x & 7) == 0) {
                p.scales[at / 32] = __half2float(__float2half_rn(dq));
                p.offsets[at / 32] = 12582912.0f + 8.0f * (float)sum;
            }
        }
    }
}

__device__ __forceinline__ void bar_consumers(int threads) { asm volatile("bar.sync 1, %0;" ::"r"(threads) : "memory"); }

// The producer's view of the line: the first place of CTA c.
__device__ __forceinline__ long long line_start(int c, long long per, int rest) { return c * per + min(c, rest); }
// The CTA that has `place`; a whole warp asks.
__device__ __forceinline__ int line_owner(long long place, int grid, long long per, int rest) {
    int before = 0;
#pragma unroll 1
    for (int c0 = 0; c0 < grid; c0 += 32) {
        const int c = c0 + (threadIdx.x & 31);
        before += __popc(__ballot_sync(0xffffffffu, c < grid && line_start(c, per, rest) <= place));
    }
    return before - 1;
}

template <int REGS>
__device__ __forceinline__ void more_registers() {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGS));
}
template <int REGS>
__device__ __forceinline__ void fewer_registers() {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS));
}

// One warp: the item's queries; lane (g, t) holds row g, elements 32 b + 8 t ..
// + 7 of each block.
template <typename T, int D, int NT, bool STEP>
__device__ __forceinline__ void load_queries(const Split &p, const Cursor<8 * NT, STEP> &at, float (&x)[NT][D / 32][8]) {
    const Attend &a = p.a;
    const int lane = threadIdx.x & 31, lt = lane & 3, row0 = at.u * 8 * NT;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const int row = row0 + nt * 8 + (lane >> 2);
        const int tok = at.n == 1 ? 0 : row / a.rep, hq = at.h * a.rep + row - tok * a.rep;
#pragma unroll
        for (int b = 0; b < D / 32; ++b)
#pragma unroll
            for (int i = 0; i < 8; ++i) x[nt][b][i] = 0.0f;
        if (row < at.n * a.rep) {
            const T *src;
            if constexpr (STEP)
                src = reinterpret_cast<const T *>(p.qkv) + ((int64_t)at.b * (a.heads + 2 * a.c.kv_heads) + hq) * D;
            else
                src = static_cast<const T *>(a.q) + (at.first + tok) * a.q_token + hq * a.q_head;
#pragma unroll
            for (int b = 0; b < D / 32; ++b) load8<T>(src + b * 32 + lt * 8, x[nt][b]);
        }
        if constexpr (STEP) {
            rotate<D>(p.rope + (int64_t)max(0, at.S - 1) * D, lt, x[nt]);
        }
    }
}

// The same warp: into the slot, as the first product's B fragments.
template <typename T, int D, int NT, bool STEP>
__device__ __forceinline__ void put_queries(const Split &p, const Cursor<8 * NT, STEP> &at, const float (&q)[NT][D / 32][8],
                                            typename Shape<T, D, NT>::Slot &slot) {
    using H = Shape<T, D, NT>;
    constexpr int NB = H::NB;
    const Attend &a = p.a;
    const int lane = threadIdx.x & 31, lt = lane & 3, row0 = at.u * 8 * NT;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const int row = row0 + nt * 8 + (lane >> 2);
        const bool live = row < at.n * a.rep;
        const int tok = at.n == 1 ? 0 : row / a.rep;
        const float(&x)[NB][8] = q[nt];
        // the row's largest magnitude goes to [2^13, 2^14): no element overflows f16, and one that loses bits there
        // lies 2^27 below it
        float scale = 1.0f, back = 1.0f;
        if constexpr (!std::is_same<T, __half>::value) {
            float amax = 0.0f;
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int i = 0; i < 8; ++i) amax = fmaxf(amax, fabsf(x[b][i]));
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
            if (amax > 0.0f && amax < INFINITY) {
                const int e = min(max(267 - (int)(__float_as_uint(amax) >> 23), 1), 253);
                scale = __uint_as_float((uint32_t)e << 23);
                back = __uint_as_float((uint32_t)(254 - e) << 23);
            }
        }
        float sums[NB];
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            uint32_t f16[H::NQ][4];
            sums[b] = 0.0f;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float x0 = x[b][2 * j] * scale, x1 = x[b][2 * j + 1] * scale;
                f16[0][j] = pack_f16(x0, x1);
                const float2 f = unpack_f16(f16[0][j]);
                if constexpr (H::NQ == 2) f16[1][j] = pack_f16(x0 - f.x, x1 - f.y);
                if (j & 1) sums[b] += f.x + f.y;
            }
#pragma unroll
            for (int k = 0; k < H::NQ; ++k) slot.q[nt][b][k][lane] = make_uint4(f16[k][0], f16[k][1], f16[k][2], f16[k][3]);
            sums[b] += __shfl_xor_sync(0xffffffffu, sums[b], 1);
            sums[b] += __shfl_xor_sync(0xffffffffu, sums[b], 2);
        }
        const int seen = live ? at.S - at.n + tok + 1 : 0;  // keys that row g sees
        const float c = a.scale * 1.4426950408889634f * back;
        const int from0 = 8 * lt, from1 = from0 + 4;  // lanes of rows 2t and 2t + 1
        slot.to_log2[nt][lane] = make_float2(__shfl_sync(0xffffffffu, c, from0), __shfl_sync(0xffffffffu, c, from1));
        slot.limit[nt][lane] = make_int2(__shfl_sync(0xffffffffu, seen, from0), __shfl_sync(0xffffffffu, seen, from1));
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const float s0 = __shfl_sync(0xffffffffu, sums[b], from0), s1 = __shfl_sync(0xffffffffu, sums[b], from1);
            slot.start[nt][b][lane] = H::F32 ? make_float2(0.0f, 0.0f) : make_float2(-72.0f * s0, -72.0f * s1);
        }
    }
}

template <typename T, int D, int NT, bool STEP>
__global__ void __launch_bounds__(32 * (Shape<T, D, NT>::W + 4), 1) sdpa_q4_kernel(const Split p) {
    using Q = KvQ4<D>;
    using H = Shape<T, D, NT>;
    constexpr int NB = Q::NB, RT = 8 * NT, W = H::W, STAGES = H::STAGES, THREADS = 32 * W;
    constexpr bool F32 = H::F32, BF = H::BF;
    constexpr int NQ = H::NQ, NP = H::NP;
    // A decode step has a warp for the new tokens. (No more than stages: a copy warp's last stage, COPY_WARPS before, was free by
    // the time its turn came, so that the one it waits for now is at most one phase of its barrier behind.)
    constexpr int COPY_WARPS = STEP ? 2 : 3;
    static_assert(COPY_WARPS <= STAGES, "a wait tells two phases apart, not three");
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ __align__(8) uint64_t full[STAGES], empty[STAGES], q_full[2], q_empty[2], new_full[2];
    __shared__ uint8_t gone_sm[STAGES][W];  // per unit, a bit for each group without a page
    __shared__ float ml_sm[W][8][2], sum_sm[8][2];
    __shared__ int is_last, stop;
    uint8_t *ring = smem;
    float *merge = reinterpret_cast<float *>(smem + H::RING);
    typename H::Slot *slots = reinterpret_cast<typename H::Slot *>(smem + H::RING + H::MERGE);

    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, lg = lane >> 2, lt = lane & 3;
    const Attend &a = p.a;
    if (tid == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], W);
        }
        for (int s = 0; s < 2; ++s) {
            mbar_init(&q_full[s], 1);
            mbar_init(&new_full[s], 1);
            mbar_init(&q_empty[s], W);
        }
        stop = 0;
        fence_mbar_init();
    }
    __syncthreads();
    pdl_launch_dependents();
    pdl_wait();

    if (warp >= W) {
        fewer_registers<H::PRODUCER_REGS>();
        // ---- a producer: this CTA's part of the line
        Cursor<RT, STEP> at;
        long long total = 0, own = 0;
#pragma unroll 1
        for (int b0 = 0; b0 < a.c.requests; b0 += 32) {
            own = 0;
            at.b = b0 + lane;
            if (at.b < a.c.requests) {
                at.load_request(p);
                own = at.request_places(a);
            }
            long long w = own;
#pragma unroll
            for (int off = 16; off; off >>= 1) w += __shfl_xor_sync(0xffffffffu, w, off);
            total += w;
        }
        const int grid = (int)min((long long)gridDim.x, max(1ll, total >> kMinPlaces));
        const int cta = blockIdx.x;
        int len = 0;
        const long long per = total >> 31 ? total / grid : (unsigned)total / (unsigned)grid;
        const int rest = (int)(total - per * grid);
        const long long lo = line_start(cta, per, rest);
        if (cta < grid && total > 0) {
            len = (int)(line_start(cta + 1, per, rest) - lo);
            long long place = 0;  // of the current request, then tile
#pragma unroll 1
            for (int b0 = 0;; b0 += 32) {
                if (a.c.requests > 32) {
                    own = 0;
                    at.b = b0 + lane;
                    if (at.b < a.c.requests) {
                        at.load_request(p);
                        own = at.request_places(a);
                    }
                }
                long long upto = own;
#pragma unroll
                for (int off = 1; off < 32; off <<= 1) {
                    const long long v = __shfl_up_sync(0xffffffffu, upto, off);
                    if (lane >= off) upto += v;
                }
                const unsigned past = __ballot_sync(0xffffffffu, place + upto > lo);
                if (past) {
                    const int l0 = __ffs(past) - 1;
                    place += __shfl_sync(0xffffffffu, upto - own, l0);
                    at.b = b0 + l0;
                    break;
                }
                place += __shfl_sync(0xffffffffu, upto, 31);
            }
            at.load_request(p);
#pragma unroll 1
            for (at.u = 0;; ++at.u) {
                at.G = at.tile_units(a, at.u);
                const long long places = (long long)(at.G + kItemCost) * a.c.kv_heads;
                if (place + places > lo) break;
                place += places;
            }
            at.h = 0;
#pragma unroll 1
            while (place + at.G + kItemCost <= lo) place += at.G + kItemCost, ++at.h;
            at.rel = (int)(place + kItemCost - lo);
        } else {
            at.rel = 0;  // len is 0: nothing to do
        }

        if (STEP && warp == W + 3) {
            // ---- new tokens, one item ahead of the consumers like their queries
#pragma unroll 1
            for (int m = 0;; ++m) {
#pragma unroll 1
                while (at.rel < len && at.from() >= at.upto(len)) at.next_item(p);
                if (at.rel >= len) return;
                const bool ok = m < 2 || mbar_wait(&q_empty[m & 1], (m / 2 - 1) & 1);
                if (__any_sync(0xffffffffu, !ok)) {
                    if (lane == 0) record_device_error(a.c.err, DEV_ERR_WAIT_EMPTY);
                    return;
                }
                if (at.upto(len) == at.G) append_new<D>(p, at.b, at.h, at.S - 1, slots[m & 1].added);
                __syncwarp();
                if (lane == 0) mbar_arrive(&new_full[m & 1]);
                at.next_item(p);
            }
        }
        if (warp > W) {
            // ---- copies, the stages in turn to two or three warps: lanes 2w and 2w + 1 find the two groups of warp w's units, every W-th of the CTA's; groups that
            // lie together (a page's) come in one copy. (A copy's addresses are a warp's, not a lane's.)
            static_assert(2 * W <= 32, "a lane for each group");
            constexpr int WARPS = COPY_WARPS;
            int k = warp - W - 1, g = at.from() + (lane >> 1) + k * W;
            bool have = lane < 2 * W && len > 0, broken = false;
#pragma unroll 1
            for (;; k += WARPS) {
#pragma unroll 1
                while (have && g >= at.upto(len)) {  // g lies behind the item's units: on to the item that has it
                    if (at.rel >= len) {
                        have = false;
                    } else {
                        g -= max(at.from(), at.upto(len));
                        at.next_item(p);
                        g += at.from();
                    }
                }
                __syncwarp();
                if (!__any_sync(0xffffffffu, have)) break;
                const uint8_t *src = nullptr;
                if (have) {
                    const int group = g * kUnitGroups + (lane & 1);
                    if (group * kKvGroup < at.S) src = a.c.group_of_row<D>(a.c.table + at.b * a.c.table_stride, at.h, group);
                    g += WARPS * W;
                }
                __syncwarp();
                const unsigned there = __ballot_sync(0xffffffffu, src != nullptr);
                const unsigned long long addr = reinterpret_cast<unsigned long long>(src);
                const unsigned long long prev = __shfl_up_sync(0xffffffffu, addr, 1);
                const bool follows = lane > 0 && src && (there >> (lane - 1) & 1) && prev + Q::GROUP_BYTES == addr;
                const unsigned stops = __ballot_sync(0xffffffffu, !follows);
                unsigned heads = there & stops;
                const int run = __ffs((stops >> lane >> 1) | (1u << (31 - lane)));  // groups from here to the next stop
                const int s = k % STAGES;
                if (k >= STAGES && !mbar_wait(&empty[s], (k / STAGES - 1) & 1)) broken = true;
                if (__any_sync(0xffffffffu, broken)) break;
                if (lane < W) gone_sm[s][lane] = (uint8_t)(~there >> (2 * lane) & 3);
                __syncwarp();
                if (lane == 0) mbar_arrive_expect_tx(&full[s], (uint32_t)__popc(there) * Q::GROUP_BYTES);
                uint8_t *dst = ring + s * W * H::UNIT;
#pragma unroll 1
                while (heads) {
                    const int j = __ffs(heads) - 1;
                    heads &= heads - 1;
                    const uint8_t *from = reinterpret_cast<const uint8_t *>(__shfl_sync(0xffffffffu, addr, j));
                    const int n = __shfl_sync(0xffffffffu, run, j);
                    if (lane == 0) bulk_g2s(dst + j * Q::GROUP_BYTES, from, (uint32_t)(n * Q::GROUP_BYTES), &full[s]);
                }
            }
            if (__any_sync(0xffffffffu, broken)) {
                // this warp's last copies (a bounded wait) before the shared memory goes
                if (lane == 0) record_device_error(a.c.err, DEV_ERR_WAIT_EMPTY);
                if (k >= WARPS) mbar_wait(&full[(k - WARPS) % STAGES], ((k - WARPS) / STAGES) & 1);
            }
            return;
        }

        // ---- items: their queries, one item ahead of the consumers
        int i0 = 0;
        bool broken = false;
#pragma unroll 1
        for (int m = 0;; ++m) {
#pragma unroll 1
            while (at.rel < len && at.from() >= at.upto(len)) at.next_item(p);
            typename H::Slot &slot = slots[m & 1];
            const bool end = at.rel >= len;
            if (m >= 2 && !mbar_wait(&q_empty[m & 1], (m / 2 - 1) & 1)) broken = true;
            if (__any_sync(0xffffffffu, broken)) {
                if (lane == 0) record_device_error(a.c.err, DEV_ERR_WAIT_EMPTY);
                return;
            }
            if (!end) {
                const int g0 = at.from(), g1 = at.upto(len), row0 = at.u * RT, rows = min(RT, at.n * a.rep - row0);
                float q[NT][NB][8];
                load_queries<T, D, NT, STEP>(p, at, q);
                put_queries<T, D, NT, STEP>(p, at, q, slot);
                Item it;
                it.end = 0;
                it.g0 = g0, it.g1 = g1, it.i0 = i0;
                it.whole = g0 == 0 && g1 == at.G;
                it.c0 = it.c1 = cta;
                if (!it.whole) {
                    it.c0 = line_owner(lo + at.rel, grid, per, rest);
                    it.c1 = line_owner(lo + at.rel + at.G - 1, grid, per, rest);
                }
                it.h = at.h, it.S = at.S;
                it.single = at.n == 1;
                it.new_unit = STEP && g1 == at.G ? at.G - 1 : -1;
                it.rows = rows, it.row0 = row0, it.first = at.first;
                it.all_see = at.S - at.n + (at.n == 1 ? 0 : row0 / a.rep) + 1;
                if (lane == 0) slot.item = it;
                i0 += g1 - g0;
            } else if (lane == 0) {
                slot.item.end = 1;
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&q_full[m & 1]);
            if (end) return;
            at.next_item(p);
        }
    }

    // ---- a consumer
    more_registers<H::CONSUMER_REGS>();
    const uint32_t f16_1024 = p.f16_1024, f16_64 = p.f16_64;
    int my_i = warp, my_k = 0;
    bool broken = false;
#pragma unroll 1
    for (int m = 0;; ++m) {
        typename H::Slot &slot = slots[m & 1];
        if (warp == 0 && !mbar_wait(&q_full[m & 1], (m / 2) & 1)) {
            record_device_error(a.c.err, DEV_ERR_WAIT_FULL);
            stop = 1;
        }
        bar_consumers(THREADS);  // and the merge buffer is free again
        if (*(volatile int *)&stop) return;
        const Item it = slot.item;
        if (it.end) return;
        uint32_t qf[NT][NB][NQ][4];
        float start[NT][NB][2];
        float to_log2[NT][2];
        int limit[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int b = 0; b < NB; ++b) {
#pragma unroll
                for (int q = 0; q < NQ; ++q) *reinterpret_cast<uint4 *>(qf[nt][b][q]) = slot.q[nt][b][q][lane];
                *reinterpret_cast<float2 *>(start[nt][b]) = slot.start[nt][b][lane];
            }
            *reinterpret_cast<float2 *>(to_log2[nt]) = slot.to_log2[nt][lane];
            *reinterpret_cast<int2 *>(limit[nt]) = slot.limit[nt][lane];
        }

        float o[NT][NB][2][4], l[NT][2], off[NT][2];
        float high[NT][2];  // the row's reference + kSlack: scores above move it
        // Value scales up to vlim = 2^voff need no lower reference. A bf16 result's probabilities are f16 themselves
        // and must stay in range; in two terms their products with the scales only.
        float vlim = NP == 1 ? 1.0f : 0.0f, voff = 0.0f;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int j = 0; j < 2; ++j) l[nt][j] = 0.0f, high[nt][j] = -INFINITY, off[nt][j] = kBias;
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int k = 0; k < 2; ++k)
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[nt][b][k][i] = 0.0f;
        }

        // One unit, tokens token0 .. + 31; `masked` where a row may not see all of them, or a group is gone.
        auto take = [&](const uint8_t *unit_buf, int token0, uint32_t gone, auto mask) {
            constexpr bool masked = decltype(mask)::value;
            float s[kUnitGroups][NT][4];
            bool low = false;
            float vmax = 0.0f;
#pragma unroll
            for (int u = 0; u < kUnitGroups; ++u) {
                const uint8_t *buf = unit_buf + u * Q::GROUP_BYTES;
                // ---- scores
                uint32_t kw[2][NB];
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const uint8_t *src = buf + Q::K_CODES + (lg + 8 * k) * (D / 2) + lt * NB * 4;
                    if constexpr (NB == 4)
                        *reinterpret_cast<uint4 *>(kw[k]) = *reinterpret_cast<const uint4 *>(src);
                    else
                        *reinterpret_cast<uint2 *>(kw[k]) = *reinterpret_cast<const uint2 *>(src);
                }
                uint32_t ks[2][NB / 2];
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const uint8_t *src = buf + Q::K_SCALES + (lg + 8 * k) * NB * 2;
                    if constexpr (NB == 4)
                        *reinterpret_cast<uint2 *>(ks[k]) = *reinterpret_cast<const uint2 *>(src);
                    else
                        ks[k][0] = *reinterpret_cast<const uint32_t *>(src);
                }
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    uint32_t e0[4], e1[4];
                    unpack_codes<!F32>(kw[0][b], e0, f16_1024, f16_64);
                    unpack_codes<!F32>(kw[1][b], e1, f16_1024, f16_64);
                    const float2 f0 = unpack_f16(ks[0][b / 2]), f1 = unpack_f16(ks[1][b / 2]);
                    const float d0 = b & 1 ? f0.y : f0.x, d1 = b & 1 ? f1.y : f1.x;
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        const float c0[4] = {start[nt][b][0], start[nt][b][1], start[nt][b][0], start[nt][b][1]};
                        float acc[4];
                        mma16816(acc, e0[0], e1[0], e0[1], e1[1], qf[nt][b][0][0], qf[nt][b][0][1], c0);
                        mma16816(acc, e0[2], e1[2], e0[3], e1[3], qf[nt][b][0][2], qf[nt][b][0][3], acc);
                        if constexpr (NQ == 2) {
                            mma16816(acc, e0[0], e1[0], e0[1], e1[1], qf[nt][b][1][0], qf[nt][b][1][1], acc);
                            mma16816(acc, e0[2], e1[2], e0[3], e1[3], qf[nt][b][1][2], qf[nt][b][1][3], acc);
                        }
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const float d = i < 2 ? d0 : d1;
                            s[u][nt][i] = b == 0 ? acc[i] * d : fmaf(acc[i], d, s[u][nt][i]);
                        }
                    }
                }
                // ---- references that are too low for a score, or for a value scale
                const uint32_t vs_word =
                    lane < 8 * NB ? *reinterpret_cast<const uint32_t *>(buf + Q::V_SCALES + lane * 4) : 0u;
                const float2 vsf = unpack_f16(vs_word & 0x7fff7fffu);
                float v = fmaxf(vsf.x, vsf.y);
                if constexpr (masked) {
                    if (token0 + u * kKvGroup + lane / (NB / 2) >= it.S || (gone >> u & 1)) v = 0.0f;
                }
                vmax = fmaxf(vmax, v);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        s[u][nt][i] *= to_log2[nt][i & 1];
                        if constexpr (masked) {
                            if (token0 + u * kKvGroup + lg + 8 * (i >> 1) >= limit[nt][i & 1] || (gone >> u & 1))
                                s[u][nt][i] = -INFINITY;
                        }
                        low |= s[u][nt][i] > high[nt][i & 1];
                    }
            }
            if (__any_sync(0xffffffffu, low || vmax > vlim)) {
#pragma unroll
                for (int o2 = 16; o2; o2 >>= 1) vmax = fmaxf(vmax, __shfl_xor_sync(0xffffffffu, vmax, o2));
                vmax = fminf(vmax, 65504.0f);
                if (vmax > vlim) {  // the power of two above it
                    const uint32_t e = (__float_as_uint(vmax) >> 23) + 1;
                    vlim = __uint_as_float(e << 23);
                    voff = (float)((int)e - 127);
                }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        float m = fmaxf(s[0][nt][j], s[0][nt][j + 2]);
#pragma unroll
                        for (int u = 1; u < kUnitGroups; ++u) m = fmaxf(m, fmaxf(s[u][nt][j], s[u][nt][j + 2]));
#pragma unroll
                        for (int o2 = 4; o2 < 32; o2 <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o2));
                        m = fmaxf(m, high[nt][j] - kSlack);
                        if (m == -INFINITY) continue;
                        const float noff = kBias - voff - m;
                        const float alpha = high[nt][j] == -INFINITY ? 1.0f : exp2_approx(noff - off[nt][j]);
                        high[nt][j] = m + kSlack;
                        off[nt][j] = noff;
                        l[nt][j] *= alpha;
#pragma unroll
                        for (int b = 0; b < NB; ++b)
#pragma unroll
                            for (int k = 0; k < 2; ++k) {
                                o[nt][b][k][j] *= alpha;
                                o[nt][b][k][j + 2] *= alpha;
                            }
                    }
            }

#pragma unroll
            for (int u = 0; u < kUnitGroups; ++u) {
                const uint8_t *buf = unit_buf + u * Q::GROUP_BYTES;
                // ---- probabilities, times the values' scales, as the second product's B fragments
                uint32_t pf[NT][NB][NP][2];
                if constexpr (BF) {
                    uint32_t vs[2][NB];  // (token 2t, token 2t + 1) of each block, and 2t + 8, 2t + 9
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        const uint8_t *src = buf + Q::V_SCALES + (2 * lt + 8 * k) * NB * 2;
                        if constexpr (NB == 4) {
                            const uint4 w = *reinterpret_cast<const uint4 *>(src);
                            vs[k][0] = __byte_perm(w.x, w.z, 0x5410);
                            vs[k][1] = __byte_perm(w.x, w.z, 0x7632);
                            vs[k][2] = __byte_perm(w.y, w.w, 0x5410);
                            vs[k][3] = __byte_perm(w.y, w.w, 0x7632);
                        } else {
                            const uint2 w = *reinterpret_cast<const uint2 *>(src);
                            vs[k][0] = __byte_perm(w.x, w.y, 0x5410);
                            vs[k][1] = __byte_perm(w.x, w.y, 0x7632);
                        }
                    }
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        float e[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            e[i] = exp2_approx(s[u][nt][i] + off[nt][i & 1]);
                            l[nt][i & 1] += e[i];
                        }
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            const uint32_t pt = transpose8x8(pack_f16(e[2 * k], e[2 * k + 1]));  // (2t, 2t + 1) of row g
#pragma unroll
                            for (int b = 0; b < NB; ++b) {
                                uint32_t v = mul_f16x2(pt, vs[k][b]);
                                if constexpr (masked) {  // what a row does not see may hold anything
                                    if (!(pt & 0x0000ffffu)) v &= 0xffff0000u;
                                    if (!(pt & 0xffff0000u)) v &= 0x0000ffffu;
                                }
                                pf[nt][b][0][k] = v;
                            }
                        }
                    }
                } else {
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        float dv[NB];
                        const uint8_t *src = buf + Q::V_SCALES + (lg + 8 * k) * NB * 2;
#pragma unroll
                        for (int b = 0; b < NB; b += 2) {
                            const float2 f = unpack_f16(*reinterpret_cast<const uint32_t *>(src + b * 2));
                            dv[b] = f.x, dv[b + 1] = f.y;
                        }
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            float e[2];
#pragma unroll
                            for (int j = 0; j < 2; ++j) {
                                e[j] = exp2_approx(s[u][nt][2 * k + j] + off[nt][j]);
                                l[nt][j] += e[j];
                            }
#pragma unroll
                            for (int b = 0; b < NB; ++b) {
                                const float x0 = masked && s[u][nt][2 * k] == -INFINITY ? 0.0f : e[0] * dv[b];
                                const float x1 = masked && s[u][nt][2 * k + 1] == -INFINITY ? 0.0f : e[1] * dv[b];
                                const uint32_t h = pack_f16(x0, x1);
                                const float2 f = unpack_f16(h);
                                pf[nt][b][0][k] = transpose8x8(h);
                                pf[nt][b][NP - 1][k] = transpose8x8(pack_f16(x0 - f.x, x1 - f.y));
                            }
                        }
                    }
                }

                // ---- values
                uint32_t vw[2][NB];
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const uint8_t *src = buf + Q::V_CODES + k * 4 * D + lane * NB * 4;
                    if constexpr (NB == 4)
                        *reinterpret_cast<uint4 *>(vw[k]) = *reinterpret_cast<const uint4 *>(src);
                    else
                        *reinterpret_cast<uint2 *>(vw[k]) = *reinterpret_cast<const uint2 *>(src);
                }
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    uint32_t e0[4], e1[4];
                    unpack_codes<false>(vw[0][b], e0, f16_1024, f16_64);
                    unpack_codes<false>(vw[1][b], e1, f16_1024, f16_64);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        if constexpr (F32) {
                            // The tensor core cuts a sum's low bits off, always toward zero: over a warp's hundreds of
                            // groups that took 1.5e-6 of a float32 result. So a group's own sum, added with rounding: 0.4e-6 (and 28.9
                            // for 28.1 us, 16 requests' 5 tokens at up to 8192).
#pragma unroll
                            for (int k = 0; k < 2; ++k) {
                                float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                                for (int q = NP - 1; q >= 0; --q)
                                    mma16816(acc, e0[2 * k], e0[2 * k + 1], e1[2 * k], e1[2 * k + 1], pf[nt][b][q][0], pf[nt][b][q][1], acc);
#pragma unroll
                                for (int i = 0; i < 4; ++i) o[nt][b][k][i] += acc[i];
                            }
                        } else {
#pragma unroll
                            for (int q = 0; q < NP; ++q) {
                                mma16816(o[nt][b][0], e0[0], e0[1], e1[0], e1[1], pf[nt][b][q][0], pf[nt][b][q][1], o[nt][b][0]);
                                mma16816(o[nt][b][1], e0[2], e0[3], e1[2], e1[3], pf[nt][b][q][0], pf[nt][b][q][1], o[nt][b][1]);
                            }
                        }
                    }
                }
            }
        };

#pragma unroll 1
        for (; my_i < it.i0 + it.g1 - it.g0; my_i += W, ++my_k) {
            const int stage = my_k % STAGES, unit = it.g0 + my_i - it.i0;
            if (!broken && !mbar_wait(&full[stage], (my_k / STAGES) & 1)) {
                record_device_error(a.c.err, DEV_ERR_WAIT_FULL);
                broken = true;
            }
            broken = __any_sync(0xffffffffu, broken);
            const uint32_t gone = gone_sm[stage][warp];
            if (!broken && gone != 3) {
                uint8_t *buf = ring + (stage * W + warp) * H::UNIT;
                if constexpr (STEP) {
                    if (unit == it.new_unit) {
                        if (!mbar_wait(&new_full[m & 1], (m / 2) & 1))
                            record_device_error(a.c.err, DEV_ERR_WAIT_FULL);
                        else if (slot.added.key >= 0)
                            patch_new<D>(slot.added, buf + ((it.S - 1) >> 4 & 1) * Q::GROUP_BYTES);
                    }
                }
                if ((unit + 1) * kUnit > it.all_see || gone)
                    take(buf, unit * kUnit, gone, std::true_type{});
                else
                    take(buf, unit * kUnit, 0u, std::false_type{});
            }
            __syncwarp();  // every lane has read the stage before a copy comes into it
            if (lane == 0) mbar_arrive(&empty[stage]);
        }

        __syncwarp();
        if (lane == 0) mbar_arrive(&q_empty[m & 1]);

        // ---- the warps' results of the item, or of this CTA's part of it
        // four finished sums of row rr, of weight `sum` against the reference `least`
        auto finish = [&](int rr, int d, float (&v)[4], float sum, float least) {
            const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] *= inv;
            const int tok = it.single ? 0 : (it.row0 + rr) / a.rep;
            const int r = it.first + tok, hq = it.h * a.rep + it.row0 + rr - tok * a.rep;
            finish4<T, D, STEP>(p, r, hq, d, v);
            if (d == 0 && a.lse)
                a.lse[(int64_t)r * a.heads + hq] = sum == 0.0f ? 0.0f : (log2f(sum) - least) * 0.6931471805599453f;
        };
        const int64_t own_slot = (int64_t)blockIdx.x * 2 + (it.g0 == 0);
        float *po = p.part_o + own_slot * RT * D;
        float *pml = p.part_ml + own_slot * RT * 2;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            if (nt) bar_consumers(THREADS);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                float sum = l[nt][j];
#pragma unroll
                for (int o2 = 4; o2 < 32; o2 <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o2);
                if (lg == 0) {
                    // a row that met no key weighs nothing (NaN scores count: they set no reference, but their sum is NaN)
                    ml_sm[warp][2 * lt + j][0] = high[nt][j] == -INFINITY && sum == 0.0f ? INFINITY : off[nt][j];
                    ml_sm[warp][2 * lt + j][1] = sum;
                }
#pragma unroll
                for (int b = 0; b < NB; ++b)
                    *reinterpret_cast<float4 *>(merge + (warp * 8 + 2 * lt + j) * H::ROW + b * 32 + lg * 4) =
                        make_float4(o[nt][b][0][j], o[nt][b][0][j + 2], o[nt][b][1][j], o[nt][b][1][j + 2]);
            }
            bar_consumers(THREADS);
#pragma unroll 1
            for (int idx = tid; idx < 8 * (D / 4); idx += THREADS) {
                const int row = idx / (D / 4), d = idx % (D / 4) * 4;
                float least = INFINITY;
#pragma unroll
                for (int w = 0; w < W; ++w) least = fminf(least, ml_sm[w][row][0]);
                float v[4] = {0.0f, 0.0f, 0.0f, 0.0f}, sum = 0.0f;
                // (a warp without keys has off = inf: weight 0)
                const float base = least < INFINITY ? least : 0.0f;
#pragma unroll
                for (int w = 0; w < W; ++w) {
                    const float f = exp2_approx(base - ml_sm[w][row][0]);
                    const float4 x = *reinterpret_cast<const float4 *>(merge + (w * 8 + row) * H::ROW + d);
                    v[0] = fmaf(f, x.x, v[0]);
                    v[1] = fmaf(f, x.y, v[1]);
                    v[2] = fmaf(f, x.z, v[2]);
                    v[3] = fmaf(f, x.w, v[3]);
                    sum = fmaf(f, ml_sm[w][row][1], sum);
                }
                const int rr = nt * 8 + row;
                if (!it.whole) {
                    __stcg(reinterpret_cast<float4 *>(po + rr * D + d), make_float4(v[0], v[1], v[2], v[3]));
                    if (d == 0) __stcg(reinterpret_cast<float2 *>(pml + rr * 2), make_float2(least, sum));
                } else if (rr < it.rows) {
                    finish(rr, d, v, sum, least);
                }
            }
        }
        if (it.whole) continue;

        // The item lies in CTAs c0 .. c1. Each sets its flag behind its part and then looks at the others': the fences
        // put one CTA's look behind everyone's flag, and that one (now and then two, with the same result) joins the
        // parts in order. A flag is this launch's number, so that what lay in the workspace does not matter, and goes
        // back to 0, so that a replay of the launch finds none set.
        const int c0 = it.c0, c1 = it.c1;
        auto part = [&](int c) { return 2 * c + (c == c0); };
        bar_consumers(THREADS);
        if (warp == 0) {
            if (lane == 0) {
                __threadfence();
                *reinterpret_cast<volatile unsigned long long *>(p.flags + own_slot) = p.nonce;
            }
            __syncwarp();
            __threadfence();
            bool all = true;
#pragma unroll 1
            for (int c = c0 + lane; c <= c1; c += 32)
                all &= *reinterpret_cast<const volatile unsigned long long *>(p.flags + part(c)) == p.nonce;
            all = __all_sync(0xffffffffu, all);
            __threadfence();
            if (lane == 0) is_last = all;
        }
        bar_consumers(THREADS);
        if (!is_last) continue;
        // eight rows at a time: 16 lanes a row find the parts' common reference and weights, then a thread adds up four
        // dimensions of a row, four parts in flight
        const int parts = c1 - c0 + 1;
#pragma unroll 1
        for (int nt = 0; nt < NT; ++nt) {
            const float *ml = p.part_ml + nt * 16, *po = p.part_o + nt * 8 * D;
            if (tid < 128) {
                const int row = tid >> 4;
                float least = INFINITY, sum = 0.0f;
#pragma unroll 1
                for (int c = tid & 15; c < parts; c += 16) {
                    const float2 x = __ldcg(reinterpret_cast<const float2 *>(ml + (part(c0 + c) * RT + row) * 2));
                    *reinterpret_cast<float2 *>(merge + (row * parts + c) * 2) = x;
                    least = fminf(least, x.x);
                }
#pragma unroll
                for (int o2 = 8; o2; o2 >>= 1) least = fminf(least, __shfl_xor_sync(0xffffffffu, least, o2));
                const float base = least < INFINITY ? least : 0.0f;
#pragma unroll 1
                for (int c = tid & 15; c < parts; c += 16) {
                    float *x = merge + (row * parts + c) * 2;
                    x[0] = exp2_approx(base - x[0]);
                    sum = fmaf(x[0], x[1], sum);
                }
#pragma unroll
                for (int o2 = 8; o2; o2 >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o2);
                if ((tid & 15) == 0) {
                    sum_sm[row][0] = least;
                    sum_sm[row][1] = sum;
                }
            }
            bar_consumers(THREADS);
#pragma unroll 1
            for (int idx = tid; idx < 8 * (D / 4); idx += THREADS) {
                const int row = idx / (D / 4), d = idx % (D / 4) * 4, rr = nt * 8 + row;
                if (rr >= it.rows) continue;
                float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                const float *w = merge + row * parts * 2;
#pragma unroll 4
                for (int c = 0; c < parts; ++c) {
                    const float4 x = __ldcg(reinterpret_cast<const float4 *>(po + (part(c0 + c) * RT + row) * D + d));
                    const float f = w[2 * c];
                    v[0] = fmaf(f, x.x, v[0]);
                    v[1] = fmaf(f, x.y, v[1]);
                    v[2] = fmaf(f, x.z, v[2]);
                    v[3] = fmaf(f, x.w, v[3]);
                }
                finish(rr, d, v, sum_sm[row][1], sum_sm[row][0]);
            }
            bar_consumers(THREADS);
        }
#pragma unroll 1
        for (int c = c0 + tid; c <= c1; c += THREADS) p.flags[part(c)] = 0;
    }
}

// The most rows that a tile of the call may have, for the size of its workspace.
int tile_rows(int64_t max_query, int64_t rep) { return max_query * rep <= 8 ? 8 : 16; }

// Whether a request's rows go in tiles of 16 rather than 8. Both read and unpack the cache once a tile; 16 rows cost 1.7
// to 1.9 times 8 (16 requests at 2055, 8 KV heads of 128, bf16: 20 rows 44.8 us in two tiles of 16, 39.4 in three of 8;
// 32 rows 45.1 and 48.3; 64 rows 74.2 and 82.5), in float32 with D 128, whose registers spill, twice (32 rows 64.8 and
// 63.6).
bool wide_tiles(int64_t rows) {
    return 7 * ((rows + 15) / 16) <= 4 * ((rows + 7) / 8);
}

int64_t workspace_bytes(int rows, int64_t dim) { return (int64_t)kMaxGrid * 2 * (rows * (dim + 2) * 4 + 8); }

unsigned long long next_nonce() {
    static std::atomic<unsigned long long> count{(unsigned long long)std::chrono::steady_clock::now().time_since_epoch().count()};
    unsigned long long z = count.fetch_add(0x9e3779b97f4a7c15ull) + 0x9e3779b97f4a7c15ull;
    z = (z ^ (z >> 30)) * 0xbf58476d1ce4e5b9ull;
    z = (z ^ (z >> 27)) * 0x94d049bb133111ebull;
    z ^= z >> 31;
    return z ? z : 1;
}

template <typename T, int D, int NT, bool STEP>
int launch_split(Split &p, void *workspace, cudaStream_t stream, const char *op) {
    DeviceFacts f{};
    int st = device_facts(&f);
    if (st) return st;
    constexpr int rows = 8 * NT;
    const int grid = std::min(f.sm_count, kMaxGrid);
    p.part_o = static_cast<float *>(workspace);
    p.part_ml = p.part_o + (int64_t)kMaxGrid * 2 * rows * D;
    p.flags = reinterpret_cast<unsigned long long *>(p.part_ml + (int64_t)kMaxGrid * 2 * rows * 2);
    p.nonce = next_nonce();
    p.f16_1024 = 0x64006400u;
    p.f16_64 = 0x54005400u;
    auto kernel = sdpa_q4_kernel<T, D, NT, STEP>;
    static std::atomic<uint64_t> ready{0};  // a bit a device
    int device = 0;
    if ((st = check_cuda(cudaGetDevice(&device), op, "cudaGetDevice"))) return st;
    if (!(ready.load(std::memory_order_relaxed) >> device & 1)) {
        st = check_cuda(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape<T, D, NT>::SMEM), op,
                        "cudaFuncSetAttribute");
        if (st) return st;
        ready.fetch_or(1ull << device, std::memory_order_relaxed);
    }
    __atomic_fetch_add(&counters().sdpa_decode_launches, 1ull, __ATOMIC_RELAXED);
    return launch_pdl(kernel, dim3((unsigned)grid), dim3(32 * (Shape<T, D, NT>::W + 4)), Shape<T, D, NT>::SMEM, stream, op, p);
}

// Whether a call's query rows are better taken 256 at a time by the tcgen05
// kernel. Both read the cache once for every tile of rows; per 64 keys of D 128
// (64) this kernel's tiles of 16 rows cost 2.8 (1.8) ns each, all SMs together,
// and the other's pairs of tiles, one an SM, 2000 (1700) ns a wave of 148 CTAs
// (1390, 1180 where the rows fill one tile of 128 only). Measured, 32 heads on 8,
// here and there: 4 requests of 64 tokens at 16384 377 and 509 us (D 64: 239 and
// 435); 4 of 96 at 8192 295 and 267 (190 and 223); 16 of 17 at 16384 465 and 355
// (294 and 301); 8 of 64 at 8192 388 and 266 (246 and 222); 16 of 256 at 4096 1577
// and 541 (999 and 445); 2 of 256 at 16384, 9 heads on 3: 227 and 507 (150 and 434).
bool fills_tiles(int64_t tokens, int64_t requests, int64_t kv_heads, int64_t rep, int64_t dim, int64_t max_query) {
    if (max_query * rep <= 64) return false;
    requests = std::min(requests, tokens);
    const int64_t rows = (tokens * rep + requests - 1) / requests;  // a request, on average
    const double here = (dim == 128 ? 2.8 : 1.8) * (double)((rows + 15) / 16 * requests * kv_heads);
    const double waves = std::max(1.0, (double)((rows + 255) / 256 * requests * kv_heads) / 148.0);
    return here > waves * (dim == 128 ? (rows > 128 ? 2000.0 : 1390.0) : (rows > 128 ? 1700.0 : 1180.0));
}

template <typename T, int D>
int launch_attend(Split &p, int64_t max_query, void *workspace, cudaStream_t stream) {
    if (std::is_same<T, __nv_bfloat16>::value && fills_tiles(p.a.tokens, p.a.c.requests, p.a.c.kv_heads, p.a.rep, D, max_query))
        return launch_sdpa_q4_prefill(p.a, D, stream);
    if constexpr (!(sizeof(T) == 4 && D == 128)) {
        if (wide_tiles(max_query * p.a.rep)) return launch_split<T, D, 2, false>(p, workspace, stream, "tn_sdpa_q4_cache");
    }
    return launch_split<T, D, 1, false>(p, workspace, stream, "tn_sdpa_q4_cache");
}

int check_cache(const char *op, const KvPool &c, int64_t requests, int64_t max_pages, int64_t table_stride,
                int64_t heads, int64_t kv_heads, int64_t tokens) {
    const std::string name(op);
    if (requests < 0 || requests > 65535 || max_pages < 0 || table_stride < max_pages ||
        max_pages > kMaxRowTokens >> c.page_shift || tokens < 0 || tokens > INT32_MAX / 2)
        return set_error(TN_ERR_SHAPE, name + ": bad request, table or token count");
    if (heads < 1 || heads > 65535 || heads % kv_heads != 0)
        return set_error(TN_ERR_SHAPE, name + ": query heads (" + std::to_string(heads) +
                                           ") must be a multiple of the cache's heads (" + std::to_string(kv_heads) + ")");
    if (requests > 0 && (!c.lengths || (max_pages > 0 && !c.table))) return set_error(TN_ERR_INVALID, name + ": null pointer");
    return TN_OK;
}

}  // namespace
}  // namespace tn

extern "C" int64_t tn_sdpa_q4_workspace_bytes(int64_t tokens, int64_t heads, int64_t kv_heads, int64_t head_dim,
                                              int64_t max_query) {
    if (kv_heads < 1 || heads < 1) return 0;
    return tn::workspace_bytes(tn::tile_rows(std::max<int64_t>(1, std::min(max_query, tokens)), heads / kv_heads), head_dim);
}

extern "C" int tn_sdpa_q4_cache(const void *q, int dtype, const int64_t *q_strides, int64_t tokens, int64_t heads,
                                const void *pool, int64_t num_pages, int64_t kv_heads, int64_t head_dim,
                                int64_t page_size, const int *page_table, int64_t table_stride, int64_t max_pages,
                                const int *lengths, int64_t requests, const int *query_start, int64_t max_query,
                                void *out, float *lse, double scale, void *workspace, int64_t workspace_bytes,
                                void *stream) {
    const char *op = "tn_sdpa_q4_cache";
    int st = tn::check_kv_pool(op, pool, num_pages, kv_heads, head_dim, page_size);
    if (st) return st;
    if (dtype != TN_F32 && dtype != TN_F16 && dtype != TN_BF16)
        return tn::set_error(TN_ERR_NOT_IMPLEMENTED, std::string(op) + ": queries must be float32, float16 or bfloat16, got " +
                                                         tn_dtype_name(dtype));
    tn::KvPool c{(uint8_t *)pool, (int)num_pages, tn::kv_page_shift(page_size), (int)kv_heads, page_table, table_stride,
                 (int)max_pages, lengths, (int)requests, tn::device_error_word()};
    st = tn::check_cache(op, c, requests, max_pages, table_stride, heads, kv_heads, tokens);
    if (st) return st;
    if (!query_start && tokens != requests)
        return tn::set_error(TN_ERR_SHAPE, std::string(op) + ": without query_start every request has one query token");
    if (tokens == 0 || requests == 0) return TN_OK;
    if (!q || !q_strides || !out) return tn::set_error(TN_ERR_INVALID, std::string(op) + ": null pointer");
    const int64_t size = (int64_t)tn_dtype_size(dtype);
    if ((uintptr_t)q % 16 || q_strides[0] * size % 16 || q_strides[1] * size % 16 || (uintptr_t)out % 16)
        return tn::set_error(TN_ERR_INVALID, std::string(op) + ": query rows must be 16-byte aligned with a unit inner stride");
    max_query = std::max<int64_t>(1, std::min(query_start ? max_query : 1, tokens));
    if (!workspace || workspace_bytes < tn_sdpa_q4_workspace_bytes(tokens, heads, kv_heads, head_dim, max_query))
        return tn::set_error(TN_ERR_SHAPE, std::string(op) + ": the workspace is smaller than tn_sdpa_q4_workspace_bytes");
    const float sc = scale > 0.0 ? (float)scale : 1.0f / sqrtf((float)head_dim);
    if ((uintptr_t)workspace % 16)
        return tn::set_error(TN_ERR_INVALID, std::string(op) + ": the workspace must be 16-byte aligned");
    tn::Split p{};
    p.a = {q, q_strides[0], q_strides[1], c, query_start, out, lse, (int)tokens, (int)heads, (int)(heads / kv_heads), sc};
    __atomic_fetch_add(&tn::counters().sdpa_calls, 1ull, __ATOMIC_RELAXED);
    cudaStream_t s = tn::stream_of(stream);
    if (head_dim == 128)
        return dtype == TN_F32   ? tn::launch_attend<float, 128>(p, max_query, workspace, s)
               : dtype == TN_F16 ? tn::launch_attend<__half, 128>(p, max_query, workspace, s)
                                 : tn::launch_attend<__nv_bfloat16, 128>(p, max_query, workspace, s);
    return dtype == TN_F32   ? tn::launch_attend<float, 64>(p, max_query, workspace, s)
           : dtype == TN_F16 ? tn::launch_attend<__half, 64>(p, max_query, workspace, s)
                             : tn::launch_attend<__nv_bfloat16, 64>(p, max_query, workspace, s);
}

extern "C" int tn_sdpa_q4_decode_step_granted(const void *qkv, const void *rope, int64_t rope_rows, void *pool,
                                              int64_t num_pages, int64_t heads, int64_t kv_heads, int64_t head_dim,
                                              int64_t page_size, const int *page_table, int64_t table_stride,
                                              int64_t max_pages, const int *lengths, int64_t requests, void *out,
                                              float *lse, int8_t *codes, float *scales, float *offsets, double scale,
                                              void *workspace, int64_t workspace_bytes, const int *granted,
                                              void *stream) {
    const char *op = "tn_sdpa_q4_decode_step";
    int st = tn::check_kv_pool(op, pool, num_pages, kv_heads, head_dim, page_size);
    if (st) return st;
    tn::KvPool c{(uint8_t *)pool, (int)num_pages, tn::kv_page_shift(page_size), (int)kv_heads, page_table, table_stride,
                 (int)max_pages, lengths, (int)requests, tn::device_error_word()};
    st = tn::check_cache(op, c, requests, max_pages, table_stride, heads, kv_heads, requests);
    if (st) return st;
    if (heads / kv_heads > 8)
        return tn::set_error(TN_ERR_NOT_IMPLEMENTED, std::string(op) + ": at most 8 query heads a KV head, got " +
                                                         std::to_string(heads / kv_heads));
    if (rope_rows < 1) return tn::set_error(TN_ERR_SHAPE, std::string(op) + ": an empty rotary table");
    if (requests == 0) return TN_OK;
    if (!qkv || !rope || !out || (codes && (!scales || !offsets)))
        return tn::set_error(TN_ERR_INVALID, std::string(op) + ": null pointer");
    if ((uintptr_t)qkv % 16 || (uintptr_t)rope % 16 || (uintptr_t)out % 16 || (uintptr_t)codes % 16)
        return tn::set_error(TN_ERR_INVALID, std::string(op) + ": tensors must be 16-byte aligned");
    const float sc = scale > 0.0 ? (float)scale : 1.0f / sqrtf((float)head_dim);
    cudaStream_t s = tn::stream_of(stream);
    if (!workspace || workspace_bytes < tn_sdpa_q4_workspace_bytes(requests, heads, kv_heads, head_dim, 1))
        return tn::set_error(TN_ERR_SHAPE, std::string(op) + ": the workspace is smaller than tn_sdpa_q4_workspace_bytes");
    if ((uintptr_t)workspace % 16)
        return tn::set_error(TN_ERR_INVALID, std::string(op) + ": the workspace must be 16-byte aligned");
    __atomic_fetch_add(&tn::counters().sdpa_calls, 1ull, __ATOMIC_RELAXED);
    tn::Split p{};
    p.a = {nullptr, 0, 0, c, nullptr, out, lse, (int)requests, (int)heads, (int)(heads / kv_heads), sc};
    p.qkv = (const __nv_bfloat16 *)qkv;
    p.rope = (const __nv_bfloat16 *)rope;
    p.places = (int)std::min<int64_t>(max_pages << c.page_shift, rope_rows);
    p.codes = codes;
    p.scales = scales;
    p.offsets = offsets;
    p.granted = granted;
    return head_dim == 128 ? tn::launch_split<__nv_bfloat16, 128, 1, true>(p, workspace, s, op)
                           : tn::launch_split<__nv_bfloat16, 64, 1, true>(p, workspace, s, op);
}

extern "C" int tn_sdpa_q4_decode_step(const void *qkv, const void *rope, int64_t rope_rows, void *pool, int64_t num_pages,
                                      int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t page_size,
                                      const int *page_table, int64_t table_stride, int64_t max_pages, const int *lengths,
                                      int64_t requests, void *out, float *lse, int8_t *codes, float *scales,
                                      float *offsets, double scale, void *workspace, int64_t workspace_bytes,
                                      void *stream) {
    return tn_sdpa_q4_decode_step_granted(qkv, rope, rope_rows, pool, num_pages, heads, kv_heads, head_dim, page_size,
                                          page_table, table_stride, max_pages, lengths, requests, out, lse, codes, scales,
                                          offsets, scale, workspace, workspace_bytes, nullptr, stream);
}
