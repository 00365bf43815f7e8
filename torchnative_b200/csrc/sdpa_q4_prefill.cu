// sdpa_q4_prefill.cu -- attention of many query tokens over the paged 4-bit KV
// cache (a prompt's next piece against everything cached before it), on tcgen05.
//
// One CTA = 256 query rows (two tiles of 128) of one (request, KV head); a row
// is a token of one of the query heads that share the KV head, so that a tile's
// rows see nearly the same keys. Key tiles of 64 are unpacked once for both
// query tiles. 16 warps:
//   warps 0-3, 4-7   softmax of query tile 0, 1: thread r owns row r (TMEM lane
//                    r) and all 64 keys of a tile; before, it lays out its row
//                    of queries
//   warp 8           MMA issuer (one thread): S_k = Q_k K_j^T, the keys' high and
//                    low terms as one product of 128 columns whose halves the
//                    softmax adds (as two of 64 columns, with the queries in TMEM,
//                    1009 us for 916 at the size below), then O_k += P_k V_{j-1} one
//                    tile behind
//   warps 9-15       unpack: the keys and the values of the tile's four groups of 16
//                    tokens in turn, from global memory (a warp's next piece is
//                    loaded before it unpacks this one); warps 12-15 alone, a group
//                    each, were what bounded it: 916 us for 866. Warp 9 owns the TMEM.
// The products are f16: an element is (code - 8) times its block's scale, the
// scale taken to [1/2, 1) by a power of two of the group's own, so that nothing
// overflows; the powers come back in the softmax, those of the keys in the
// exponent's factor, those of the values in the probabilities (and out of their
// sum). Queries have a power of two a row. A key's product has 15 bits and is
// held in two f16 terms, exactly, so that scores and the logsumexp are as exact
// as float32 sums are; a value's and a probability's roundings to 2^-11 are an
// eighth of the bf16 result's own. (bf16 operands would lose 2^-8 three times
// over. For f16 results those roundings would be as large as the result's: they
// take the other kernel.) A key is exact where its block's scale lies above 2^-14
// of its group's largest: a smaller one is below f16's normal numbers here, and
// rounded to a multiple of 2^-24 of at most twice that largest scale.
// An infinite or NaN value scale counts as 0 in the products, since 0 times it
// would be NaN in the rows that do not see its token; the rows that do add it at
// the end, from the cache.
// What bounds it: the stream of products, of which hardly a moment is without one,
// but each of 128 x 128 x 16 takes 110 to 160 cycles for the 64 of the pipe's peak
// (which was active 41% of the cycles at 866 us); two terms of K make half as many
// again; and the last wave of items (384 on 148 SMs), an eighth. 2 x 1536 tokens at
// 9728, 32/8 heads of 128: 824 us, 547 TFLOP/s.
// Every wait is bounded; one that gives up raises a CTA-wide abort flag.
#include <algorithm>
#include <atomic>

#include "sdpa_q4.cuh"
#include "tc05.cuh"

namespace tn {
namespace {

constexpr int BM = 128, NQT = 2, BN = 64, NK = 2, NV = 3, NINFO = 8, UNPACKERS = 7;
constexpr int THREADS = 16 * 32, SOFTMAX_REGS = 168, OTHER_REGS = 88;
static_assert(256 * SOFTMAX_REGS + 256 * OTHER_REGS <= THREADS * 128, "what the CTA is launched with");
constexpr int KPANEL = BN * 128, PTILE = BM * 128;  // rows of 64 16-bit elements
// TMEM columns (512): scores (the keys' high terms, their low ones), results
constexpr int TS = 0, TO = 256;
constexpr float kBias = 10.0f, kSlack = 5.0f;  // a probability is 2^10 at its row's reference, 2^15 at most

// What the unpacking warps say of a key tile, a value for each of its groups.
struct Info {
    float k[4];     // the keys' power of two; -1: the group has no page
    float v[4];     // the values' power of two: its exponent,
    float vinv[4];  // and 2^-exponent
};

template <int D>
struct Layout {
    static constexpr int P = D / 64;  // panels of 64 columns
    static constexpr int KTILE = P * KPANEL;
    static constexpr int Q = 0, K = Q + NQT * P * PTILE, V = K + NK * 2 * KTILE, PR = V + NV * KTILE, INFO = PR + NQT * PTILE,
                         BAR = INFO + NINFO * (int)sizeof(Info);
    static constexpr int SMEM = BAR + 512 + 1024;
};

__device__ __forceinline__ bool wait_or_abort(uint64_t *bar, uint32_t parity, volatile int *abort, int *err) {
    if (mbar_try_wait(bar, parity)) return true;
    const long long start = clock64();
    while (!mbar_try_wait(bar, parity)) {
        if (*abort) return false;
        if (clock64() - start > kWaitBudgetCycles) {
            *abort = 1;
            record_device_error(err, DEV_ERR_WAIT_FULL);
            return false;
        }
    }
    return true;
}

// The same by a whole warp, of one mind afterwards.
__device__ __forceinline__ bool warp_wait(uint64_t *bar, uint32_t parity, volatile int *abort, int *err) {
    return __all_sync(0xffffffffu, wait_or_abort(bar, parity, abort, err));
}

__device__ __forceinline__ void st_shared_v4(uint32_t a, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
__device__ __forceinline__ uint64_t pk2(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void upk2(uint64_t r, float &a, float &b) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(r));
}
__device__ __forceinline__ uint64_t fma2p(uint64_t x, uint64_t y, uint64_t z) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(x), "l"(y), "l"(z));
    return d;
}
__device__ __forceinline__ uint64_t add2p(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
// A lane's codes and scales of the keys, or of the values, of one group (16 tokens). Keys: two vectors, tokens lane / 4
// and + 8, t = lane % 4. Values: the two vectors of elements 8 q .. 8 q + 7 of each block, tokens 8 h + 2 t and + 1;
// lane = 16 h + 4 q + t.
template <int D>
struct Words {
    uint32_t codes[2][D / 32], scales[2][D / 64];
    bool gone;

    __device__ __forceinline__ void load(const KvPool &c, const int *row, int head, int group, bool values, int S, int lane) {
        using Q = KvQ4<D>;
        constexpr int NB = D / 32;
#pragma unroll
        for (int b = 0; b < NB; ++b) codes[0][b] = codes[1][b] = 0;
#pragma unroll
        for (int b = 0; b < NB / 2; ++b) scales[0][b] = scales[1][b] = 0;
        gone = false;
        if (group * kKvGroup >= S) return;
        const uint8_t *src = c.group_of_row<D>(row, head, group);
        gone = !src;
        if (!src) return;
        const int t = lane & 3, q = lane >> 2 & 3, h = lane >> 4, left = S - group * kKvGroup;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int token = values ? 8 * h + 2 * t + i : (lane >> 2) + 8 * i;
            const uint8_t *p = src + (values ? Q::V_CODES + h * 4 * D + ((2 * q + i) * 4 + t) * NB * 4
                                             : Q::K_CODES + token * (D / 2) + t * NB * 4);
            const uint8_t *d = src + (values ? Q::v_scale(token, 0) : Q::k_scale(token, 0));
            // what lies behind the last token may be anything: its scales are 0
            if constexpr (NB == 4) {
                *reinterpret_cast<uint4 *>(codes[i]) = *reinterpret_cast<const uint4 *>(p);
                if (token < left) *reinterpret_cast<uint2 *>(scales[i]) = *reinterpret_cast<const uint2 *>(d);
            } else {
                *reinterpret_cast<uint2 *>(codes[i]) = *reinterpret_cast<const uint2 *>(p);
                if (token < left) scales[i][0] = *reinterpret_cast<const uint32_t *>(d);
            }
        }
    }
};

// The largest exponent field (1 .. 30) of two half2's magnitudes, kept with `e`.
__device__ __forceinline__ int most_exponent(int e, uint32_t w) {
    return max(e, max((int)(w >> 10 & 31), (int)(w >> 26 & 31)));
}
// 2^(14 - e) as half2: takes scales of at most that exponent to [1/2, 1)
__device__ __forceinline__ uint32_t power_f16x2(int e) {
    const uint32_t h = e < 29 ? (uint32_t)(29 - e) << 10 : 0x400u >> (e - 28);
    return h | h << 16;
}

template <int D>
__global__ void __launch_bounds__(THREADS, 1) sdpa_q4_prefill_kernel(const Attend a, int slots, uint32_t f16_1024,
                                                                     uint32_t f16_64) {
    using L = Layout<D>;
    using T = __nv_bfloat16;
    constexpr int NB = D / 32;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t *base = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const uint32_t sb = smem_u32(base);
    volatile Info *info = reinterpret_cast<volatile Info *>(base + L::INFO);
    uint64_t *bars = reinterpret_cast<uint64_t *>(base + L::BAR);
    uint64_t *q_full = bars, *k_full = q_full + 1, *k_empty = k_full + NK, *v_full = k_empty + NK, *v_empty = v_full + NV,
             *s_full = v_empty + NV /*[2]*/, *s_free = s_full + 2 /*[2]*/, *p_full = s_free + 2 /*[2]*/,
             *o_done = p_full + 2 /*[2]*/, *info_full = o_done + 2 /*[NINFO]*/, *mma_done = info_full + NINFO;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(mma_done + 1);
    volatile int *abort = reinterpret_cast<volatile int *>(tmem_slot + 1);
    volatile int *where = reinterpret_cast<volatile int *>(tmem_slot + 2);  // request, pair of tiles
    int *odd_tiles = reinterpret_cast<int *>(tmem_slot + 4);  // first and last with value scales that are not finite
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    pdl_launch_dependents();
    pdl_wait();
    // ---- which request and pair of tiles: the last ones, which see the most keys, go first
    const int head = blockIdx.x % a.c.kv_heads;
    int want = slots - 1 - blockIdx.x / a.c.kv_heads;
    if (warp == 0) {
        int at = -1, pair = 0;
        for (int b0 = 0; b0 < a.c.requests && at < 0; b0 += 32) {
            int first, pairs = 0;
            if (b0 + lane < a.c.requests) {
                const long long rows = (long long)a.query_tokens(b0 + lane, &first) * a.rep;
                pairs = (int)((rows + NQT * BM - 1) / (NQT * BM));
            }
            int upto = pairs;
#pragma unroll
            for (int off = 1; off < 32; off <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, upto, off);
                if (lane >= off) upto += v;
            }
            const unsigned past = __ballot_sync(0xffffffffu, upto > want);
            if (past) {
                const int l0 = __ffs(past) - 1;
                at = b0 + l0;
                pair = want - __shfl_sync(0xffffffffu, upto - pairs, l0);
            } else {
                want -= __shfl_sync(0xffffffffu, upto, 31);
            }
        }
        if (lane == 0) {
            where[0] = at;
            where[1] = pair;
        }
    }
    if (tid == 32) {
        mbar_init(q_full, 8);
        for (int i = 0; i < NK; ++i) {
            mbar_init(&k_full[i], 4);
            mbar_init(&k_empty[i], 1);
        }
        for (int i = 0; i < NV; ++i) {
            mbar_init(&v_full[i], 4);
            mbar_init(&v_empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&s_full[i], 1);
            mbar_init(&s_free[i], 4);
            mbar_init(&p_full[i], 4);
            mbar_init(&o_done[i], 1);
        }
        for (int i = 0; i < NINFO; ++i) mbar_init(&info_full[i], 8);
        mbar_init(mma_done, 1);
        *abort = 0;
        odd_tiles[0] = INT32_MAX;
        odd_tiles[1] = -1;
        fence_mbar_init();
    }
    __syncthreads();
    const int b = where[0], row_first = where[1] * (NQT * BM);
    if (b < 0) return;  // fewer pairs than the grid was sized for
    if (warp == 9) tc05::alloc(tmem_slot, 512);
    tc05::fence_before();
    __syncthreads();
    tc05::fence_after();
    const uint32_t tmem = *tmem_slot;

    int first;
    const int n = a.query_tokens(b, &first), S = a.c.length(b), rows = n * a.rep;
    // key tiles of query tile k: up to the last key that its last row sees
    auto tiles_of = [&](int k) {
        const int r0 = row_first + BM * k;
        if (r0 >= rows) return 0;
        const int keys = S - n + min(r0 + BM - 1, rows - 1) / a.rep + 1;
        return max(0, (keys + BN - 1) / BN);
    };
    const int nt0 = tiles_of(0), nt1 = tiles_of(1), ntm = max(nt0, nt1);

    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(OTHER_REGS));
        if (warp >= 9) {
            // ---------------- unpack: a key tile is eight pieces, the keys and the values of its four groups, and the pieces
            // go to the seven warps in turn. A piece waits only for what pieces before it make possible. A parity names a phase
            // only to a warp that knows the one before to be over: its last piece, seven back, tells it. That was a tile's
            // K_1 .. V_3 before, so S_{j-3} or PV_{j-4} is over, or K_0 of the same tile, so S_{j-2} and PV_{j-3}, which
            // was issued before it; and the phases before the ones waited for are S_{j-4} and PV_{j-6}.
            static_assert(UNPACKERS == 7 && NK == 2 && NV == 3, "or the above has to be shown again");
            const int *table = a.c.table + b * a.c.table_stride;
            const int t = lane & 3, q = lane >> 2 & 3, pieces = 8 * ntm;
            Words<D> x;
            auto load = [&](int piece) { x.load(a.c, table, head, 4 * (piece >> 3) + (piece & 3), piece & 4, S, lane); };
            if (warp - 9 < pieces) load(warp - 9);
            for (int piece = warp - 9; piece < pieces; piece += UNPACKERS) {
                Words<D> y = x;
                if (piece + UNPACKERS < pieces) load(piece + UNPACKERS);
                const int j = piece >> 3, w = piece & 3, slot = j % NINFO, ks = j % NK, vs = j % NV;
                // the group's power of two
                int e = 1;
#pragma unroll
                for (int c = 0; c < NB / 2; ++c) e = most_exponent(most_exponent(e, y.scales[0][c]), y.scales[1][c]);
                e = (int)__reduce_max_sync(0xffffffffu, (unsigned)e);
                const bool odd = e > 30;
                if (odd) {
                    // infinite and NaN scales. A score that is not finite is its own row's matter; a value times 0 would
                    // reach the rows that do not see it, so it counts as 0 here, and what it adds to the others' results
                    // comes in at the end.
                    e = 30;
                    if (piece & 4) {
                        e = 1;
#pragma unroll
                        for (int c = 0; c < NB / 2; ++c)
#pragma unroll
                            for (int i = 0; i < 2; ++i) {
                                const uint32_t w = y.scales[i][c];
                                if ((w & 0x7c00u) == 0x7c00u) y.scales[i][c] &= 0xffff0000u;
                                if ((w & 0x7c000000u) == 0x7c000000u) y.scales[i][c] &= 0xffffu;
                                e = most_exponent(e, y.scales[i][c]);
                            }
                        e = (int)__reduce_max_sync(0xffffffffu, (unsigned)e);
                    }
                }
                const uint32_t power = power_f16x2(e);
                if (!(piece & 4)) {
                    if (j >= NK && !warp_wait(&k_empty[ks], (j / NK - 1) & 1, abort, a.c.err)) break;
                    if (lane == 0) {
                        info[slot].k[w] = y.gone ? -1.0f : __uint_as_float((uint32_t)(e + 113) << 23);
                        mbar_arrive(&info_full[slot]);
                    }
                    const int krow = 16 * w + (lane >> 2);
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const uint32_t dst = sb + L::K + ks * 2 * L::KTILE + (krow + 8 * i) * 128;
#pragma unroll
                        for (int c = 0; c < NB; ++c) {
                            const uint32_t d = mul_f16x2(__byte_perm(y.scales[i][c / 2], 0, c & 1 ? 0x3232 : 0x1010), power);
                            uint32_t e4[4];
                            unpack_codes<false>(y.codes[i][c], e4, f16_1024, f16_64);
                            uint32_t hi[4], lo[4];
#pragma unroll
                            for (int k = 0; k < 4; ++k) {
                                hi[k] = mul_f16x2(e4[k], d);
                                lo[k] = fma_f16x2(e4[k], d, hi[k] ^ 0x80008000u);
                            }
                            const int chunk = 4 * c + t;
                            const uint32_t at = dst + (chunk >> 3) * 2 * KPANEL + (((chunk & 7) ^ (krow & 7)) << 4);
                            st_shared_v4(at, hi[0], hi[1], hi[2], hi[3]);
                            st_shared_v4(at + KPANEL, lo[0], lo[1], lo[2], lo[3]);
                        }
                    }
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&k_full[ks]);
                } else {
                    if (lane == 0) {
                        if (odd) {
                            atomicMin(odd_tiles, j);
                            atomicMax(odd_tiles + 1, j);
                        }
                        info[slot].v[w] = (float)(e - 14);
                        info[slot].vinv[w] = __uint_as_float((uint32_t)(141 - e) << 23);
                        mbar_arrive(&info_full[slot]);
                    }
                    if (j >= NV && !warp_wait(&v_empty[vs], (j / NV - 1) & 1, abort, a.c.err)) break;
                    const int vrow = 16 * w + 8 * (lane >> 4) + 2 * t;
                    const uint32_t dst = sb + L::V + vs * L::KTILE + vrow * 128;
#pragma unroll
                    for (int c = 0; c < NB; ++c) {
                        // the block's scales of the two tokens
                        const uint32_t d = mul_f16x2(__byte_perm(y.scales[0][c / 2], y.scales[1][c / 2], c & 1 ? 0x7632 : 0x5410), power);
                        uint32_t e0[4], e1[4];
                        unpack_codes<false>(y.codes[0][c], e0, f16_1024, f16_64);
                        unpack_codes<false>(y.codes[1][c], e1, f16_1024, f16_64);
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            e0[i] = mul_f16x2(e0[i], d);
                            e1[i] = mul_f16x2(e1[i], d);
                        }
                        const int chunk = 4 * c + q;
                        const uint32_t at = dst + (chunk >> 3) * KPANEL;
                        st_shared_v4(at + (((chunk & 7) ^ (vrow & 7)) << 4), __byte_perm(e0[0], e0[1], 0x5410),
                                     __byte_perm(e0[2], e0[3], 0x5410), __byte_perm(e1[0], e1[1], 0x5410),
                                     __byte_perm(e1[2], e1[3], 0x5410));
                        st_shared_v4(at + 128 + (((chunk & 7) ^ ((vrow + 1) & 7)) << 4), __byte_perm(e0[0], e0[1], 0x7632),
                                     __byte_perm(e0[2], e0[3], 0x7632), __byte_perm(e1[0], e1[1], 0x7632),
                                     __byte_perm(e1[2], e1[3], 0x7632));
                    }
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&v_full[vs]);
                }
            }
        } else {
            {
                // ---------------- MMA issuer: the whole warp comes along, its first lane's instructions count
                const uint32_t one = lane == 0;
                const uint32_t id_qk = tc05::idesc_f16(false, BM, 2 * BN, false);
                const uint32_t id_pv = tc05::idesc_f16(false, BM, D, true);
                const int nt[2] = {nt0, nt1};
                bool ok = warp_wait(q_full, 0, abort, a.c.err);
                const uint64_t q_desc = tc05::desc_sw128(sb + L::Q, 16, 1024);
                const uint64_t k_desc = tc05::desc_sw128(sb + L::K, 16, 1024), p_desc = tc05::desc_sw128(sb + L::PR, 16, 1024),
                               v_desc = tc05::desc_sw128(sb + L::V, KPANEL, 1024);
                auto pv = [&](int t) -> bool {
                    const int vs = t % NV;
                    if (!warp_wait(&v_full[vs], (t / NV) & 1, abort, a.c.err)) return false;
                    for (int k = 0; k < NQT; ++k) {
                        if (t >= nt[k]) continue;
                        if (!warp_wait(&p_full[k], t & 1, abort, a.c.err)) return false;
                        tc05::fence_after();
                        const uint64_t pd = p_desc + (k * PTILE >> 4), vd = v_desc + (vs * L::KTILE >> 4);
#pragma unroll
                        for (int kk = 0; kk < BN / 16; ++kk)
                            tc05::mma_ss_if(one, tmem + TO + k * 128, pd + (kk * 32 >> 4), vd + (kk * 2048 >> 4), id_pv,
                                            (t > 0 || kk > 0) ? 1u : 0u);
                        tc05::commit_if(one, &o_done[k]);
                    }
                    tc05::commit_if(one, &v_empty[vs]);
                    return true;
                };
                for (int j = 0; j < ntm && ok; ++j) {
                    const int ks = j % NK;
                    if (!warp_wait(&k_full[ks], (j / NK) & 1, abort, a.c.err)) break;
                    for (int k = 0; k < NQT && ok; ++k)
                        if (j >= 1 && j < nt[k]) ok = warp_wait(&s_free[k], (j - 1) & 1, abort, a.c.err);
                    if (!ok) break;
                    tc05::fence_after();
                    // The two tiles' products in turn: 864 us one tile after the other, 820 so. (The results' in turn,
                    // too: 832, since the first tile's then wait for the second's probabilities.)
                    const uint64_t kd = k_desc + (ks * 2 * L::KTILE >> 4);
                    const uint32_t go[2] = {one && j < nt0, one && j < nt1};
#pragma unroll
                    for (int kk = 0; kk < D / 16; ++kk)
#pragma unroll
                        for (int k = 0; k < NQT; ++k) {
                            const uint32_t p = kk >> 2, at = kk & 3;
                            tc05::mma_ss_if(go[k], tmem + TS + k * 2 * BN, q_desc + (((k * L::P + p) * PTILE + at * 32) >> 4),
                                            kd + ((p * 2 * KPANEL + at * 32) >> 4), id_qk, kk > 0);
                        }
#pragma unroll
                    for (int k = 0; k < NQT; ++k) tc05::commit_if(go[k], &s_full[k]);
                    tc05::commit_if(one, &k_empty[ks]);
                    if (ok && j >= 1) ok = pv(j - 1);
                }
                if (ok && ntm > 0) pv(ntm - 1);
                tc05::commit_if(one, mma_done);
                if (!mbar_wait(mma_done, 0)) record_device_error(a.c.err, DEV_ERR_DRAIN);
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(SOFTMAX_REGS));
        // ---------------- softmax of query tile k: thread r owns row 128 k + r of the pair
        const int k = warp >> 2, r = tid & 127, row = row_first + BM * k + r;
        const int nt = k == 0 ? nt0 : nt1;
        const int tok = min(row, max(rows - 1, 0)) / a.rep;
        const int sees = S - n + tok + 1;                                   // keys of this row
        const int all_see = S - n + (row_first + BM * k) / a.rep + 1;       // keys of every row of the tile
        const uint32_t lane_off = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t tO = tmem + lane_off + TO + k * 128;
        // ---- this row's queries, in f16 into shared memory: the largest magnitude taken to [2^13, 2^14) by a power of two
        float inv_q = 1.0f;
        {
            uint4 q[D / 8];
            const T *src = static_cast<const T *>(a.q) + (first + tok) * a.q_token + (head * a.rep + row - tok * a.rep) * a.q_head;
            uint32_t most = 0;  // of the magnitudes of a word's two elements (16-bit integers order as they do)
#pragma unroll
            for (int c = 0; c < D / 8; ++c) {
                q[c] = row < rows ? *reinterpret_cast<const uint4 *>(src + c * 8) : make_uint4(0, 0, 0, 0);
                const uint32_t w[4] = {q[c].x, q[c].y, q[c].z, q[c].w};
#pragma unroll
                for (int i = 0; i < 4; ++i) most = __vmaxu2(most, w[i] & 0x7fff7fffu);
            }
            most = max(most & 0xffffu, most >> 16);
            float scale = 1.0f;
            if (most > 0 && most < 0x7f80u) {
                const int e = min(max(267 - (int)(most >> 7), 1), 253);
                scale = __uint_as_float((uint32_t)e << 23);
                inv_q = __uint_as_float((uint32_t)(254 - e) << 23);
            }
#pragma unroll
            for (int c = 0; c < D / 8; ++c) {
                const uint32_t w[4] = {q[c].x, q[c].y, q[c].z, q[c].w};
                uint32_t v[4];
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    v[i] = pack_f16(__uint_as_float(w[i] << 16) * scale, __uint_as_float(w[i] & 0xffff0000u) * scale);
                st_shared_v4(sb + L::Q + (k * L::P + (c >> 3)) * PTILE + r * 128 + (((c & 7) ^ (r & 7)) << 4), v[0], v[1], v[2], v[3]);
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(q_full);
        }
        float m_used = -INFINITY, l = 0.0f;
        bool ok = true;
        // p = 2^(s c2 - m); above 0, so that what is masked stays -inf
        const float c2 = fmaxf(a.scale * 1.4426950408889634f * inv_q, 1.1754944e-38f);
        for (int t = 0; t < nt && ok; ++t) {
            if (!warp_wait(&s_full[k], t & 1, abort, a.c.err) ||
                !warp_wait(&info_full[t % NINFO], (t / NINFO) & 1, abort, a.c.err)) {
                ok = false;
                break;
            }
            tc05::fence_after();
            float ck[4], cv[4], ci[4];
            bool full = (t + 1) * BN <= all_see;
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                ck[g] = info[t % NINFO].k[g];
                cv[g] = info[t % NINFO].v[g];
                ci[g] = info[t % NINFO].vinv[g];
                full &= ck[g] > 0.0f;
            }
            float sv[64];
            {
                float hi[32], lo[32];
                const uint32_t tS = tmem + lane_off + TS + k * 2 * BN;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    tc05::ld32(tS + 32 * h, hi);
                    tc05::ld32(tS + BN + 32 * h, lo);
                    tc05::wait_ld();
#pragma unroll
                    for (int i = 0; i < 32; i += 2) upk2(add2p(pk2(hi[i], hi[i + 1]), pk2(lo[i], lo[i + 1])), sv[32 * h + i], sv[32 * h + i + 1]);
                }
            }
            tc05::fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&s_free[k]);
            if (!full) {
#pragma unroll
                for (int c = 0; c < 64; ++c)
                    if (t * BN + c >= sees || ck[c / 16] < 0.0f) sv[c] = -INFINITY;
            }
            float mx = -INFINITY;
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                float mq[2] = {-INFINITY, -INFINITY};
#pragma unroll
                for (int c = 0; c < 16; c += 2) mq[(c >> 1) & 1] = max3(mq[(c >> 1) & 1], sv[16 * g + c], sv[16 * g + c + 1]);
                ck[g] = c2 * fabsf(ck[g]);
                mx = fmaxf(mx, fmaf(fmaxf(mq[0], mq[1]), ck[g], cv[g]));
            }
            // the reference follows the maximum by more than 2^kSlack only
            float alpha = 1.0f;
            if (mx > m_used + kSlack) {
                alpha = (m_used == -INFINITY) ? 0.0f : exp2f(m_used - mx);
                m_used = mx;
            }
            float sum = 0.0f;
            if (m_used == -INFINITY) {
#pragma unroll
                for (int c = 0; c < 64; ++c) sv[c] = sv[c] == sv[c] ? 0.0f : sv[c];
            } else {
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const float o = cv[g] - m_used + kBias;
                    const uint64_t cp = pk2(ck[g], ck[g]), op = pk2(o, o);
                    uint64_t sp = pk2(0.0f, 0.0f);
#pragma unroll
                    for (int c = 16 * g; c < 16 * g + 16; c += 2) {
                        float e0, e1;
                        upk2(fma2p(pk2(sv[c], sv[c + 1]), cp, op), e0, e1);
                        sv[c] = exp2_approx(e0);
                        sv[c + 1] = exp2_approx(e1);
                        sp = add2p(sp, pk2(sv[c], sv[c + 1]));
                    }
                    float s0, s1;
                    upk2(sp, s0, s1);
                    sum = fmaf(s0 + s1, ci[g], sum);
                }
            }
            l = l * alpha + sum;
            // PV_{t-1} has read P and written O: P may be rewritten, O rescaled
            if (t > 0) {
                if (!warp_wait(&o_done[k], (t - 1) & 1, abort, a.c.err)) {
                    ok = false;
                    break;
                }
                tc05::fence_after();
                if (__any_sync(0xffffffffu, alpha != 1.0f)) {
#pragma unroll
                    for (int c = 0; c < D / 32; ++c) {
                        float v[32];
                        tc05::ld32(tO + c * 32, v);
                        tc05::wait_ld();
#pragma unroll
                        for (int i = 0; i < 32; ++i) v[i] *= alpha;
                        tc05::st32(tO + c * 32, v);
                    }
                    tc05::wait_st();
                }
            }
            {
                const uint32_t prow = sb + L::PR + k * PTILE + r * 128;
#pragma unroll
                for (int cc = 0; cc < 8; ++cc)
                    st_shared_v4(prow + ((cc ^ (r & 7)) << 4), pack_f16(sv[cc * 8 + 0], sv[cc * 8 + 1]),
                                 pack_f16(sv[cc * 8 + 2], sv[cc * 8 + 3]), pack_f16(sv[cc * 8 + 4], sv[cc * 8 + 5]),
                                 pack_f16(sv[cc * 8 + 6], sv[cc * 8 + 7]));
            }
            fence_proxy_async_smem();
            tc05::fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_full[k]);
        }
        // ---- out = O / l, lse = m ln 2 + ln l; a row that sees no key gives zeros
        if (ok && (nt == 0 || warp_wait(&o_done[k], (nt - 1) & 1, abort, a.c.err))) {
            tc05::fence_after();
            const bool live = row < rows;
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
            // (of this row's tiles all is written: their info_full says so)
            const int odd0 = *(volatile int *)odd_tiles, odd1 = *(volatile int *)(odd_tiles + 1);
            const int64_t at = (int64_t)(first + tok) * a.heads + head * a.rep + (row - tok * a.rep);
#pragma unroll
            for (int c = 0; c < D / 32; ++c) {
                float v[32];
                if (nt > 0) {
                    tc05::ld32(tO + c * 32, v);
                    tc05::wait_ld();
                } else {
#pragma unroll
                    for (int i = 0; i < 32; ++i) v[i] = 0.0f;
                }
                if (live && odd1 >= odd0) {
                    // the block's elements of the keys that were left out, as they are: infinite, or NaN
                    const int *table = a.c.table + b * a.c.table_stride;
#pragma unroll 1
                    for (int key = odd0 * BN; key < min(sees, (odd1 + 1) * BN); ++key) {
                        const uint8_t *src = a.c.group_of_row<D>(table, head, key >> 4);
                        if (!src) continue;
                        const float d = __half2float(*reinterpret_cast<const __half *>(src + KvQ4<D>::v_scale(key & 15, c)));
                        if (fabsf(d) < INFINITY) continue;
#pragma unroll
                        for (int g = 0; g < 8; ++g) {
                            const uint32_t w = *reinterpret_cast<const uint16_t *>(src + KvQ4<D>::v_half(key & 15, g, c));
#pragma unroll
                            for (int i = 0; i < 4; ++i) v[4 * g + i] = fmaf((float)(int)(w >> (4 * i) & 15) - 8.0f, d, v[4 * g + i]);
                        }
                    }
                }
                if (live) {
                    uint32_t w[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i] * inv, v[2 * i + 1] * inv);
                        w[i] = *reinterpret_cast<const uint32_t *>(&h);
                    }
                    uint4 *dst = reinterpret_cast<uint4 *>(static_cast<T *>(a.out) + at * D + c * 32);
#pragma unroll
                    for (int i = 0; i < 4; ++i) dst[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
                }
            }
            if (live && a.lse) a.lse[at] = l == 0.0f ? 0.0f : (m_used - kBias) * 0.6931471805599453f + logf(l);
        }
    }

    tc05::fence_before();
    __syncthreads();
    if (warp == 9) {
        tc05::fence_after();
        tc05::dealloc(tmem, 512);
    }
}

template <int D>
int launch(const Attend &a, cudaStream_t stream) {
    const char *op = "tn_sdpa_q4_cache";
    static std::atomic<uint64_t> ready{0};  // a bit a device
    int device = 0;
    int st = check_cuda(cudaGetDevice(&device), op, "cudaGetDevice");
    if (st) return st;
    auto kernel = sdpa_q4_prefill_kernel<D>;
    if (!(ready.load(std::memory_order_relaxed) >> device & 1)) {
        st = check_cuda(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Layout<D>::SMEM), op,
                        "cudaFuncSetAttribute");
        if (st) return st;
        ready.fetch_or(1ull << device, std::memory_order_relaxed);
    }
    // the requests' pairs of tiles: every one of its own may be part full
    const int64_t slots = (int64_t)a.tokens * a.rep / (NQT * BM) + std::min<int64_t>(a.c.requests, a.tokens);
    if (slots * a.c.kv_heads > INT32_MAX)
        return set_error(TN_ERR_SHAPE, std::string(op) + ": too many query rows for one call");
    __atomic_fetch_add(&counters().sdpa_prefill_launches, 1ull, __ATOMIC_RELAXED);
    return launch_pdl(kernel, dim3((unsigned)(slots * a.c.kv_heads)), dim3(THREADS), Layout<D>::SMEM, stream, op, a,
                      (int)slots, 0x64006400u, 0x54005400u);
}

}  // namespace

int launch_sdpa_q4_prefill(const Attend &a, int head_dim, cudaStream_t stream) {
    return head_dim == 128 ? launch<128>(a, stream) : launch<64>(a, stream);
}

}  // namespace tn
