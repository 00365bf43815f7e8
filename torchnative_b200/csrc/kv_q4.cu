// kv_q4.cu -- the quantising append of the paged 4-bit KV cache.
//
// Per 32 elements of a key or value row: m the element of largest magnitude,
// d = m / -8, code = min(15, trunc(x / d + 8.5)), stored as codes and f16(d):
// the bytes of tn_q4_0_quantize in the cache's order. Four lanes hold a block,
// eight elements each, which are one whole K word (two V pieces), so that no
// lane needs another's codes.
#include "kv_q4.cuh"

namespace tn {
namespace {

constexpr int kThreads = 256;

struct Append {
    const void *k, *v;
    int64_t k_token, k_head, v_token, v_head;  // element strides
    const int64_t *slots;
    int64_t tokens, num_slots;
    uint8_t *pool;
    int kv_heads, page_shift;
    int *err;
};

// One warp: 256 / D neighbouring tokens of one head, keys and values; a lane has
// eight elements of a row. 2 D elements read and 9 D / 8 bytes written
// a token and head; bound by the quantiser's instructions where there are many: 8192 tokens of 8 x 128 bf16 take 13.7
// us, 3.1 TB/s (half a copy's rate), 342 instructions a warp, issue active in 79% of the cycles; 32 tokens take 1.8 us,
// a launch.
template <typename T, int D>
__global__ void __launch_bounds__(kThreads) kv_q4_append_kernel(const Append p) {
    using Q = KvQ4<D>;
    constexpr int ROW_LANES = D / 8, TOKENS = 32 / ROW_LANES;
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x & 31, t = lane & 3, block = lane % ROW_LANES >> 2, head = blockIdx.y;
    const int64_t token = (blockIdx.x * (int64_t)(kThreads / 32) + (threadIdx.x >> 5)) * TOKENS + lane / ROW_LANES;
    const bool live = token < p.tokens;
    float k[8], v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) k[i] = v[i] = 0.0f;
    int64_t slot = -1;
    if (live) {
        slot = p.slots[token];
        const int64_t e = block * 32 + t * 8;
        load8<T>(static_cast<const T *>(p.k) + token * p.k_token + head * p.k_head + e, k);
        load8<T>(static_cast<const T *>(p.v) + token * p.v_token + head * p.v_head + e, v);
    }
    const float kd = q4_0_scale(q4_0_extreme(k)), vd = q4_0_scale(q4_0_extreme(v));
    const uint32_t kw = q4_0_k_word(k, q4_0_inverse(kd)), vw = q4_0_v_halves(v, q4_0_inverse(vd));
    // an even token whose odd neighbour's row is in the other half of the lanes: their 16-bit pieces as words
    const uint32_t vw2 = __shfl_xor_sync(0xffffffffu, vw, ROW_LANES);
    const int64_t slot2 = __shfl_xor_sync(0xffffffffu, slot, ROW_LANES);
    if (slot >= p.num_slots) {  // never followed
        record_bad_page(p.err);
        return;
    }
    if (slot < 0) return;
    const int64_t page = slot >> p.page_shift;
    const int in_page = (int)(slot & ((1 << p.page_shift) - 1)), key = in_page & 15;
    uint8_t *g = p.pool + (((page * p.kv_heads + head) << (p.page_shift - 4)) + (in_page >> 4)) * Q::GROUP_BYTES;
    *reinterpret_cast<uint32_t *>(g + Q::k_word(key, t, block)) = kw;
    if ((slot ^ 1) == slot2) {
        const int odd = key & 1;
        const uint32_t word = odd ? (vw2 >> 16) | (vw & 0xffff0000u) : (vw & 0xffffu) | (vw2 << 16);
        *reinterpret_cast<uint32_t *>(g + Q::v_half(key & ~1, 2 * t + odd, block)) = word;
    } else {
        *reinterpret_cast<unsigned short *>(g + Q::v_half(key, 2 * t, block)) = (unsigned short)vw;
        *reinterpret_cast<unsigned short *>(g + Q::v_half(key, 2 * t + 1, block)) = (unsigned short)(vw >> 16);
    }
    if (t == 0) {
        *reinterpret_cast<__half *>(g + Q::k_scale(key, block)) = __float2half_rn(kd);
        *reinterpret_cast<__half *>(g + Q::v_scale(key, block)) = __float2half_rn(vd);
    }
}

template <typename T, int D>
int launch_append(const Append &p, cudaStream_t stream) {
    constexpr int tokens = kThreads / 32 * (256 / D);  // of a CTA
    return launch_pdl(kv_q4_append_kernel<T, D>, dim3((unsigned)((p.tokens + tokens - 1) / tokens), (unsigned)p.kv_heads),
                      dim3(kThreads), 0, stream, "tn_kv_q4_append", p);
}

bool aligned(const void *p, int64_t token, int64_t head, int64_t size) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && token * size % 16 == 0 && head * size % 16 == 0;
}

}  // namespace
}  // namespace tn

extern "C" int tn_kv_q4_append(const void *k, const void *v, int dtype, const int64_t *k_strides,
                               const int64_t *v_strides, int64_t tokens, const int64_t *slots, void *pool,
                               int64_t num_pages, int64_t kv_heads, int64_t head_dim, int64_t page_size, void *stream) {
    const std::string op("tn_kv_q4_append");
    int st = tn::check_kv_pool("tn_kv_q4_append", pool, num_pages, kv_heads, head_dim, page_size);
    if (st) return st;
    if (dtype != TN_F32 && dtype != TN_F16 && dtype != TN_BF16)
        return tn::set_error(TN_ERR_NOT_IMPLEMENTED, op + ": keys and values must be float32, float16 or bfloat16, got " +
                                                         tn_dtype_name(dtype));
    if (tokens < 0 || tokens > ((int64_t)1 << 40) / (kv_heads * head_dim))
        return tn::set_error(TN_ERR_SHAPE, op + ": bad token count");
    if (tokens == 0) return TN_OK;
    if (!k || !v || !slots || !k_strides || !v_strides) return tn::set_error(TN_ERR_INVALID, op + ": null pointer");
    const int64_t size = (int64_t)tn_dtype_size(dtype);
    if (!tn::aligned(k, k_strides[0], k_strides[1], size) || !tn::aligned(v, v_strides[0], v_strides[1], size))
        return tn::set_error(TN_ERR_INVALID, op + ": key and value rows must be 16-byte aligned with a unit inner stride");
    tn::Append p{k, v, k_strides[0], k_strides[1], v_strides[0], v_strides[1], slots, tokens, num_pages * page_size,
                 static_cast<uint8_t *>(pool), (int)kv_heads, tn::kv_page_shift(page_size), tn::device_error_word()};
    __atomic_fetch_add(&tn::counters().q4_codec_launches, 1ull, __ATOMIC_RELAXED);
    cudaStream_t s = tn::stream_of(stream);
    if (head_dim == 128)
        return dtype == TN_F32   ? tn::launch_append<float, 128>(p, s)
               : dtype == TN_F16 ? tn::launch_append<__half, 128>(p, s)
                                 : tn::launch_append<__nv_bfloat16, 128>(p, s);
    return dtype == TN_F32   ? tn::launch_append<float, 64>(p, s)
           : dtype == TN_F16 ? tn::launch_append<__half, 64>(p, s)
                             : tn::launch_append<__nv_bfloat16, 64>(p, s);
}
