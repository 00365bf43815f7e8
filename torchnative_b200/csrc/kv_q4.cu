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

// Work item: one block of one row, four lanes. Items run over blocks, then K
// and V, then heads, then tokens.
template <typename T, int D>
__global__ void __launch_bounds__(kThreads) kv_q4_append_kernel(const Append p) {
    using Q = KvQ4<D>;
    pdl_launch_dependents();
    pdl_wait();
    const int64_t item = (blockIdx.x * (int64_t)kThreads + threadIdx.x) >> 2;
    const int t = threadIdx.x & 3;
    const int block = (int)(item % Q::NB);
    const int is_v = (int)(item / Q::NB % 2);
    const int64_t row = item / (2 * Q::NB);
    const int head = (int)(row % p.kv_heads);
    const int64_t token = row / p.kv_heads;
    const bool live = token < p.tokens;
    int64_t slot = live ? p.slots[token] : -1;
    if (slot >= p.num_slots) {  // never followed
        record_device_error(p.err, DEV_ERR_BAD_PAGE);
        slot = -1;
    }
    float x[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
    if (slot >= 0) {
        const T *src = is_v ? static_cast<const T *>(p.v) + token * p.v_token + head * p.v_head
                            : static_cast<const T *>(p.k) + token * p.k_token + head * p.k_head;
        load8<T>(src + block * 32 + t * 8, x);
    }
    const float d = __fdiv_rn(q4_0_extreme(x), -8.0f);
    const float inv = (d != 0.0f) ? __fdiv_rn(1.0f, d) : 0.0f;
    if (slot < 0) return;
    const int64_t page = slot >> p.page_shift;
    const int in_page = (int)(slot & ((1 << p.page_shift) - 1)), key = in_page & 15;
    uint8_t *g = p.pool + (((page * p.kv_heads + head) << (p.page_shift - 4)) + (in_page >> 4)) * Q::GROUP_BYTES;
    if (is_v) {
        const uint32_t w = q4_0_v_halves(x, inv);
        *reinterpret_cast<unsigned short *>(g + Q::v_half(key, 2 * t, block)) = (unsigned short)w;
        *reinterpret_cast<unsigned short *>(g + Q::v_half(key, 2 * t + 1, block)) = (unsigned short)(w >> 16);
    } else {
        *reinterpret_cast<uint32_t *>(g + Q::k_word(key, t, block)) = q4_0_k_word(x, inv);
    }
    if (t == 0)
        *reinterpret_cast<__half *>(g + (is_v ? Q::v_scale(key, block) : Q::k_scale(key, block))) = __float2half_rn(d);
}

template <typename T, int D>
int launch_append(const Append &p, cudaStream_t stream) {
    const int64_t threads = p.tokens * p.kv_heads * 2 * KvQ4<D>::NB * 4;
    return launch_pdl(kv_q4_append_kernel<T, D>, dim3((unsigned)((threads + kThreads - 1) / kThreads)), dim3(kThreads),
                      0, stream, "tn_kv_q4_append", p);
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
