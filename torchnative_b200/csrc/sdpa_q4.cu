// sdpa_q4.cu -- attention over the paged 4-bit KV cache.
//
// Token i of the n query tokens of a request whose cache holds S tokens (its
// own included) attends keys 0 .. S - n + i:
//   s_j = scale * q . (d_j * (code_j - 8)),  out = sum_j e^(s_j - m) v_j / l,
//   lse = m + log l;
// a token that sees no key gives zeros and lse 0, as the dense operator does.
#include "kv_q4.cuh"

namespace tn {
namespace {

struct Attend {
    const void *q;
    int64_t q_token, q_head;  // element strides
    KvPool c;
    const int *query_start;  // [requests + 1], or NULL: token r is request r's only one
    void *out;               // [tokens][heads][D]
    float *lse;              // [tokens][heads] or NULL
    int tokens, heads, rep;
    float scale;
};

// The request of packed token r and the number of its keys that r sees; -1 for
// a row behind the last request's.
__device__ __forceinline__ int request_of(const Attend &p, int r, int *keys) {
    int b = r, first = r, n = 1;
    if (p.query_start) {
        int lo = 0, hi = p.c.requests;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (p.query_start[mid] <= r)
                lo = mid;
            else
                hi = mid;
        }
        b = lo;
        first = p.query_start[b];
        n = p.query_start[b + 1] - first;
        if (r < first || r >= first + n) return -1;
    }
    *keys = p.c.length(b) - n + (r - first) + 1;
    return b;
}

constexpr int kSimpleThreads = 128;

// One CTA for one (token, head): a thread per key, then a thread per dimension.
template <typename T, int D>
__global__ void __launch_bounds__(kSimpleThreads) sdpa_q4_simple_kernel(const Attend p) {
    using Q = KvQ4<D>;
    __shared__ float q[D], s[kSimpleThreads], part[kSimpleThreads], red[4];
    __shared__ const uint8_t *groups[kSimpleThreads / 16];
    const int tid = threadIdx.x, r = blockIdx.x, h = blockIdx.y, lane = tid & 31, warp = tid >> 5;
    pdl_launch_dependents();
    pdl_wait();
    int keys = 0;
    const int b = request_of(p, r, &keys);
    if (b < 0) return;
    for (int d = tid; d < D; d += kSimpleThreads)
        q[d] = to_f32<T>(static_cast<const T *>(p.q)[r * p.q_token + h * p.q_head + d]);
    constexpr int HALVES = kSimpleThreads / D;  // key halves of the second product
    const int dim = tid % D, half = tid / D;
    float m = -INFINITY, l = 0.0f, o = 0.0f;
    for (int j0 = 0; j0 < keys; j0 += kSimpleThreads) {
        __syncthreads();
        if (tid < kSimpleThreads / 16)
            groups[tid] = j0 + tid * 16 < keys ? p.c.group<D>(b, h / p.rep, j0 / 16 + tid) : nullptr;
        __syncthreads();
        const uint8_t *g = groups[tid / 16];
        float x = -INFINITY;
        if (j0 + tid < keys && g) {
            x = 0.0f;
            for (int block = 0; block < Q::NB; ++block) {
                float dot = 0.0f;
                for (int t = 0; t < 4; ++t) {
                    const uint32_t w = *reinterpret_cast<const uint32_t *>(g + Q::k_word(tid & 15, t, block));
#pragma unroll
                    for (int n = 0; n < 8; ++n)
                        dot = fmaf((float)((int)((w >> (4 * n)) & 15) - 8), q[block * 32 + t * 8 + 2 * (n & 3) + (n >> 2)],
                                   dot);
                }
                x = fmaf(dot, __half2float(*reinterpret_cast<const __half *>(g + Q::k_scale(tid & 15, block))), x);
            }
            x *= p.scale;
        }
        float mx = x;
#pragma unroll
        for (int off = 16; off; off >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
        if (lane == 0) red[warp] = mx;
        __syncthreads();
        mx = fmaxf(m, fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])));
        const float alpha = mx == -INFINITY ? 1.0f : expf(m - mx);
        s[tid] = x == -INFINITY ? 0.0f : expf(x - mx);
        m = mx;
        __syncthreads();
        l *= alpha;
        o *= alpha;
        for (int j = 0; j < kSimpleThreads; ++j) l += s[j];
        for (int j = half; j < min(kSimpleThreads, keys - j0); j += HALVES) {
            const uint8_t *v = groups[j / 16];
            if (!v) continue;
            const uint32_t w = *reinterpret_cast<const unsigned short *>(v + Q::v_half(j & 15, dim % 32 / 4, dim / 32));
            const float d = __half2float(*reinterpret_cast<const __half *>(v + Q::v_scale(j & 15, dim / 32)));
            o = fmaf(s[j] * d, (float)((int)((w >> (4 * (dim & 3))) & 15) - 8), o);
        }
    }
    part[tid] = o;
    __syncthreads();
    if (tid < D) {
        float v = 0.0f;
        for (int i = 0; i < HALVES; ++i) v += part[i * D + tid];
        const int64_t at = ((int64_t)r * p.heads + h) * D + tid;
        v = l == 0.0f ? 0.0f : v / l;
        if constexpr (sizeof(T) == 4)
            static_cast<float *>(p.out)[at] = v;
        else if constexpr (std::is_same<T, __half>::value)
            static_cast<__half *>(p.out)[at] = __float2half_rn(v);
        else
            static_cast<__nv_bfloat16 *>(p.out)[at] = __float2bfloat16_rn(v);
        if (tid == 0 && p.lse) p.lse[(int64_t)r * p.heads + h] = l == 0.0f ? 0.0f : m + logf(l);
    }
}

template <typename T, int D>
int launch_attend(const Attend &p, cudaStream_t stream) {
    return launch_pdl(sdpa_q4_simple_kernel<T, D>, dim3((unsigned)p.tokens, (unsigned)p.heads), dim3(kSimpleThreads), 0,
                      stream, "tn_sdpa_q4_cache", p);
}

// Rotates the q and k heads of one projection row at the request's last
// position and appends k and v there: q_out [B][heads][D].
template <int D>
__global__ void rope_append_q4_kernel(const __nv_bfloat16 *qkv, const __nv_bfloat16 *rope, int64_t rope_rows, KvPool c,
                                      int heads, __nv_bfloat16 *q_out) {
    using Q = KvQ4<D>;
    __shared__ float row[D];
    pdl_launch_dependents();
    pdl_wait();
    const int b = blockIdx.y, h = blockIdx.x, W = heads + 2 * c.kv_heads, i = threadIdx.x;
    const __nv_bfloat16 *x = qkv + ((int64_t)b * W + h) * D;
    const int pos = c.length(b) - 1;
    if (pos >= 0 && pos >= rope_rows) record_device_error(c.err, DEV_ERR_BAD_PAGE);
    const int at = (int)max((int64_t)0, min((int64_t)pos, rope_rows - 1));
    if (i < D / 2) {
        const float cs = __bfloat162float(rope[(int64_t)at * D + i]), sn = __bfloat162float(rope[(int64_t)at * D + D / 2 + i]);
        float a = __bfloat162float(x[i]), e = __bfloat162float(x[i + D / 2]);
        if (h < heads + c.kv_heads) {
            const float a2 = a * cs - e * sn, e2 = e * cs + a * sn;
            a = a2, e = e2;
        }
        row[i] = __bfloat162float(__float2bfloat16_rn(a));
        row[i + D / 2] = __bfloat162float(__float2bfloat16_rn(e));
    }
    __syncthreads();
    if (h < heads) {
        for (int d = i; d < D; d += blockDim.x) q_out[((int64_t)b * heads + h) * D + d] = __float2bfloat16_rn(row[d]);
        return;
    }
    if (pos < 0 || pos >= rope_rows) return;
    const int kvh = (h - heads) % c.kv_heads, is_v = h >= heads + c.kv_heads, key = pos & 15;
    uint8_t *g = c.group<D>(b, kvh, pos >> 4);
    if (!g || i >= 32) return;
    float v[8];
    const int block = (i >> 2) % Q::NB, t = i & 3;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = row[block * 32 + t * 8 + e];
    const float d = __fdiv_rn(q4_0_extreme(v), -8.0f);
    const float inv = (d != 0.0f) ? __fdiv_rn(1.0f, d) : 0.0f;
    if (i >= 4 * Q::NB) return;
    if (is_v) {
        const uint32_t w = q4_0_v_halves(v, inv);
        *reinterpret_cast<unsigned short *>(g + Q::v_half(key, 2 * t, block)) = (unsigned short)w;
        *reinterpret_cast<unsigned short *>(g + Q::v_half(key, 2 * t + 1, block)) = (unsigned short)(w >> 16);
    } else {
        *reinterpret_cast<uint32_t *>(g + Q::k_word(key, t, block)) = q4_0_k_word(v, inv);
    }
    if (t == 0)
        *reinterpret_cast<__half *>(g + (is_v ? Q::v_scale(key, block) : Q::k_scale(key, block))) = __float2half_rn(d);
}

int check_cache(const char *op, const KvPool &c, int64_t requests, int64_t max_pages, int64_t table_stride,
                int64_t heads, int64_t kv_heads, int64_t tokens) {
    const std::string name(op);
    if (requests < 0 || requests > 65535 || max_pages < 0 || table_stride < max_pages ||
        max_pages > (int64_t)INT32_MAX >> c.page_shift || tokens < 0 || tokens > INT32_MAX / 2)
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
    (void)kv_heads, (void)max_query;
    return tokens * heads * head_dim * 2 + 256;
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
    (void)max_query;
    if (!workspace || workspace_bytes < tn_sdpa_q4_workspace_bytes(tokens, heads, kv_heads, head_dim, max_query))
        return tn::set_error(TN_ERR_SHAPE, std::string(op) + ": the workspace is smaller than tn_sdpa_q4_workspace_bytes");
    const float sc = scale > 0.0 ? (float)scale : 1.0f / sqrtf((float)head_dim);
    tn::Attend p{q, q_strides[0], q_strides[1], c, query_start, out, lse, (int)tokens, (int)heads, (int)(heads / kv_heads), sc};
    __atomic_fetch_add(&tn::counters().sdpa_calls, 1ull, __ATOMIC_RELAXED);
    __atomic_fetch_add(&tn::counters().sdpa_decode_launches, 1ull, __ATOMIC_RELAXED);
    cudaStream_t s = tn::stream_of(stream);
    if (head_dim == 128)
        return dtype == TN_F32   ? tn::launch_attend<float, 128>(p, s)
               : dtype == TN_F16 ? tn::launch_attend<__half, 128>(p, s)
                                 : tn::launch_attend<__nv_bfloat16, 128>(p, s);
    return dtype == TN_F32   ? tn::launch_attend<float, 64>(p, s)
           : dtype == TN_F16 ? tn::launch_attend<__half, 64>(p, s)
                             : tn::launch_attend<__nv_bfloat16, 64>(p, s);
}

extern "C" int tn_sdpa_q4_decode_step(const void *qkv, const void *rope, int64_t rope_rows, void *pool, int64_t num_pages,
                                      int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t page_size,
                                      const int *page_table, int64_t table_stride, int64_t max_pages, const int *lengths,
                                      int64_t requests, void *out, float *lse, int8_t *codes, float *scales,
                                      float *offsets, double scale, void *workspace, int64_t workspace_bytes,
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
    void *q = workspace;
    __atomic_fetch_add(&tn::counters().sdpa_calls, 1ull, __ATOMIC_RELAXED);
    __atomic_fetch_add(&tn::counters().sdpa_decode_launches, 1ull, __ATOMIC_RELAXED);
    tn::Attend p{q, heads * head_dim, head_dim, c, nullptr, out, lse, (int)requests, (int)heads, (int)(heads / kv_heads), sc};
    const dim3 grid((unsigned)(heads + 2 * kv_heads), (unsigned)requests);
    auto kernel = head_dim == 128 ? tn::rope_append_q4_kernel<128> : tn::rope_append_q4_kernel<64>;
    st = tn::launch_pdl(kernel, grid, dim3(64), 0, s, op, (const __nv_bfloat16 *)qkv, (const __nv_bfloat16 *)rope, rope_rows,
                        c, (int)heads, (__nv_bfloat16 *)q);
    if (st) return st;
    st = head_dim == 128 ? tn::launch_attend<__nv_bfloat16, 128>(p, s) : tn::launch_attend<__nv_bfloat16, 64>(p, s);
    if (st || !codes) return st;
    return tn_q8_0_quantize_planar(out, TN_BF16, heads * head_dim, codes, heads * head_dim, scales, offsets, requests,
                                   heads * head_dim, stream);
}
