// sdpa_q4.cuh -- what the attention kernels over the paged 4-bit cache share.
#pragma once

#include "kv_q4.cuh"

namespace tn {

// One call.
struct Attend {
    const void *q;
    int64_t q_token, q_head;  // element strides
    KvPool c;
    const int *query_start;  // [requests + 1], or NULL: token r is request r's only one
    void *out;               // [tokens][heads][D]
    float *lse;              // [tokens][heads] or NULL
    int tokens, heads, rep;
    float scale;
    // Where the query tokens of request b lie: rows first .. first + n, within the call's.
    __device__ __forceinline__ int query_tokens(int b, int *first) const {
        *first = b;
        if (!query_start) return 1;
        *first = min(max(query_start[b], 0), tokens);
        return max(min(query_start[b + 1], tokens) - *first, 0);
    }
};

__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

__device__ __forceinline__ uint32_t sub_f16x2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
__device__ __forceinline__ uint32_t mul_f16x2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
__device__ __forceinline__ uint32_t fma_f16x2(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t r;
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
    return r;
}
__device__ __forceinline__ float2 unpack_f16(uint32_t v) {
    return __half22float2(*reinterpret_cast<const __half2 *>(&v));
}

// (a & mask) | bits as one instruction: `bits` in a register of its own, since an instruction takes one constant only.
__device__ __forceinline__ uint32_t and_or(uint32_t a, uint32_t mask, uint32_t bits) {
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(a), "r"(mask), "r"(bits));
    return r;
}

// The nibbles n and n + 4 of a word as half2, n = 0 .. 3: codes minus 8, except
// that with RAW the odd ones come as 64 + code.
template <bool RAW>
__device__ __forceinline__ void unpack_codes(uint32_t w, uint32_t (&e)[4], uint32_t low, uint32_t high) {
    constexpr uint32_t kLow = 0x64086408u, kHigh = 0x54805480u;  // 1032, 72
    const uint32_t u = w >> 8;
    e[0] = sub_f16x2(and_or(w, 0x000f000fu, low), kLow);
    e[1] = and_or(w, 0x00f000f0u, high);
    e[2] = sub_f16x2(and_or(u, 0x000f000fu, low), kLow);
    e[3] = and_or(u, 0x00f000f0u, high);
    if constexpr (!RAW) {
        e[1] = sub_f16x2(e[1], kHigh);
        e[3] = sub_f16x2(e[3], kHigh);
    }
}

// Many bf16 query tokens a request, on tcgen05 (sdpa_q4_prefill.cu).
int launch_sdpa_q4_prefill(const Attend &a, int head_dim, cudaStream_t stream);

}  // namespace tn
