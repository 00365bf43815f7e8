// kv_q4.cuh -- the paged 4-bit KV cache: its layout in memory, and what the
// kernels that fill and read it share.
//
// A pool holds pages of `page_size` tokens (a power of two from 16 on) for
// every KV head; a page of one head is page_size / 16 groups of 16 tokens, and
// a group is 18 * D contiguous bytes:
//   [0, 8D)     K codes   [16 tokens][4 t][D/32 blocks] words of 8 nibbles: nibble
//                         n < 4 of word (t, block) is element 8t + 2n of the block's
//                         32, nibble 4 + n is element 8t + 2n + 1
//   [8D, 9D)    K scales  [16 tokens][D/32] f16
//   [9D, 17D)   V codes   [2 h][8 g][4 t][D/32] words of two 16-bit halves: half p
//                         is token 8h + 2t + p, its nibble n is element 4g + n
//   [17D, 18D)  V scales  [16 tokens][D/32] f16
// Codes and scales are GGML Q4_0's (BlockQ4_0::from_float, k_quants.rs:241-277),
// only their order differs. It is the order in which a warp's m16n8k16 tensor
// instructions take them: lane 4g + t finds the 8D / 32 bytes of its K rows
// (tokens g and g + 8) and of its V columns (tokens 2t, 2t + 1, 2t + 8, 2t + 9)
// as whole 16-byte (D = 64: 8-byte) vectors, neighbouring lanes next to each
// other, and each extraction mask yields the two elements of one operand
// register. A group's bytes are a multiple of 16, so that one bulk copy brings
// it to shared memory.
#pragma once

#include <string>
#include <type_traits>

#include "tn_common.cuh"

namespace tn {

constexpr int kKvGroup = 16;
// Tokens that a table's row may name: 32-bit positions with room for a tile behind the last one.
constexpr int64_t kMaxRowTokens = ((int64_t)1 << 31) - 1024;

template <int D>
struct KvQ4 {
    static constexpr int NB = D / 32;           // blocks a row
    static constexpr int GROUP_BYTES = 18 * D;  // 16 tokens of one head, K and V
    static constexpr int K_CODES = 0, K_SCALES = 8 * D, V_CODES = 9 * D, V_SCALES = 17 * D;
    // byte of the K word (t, block) of token `key` of a group
    __host__ __device__ static constexpr int k_word(int key, int t, int block) {
        return K_CODES + key * (D / 2) + (t * NB + block) * 4;
    }
    // byte of the 16-bit V piece (elements 4g .. 4g + 3 of a block) of token `key`
    __host__ __device__ static constexpr int v_half(int key, int g, int block) {
        return V_CODES + (key >> 3) * 4 * D + ((g * 4 + ((key & 7) >> 1)) * NB + block) * 4 + (key & 1) * 2;
    }
    __host__ __device__ static constexpr int k_scale(int key, int block) { return K_SCALES + (key * NB + block) * 2; }
    __host__ __device__ static constexpr int v_scale(int key, int block) { return V_SCALES + (key * NB + block) * 2; }
};

// The cache as a call gives it. Page ids, lengths and slots live on the device,
// so the kernels check them: an id outside [0, num_pages) is never followed.
struct KvPool {
    uint8_t *pool;
    int num_pages, page_shift, kv_heads;
    const int *table;  // [requests][table_stride] page ids
    int64_t table_stride;
    int max_pages;
    const int *lengths;  // [requests] cached tokens
    int requests;
    int *err;

    // The cached tokens of request b, within what its table row can name.
    __device__ __forceinline__ int length(int b) const {
        const int64_t cap = (int64_t)max_pages << page_shift;
        const int n = lengths[b];
        return n < 0 ? 0 : (n > cap ? (int)cap : n);
    }
    // The group of tokens [16 group, 16 group + 16) of request b, or NULL (and
    // the word for bad pages set) where the table names no page of the pool.
    // (A pool holds fewer than 2^31 groups: 4.9 TB.)
    template <int D>
    __device__ __forceinline__ uint8_t *group(int b, int kvh, int group) const {
        return group_of_row<D>(table + b * table_stride, kvh, group);
    }
    template <int D>
    __device__ __forceinline__ uint8_t *group_of_row(const int *row, int kvh, int group) const {
        const int shift = page_shift - 4, page = row[group >> shift];
        if ((unsigned)page >= (unsigned)num_pages) {
            record_bad_page(err);
            return nullptr;
        }
        return pool + (int64_t)(((page * kv_heads + kvh) << shift) + (group & ((1 << shift) - 1))) * KvQ4<D>::GROUP_BYTES;
    }
};

// A launch that may begin while the kernel before it ends (programmatic
// dependent launch): every kernel of the cache waits for that kernel's memory
// itself, before it reads or writes anything.
template <typename K, typename... Args>
int launch_pdl_cluster(K kernel, dim3 grid, dim3 block, int smem, cudaStream_t stream, const char *what, int cluster,
                       Args... args) {
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = (size_t)smem;
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    return check_cuda(cudaLaunchKernelEx(&cfg, kernel, args...), what, "cudaLaunchKernelEx");
}
template <typename K, typename... Args>
int launch_pdl(K kernel, dim3 grid, dim3 block, int smem, cudaStream_t stream, const char *what, Args... args) {
    return launch_pdl_cluster(kernel, grid, block, smem, stream, what, 1, args...);
}

int check_kv_pool(const char *op, const void *pool, int64_t num_pages, int64_t kv_heads, int64_t head_dim,
                  int64_t page_size);
int kv_page_shift(int64_t page_size);  // log2 of a page size the cache takes, else -1

// Eight neighbouring elements (16-byte aligned), widened.
template <typename T>
__device__ __forceinline__ void load8(const T *src, float (&x)[8]) {
    if constexpr (sizeof(T) == 4) {
        const float4 a = *reinterpret_cast<const float4 *>(src), b = *reinterpret_cast<const float4 *>(src + 4);
        x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
    } else {
        const uint4 a = *reinterpret_cast<const uint4 *>(src);
        const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const unsigned short u = (unsigned short)(w[i >> 1] >> (16 * (i & 1)));
            T e;
            memcpy(&e, &u, 2);
            x[i] = to_f32<T>(e);
        }
    }
}

__device__ __forceinline__ float round_bf16(float x) { return __bfloat162float(__float2bfloat16_rn(x)); }

// The Q4_0 code of x in a block with reciprocal scale `inv`: trunc(x * inv + 8.5)
// in [0, 15], NaN to 0 (Rust's `as u8`, then min 15), in the low bits of a float
// at 2^23, whose last place is 1 and whose sum rounds toward zero. Explicitly
// rounded, so that no contraction changes a byte.
constexpr uint32_t kCodeBase = 0x4b000000u;  // the bits of 2^23
__device__ __forceinline__ uint32_t q4_0_code_at_2_23(float x, float inv) {
    const float v = __fadd_rn(__fmul_rn(x, inv), 8.5f);
    return __float_as_uint(__fadd_rz(fminf(fmaxf(v, 0.0f), 15.0f), 8388608.0f));
}
// Codes at the nibbles `at[i]` of a word; the floats' upper bits, the same of every one, go off at the end.
template <int N>
__device__ __forceinline__ uint32_t q4_0_word(const float (&x)[8], float inv, const int (&at)[N]) {
    uint32_t w = 0, base = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        w += q4_0_code_at_2_23(x[i], inv) * (1u << (4 * at[i]));
        base += kCodeBase * (1u << (4 * at[i]));
    }
    return w - base;
}
// d = m / -8 and 1 / d (0 where d is 0) of a block, as IEEE float32 divisions give them: the first is a product by a
// power of two.
__device__ __forceinline__ float q4_0_scale(float m) { return __fmul_rn(m, -0.125f); }
__device__ __forceinline__ float q4_0_inverse(float d) { return d != 0.0f ? __frcp_rn(d) : 0.0f; }

__device__ __forceinline__ float max3(float a, float b, float c) {
    float y;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
    return y;
}
__device__ __forceinline__ float min3(float a, float b, float c) {
    float y;
    asm("min.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
    return y;
}

// The element of largest magnitude of a block of 32 held 8 a lane by 4
// neighbouring lanes in element order; the first of equals, as
// BlockQ4_0::from_float's loop finds it (NaN never wins its comparison): the
// block's maximum or its minimum, and only where their magnitudes are the same,
// which is looked at by the whole warp, the elements one after the other.
__device__ __forceinline__ float q4_0_extreme(const float (&x)[8]) {
    float hi = max3(0.0f, x[0], x[1]), lo = min3(0.0f, x[0], x[1]);
#pragma unroll
    for (int i = 2; i < 8; i += 2) {
        hi = max3(hi, x[i], x[i + 1]);
        lo = min3(lo, x[i], x[i + 1]);
    }
#pragma unroll
    for (int off = 1; off < 4; off <<= 1) {
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, off));
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, off));
    }
    float m = hi > -lo ? hi : lo;
    if (__any_sync(0xffffffffu, hi == -lo)) {
        float amax = 0.0f, first = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float a = fabsf(x[i]);
            if (amax < a) amax = a, first = x[i];
        }
#pragma unroll
        for (int off = 1; off < 4; off <<= 1) {
            const float oa = __shfl_xor_sync(0xffffffffu, amax, off), om = __shfl_xor_sync(0xffffffffu, first, off);
            // the lower lane's element comes first: of equals it wins
            const bool other = (threadIdx.x & off) ? !(oa < amax) : (amax < oa);
            if (other) amax = oa, first = om;
        }
        m = first;
    }
    return m;
}

// 8 elements a lane (lane t of the block's 4) -> the lane's K word, or its two
// V pieces (g = 2t low, g = 2t + 1 high).
__device__ __forceinline__ uint32_t q4_0_k_word(const float (&x)[8], float inv) {
    constexpr int at[8] = {0, 4, 1, 5, 2, 6, 3, 7};
    return q4_0_word<8>(x, inv, at);
}
__device__ __forceinline__ uint32_t q4_0_v_halves(const float (&x)[8], float inv) {
    constexpr int at[8] = {0, 1, 2, 3, 4, 5, 6, 7};
    return q4_0_word<8>(x, inv, at);
}

}  // namespace tn
