// kv_pages.cu -- block tables and slot maps from request lengths.
//
// One call takes every request from its old length to its new one: pages of
// requests that shrink go back on the free stack, requests that grow take pages
// from its top, and every new token gets its slot, position and place in the
// packed rows. All of it is prefix sums over the requests (pages given, pages
// taken, tokens new), so the result does not depend on any order of execution.
#include <algorithm>
#include <atomic>

#include "kv_q4.cuh"

namespace tn {

int kv_page_shift(int64_t page_size) {
    for (int s = 4; s <= 10; ++s)
        if (page_size == (int64_t)1 << s) return s;
    return -1;
}

int check_kv_pool(const char *op, const void *pool, int64_t num_pages, int64_t kv_heads, int64_t head_dim,
                  int64_t page_size) {
    const std::string name(op);
    if (kv_page_shift(page_size) < 0)
        return set_error(TN_ERR_NOT_IMPLEMENTED, name + ": a page holds 16, 32, 64, 128, 256, 512 or 1024 tokens, got " +
                                                     std::to_string(page_size));
    if (head_dim != 64 && head_dim != 128)
        return set_error(TN_ERR_NOT_IMPLEMENTED, name + ": the 4-bit KV cache takes head dimensions 64 and 128, got " +
                                                     std::to_string(head_dim));
    if (num_pages < 0 || kv_heads < 1 || kv_heads > 65535 ||
        num_pages > INT32_MAX / (kv_heads * (page_size / kKvGroup)))
        return set_error(TN_ERR_SHAPE, name + ": bad page or head count");
    if ((!pool && num_pages > 0) || reinterpret_cast<uintptr_t>(pool) % 16 != 0)
        return set_error(TN_ERR_INVALID, name + ": the pool must be a 16-byte aligned device pointer");
    return TN_OK;
}

namespace {

constexpr int kThreads = 1024;
constexpr int kMaxRequests = 8192;
// Where more pages than this may move, a cluster of CTAs shares the moves; all of them compute the sums. Two calls, there
// and back, in one CTA and in the cluster: 512 requests of up to 256 pages, of which 13,300 are taken and 5,800 given, 42.7
// and 20.1 us; 512 of up to 64 pages 21.9 and 18.0, 256 of them 16.4 and 17.0; a step of 128 requests 6.4 and 8.9. (A
// thread moves one page at a time: four at once, for their loads, took 21.4 us where this takes 20.1, and 13.7 for 13.2
// with 16 requests of 1000 pages in one CTA.)
constexpr int64_t kMovesInOne = 16384;
constexpr int kCtas = 8;
// Up to here the launch that moves the pages writes the slots too; above, a second one over the whole GPU does (210,000
// new tokens of 512 requests: 144 us in one CTA, 21 in two launches).
constexpr int kSlotsInOne = 4096;

enum : int { BAD_NONE = 0, BAD_POOL = 1, BAD_LENGTH = 2, BAD_TOKENS = 3, BAD_STACK = 4 };

struct Resize {
    int *table;
    int64_t table_stride;
    int max_pages;
    int *lengths;
    const int *new_lengths;  // NULL: every request with tokens grows by `grow`
    int grow, requests;
    int *free_pages, *free_count;
    int num_pages, page_shift;
    int64_t *slots;
    int *positions;
    int max_tokens;
    int *query_start, *status;
    int *granted;  // [requests] or NULL
    int aligned;  // slots and positions may be written in 16-byte vectors
    int *err;
};

// Every thread of the cluster's CTAs, and what they wrote to global memory before; one CTA needs its own barrier only.
__device__ __forceinline__ void sync_all(int ctas) {
    if (ctas == 1) {
        __syncthreads();
    } else {
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    }
}

__device__ __forceinline__ int pages_of(int n, int shift) { return (n + (1 << shift) - 1) >> shift; }

// The last of the `n` ascending starts that is at most x (x >= starts[0] = 0).
__device__ __forceinline__ int find(const int *starts, int n, int x) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (starts[mid] <= x)
            lo = mid;
        else
            hi = mid;
    }
    return lo;
}

// A token's slot; -1, and reported, where the table names no page of the pool.
__device__ __forceinline__ int64_t slot_of(const Resize &p, int b, int position) {
    const int page = p.table[b * p.table_stride + (position >> p.page_shift)];
    if ((unsigned)page >= (unsigned)p.num_pages) {
        record_bad_page(p.err);
        return -1;
    }
    return ((int64_t)page << p.page_shift) + (position & ((1 << p.page_shift) - 1));
}

// Latency bounds it: a launch, and inside it a chain of dependent loads
// (lengths, prefix sums, stack entries). A decode step and its way back, two calls:
// 6.3 us of 32 requests, 9.0 of 700.
__global__ void __launch_bounds__(kThreads) kv_pages_resize_kernel(const Resize p) {
    extern __shared__ int sm[];
    const int B = p.requests, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int ctas = gridDim.x, all = ctas * kThreads, me = blockIdx.x * kThreads + tid;
    int *old_len = sm, *new_len = sm + B, *give_at = sm + 2 * B, *take_at = give_at + B + 1, *tok_at = take_at + B + 1;
    __shared__ long long warp_sum[3][kThreads / 32];
    __shared__ long long total[3];
    __shared__ int bad_length;

    pdl_launch_dependents();
    pdl_wait();
    if (tid == 0) bad_length = 0;
    __syncthreads();
    const int top0 = *p.free_count;
    const int64_t cap = (int64_t)p.max_pages << p.page_shift;
    // each thread takes `per` neighbouring requests
    const int per = (B + kThreads - 1) / kThreads, b0 = min(B, tid * per), b1 = min(B, b0 + per);
    long long sum[3] = {0, 0, 0};
    for (int b = b0; b < b1; ++b) {
        const int o = p.lengths[b];
        const long long n = p.new_lengths ? p.new_lengths[b] : (o > 0 ? (long long)o + p.grow : 0);
        if (o < 0 || o > cap || n < 0 || n > cap) {
            bad_length = 1;
            old_len[b] = new_len[b] = 0;
            continue;
        }
        old_len[b] = o;
        new_len[b] = (int)n;
        const int have = pages_of(o, p.page_shift), want = pages_of((int)n, p.page_shift);
        sum[0] += max(0, have - want);
        sum[1] += max(0, want - have);
        sum[2] += max(0, (int)n - o);
    }
    long long before[3];
#pragma unroll
    for (int k = 0; k < 3; ++k) {
        long long v = sum[k];
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const long long u = __shfl_up_sync(0xffffffffu, v, off);
            if (lane >= off) v += u;
        }
        if (lane == 31) warp_sum[k][warp] = v;
        before[k] = v - sum[k];
    }
    __syncthreads();
    if (warp < 3) {
        long long v = warp_sum[warp][lane];
        const long long own = v;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const long long u = __shfl_up_sync(0xffffffffu, v, off);
            if (lane >= off) v += u;
        }
        warp_sum[warp][lane] = v - own;
        if (lane == 31) total[warp] = v;
    }
    sync_all(ctas);  // every CTA has read the lengths and the count
    const long long gives = total[0], takes = total[1], tokens = total[2];
    const int bad = bad_length                                            ? BAD_LENGTH
                    : top0 < 0 || top0 + gives > (long long)p.num_pages   ? BAD_STACK
                    : takes > top0 + gives                                ? BAD_POOL
                    : tokens > (long long)p.max_tokens                    ? BAD_TOKENS
                                                                          : BAD_NONE;
    if (bad) {  // nothing changes; no token has a slot
        if (me == 0 && *p.status == 0) *p.status = bad;
        for (int b = me; b <= B; b += all) {
            p.query_start[b] = 0;
            if (p.granted && b < B) p.granted[b] = 0;
        }
        if (p.max_tokens <= kSlotsInOne) {
            for (int r = me; r < p.max_tokens; r += all) {
                p.slots[r] = -1;
                p.positions[r] = -1;
            }
        }
        return;
    }
    for (int b = b0; b < b1; ++b) {
        const int o = old_len[b], n = new_len[b];
        const int have = pages_of(o, p.page_shift), want = pages_of(n, p.page_shift);
        give_at[b] = (int)(before[0] + warp_sum[0][warp]);
        take_at[b] = (int)(before[1] + warp_sum[1][warp]);
        tok_at[b] = (int)(before[2] + warp_sum[2][warp]);
        before[0] += max(0, have - want);
        before[1] += max(0, want - have);
        before[2] += max(0, n - o);
        if (blockIdx.x == 0) {
            p.query_start[b] = tok_at[b];
            p.lengths[b] = n;
            if (p.granted && n != o) p.granted[b] = max(0, n - o);
        }
    }
    const int top = top0 + (int)gives;
    if (tid == 0) {
        give_at[B] = (int)gives;
        take_at[B] = (int)takes;
    }
    if (me == 0) {
        p.query_start[B] = (int)tokens;
        *p.free_count = top - (int)takes;
    }
    __syncthreads();
    // Pages given back, the last one first, so that a roll-back leaves the stack as it was; then the pages taken.
    for (int i = me; i < (int)gives; i += all) {
        const int b = find(give_at, B, i);
        int *at = p.table + b * p.table_stride + pages_of(new_len[b], p.page_shift) + (i - give_at[b]);
        p.free_pages[top - 1 - i] = *at;
        *at = -1;
    }
    sync_all(ctas);
    for (int i = me; i < (int)takes; i += all) {
        const int b = find(take_at, B, i);
        p.table[b * p.table_stride + pages_of(old_len[b], p.page_shift) + (i - take_at[b])] = p.free_pages[top - 1 - i];
    }
    if (p.max_tokens > kSlotsInOne) return;
    sync_all(ctas);
    for (int r = me; r < p.max_tokens; r += all) {
        int64_t slot = -1;
        int position = -1;
        if (r < (int)tokens) {
            const int b = find(tok_at, B, r);
            position = old_len[b] + r - tok_at[b];
            slot = slot_of(p, b, position);
        }
        p.slots[r] = slot;
        p.positions[r] = position;
    }
}

// The slots and positions of many new tokens, from the tables and lengths that
// the launch before left; four neighbouring tokens a thread.
__global__ void __launch_bounds__(256) kv_pages_slots_kernel(const Resize p) {
    extern __shared__ int sm[];
    pdl_launch_dependents();
    pdl_wait();
    const int B = p.requests;
    for (int b = threadIdx.x; b <= B; b += 256) sm[b] = p.query_start[b];
    __syncthreads();
    const int64_t r0 = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;  // r0 + 4 may be 2^31
    if (r0 >= p.max_tokens) return;
    const int tokens = sm[B];
    int b = r0 < tokens ? find(sm, B, (int)r0) : 0;
    int64_t slots[4];
    int positions[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        slots[i] = -1;
        positions[i] = -1;
        if (r0 + i < tokens) {
            const int r = (int)r0 + i;
            while (sm[b + 1] <= r) ++b;
            positions[i] = p.lengths[b] - (sm[b + 1] - r);
            slots[i] = slot_of(p, b, positions[i]);
        }
    }
    if (r0 + 4 <= p.max_tokens && p.aligned) {
        *reinterpret_cast<longlong2 *>(p.slots + r0) = make_longlong2(slots[0], slots[1]);
        *reinterpret_cast<longlong2 *>(p.slots + r0 + 2) = make_longlong2(slots[2], slots[3]);
        *reinterpret_cast<int4 *>(p.positions + r0) = make_int4(positions[0], positions[1], positions[2], positions[3]);
    } else {
        for (int i = 0; i < 4 && r0 + i < p.max_tokens; ++i) {
            p.slots[r0 + i] = slots[i];
            p.positions[r0 + i] = positions[i];
        }
    }
}

}  // namespace
}  // namespace tn

extern "C" int64_t tn_kv_q4_page_bytes(int64_t kv_heads, int64_t head_dim, int64_t page_size) {
    if (tn::check_kv_pool("tn_kv_q4_page_bytes", nullptr, 0, kv_heads, head_dim, page_size)) return -1;
    return kv_heads * (page_size / tn::kKvGroup) * 18 * head_dim;
}

extern "C" int tn_kv_pages_resize_granted(int *page_table, int64_t table_stride, int64_t max_pages, int *lengths,
                                          const int *new_lengths, int64_t grow, int64_t requests, int *free_pages,
                                          int *free_count, int64_t num_pages, int64_t page_size, int64_t *slots,
                                          int *positions, int64_t max_tokens, int *query_start, int *status,
                                          int *granted, void *stream) {
    const std::string op("tn_kv_pages_resize");
    const int shift = tn::kv_page_shift(page_size);
    if (shift < 0)
        return tn::set_error(TN_ERR_NOT_IMPLEMENTED, op + ": a page holds 16, 32, 64, 128, 256, 512 or 1024 tokens, got " +
                                                         std::to_string(page_size));
    if (requests < 0 || max_pages < 0 || table_stride < max_pages || num_pages < 0 || num_pages > INT32_MAX ||
        max_tokens < 0 || max_tokens > INT32_MAX || max_pages > tn::kMaxRowTokens >> shift)
        return tn::set_error(TN_ERR_SHAPE, op + ": bad table, pool or token count");
    if (grow < 0 || grow > INT32_MAX)
        return tn::set_error(TN_ERR_SHAPE, op + ": grow must be a token count (new_lengths shrinks requests)");
    if (requests > tn::kMaxRequests)
        return tn::set_error(TN_ERR_NOT_IMPLEMENTED, op + ": at most " + std::to_string(tn::kMaxRequests) + " requests");
    if (!free_count || !query_start || !status || (requests > 0 && !lengths) ||
        (requests > 0 && max_pages > 0 && !page_table) || (num_pages > 0 && !free_pages) ||
        (max_tokens > 0 && (!slots || !positions)))
        return tn::set_error(TN_ERR_INVALID, op + ": null pointer");
    if (new_lengths && new_lengths == lengths)
        return tn::set_error(TN_ERR_INVALID, op + ": new_lengths must not be lengths");
    tn::Resize p{page_table, table_stride, (int)max_pages, lengths, new_lengths, (int)grow, (int)requests, free_pages,
                 free_count, (int)num_pages, shift, slots, positions, (int)max_tokens, query_start, status,
                 granted, ((uintptr_t)slots | (uintptr_t)positions) % 16 == 0, tn::device_error_word()};
    const int smem = (int)((5 * requests + 2) * sizeof(int));
    if (smem > 48 * 1024 - 1024) {
        // once a device, for the most requests: the limit is the kernel's, not the call's
        static std::atomic<uint64_t> ready{0};  // a bit a device
        int device = 0;
        int st = tn::check_cuda(cudaGetDevice(&device), "tn_kv_pages_resize", "cudaGetDevice");
        if (st) return st;
        if (!(ready.load(std::memory_order_relaxed) >> device & 1)) {
            st = tn::check_cuda(cudaFuncSetAttribute(tn::kv_pages_resize_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                     (int)((5 * tn::kMaxRequests + 2) * sizeof(int))),
                                "tn_kv_pages_resize", "cudaFuncSetAttribute");
            if (st) return st;
            ready.fetch_or(1ull << device, std::memory_order_relaxed);
        }
    }
    cudaStream_t s = tn::stream_of(stream);
    const int64_t moves = new_lengths ? max_pages : std::min(max_pages, (grow >> shift) + 1);
    const int ctas = requests * moves > tn::kMovesInOne ? tn::kCtas : 1;
    int st = tn::launch_pdl_cluster(tn::kv_pages_resize_kernel, dim3(ctas), dim3(tn::kThreads), smem, s,
                                    "tn_kv_pages_resize", ctas, p);
    if (st || max_tokens <= tn::kSlotsInOne) return st;
    return tn::launch_pdl(tn::kv_pages_slots_kernel, dim3((unsigned)((max_tokens + 1023) / 1024)), dim3(256),
                          (int)((requests + 1) * sizeof(int)), s, "tn_kv_pages_resize", p);
}

extern "C" int tn_kv_pages_resize(int *page_table, int64_t table_stride, int64_t max_pages, int *lengths,
                                  const int *new_lengths, int64_t grow, int64_t requests, int *free_pages,
                                  int *free_count, int64_t num_pages, int64_t page_size, int64_t *slots, int *positions,
                                  int64_t max_tokens, int *query_start, int *status, void *stream) {
    return tn_kv_pages_resize_granted(page_table, table_stride, max_pages, lengths, new_lengths, grow, requests, free_pages,
                                      free_count, num_pages, page_size, slots, positions, max_tokens, query_start, status,
                                      nullptr, stream);
}
