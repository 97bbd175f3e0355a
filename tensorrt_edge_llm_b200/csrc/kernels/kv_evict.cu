// Shortening a paged cache by accumulated attention weight.  For every sequence and KV head
//
//   kv_evict_select  the rows that stay: the first ones, the latest ones, and of those between them the heaviest (equal weights: the earlier row),
//                    in ascending order.  A radix selection over the weights' bit patterns, eight bits a pass, then an ordered compaction.
//   kv_evict_move    copies of those rows (keys, values, block scales, weights) into the rows 0, 1, 2 .. of other pages.
#include "host_utils.h"
#include "tc5_common.cuh"

namespace telb {

struct EvictParams {
    uint8_t* pool;
    float* weights;
    const int *page_table, *lengths, *to_table;
    int* kept;
    int num_seqs, hkv, num_pages, max_pages, to_pages, page_size, row_bytes, scale_bytes, keep, first, recent;
};

constexpr int kEvictThreads = 1024;

// Larger weight, larger key; NaN above everything, rows without a page below.
__device__ __forceinline__ uint32_t weight_key(float w) {
    if (w != w) return 0xffffffffu;
    const uint32_t u = __float_as_uint(w + 0.f);               // -0 counts as 0
    return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

__global__ void __launch_bounds__(kEvictThreads) kv_evict_select_kernel(const EvictParams p) {
    pdl_prologue();
    __shared__ int hist[256];
    __shared__ uint32_t s_prefix;
    __shared__ int s_left;
    __shared__ int s_gt[32], s_eq[32];
    const int head = blockIdx.x, seq = blockIdx.y, tid = threadIdx.x;
    const int* table = p.page_table + (size_t)seq * p.max_pages;
    const int n = (int)min((long long)max(p.lengths[seq], 0), (long long)p.max_pages * p.page_size);
    int* kept = p.kept + ((size_t)seq * p.hkv + head) * p.keep;
    if (n <= p.keep) {
        for (int i = tid; i < p.keep; i += kEvictThreads) kept[i] = i < n ? i : -1;
        return;
    }
    const int lo = p.first, hi = n - p.recent, want = p.keep - p.first - p.recent;
    auto key_of = [&](int i) -> uint32_t {
        const int page = table[i / p.page_size];
        if ((unsigned)page >= (unsigned)p.num_pages) return 0u;
        return weight_key(p.weights[((size_t)page * p.hkv + head) * p.page_size + i % p.page_size]);
    };
    uint32_t prefix = 0;
    int left = want;                                            // still to be found among the keys that begin with the prefix
    if (want > 0) {
        for (int shift = 24; shift >= 0; shift -= 8) {
            for (int i = tid; i < 256; i += kEvictThreads) hist[i] = 0;
            __syncthreads();
            for (int i = lo + tid; i < hi; i += kEvictThreads) {
                const uint32_t k = key_of(i);
                if (shift == 24 || (k >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&hist[(k >> shift) & 255u], 1);
            }
            __syncthreads();
            if (tid == 0) {
                int rest = left, d = 255;
                for (; d > 0 && hist[d] < rest; --d) rest -= hist[d];
                s_prefix = prefix | ((uint32_t)d << shift);
                s_left = rest;
            }
            __syncthreads();
            prefix = s_prefix;
            left = s_left;
        }
    } else {
        prefix = 0xffffffffu;
        left = 0;
    }
    // every thread takes a contiguous part of the rows between; how many of them are above the border and on it
    const int per = (hi - lo + kEvictThreads - 1) / kEvictThreads;
    const int a = min(hi, lo + tid * per), b = min(hi, a + per);
    int gt = 0, eq = 0;
    for (int i = a; i < b; ++i) {
        const uint32_t k = key_of(i);
        gt += k > prefix;
        eq += k == prefix;
    }
    int gt_in = gt, eq_in = eq;                                 // inclusive sums over the threads
    const int lane = tid & 31, warp = tid >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, gt_in, o), y = __shfl_up_sync(0xffffffffu, eq_in, o);
        if (lane >= o) gt_in += x, eq_in += y;
    }
    if (lane == 31) s_gt[warp] = gt_in, s_eq[warp] = eq_in;
    __syncthreads();
    if (warp == 0) {
        int x = s_gt[lane], y = s_eq[lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(0xffffffffu, x, o), v = __shfl_up_sync(0xffffffffu, y, o);
            if (lane >= o) x += u, y += v;
        }
        s_gt[lane] = x;
        s_eq[lane] = y;
    }
    __syncthreads();
    const int gt_before = gt_in - gt + (warp ? s_gt[warp - 1] : 0);
    int eq_before = eq_in - eq + (warp ? s_eq[warp - 1] : 0);
    int at = p.first + gt_before + min(eq_before, left);
    for (int i = a; i < b; ++i) {
        const uint32_t k = key_of(i);
        if (k > prefix || (k == prefix && eq_before++ < left)) kept[at++] = i;
    }
    for (int i = tid; i < p.first; i += kEvictThreads) kept[i] = i;
    for (int i = tid; i < p.recent; i += kEvictThreads) kept[p.keep - p.recent + i] = hi + i;
}

// grid (groups of 64 rows, 2 x KV heads, sequences)
__global__ void __launch_bounds__(256) kv_evict_move_kernel(const EvictParams p) {
    pdl_prologue();
    __shared__ long long s_src[64];                             // slab row of every kept row: page * page_size + place, -1: none
    const int seq = blockIdx.z, kv = blockIdx.y / p.hkv, head = blockIdx.y - kv * p.hkv, j0 = blockIdx.x * 64;
    const int rows = min(64, p.keep - j0);
    const int* table = p.page_table + (size_t)seq * p.max_pages;
    const int* to = p.to_table + (size_t)seq * p.to_pages;
    const size_t slab = (size_t)p.page_size * (p.row_bytes + p.scale_bytes);
    if (threadIdx.x < rows) {
        const int i = p.kept[((size_t)seq * p.hkv + head) * p.keep + j0 + threadIdx.x];
        const int page = i >= 0 ? table[i / p.page_size] : -1;
        s_src[threadIdx.x] = (unsigned)page < (unsigned)p.num_pages ? (long long)page * p.page_size + i % p.page_size : -1;
    }
    __syncthreads();
    const int pieces = p.row_bytes / 16, words = p.scale_bytes / 4, each = pieces + words;
    for (int i = threadIdx.x; i < rows * each; i += blockDim.x) {
        const int r = i / each, c = i - r * each, j = j0 + r;
        const long long src = s_src[r];
        const int page = j / p.page_size < p.to_pages ? to[j / p.page_size] : -1;
        if (src < 0 || (unsigned)page >= (unsigned)p.num_pages) continue;
        const int from_at = (int)(src % p.page_size), at = j % p.page_size;
        const uint8_t* sp = p.pool + (((size_t)(src / p.page_size) * 2 + kv) * p.hkv + head) * slab;
        uint8_t* dp = p.pool + (((size_t)page * 2 + kv) * p.hkv + head) * slab;
        if (c < pieces) {
            *reinterpret_cast<uint4*>(dp + (size_t)at * p.row_bytes + c * 16) = *reinterpret_cast<const uint4*>(sp + (size_t)from_at * p.row_bytes + c * 16);
        } else {
            const size_t base = (size_t)p.page_size * p.row_bytes + (c - pieces) * 4;
            *reinterpret_cast<uint32_t*>(dp + base + (size_t)at * p.scale_bytes) = *reinterpret_cast<const uint32_t*>(sp + base + (size_t)from_at * p.scale_bytes);
        }
    }
    if (kv == 0 && threadIdx.x < rows) {
        const int j = j0 + threadIdx.x;
        const long long src = s_src[threadIdx.x];
        const int page = j / p.page_size < p.to_pages ? to[j / p.page_size] : -1;
        if (src >= 0 && (unsigned)page < (unsigned)p.num_pages)
            p.weights[((size_t)page * p.hkv + head) * p.page_size + j % p.page_size] = p.weights[((size_t)(src / p.page_size) * p.hkv + head) * p.page_size + src % p.page_size];
    }
}

}  // namespace telb

using namespace telb;

// row_bytes: a row of one head's keys (or values) without its block scales, scale_bytes: those (0: none), which lie behind all rows of a slab.
extern "C" int telb_kv_evict(const EvictParams* params, cudaStream_t stream) {
    const EvictParams& p = *params;
    if (p.num_seqs <= 0 || p.hkv <= 0) return 0;
    if (p.row_bytes <= 0 || p.row_bytes % 16 || p.scale_bytes % 4) return fail("telb_kv_evict: rows must be multiples of 16 bytes, block scales of 4");
    if ((long long)p.page_size * (p.row_bytes + p.scale_bytes) % 16) return fail("telb_kv_evict: a head's part of a page must be a multiple of 16 bytes");
    if (p.first < 0 || p.recent < 0 || p.keep < 1 || p.first + p.recent > p.keep) return fail("telb_kv_evict: first and recent rows must fit into those that stay");
    if (p.num_seqs > 65535 || 2 * p.hkv > 65535) return fail("telb_kv_evict: more than 65535 sequences or planes");
    TELB_LAUNCH("kv_evict_select_kernel", kv_evict_select_kernel, dim3(p.hkv, p.num_seqs), dim3(kEvictThreads), 0, stream, p);
    TELB_LAUNCH("kv_evict_move_kernel", kv_evict_move_kernel, dim3((p.keep + 63) / 64, 2 * p.hkv, p.num_seqs), dim3(256), 0, stream, p);
    return 0;
}
