// Shortening a paged cache by accumulated attention weight.  For every sequence and KV head
//
//   kv_evict_select  the rows that stay: the first ones, the latest ones, and of those between them the heaviest (equal weights: the earlier row),
//                    in ascending order.  A radix selection over the bit patterns of the weights, then an ordered compaction.
//   kv_evict_move    copies of those rows (keys, values, block scales, weights) into the rows 0, 1, 2 .. of other pages.
#include "host_utils.h"
#include "tc5_common.cuh"

namespace telb {

struct EvictParams {
    uint8_t* pool;
    float* weights;
    const int *page_table, *lengths, *to_table;
    int* kept;
    int num_seqs, hkv, num_pages, max_pages, to_pages, page_size, page_shift, row_bytes, scale_bytes, keep, first, recent;
};

constexpr int kEvictThreads = 512;
constexpr int kEvictRanks = 16, kEvictBins = 2048;
constexpr int kEvictHeld = 24576;                               // keys that a CTA holds in shared memory; those behind them are made anew in every pass

// Larger weight, larger key; NaN above everything, rows without a page below.
__device__ __forceinline__ uint32_t weight_key(float w) {
    if (w != w) return 0xffffffffu;
    const uint32_t u = __float_as_uint(w + 0.f);               // -0 counts as 0
    return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ uint32_t cluster_map(const void* p, uint32_t rank) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(p)), "r"(rank));
    return r;
}
__device__ __forceinline__ int cluster_load(uint32_t at) {
    int v;
    asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ void cluster_sync_all() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// A cluster per (KV head, sequence); its CTAs take equal parts of the sequence's rows, whose keys they keep in shared memory.  The border key is found
// from the histograms of all of them, 11, 11 and 10 bits at a time (mostly the first two passes do); then every CTA writes its part of the
// rows that stay, in order.
__global__ void __launch_bounds__(kEvictThreads) kv_evict_select_kernel(const EvictParams p) {
    extern __shared__ __align__(16) uint32_t held[];
    __shared__ __align__(16) int hist[2][kEvictBins];           // of two passes in turn: one is read by the cluster while the next is cleared
    __shared__ int coarse[2][256];                              // sums of eight neighbours
    __shared__ int s_warp[8], s_found[3], s_counts[2];
    __shared__ int s_gt[kEvictThreads / 32], s_eq[kEvictThreads / 32];
    pdl_prologue();
    const int ranks = gridDim.x, rank = blockIdx.x, head = blockIdx.y, seq = blockIdx.z, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    constexpr int threads = kEvictThreads;
    const int* table = p.page_table + (size_t)seq * p.max_pages;
    const int n = (int)min((long long)max(p.lengths[seq], 0), (long long)p.max_pages * p.page_size);
    int* kept = p.kept + ((size_t)seq * p.hkv + head) * p.keep;
    if (n <= p.keep) {                                          // the whole cluster
        for (int i = rank * threads + tid; i < p.keep; i += ranks * threads) kept[i] = i < n ? i : -1;
        return;
    }
    const int lo = p.first, hi = n - p.recent, want = p.keep - p.first - p.recent;
    const int per = ((n + ranks - 1) / ranks + 3) & ~3, begin = min(n, rank * per), count = min(n, begin + per) - begin;
    const int a0 = max(lo - begin, 0), a1 = min(hi - begin, count);       // the rows of this part that are not sure to stay
    for (int i = tid; i < kEvictBins; i += threads) hist[0][i] = 0;
    __syncthreads();
    auto sync = [&]() {
        if (ranks > 1) cluster_sync_all();
        else __syncthreads();
    };
    // Keys of the rows begin + i .. + 3 (i a multiple of four, as is a page's number of rows).
    auto fresh = [&](int i) -> uint4 {
        const int row = begin + i, lp = p.page_shift >= 0 ? row >> p.page_shift : row / p.page_size, page = table[lp];
        uint4 k = make_uint4(0u, 0u, 0u, 0u);
        if ((unsigned)page < (unsigned)p.num_pages) {
            const float4 w = *reinterpret_cast<const float4*>(p.weights + ((size_t)page * p.hkv + head) * p.page_size + row - lp * p.page_size);
            k = make_uint4(weight_key(w.x), weight_key(w.y), weight_key(w.z), weight_key(w.w));
        }
        return k;
    };
    auto keys_of = [&](int i) -> uint4 { return i < kEvictHeld ? *reinterpret_cast<const uint4*>(held + i) : fresh(i); };
    uint32_t prefix = want > 0 ? 0u : 0xffffffffu;
    int left = max(want, 0);                                    // still to be found among the keys that begin with the prefix
    auto add = [&](int pass, uint32_t k) {
        if (pass == 0) atomicAdd(&hist[0][k >> 21], 1);
        else if (pass == 1 && k >> 21 == prefix >> 21) atomicAdd(&hist[1][(k >> 10) & 2047u], 1);
        else if (pass == 2 && k >> 10 == prefix >> 10) atomicAdd(&hist[0][k & 1023u], 1);
    };
    auto digits = [&](int pass, int i, const uint4& k4) {
        const uint32_t k[4] = {k4.x, k4.y, k4.z, k4.w};
        if (i >= a0 && i + 3 < a1) {
#pragma unroll
            for (int e = 0; e < 4; ++e) add(pass, k[e]);
        } else {
            for (int e = 0; e < 4; ++e)
                if (i + e >= a0 && i + e < a1) add(pass, k[e]);
        }
    };
#pragma unroll 4
    for (int i = 4 * tid; i < count; i += 4 * threads) {
        const uint4 k = fresh(i);
        if (i < kEvictHeld) *reinterpret_cast<uint4*>(held + i) = k;
        digits(0, i, k);
    }
    // After a pass: the digit of the border key, its upper eight bits first, from sums of eight bins.  True where nothing is left to be found.
    auto find = [&](int pass, int shift) -> bool {
        const int* h = hist[pass & 1];
        int* sums = coarse[pass & 1];
        __syncthreads();
        if (warp < 8) {
            const int4 x = *reinterpret_cast<const int4*>(h + 8 * tid), y = *reinterpret_cast<const int4*>(h + 8 * tid + 4);
            sums[tid] = x.x + x.y + x.z + x.w + y.x + y.y + y.z + y.w;
        }
        sync();
        int mine = 0, incl = 0;
        if (warp < 8) {
            // thread t: sum 255 - t over the whole cluster (all loads on their way before the first addition), then with all sums above
            int part[kEvictRanks];
#pragma unroll
            for (int r = 0; r < kEvictRanks; ++r) part[r] = r < ranks ? cluster_load(cluster_map(&sums[255 - tid], r)) : 0;
#pragma unroll
            for (int r = 0; r < kEvictRanks; ++r) mine += part[r];
            incl = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o) incl += v;
            }
            if (lane == 31) s_warp[warp] = incl;
        }
        *reinterpret_cast<int4*>(&hist[(pass + 1) & 1][4 * tid]) = make_int4(0, 0, 0, 0);          // read by the others in the pass before this one
        __syncthreads();
        if (warp < 8) {
            for (int w = 0; w < warp; ++w) incl += s_warp[w];
            if (incl >= left && incl - mine < left) {
                s_found[0] = 255 - tid;
                s_found[1] = left - (incl - mine);
            }
        }
        __syncthreads();
        if (warp == 0) {
            // lane: bin 7 - lane % 8 of that sum, of the ranks lane / 8, + 4 ..
            const int top = s_found[0] * 8 + 7, rest = s_found[1], e = lane & 7;
            int part[kEvictRanks / 4], bin = 0;
#pragma unroll
            for (int r = 0; r < kEvictRanks / 4; ++r) part[r] = 4 * r + (lane >> 3) < ranks ? cluster_load(cluster_map(h + top - e, 4 * r + (lane >> 3))) : 0;
#pragma unroll
            for (int r = 0; r < kEvictRanks / 4; ++r) bin += part[r];
            bin += __shfl_xor_sync(0xffffffffu, bin, 8);
            bin += __shfl_xor_sync(0xffffffffu, bin, 16);
            int to = bin;
#pragma unroll
            for (int o = 1; o < 8; o <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, to, o);
                if (e >= o) to += v;
            }
            __syncwarp();
            if (lane < 8 && to >= rest && to - bin < rest) {
                s_found[0] = top - e;
                s_found[1] = rest - (to - bin);
                s_found[2] = to == rest;
            }
        }
        __syncthreads();
        prefix |= (uint32_t)s_found[0] << shift;
        left = s_found[1];
        if (!s_found[2]) return false;
        --prefix;                                               // every key that begins so stays: the border lies just below.  Not below zero: then all
        left = 0;                                               // rows between would stay, and there are more of them
        return true;
    };
    if (want > 0 && !find(0, 21)) {
#pragma unroll 4
        for (int i = 4 * tid; i < count; i += 4 * threads) digits(1, i, keys_of(i));
        if (!find(1, 10)) {
#pragma unroll 4
            for (int i = 4 * tid; i < count; i += 4 * threads) digits(2, i, keys_of(i));
            find(2, 0);
        }
    }
    // Keys above the border and on it, per warp: contiguous parts, 128 rows at a time.
    const int chunk = (count + 4 * threads - 1) / (4 * threads) * 128;
    const int w0 = min(count, warp * chunk), w1 = min(count, w0 + chunk);
    auto sort_out = [&](int i, const uint4& k4, int (&is)[4]) {          // 1 above, 1 << 16 on the border
        const uint32_t k[4] = {k4.x, k4.y, k4.z, k4.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) is[e] = i < w1 && i + e >= a0 && i + e < a1 ? k[e] > prefix ? 1 : k[e] == prefix ? 1 << 16 : 0 : 0;
    };
    int gt = 0, eq = 0;
#pragma unroll 4
    for (int i = w0 + 4 * lane; i < w1; i += 128) {
        int is[4];
        sort_out(i, keys_of(i), is);
        const int sum = is[0] + is[1] + is[2] + is[3];
        gt += sum & 0xffff;
        eq += sum >> 16;
    }
    gt = __reduce_add_sync(0xffffffffu, gt);
    eq = __reduce_add_sync(0xffffffffu, eq);
    if (lane == 0) s_gt[warp] = gt, s_eq[warp] = eq;
    __syncthreads();
    const int mine_gt = lane < threads / 32 ? s_gt[lane] : 0, mine_eq = lane < threads / 32 ? s_eq[lane] : 0;
    int gt_before = __reduce_add_sync(0xffffffffu, lane < warp ? mine_gt : 0), eq_before = __reduce_add_sync(0xffffffffu, lane < warp ? mine_eq : 0);
    if (ranks > 1) {
        if (warp == 0) {
            const int all_gt = __reduce_add_sync(0xffffffffu, mine_gt), all_eq = __reduce_add_sync(0xffffffffu, mine_eq);
            if (lane == 0) s_counts[0] = all_gt, s_counts[1] = all_eq;
        }
        cluster_sync_all();
        if (rank > 0) {                                         // and of the CTAs before
            gt_before += __reduce_add_sync(0xffffffffu, lane < rank ? cluster_load(cluster_map(&s_counts[0], lane)) : 0);
            eq_before += __reduce_add_sync(0xffffffffu, lane < rank ? cluster_load(cluster_map(&s_counts[1], lane)) : 0);
        }
    }
    for (int i0 = w0; i0 < w1; i0 += 128) {
        const int i = i0 + 4 * lane;
        int is[4];
        sort_out(i, i < w1 ? keys_of(i) : make_uint4(0u, 0u, 0u, 0u), is);
        const int mine = is[0] + is[1] + is[2] + is[3];
        int incl = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += v;
        }
        const int all = __shfl_sync(0xffffffffu, incl, 31);
        int gt_at = gt_before + ((incl - mine) & 0xffff), eq_at = eq_before + ((incl - mine) >> 16);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (is[e] == 1 || (is[e] != 0 && eq_at < left)) kept[p.first + gt_at + min(eq_at, left)] = begin + i + e;
            gt_at += is[e] & 0xffff;
            eq_at += is[e] >> 16;
        }
        gt_before += all & 0xffff;
        eq_before += all >> 16;
    }
    if (rank == 0)
        for (int i = tid; i < p.first; i += threads) kept[i] = i;
    if (rank == ranks - 1)
        for (int i = tid; i < p.recent; i += threads) kept[p.keep - p.recent + i] = hi + i;
    if (ranks > 1) cluster_sync_all();                          // nobody leaves while its counts may be read
}

constexpr int kMoveRows = 128;

// Reads that bring 64 bytes from memory: rows that stay lie apart, and the 128 of a plain load are twice a four-bit row of 128 features.
__device__ __forceinline__ uint4 load_apart(const uint4* p) {
    uint4 v;
    asm volatile("ld.global.L2::64B.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
    return v;
}
__device__ __forceinline__ uint2 load_apart(const uint2* p) {
    uint2 v;
    asm volatile("ld.global.L2::64B.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p) : "memory");
    return v;
}
__device__ __forceinline__ uint32_t load_apart(const uint32_t* p) {
    uint32_t v;
    asm volatile("ld.global.L2::64B.u32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
    return v;
}

// grid (groups of 128 rows, KV heads, sequences): keys, values and weights of these rows.  Every thread has four copies on their way.
__global__ void __launch_bounds__(256, 6) kv_evict_move_kernel(const EvictParams p) {
    __shared__ const uint8_t *s_src[kMoveRows], *s_ssrc[kMoveRows];       // a row's key codes and key scales; null: no copy
    __shared__ uint8_t *s_dst[kMoveRows], *s_sdst[kMoveRows];
    pdl_prologue();
    const int seq = blockIdx.z, head = blockIdx.y, j0 = blockIdx.x * kMoveRows, rows = min(kMoveRows, p.keep - j0), tid = threadIdx.x;
    const size_t slab = (size_t)p.page_size * (p.row_bytes + p.scale_bytes);
    const float* w_src = nullptr;
    float* w_dst = nullptr;
    if (tid < rows) {
        const int j = j0 + tid, i = p.kept[((size_t)seq * p.hkv + head) * p.keep + j];
        const int lp = j / p.page_size, at = j - lp * p.page_size;
        const int dst = lp < p.to_pages ? p.to_table[(size_t)seq * p.to_pages + lp] : -1;
        const int page = i >= 0 ? p.page_table[(size_t)seq * p.max_pages + i / p.page_size] : -1;
        const bool ok = (unsigned)page < (unsigned)p.num_pages && (unsigned)dst < (unsigned)p.num_pages;
        const int from = ok ? i % p.page_size : 0;
        const uint8_t* sb = p.pool + ((size_t)page * 2 * p.hkv + head) * slab;
        uint8_t* db = p.pool + ((size_t)dst * 2 * p.hkv + head) * slab;
        const size_t scales = (size_t)p.page_size * p.row_bytes;
        s_src[tid] = ok ? sb + (size_t)from * p.row_bytes : nullptr;
        s_dst[tid] = db + (size_t)at * p.row_bytes;
        s_ssrc[tid] = sb + scales + (size_t)from * p.scale_bytes;
        s_sdst[tid] = db + scales + (size_t)at * p.scale_bytes;
        if (ok) {
            w_src = p.weights + ((size_t)page * p.hkv + head) * p.page_size + from;
            w_dst = p.weights + ((size_t)dst * p.hkv + head) * p.page_size + at;
        }
    }
    __syncthreads();
    const float w = w_src ? *w_src : 0.f;
    const size_t value_at = (size_t)p.hkv * slab;
    // neighbouring threads copy neighbouring pieces of a row; a thread has one place in the row
    auto copy = [&](auto unit, int pieces, const uint8_t* const* src, uint8_t* const* dst) {
        using U = decltype(unit);
        for (int c0 = 0; c0 < pieces; c0 += 256) {
            const int wide = min(256, pieces - c0), step = 256 / wide, c = c0 + tid % wide;
            for (int r = tid / wide; r < rows && tid < step * wide; r += 2 * step) {
                U v[4];
                const bool one = s_src[r] != nullptr, two = r + step < rows && s_src[r + step] != nullptr;
                if (one) {
                    const U* f = reinterpret_cast<const U*>(src[r]) + c;
                    v[0] = load_apart(f);
                    v[1] = load_apart(reinterpret_cast<const U*>(reinterpret_cast<const uint8_t*>(f) + value_at));
                }
                if (two) {
                    const U* f = reinterpret_cast<const U*>(src[r + step]) + c;
                    v[2] = load_apart(f);
                    v[3] = load_apart(reinterpret_cast<const U*>(reinterpret_cast<const uint8_t*>(f) + value_at));
                }
                if (one) {
                    U* o = reinterpret_cast<U*>(dst[r]) + c;
                    *o = v[0];
                    *reinterpret_cast<U*>(reinterpret_cast<uint8_t*>(o) + value_at) = v[1];
                }
                if (two) {
                    U* o = reinterpret_cast<U*>(dst[r + step]) + c;
                    *o = v[2];
                    *reinterpret_cast<U*>(reinterpret_cast<uint8_t*>(o) + value_at) = v[3];
                }
            }
        }
    };
    copy(uint4(), p.row_bytes / 16, s_src, s_dst);
    if (p.scale_bytes % 8 == 0 && p.scale_bytes) copy(uint2(), p.scale_bytes / 8, s_ssrc, s_sdst);
    else if (p.scale_bytes) copy(uint32_t(), p.scale_bytes / 4, s_ssrc, s_sdst);
    if (w_dst) *w_dst = w;
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
    if (p.num_seqs > 65535 || p.hkv > 65535) return fail("telb_kv_evict: more than 65535 sequences or heads");
    if (p.page_size % 4 || p.page_size > 32764) return fail("telb_kv_evict: pages of a multiple of four rows, at most 32764");
    static int most_ranks[64] = {};                              // clusters of 16 where the device places them
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64) return fail("telb_kv_evict: device index above 63");
    if (!most_ranks[dev]) {
        cudaError_t e = cudaFuncSetAttribute(kv_evict_select_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kEvictHeld * 4 + 16);
        if (e != cudaSuccess) return fail("cudaFuncSetAttribute(kv_evict_select)", e);
        int ranks = 8;
        if (cudaFuncSetAttribute(kv_evict_select_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) == cudaSuccess) {
            cudaLaunchConfig_t c{};
            c.gridDim = dim3(kEvictRanks);
            c.blockDim = dim3(kEvictThreads);
            c.dynamicSmemBytes = kEvictHeld * 4 + 16;
            cudaLaunchAttribute a;
            a.id = cudaLaunchAttributeClusterDimension;
            a.val.clusterDim.x = kEvictRanks;
            a.val.clusterDim.y = a.val.clusterDim.z = 1;
            c.attrs = &a;
            c.numAttrs = 1;
            int clusters = 0;
            if (cudaOccupancyMaxActiveClusters(&clusters, kv_evict_select_kernel, &c) == cudaSuccess && clusters > 0) ranks = kEvictRanks;
        }
        cudaGetLastError();
        most_ranks[dev] = ranks;
    }
    // CTAs of a cluster: up to two an SM in all, each with 4096 rows or more.  16 sequences of 8192 rows, 8 heads: 1, 2, 4 CTAs 40, 37, 42 us (both kernels);
    // one sequence of 131000, 4 heads: 4, 8, 16 CTAs 63, 34, 28.
    const long long most = (long long)p.max_pages * p.page_size, items = (long long)p.num_seqs * p.hkv;
    int ranks = 1;
    while (ranks < most_ranks[dev] && items * ranks * 2 <= 2 * sm_count() && most >= 8192LL * ranks) ranks *= 2;
    const long long per = (most + ranks - 1) / ranks + 4;
    const int smem = (int)(per < kEvictHeld ? per : kEvictHeld) * 4 + 16;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(ranks, p.hkv, p.num_seqs);
    cfg.blockDim = dim3(kEvictThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = ranks;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl_enabled() ? 2 : 1;
    cudaError_t e = cudaLaunchKernelEx(&cfg, kv_evict_select_kernel, p);
    if (e != cudaSuccess) return fail("kv_evict_select_kernel", e);
    TELB_LAUNCH("kv_evict_move_kernel", kv_evict_move_kernel, dim3((p.keep + kMoveRows - 1) / kMoveRows, p.hkv, p.num_seqs), dim3(256), 0, stream, p);
    return 0;
}
