// Attention of few query rows a sequence over four-bit cache pages (layout: kv_fp4_common.cuh), read in place.
//
// The rows of a sequence and the query heads of a KV head make `columns`; 16 keys, 16 features and 8 columns make one fp16 matrix instruction.
//   scores  S[key, column] = sum over d of K[key, d] q[column, d]       A = keys, 16 bytes a lane from a key's row, B = queries in registers
//   output  O[d, column]  += sum over keys of V[key, d] P[key, column]  A = values, the nibbles of two keys joined before they become half2
// Features and keys may come in any order inside a sum, so both operands are taken from the pages in the order in which they lie there; no
// data crosses lanes but the probabilities (one 8 x 8 transposition per 8 keys).  code * block scale is exact in fp16; scales[] and the softmax scale
// multiply the 32-bit sums.  Probabilities are exp2(score - reference), the reference 8 to 16 below the maximum: fp16 keeps eleven bits of
// those down to 2^-22 of the largest, and the accumulators are rescaled only when a score outgrows the reference by 2^15.
//
// What bounds it is the issue of instructions: 16 keys of 128 features are some 290 of them for 8 columns, 224 alone for codes to half2 (4 ALU
// instructions a word of eight codes), block scales and products; the pages' bytes would take a third to a half of the time.  So tiles that every
// column sees whole have code without masks, and a ring of asynchronous copies per warp keeps three tiles on their way.  Measured with heads of 128:
// 64 sequences of 1088 keys, 32 / 8 heads, 26.0 us (3.0 TB/s, 0.46 of the copy rate; 16-bit pages 55, E4M3 pages 35); 30 of up to 4000 38.9 us; one of 131000,
// 32 / 4 heads, 34 us; one of 700 8.2 us, which is latency: launch, page table, first tile, join.  Taken back: bulk copies with mbarriers in place of the
// lanes' copies; 32 columns a warp (half the occupancy); operands expanded once for all warps of a CTA, in shared memory (half the instructions, but two
// barriers for every 128 keys: 2 sequences of 4000 keys, 128 columns, 49 us against 50, one of 8000, 64 columns, 28 against 24).
#include <type_traits>

#include "host_utils.h"
#include "kv_fp4_common.cuh"

namespace telb {

struct Fp4AttnParams {
    const void* q;
    const uint8_t* pool;
    void* out;
    float *part_o, *part_ml, *stat;
    const int *q_start, *q_len, *past_len, *page_table;
    const float *scales, *sinks;
    float* weights;
    int2* spans;
    float4* scores;
    int num_seqs, tokens, max_q_len, num_pages, max_pages, page_size, page_shift, hq, hkv, window, ctas, ranks, max_items, tiles, pairs;
    float scale, decay;
};

constexpr int kFp4Warps = 4, kFp4Tile = 32;               // warps of a CTA; keys that a warp takes at a time
constexpr float kRefStart = -1e30f;

__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16_first(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ uint32_t hmul2u(uint32_t a, uint32_t b) {
    const __half2 r = __hmul2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ float exp2_approx(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// Where row r of a 16-key tile lies in it: neighbours in memory alternate, so that the four rows that a warp's lanes read together differ in parity.
__device__ __forceinline__ int key_place(int r) { return r ^ ((r >> 1) & 1); }

// Queries of column `g` (lane = 4 g + t), features t * D/4 ..: B operands of all D/16 steps.  Returns the power of two that they were divided by.
template <typename T, int D>
__device__ __forceinline__ float load_query(const T* src, bool real, uint32_t (&b)[D / 16][2]) {
    constexpr int N = D / 4;
    alignas(16) T x[N];
#pragma unroll
    for (int i = 0; i < N / 8; ++i)
        *reinterpret_cast<uint4*>(x + 8 * i) = real ? *reinterpret_cast<const uint4*>(src + 8 * i) : make_uint4(0, 0, 0, 0);
    float up = 1.f;
    if constexpr (std::is_same<T, __half>::value) {
#pragma unroll
        for (int j = 0; j < D / 16; ++j) {
            b[j][0] = *reinterpret_cast<const uint32_t*>(x + 4 * j);
            b[j][1] = *reinterpret_cast<const uint32_t*>(x + 4 * j + 2);
        }
    } else {
        // bf16 queries enter as fp16, divided by the power of two below their column's largest: exact down to 2^-17 of it, off by 2^-25 of it at most below
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) m = max(m, __float_as_uint(Cvt<T>::to_f(x[i])) & 0x7fffffffu);
        m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
        m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
        const int e = m == 0 ? 0 : min(max((int)(m >> 23) - 127, -126), 126);
        up = __uint_as_float((uint32_t)(127 + e) << 23);
        const float down = __uint_as_float((uint32_t)(127 - e) << 23);
#pragma unroll
        for (int j = 0; j < D / 16; ++j) {
            b[j][0] = Cvt<__half>::pack2(Cvt<T>::to_f(x[4 * j]) * down, Cvt<T>::to_f(x[4 * j + 1]) * down);
            b[j][1] = Cvt<__half>::pack2(Cvt<T>::to_f(x[4 * j + 2]) * down, Cvt<T>::to_f(x[4 * j + 3]) * down);
        }
    }
    return up;
}

// A 16-key tile of keys: codes and scales of the rows key_place(g) and + 8, features t * D/4 ...
template <int D>
struct KeyTile {
    uint32_t w[2][D / 32];
    uint16_t s[2][(D + 127) / 128];
    __device__ __forceinline__ void load(const uint8_t* codes, const uint8_t* sf, int g, int t) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const int at = key_place(g) + 8 * r;
            const uint8_t* c = codes + at * (D / 2) + t * (D / 8);
            const uint8_t* f = sf + at * (D / 16) + t * (D / 64);
            if constexpr (D == 64) {
                *reinterpret_cast<uint2*>(w[r]) = *reinterpret_cast<const uint2*>(c);
                s[r][0] = *f;
            } else {
#pragma unroll
                for (int i = 0; i < D / 128; ++i) *reinterpret_cast<uint4*>(w[r] + 4 * i) = *reinterpret_cast<const uint4*>(c + 16 * i);
#pragma unroll
                for (int i = 0; i < D / 128; ++i) s[r][i] = *reinterpret_cast<const uint16_t*>(f + 2 * i);
            }
        }
    }
    // A operands: of word j, [0..3] of the step over its features 0..3 of every lane, [4..7] of the step over its features 4..7.
    __device__ __forceinline__ void operands(uint32_t (&a)[D / 32][8]) const {
        uint32_t two[2][(D + 127) / 128];
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
            for (int i = 0; i < (D + 127) / 128; ++i) two[r][i] = e4m3x2_to_half(s[r][i]);
#pragma unroll
        for (int j = 0; j < D / 32; ++j)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                e2m1x8_to_half(w[r][j], a[j][r], a[j][2 + r], a[j][4 + r], a[j][6 + r]);
                const uint32_t sc = __byte_perm(two[r][j / 4], 0u, (j / 2) % 2 ? 0x3232 : 0x1010);       // blocks of 16 features: two words each
#pragma unroll
                for (int i = 0; i < 4; ++i) a[j][2 * i + r] = hmul2u(a[j][2 * i + r], sc);
            }
    }
    template <int NT>
    __device__ __forceinline__ void scores(const uint32_t (&b)[NT][D / 16][2], float (&acc)[NT][4]) const {
        uint32_t a[D / 32][8];
        operands(a);
#pragma unroll
        for (int j = 0; j < D / 32; ++j)
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                if (j == 0) mma_f16_first(acc[n], *reinterpret_cast<const uint32_t(*)[4]>(&a[j][0]), b[n][2 * j][0], b[n][2 * j][1]);
                else mma_f16(acc[n], *reinterpret_cast<const uint32_t(*)[4]>(&a[j][0]), b[n][2 * j][0], b[n][2 * j][1]);
                mma_f16(acc[n], *reinterpret_cast<const uint32_t(*)[4]>(&a[j][4]), b[n][2 * j + 1][0], b[n][2 * j + 1][1]);
            }
    }
};

// A 16-key tile of values: of the keys key_place(2t), (2t + 1), (2t + 8), (2t + 9), features g * D/8 ...
template <int D>
struct ValueTile {
    uint32_t w[4][D / 64];
    uint32_t s[4];
    __device__ __forceinline__ static int place(int i, int t) { return key_place(2 * t + (i & 1) + 8 * (i >> 1)); }
    __device__ __forceinline__ void load(const uint8_t* codes, const uint8_t* sf, int g, int t) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int at = place(i, t);
            const uint8_t* c = codes + at * (D / 2) + g * (D / 16);
            if constexpr (D == 64) w[i][0] = *reinterpret_cast<const uint32_t*>(c);
            else if constexpr (D == 128) *reinterpret_cast<uint2*>(w[i]) = *reinterpret_cast<const uint2*>(c);
            else *reinterpret_cast<uint4*>(w[i]) = *reinterpret_cast<const uint4*>(c);
            const uint8_t* f = sf + at * (D / 16);
            if constexpr (D == 64) s[i] = f[g / 2];
            else if constexpr (D == 128) s[i] = f[g];
            else s[i] = *reinterpret_cast<const uint16_t*>(f + 2 * g);
        }
    }
    // Keys but the `span` ones from `from` on, which no row sees: what lies there may be anything, NaN scales too (a zero scale takes them out).
    __device__ __forceinline__ void clear(int t, int from, int span) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if ((unsigned)(place(i, t) - from) >= (unsigned)span) s[i] = 0;
    }
    template <int NT>
    __device__ __forceinline__ void add(const uint32_t (&pb)[NT][2], float (&o)[NT][D / 16][4]) const {
#pragma unroll
        for (int half = 0; half < (D == 256 ? 2 : 1); ++half) {                  // D = 256: two blocks of 16 features a lane
            const uint32_t s01 = e4m3x2_to_half((uint16_t)__byte_perm(s[0], s[1], half ? 0x4451 : 0x4440));
            const uint32_t s23 = e4m3x2_to_half((uint16_t)__byte_perm(s[2], s[3], half ? 0x4451 : 0x4440));
#pragma unroll
            for (int ww = 0; ww < (D == 64 ? 1 : 2); ++ww) {
                const int word = half * 2 + ww;
                uint32_t ev[2][4], od[2][4];
#pragma unroll
                for (int pr = 0; pr < 2; ++pr) {                                  // keys (2t, 2t + 1) and (2t + 8, 2t + 9)
                    const uint32_t w0 = w[2 * pr][word], w1 = w[2 * pr + 1][word];
                    const uint32_t even = (w0 & 0x0f0f0f0fu) | ((w1 << 4) & 0xf0f0f0f0u), odd = ((w0 >> 4) & 0x0f0f0f0fu) | (w1 & 0xf0f0f0f0u);
                    e2m1x8_to_half(even, ev[pr][0], ev[pr][1], ev[pr][2], ev[pr][3]);
                    e2m1x8_to_half(odd, od[pr][0], od[pr][1], od[pr][2], od[pr][3]);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        ev[pr][i] = hmul2u(ev[pr][i], pr ? s23 : s01);
                        od[pr][i] = hmul2u(od[pr][i], pr ? s23 : s01);
                    }
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t a[4] = {ev[0][i], od[0][i], ev[1][i], od[1][i]};
#pragma unroll
                    for (int n = 0; n < NT; ++n) mma_f16(o[n][word * 4 + i], a, pb[n][0], pb[n][1]);
                }
            }
        }
    }
};

// Limits of a column: keys [low, high) are visible to it; none where the column is not one of the step's.
struct ColumnLimits {
    int low, high;
    __device__ __forceinline__ ColumnLimits(int col, int columns, int group, int past, int window) {
        const int r = col / group;
        high = col < columns ? past + r + 1 : 0;
        low = window > 0 ? max(0, high - window) : 0;
    }
};

// ---- which keys a CTA takes ---------------------------------------------------------------------------------------------------
//
// An item is a sequence, a KV head and a chunk of C columns; its keys come in tiles of 32.  All tiles of all items stand in one line, which is cut into
// equal parts, one per CTA, so that sequences of any lengths load the SMs alike.  A CTA meets whole items, whose results it writes, and parts
// of an item at its ends, which the merge kernel joins in their order.

struct Fp4Line {
    int total, per;                                                             // tiles in the line; tiles of a CTA
};

__device__ __forceinline__ int fp4_first_tile(int past, int window) { return window > 0 ? max(0, past + 1 - window) / kFp4Tile : 0; }
__device__ __forceinline__ int fp4_tiles(int past, int ql, int window) {
    return ql > 0 ? (past + ql + kFp4Tile - 1) / kFp4Tile - fp4_first_tile(past, window) : 0;
}
__device__ __forceinline__ int fp4_items(int ql, int group, int hkv, int cols) { return (ql * group + cols - 1) / cols * hkv; }

// Lengths of the line, by all lanes of a warp.
__device__ __forceinline__ Fp4Line fp4_line(const Fp4AttnParams& p, int cols, int lane) {
    int sum = 0;
    const int group = p.hq / p.hkv;
    for (int s = lane; s < p.num_seqs; s += 32) {
        const int ql = p.q_len[s];
        sum += fp4_tiles(p.past_len[s], ql, p.window) * fp4_items(ql, group, p.hkv, cols);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    return {sum, max((sum + (int)gridDim.x - 1) / (int)gridDim.x, kFp4Warps)};
}

// The sequence that holds place `at` of the line, and its first place.
__device__ __forceinline__ int fp4_locate(const Fp4AttnParams& p, int cols, int lane, int at, int& start) {
    const int group = p.hq / p.hkv;
    int base = 0;
    for (int s0 = 0; s0 < p.num_seqs; s0 += 32) {
        const int s = s0 + lane;
        int n = 0;
        if (s < p.num_seqs) {
            const int ql = p.q_len[s];
            n = fp4_tiles(p.past_len[s], ql, p.window) * fp4_items(ql, group, p.hkv, cols);
        }
        int incl = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += v;
        }
        const unsigned here = __ballot_sync(0xffffffffu, at < base + incl);
        if (here) {
            const int l = __ffs(here) - 1;
            start = base + __shfl_sync(0xffffffffu, incl - n, l);
            return s0 + l;
        }
        base += __shfl_sync(0xffffffffu, incl, 31);
    }
    return -1;
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
// The tiles of a warp on their way into its own ring in shared memory.  A stage: key codes [32][D/2], value codes, key scales [32][D/16], value scales.
template <int D>
struct Fp4Ring {
    static constexpr int kStages = 3, kCodes = kFp4Tile * D / 2, kScales = kFp4Tile * D / 16, kBytes = 2 * (kCodes + kScales);
    static constexpr int kScaleLanes = kScales / 16 < 32 ? kScales / 16 : 32;    // lanes that copy one plane's scales
    // A lane copies its 16 bytes of every 512 of codes, and 16 bytes of scales (or, of wide heads, of every 512): where they lie in page 0, row 0.
    const uint8_t *keys, *values, *scales;
    const int* table;
    uint32_t page_bytes, smem;
    int page_shift, max_pages, num_pages, ids_at, ids, end, lane;

    // `first_ids`: the lane's entry of the first 32 of the table.
    __device__ __forceinline__ void begin(const Fp4AttnParams& p, int seq, int kvh, int end_, uint32_t smem_, int lane_, int first_ids) {
        const size_t slab = fp4_slab_bytes(p.page_size, D);
        lane = lane_;
        keys = p.pool + kvh * slab + lane * 16;
        values = keys + p.hkv * slab;
        scales = p.pool + (kvh + (lane / kScaleLanes) * p.hkv) * slab + (size_t)p.page_size * (D / 2) + lane % kScaleLanes * 16;
        page_bytes = (uint32_t)(2 * p.hkv * slab);
        table = p.page_table + (size_t)seq * p.max_pages;
        page_shift = p.page_shift;
        max_pages = p.max_pages;
        num_pages = p.num_pages;
        ids_at = 0;
        ids = first_ids;
        end = end_;
        smem = smem_;
    }
    // Pages of the table are looked up 32 at a time.
    __device__ __forceinline__ int page_of(int key) {
        const int lp = key >> page_shift;
        if (lp < ids_at || lp >= ids_at + 32) {
            ids_at = lp;
            const int i = lp + lane;
            ids = i < max_pages ? table[i] : -1;
        }
        const int page = __shfl_sync(0xffffffffu, ids, lp - ids_at);
        return key < end && (unsigned)page < (unsigned)num_pages ? page : -1;
    }
    // Starts the copies of a tile; returns a bit per half that has no page (keys from `end` on count as having none).
    __device__ __forceinline__ uint32_t load(int stage, int tile, bool real) {
        uint32_t missing = 0;
        if (real) {
            const int kb = tile * kFp4Tile, page0 = page_of(kb), at = kb & ((1 << page_shift) - 1);
            const uint32_t dst = smem + stage * kBytes + lane * 16;
            if (page_shift >= 5 && page0 >= 0 && kb + 16 < end) {                 // the whole tile lies in one page
                const uint64_t off = (uint64_t)(uint32_t)page0 * page_bytes;
                const uint8_t *k = keys + off + at * (D / 2), *v = values + off + at * (D / 2), *f = scales + off + at * (D / 16);
#pragma unroll
                for (int i = 0; i < kCodes / 512; ++i) cp_async16(dst + i * 512, k + i * 512);
#pragma unroll
                for (int i = 0; i < kCodes / 512; ++i) cp_async16(dst + kCodes + i * 512, v + i * 512);
                if constexpr (kScaleLanes == 32) {                                // D = 256: a plane's scales are 512 bytes
                    cp_async16(dst + 2 * kCodes, f);
                    cp_async16(dst + 2 * kCodes + kScales, f + (values - keys));
                } else if (2 * kScaleLanes == 32 || lane < 2 * kScaleLanes) {
                    cp_async16(dst + 2 * kCodes, f);                              // the planes' scales follow one another in the stage
                }
            } else {
#pragma unroll 1
                for (int h = 0; h < 2; ++h) {
                    const int key = kb + 16 * h, page = page_of(key), in = key & ((1 << page_shift) - 1);
                    if (page < 0) {
                        missing |= 1u << h;
                        continue;
                    }
                    const uint64_t off = (uint64_t)(uint32_t)page * page_bytes;
#pragma unroll
                    for (int v = 0; v < 2; ++v) {
                        const uint8_t* c = (v ? values : keys) + off + in * (D / 2);
                        const uint8_t* f = (v ? values : keys) + off + ((size_t)(D / 2) << page_shift) + in * (D / 16);
#pragma unroll
                        for (int i = 0; i < kCodes / 1024; ++i) cp_async16(dst + v * kCodes + h * (kCodes / 2) + i * 512, c + i * 512);
                        if (lane < kScales / 32) cp_async16(dst + 2 * kCodes + v * kScales + h * (kScales / 2), f);
                    }
                }
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        return missing;
    }
};

__device__ __forceinline__ int fp4_first_ids(const Fp4AttnParams& p, int seq) {
    const int lane = threadIdx.x & 31;
    return lane < p.max_pages ? p.page_table[(size_t)seq * p.max_pages + lane] : -1;
}

template <typename T, int D, int NT>
struct Fp4Occupancy {
    // CTAs an SM: registers for the accumulators (4 NT D/16) and the queries (2 NT D/16) besides some 60; three stages of a ring a warp
    static constexpr int kCtas = D * NT <= 128 ? 4 : D * NT <= 256 && D < 256 ? 3 : 2;
};

// One item's tiles [tile0, tile1), every fourth of them this warp's: outputs of the warp over its keys, the references of their probabilities and their sums.
// kVotes: the scores are kept for the accumulated weights.
template <typename T, int D, int NT, bool kVotes>
__device__ __forceinline__ void fp4_keys(const Fp4AttnParams& p, int seq, int kvh, int chunk, int q0, int past, int columns, int tile0, int tile1, int first_ids,
                                         uint32_t ring_at, const uint8_t* ring_ptr, float base, float (&o)[NT][D / 16][4], float (&ref)[NT][2], float (&sum)[NT][2]) {
    constexpr int C = 8 * NT;
    using Ring = Fp4Ring<D>;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int group = p.hq / p.hkv;
    const int r_first = chunk * C / group, r_last = (min(columns, chunk * C + C) - 1) / group;
    const int end = past + r_last + 1, begin = p.window > 0 ? max(0, past + r_first + 1 - p.window) : 0;      // the keys that some column sees
    const int all_low = p.window > 0 ? max(0, past + r_last + 1 - p.window) : 0, all_high = past + r_first + 1;      // visible to every column
    Ring ring;
    ring.begin(p, seq, kvh, end, ring_at, lane, first_ids);
    uint32_t flags = 0;                                                      // two bits a stage
    int next = tile0 + warp;
#pragma unroll
    for (int s = 0; s < Ring::kStages - 1; ++s, next += kFp4Warps) flags |= ring.load(s, next, next < tile1) << (2 * s);

    uint32_t qb[NT][D / 16][2];
    float factor[NT][2];
    int low[NT][2], high[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const int c = chunk * C + n * 8 + g;
        const int r = c / group, h = kvh * group + c - r * group;
        const float up = load_query<T, D>(reinterpret_cast<const T*>(p.q) + ((size_t)(q0 + r) * p.hq + h) * D + t * (D / 4), c < columns, qb[n]);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            factor[n][i] = base * __shfl_sync(0xffffffffu, up, (2 * t + i) * 4);
            const ColumnLimits lim(chunk * C + n * 8 + 2 * t + i, columns, group, past, p.window);
            low[n][i] = lim.low;
            high[n][i] = lim.high;
        }
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int i = 0; i < D / 16; ++i)
#pragma unroll
            for (int k = 0; k < 4; ++k) o[n][i][k] = 0.f;
        ref[n][0] = ref[n][1] = kRefStart;
        sum[n][0] = sum[n][1] = 0.f;
    }
    const int all_chunks = (p.max_q_len * group + 7) / 8;
    const int first_tile = fp4_first_tile(past, p.window);
    float4* keep = nullptr;                                                      // of the sequence's first tile
    if (kVotes && t < p.pairs) keep = p.scores + (((size_t)seq * p.hkv + kvh) * all_chunks + chunk * NT) * p.tiles * 16 * p.pairs + g * p.pairs + t;
    // Scores of a tile to probabilities, and those times its values.
    auto take = [&](auto open, const uint8_t* st, int kb, uint32_t missing, const float (&s)[2][NT][4]) {
        float x[2][NT][4];
        auto shifted = [&]() {
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int i = 0; i < 4; ++i) x[m][n][i] = fmaf(s[m][n][i], factor[n][i & 1], -ref[n][i & 1]);
            if constexpr (!decltype(open)::value) {
#pragma unroll
                for (int m = 0; m < 2; ++m)
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int key = kb + 16 * m + key_place(g) + 8 * (i >> 1);
                            if (((missing >> m) & 1u) || key < low[n][i & 1] || key >= high[n][i & 1]) x[m][n][i] = -INFINITY;
                        }
            }
        };
        shifted();
        const int nth = kb / kFp4Tile - first_tile;
        if (kVotes && keep != nullptr && nth < p.tiles) {
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    float v[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        v[i] = s[m][n][i] * factor[n][i & 1];
                        if constexpr (!decltype(open)::value)
                            if (x[m][n][i] == -INFINITY) v[i] = -INFINITY;
                    }
                    if (NT == 1 || chunk * NT + n < all_chunks)
                        keep[((size_t)n * p.tiles + nth) * 16 * p.pairs + m * 8 * p.pairs] = make_float4(v[0], v[1], v[2], v[3]);
                }
        }
        float most = -INFINITY;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) most = fmaxf(most, fmaxf(x[0][n][i], x[1][n][i]));
        if (__any_sync(0xffffffffu, most > 15.f)) {
            float up[NT][2];
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    // scores themselves: x has lost them where the reference is the first one
                    float top = -INFINITY;
#pragma unroll
                    for (int m = 0; m < 2; ++m)
#pragma unroll
                        for (int i = c; i < 4; i += 2)
                            if (x[m][n][i] > -INFINITY) top = fmaxf(top, s[m][n][i] * factor[n][c]);
#pragma unroll
                    for (int d = 4; d < 32; d *= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
                    const float next_ref = top - ref[n][c] > 15.f ? top - 8.f : ref[n][c];
                    up[n][c] = exp2_approx(ref[n][c] - next_ref);
                    ref[n][c] = next_ref;
                    sum[n][c] *= up[n][c];
                }
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int i = 0; i < D / 16; ++i)
#pragma unroll
                    for (int k = 0; k < 4; ++k) o[n][i][k] *= up[n][k & 1];
            shifted();
        }
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            uint32_t pb[NT][2];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    x[m][n][i] = exp2_approx(x[m][n][i]);
                    sum[n][i & 1] += x[m][n][i];
                }
                pb[n][0] = transpose8(Cvt<__half>::pack2(x[m][n][0], x[m][n][1]));
                pb[n][1] = transpose8(Cvt<__half>::pack2(x[m][n][2], x[m][n][3]));
            }
            ValueTile<D> vt;
            vt.load(st + Ring::kCodes + m * (16 * D / 2), st + 2 * Ring::kCodes + Ring::kScales + m * D, g, t);
            if constexpr (!decltype(open)::value) vt.clear(t, begin - kb - 16 * m, (missing >> m) & 1u ? 0 : end - begin);
            vt.template add<NT>(pb, o);
        }
    };
    int stage = 0;
    for (int tile = tile0 + warp; tile < tile1; tile += kFp4Warps) {
        const int ahead = stage == 0 ? Ring::kStages - 1 : stage - 1;
        __syncwarp();                                                        // the stage to be filled has been read by all lanes
        flags = (flags & ~(3u << (2 * ahead))) | (ring.load(ahead, next, next < tile1) << (2 * ahead));
        next += kFp4Warps;
        asm volatile("cp.async.wait_group %0;" ::"n"(Ring::kStages - 1) : "memory");
        __syncwarp();
        const uint8_t* st = ring_ptr + stage * Ring::kBytes;
        const uint32_t missing = (flags >> (2 * stage)) & 3u;
        const int kb = tile * kFp4Tile;
        float s[2][NT][4];
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            KeyTile<D> kt;
            kt.load(st + m * (16 * D / 2), st + 2 * Ring::kCodes + m * D, g, t);
            kt.template scores<NT>(qb, s[m]);
        }
        // A tile that every column sees whole takes no masks; the code for the others stands apart
        if (kb >= all_low && kb + kFp4Tile <= all_high && missing == 0u) take(std::true_type(), st, kb, missing, s);
        else take(std::false_type(), st, kb, missing, s);
        stage = stage + 1 == Ring::kStages ? 0 : stage + 1;
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
}

// The warps' results joined where their rings were: smem [warps][C][D] outputs and [warps][C][2]; `use(column, first feature, four outputs, reference, sum)`.
template <int D, int NT, typename Use>
__device__ __forceinline__ void fp4_join(float* smem_f, int live, float (&o)[NT][D / 16][4], float (&ref)[NT][2], float (&sum)[NT][2], Use use) {
    constexpr int C = 8 * NT;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    float* so = smem_f + warp * C * D;
    float* sml = smem_f + kFp4Warps * C * D;
    __syncthreads();                                                             // the rings have been read
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
#pragma unroll
            for (int d = 4; d < 32; d *= 2) sum[n][c] += __shfl_xor_sync(0xffffffffu, sum[n][c], d);
            const int col = n * 8 + 2 * t + c;
            if (col >= live) continue;
            if (g == 0) *reinterpret_cast<float2*>(sml + (warp * C + col) * 2) = make_float2(ref[n][c], sum[n][c]);
#pragma unroll
            for (int i = 0; i < D / 16; ++i) *reinterpret_cast<float2*>(so + col * D + g * (D / 8) + 2 * i) = make_float2(o[n][i][c], o[n][i][c + 2]);
        }
    __syncthreads();
    for (int i = threadIdx.x; i < live * (D / 4); i += blockDim.x) {
        const int col = i / (D / 4), d = (i - col * (D / 4)) * 4;
        float2 ml[kFp4Warps];
        float top = kRefStart, l = 0.f;
#pragma unroll
        for (int w = 0; w < kFp4Warps; ++w) {
            ml[w] = *reinterpret_cast<const float2*>(sml + (w * C + col) * 2);
            top = fmaxf(top, ml[w].x);
        }
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kFp4Warps; ++w) {
            const float f = exp2_approx(ml[w].x - top);
            const float4 v = *reinterpret_cast<const float4*>(smem_f + (w * C + col) * D + d);
            acc.x += f * v.x, acc.y += f * v.y, acc.z += f * v.z, acc.w += f * v.w;
            l += f * ml[w].y;
        }
        use(col, d, acc, top, l);
    }
}

// A column's sink joins its sum: the factor of what came before; `l` becomes 1 / sum.
__device__ __forceinline__ float fp4_sink(const Fp4AttnParams& p, int h, float& top, float& l) {
    float f = 1.f;
    if (p.sinks) {
        const float z = p.sinks[h] * 1.4426950408889634f, m = fmaxf(top, z);
        f = exp2_approx(top - m);
        l = l * f + exp2_approx(z - m);
        top = m;
    }
    l = l == 0.f ? 0.f : 1.f / l;                                                // a row that sees nothing gives zeros
    return f;
}

// Four outputs of a column whose keys have all been joined: the sink, the sum and the values' scale, then the one rounding.
template <typename T, int D>
__device__ __forceinline__ void fp4_finish(const Fp4AttnParams& p, size_t row, int h, int d, float4 acc, float top, float l) {
    const float keep = fp4_sink(p, h, top, l), inv = l, f = inv * keep * p.scales[1];
    *reinterpret_cast<uint2*>(reinterpret_cast<T*>(p.out) + row * D + d) = make_uint2(Cvt<T>::pack2(acc.x * f, acc.y * f), Cvt<T>::pack2(acc.z * f, acc.w * f));
    if (p.stat && d == 0) *reinterpret_cast<float2*>(p.stat + row * 2) = make_float2(top, inv);
}

__device__ __forceinline__ float4 cluster_load_f4(const void* at, uint32_t rank) {
    uint32_t a;
    float4 v;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(at)), "r"(rank));
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ void fp4_cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// Accumulated attention weights: weights[page, head, slot] = decay * weights + the sum over the step's rows and the group's heads of
// exp2(score - top) / sum, for keys that some row sees; the step's own keys start from zero.  fp4_keys has left its scores (4 bytes for each
// key and column, mostly still in the L2 cache); making them again took the keys, their expansion and the products a second time (16 sequences of 8192:
// 36 us against 8).  A warp owns 32 keys, so that every sum has one order.  Where a CTA's columns are all that the step has, it adds them itself
// once the sums are known, and every lane reads what it wrote (16 sequences of 8192: 55 us for the step, with a kernel for the weights 59).
// U tiles at a time: first, first + stride ... of those below `tiles`; `stat(column)` gives (top, 1 / sum).
template <int U, typename Stat>
__device__ __forceinline__ void fp4_weigh(const Fp4AttnParams& p, int seq, int kvh, int ql, int past, int index, int stride, int tiles, Stat stat) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, columns = ql * (p.hq / p.hkv);
    if (index >= tiles) return;
    const int first_tile = fp4_first_tile(past, p.window), first = p.window > 0 ? max(0, past + 1 - p.window) : 0;
    float* w[U];
    float old[U], given[U][2][2];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        // a lane's own key: half t / 2, row g or g + 8 of it
        const int at = index + u * stride, mine = (first_tile + at) * kFp4Tile + 16 * (t >> 1) + key_place(g) + 8 * (t & 1), lp = mine >> p.page_shift;
        const int page = at < tiles && mine >= first && mine < past + ql && lp < p.max_pages ? p.page_table[(size_t)seq * p.max_pages + lp] : -1;
        w[u] = (unsigned)page < (unsigned)p.num_pages ? p.weights + ((size_t)page * p.hkv + kvh) * p.page_size + (mine & (p.page_size - 1)) : nullptr;
        old[u] = w[u] && mine < past ? p.decay * *w[u] : 0.f;
        given[u][0][0] = given[u][0][1] = given[u][1][0] = given[u][1][1] = 0.f;
    }
    const int all_chunks = (p.max_q_len * (p.hq / p.hkv) + 7) / 8, chunks = min((columns + 7) / 8, all_chunks);
    const float4* src = p.scores + (((size_t)seq * p.hkv + kvh) * all_chunks * p.tiles + index) * 16 * p.pairs + g * p.pairs + t;
    if (t < p.pairs) {
#pragma unroll 4 / U
        for (int ch = 0; ch < chunks; ++ch) {
            float4 s[U][2];
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int m = 0; m < 2; ++m)
                    s[u][m] = index + u * stride < tiles ? src[((size_t)ch * p.tiles + u * stride) * 16 * p.pairs + m * 8 * p.pairs]
                                                         : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
            float2 st[2];
#pragma unroll
            for (int c = 0; c < 2; ++c) st[c] = ch * 8 + 2 * t + c < columns ? stat(ch * 8 + 2 * t + c) : make_float2(0.f, 0.f);
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int m = 0; m < 2; ++m) {
                    given[u][m][0] += exp2_approx(s[u][m].x - st[0].x) * st[0].y;
                    given[u][m][1] += exp2_approx(s[u][m].z - st[0].x) * st[0].y;
                    if (ch * 8 + 2 * t + 1 < columns) {                          // the last column may have no neighbour
                        given[u][m][0] += exp2_approx(s[u][m].y - st[1].x) * st[1].y;
                        given[u][m][1] += exp2_approx(s[u][m].w - st[1].x) * st[1].y;
                    }
                }
        }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                given[u][m][r] += __shfl_xor_sync(0xffffffffu, given[u][m][r], 1);
                given[u][m][r] += __shfl_xor_sync(0xffffffffu, given[u][m][r], 2);
            }
        const float sum = t & 2 ? (t & 1 ? given[u][1][1] : given[u][1][0]) : (t & 1 ? given[u][0][1] : given[u][0][0]);
        if (w[u]) *w[u] = old[u] + sum;
    }
}

// Many items: a cluster per item, its CTAs take equal parts of the item's tiles and join their results through shared memory.
// grid (CTAs of a cluster, items of a sequence, sequences)
template <typename T, int D, int NT, bool kVotes>
__global__ void __launch_bounds__(kFp4Warps * 32, (Fp4Occupancy<T, D, NT>::kCtas)) attention_fp4_cluster_kernel(const Fp4AttnParams p) {
    pdl_prologue();
    constexpr int C = 8 * NT;
    using Ring = Fp4Ring<D>;
    extern __shared__ __align__(16) uint8_t smem[];
    const int warp = threadIdx.x >> 5, ranks = gridDim.x, rank = blockIdx.x, seq = blockIdx.z;
    const int chunk = blockIdx.y / p.hkv, kvh = blockIdx.y - chunk * p.hkv;
    const int first_ids = fp4_first_ids(p, seq);                                 // on its way with the lengths, not behind them
    const int group = p.hq / p.hkv, ql = p.q_len[seq], past = p.past_len[seq], q0 = p.q_start[seq], columns = ql * group;
    if (chunk * C >= columns) return;                                            // the whole cluster
    const int first = fp4_first_tile(past, p.window), tiles = fp4_tiles(past, ql, p.window);
    const int tile0 = first + tiles * rank / ranks, tile1 = first + tiles * (rank + 1) / ranks;
    float o[NT][D / 16][4], ref[NT][2], sum[NT][2];
    fp4_keys<T, D, NT, kVotes>(p, seq, kvh, chunk, q0, past, columns, tile0, tile1, first_ids, smem_u32(smem) + warp * Ring::kStages * Ring::kBytes,
                       smem + warp * Ring::kStages * Ring::kBytes, p.scale * 1.4426950408889634f * p.scales[0], o, ref, sum);
    float* smem_f = reinterpret_cast<float*>(smem);
    const int live = min(C, columns - chunk * C);
    // the CTA's own references and sums lie behind all warps' results, (top, 1 / sum) of the item's columns behind those
    float4* own_ml = reinterpret_cast<float4*>(smem_f + kFp4Warps * C * (D + 2));
    float2* s_stat = reinterpret_cast<float2*>(own_ml + C);
    const bool weigh = kVotes && p.max_items == p.hkv;
    auto weights = [&]() {
        const int limit = min(tiles, p.tiles);
        constexpr int U = NT == 1 ? 4 : 2;
        for (int i = tile0 + warp - first; i < tile1 - first; i += U * kFp4Warps)
            fp4_weigh<U>(p, seq, kvh, ql, past, i, kFp4Warps, min(limit, tile1 - first), [&](int col) { return s_stat[col]; });
    };
    auto finish = [&](int col, int d, float4 acc, float top, float l) {
        const int c = chunk * C + col, r = c / group, h = kvh * group + c - r * group;
        fp4_finish<T, D>(p, (size_t)(q0 + r) * p.hq + h, h, d, acc, top, l);
    };
    auto stat_of = [&](int col, float top, float l) {
        const int c = chunk * C + col, r = c / group;
        fp4_sink(p, kvh * group + c - r * group, top, l);
        s_stat[col] = make_float2(top, l);
    };
    if (ranks == 1) {
        fp4_join<D, NT>(smem_f, live, o, ref, sum, [&](int col, int d, float4 acc, float top, float l) {
            finish(col, d, acc, top, l);
            if (weigh && d == 0) stat_of(col, top, l);
        });
        if (weigh) {
            __syncthreads();
            weights();
        }
        return;
    }
    // the CTA's own results take the first warp's place (a thread reads what it replaces)
    fp4_join<D, NT>(smem_f, live, o, ref, sum, [&](int col, int d, float4 acc, float top, float l) {
        *reinterpret_cast<float4*>(smem_f + col * D + d) = acc;
        if (d == 0) own_ml[col] = make_float4(top, l, 0.f, 0.f);
    });
    fp4_cluster_sync();
    for (int i = rank * blockDim.x + threadIdx.x; i < live * (D / 4); i += ranks * blockDim.x) {
        const int col = i / (D / 4), d = (i - col * (D / 4)) * 4;
        float top = kRefStart, l = 0.f;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int r0 = 0; r0 < ranks; r0 += 4) {
            float4 ml[4], v[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                ml[r] = r0 + r < ranks ? cluster_load_f4(own_ml + col, r0 + r) : make_float4(kRefStart, 0.f, 0.f, 0.f);
                v[r] = r0 + r < ranks ? cluster_load_f4(smem_f + col * D + d, r0 + r) : make_float4(0.f, 0.f, 0.f, 0.f);
            }
            const float next = fmaxf(fmaxf(fmaxf(ml[0].x, ml[1].x), fmaxf(ml[2].x, ml[3].x)), top), keep = exp2_approx(top - next);
            acc.x *= keep, acc.y *= keep, acc.z *= keep, acc.w *= keep;
            l *= keep;
            top = next;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float f = exp2_approx(ml[r].x - top);
                acc.x += f * v[r].x, acc.y += f * v[r].y, acc.z += f * v[r].z, acc.w += f * v[r].w;
                l += f * ml[r].y;
            }
        }
        finish(col, d, acc, top, l);
    }
    if (weigh && threadIdx.x < live) {
        float top = kRefStart, l = 0.f;
        float4 ml[16];
#pragma unroll
        for (int r = 0; r < 16; ++r) ml[r] = r < ranks ? cluster_load_f4(own_ml + threadIdx.x, r) : make_float4(kRefStart, 0.f, 0.f, 0.f);
#pragma unroll
        for (int r = 0; r < 16; ++r) top = fmaxf(top, ml[r].x);
#pragma unroll
        for (int r = 0; r < 16; ++r) l += exp2_approx(ml[r].x - top) * ml[r].y;
        stat_of(threadIdx.x, top, l);
    }
    fp4_cluster_sync();                                                          // nobody leaves while its results may be read
    if (weigh) weights();
}

// Few items and many keys: the line.
template <typename T, int D, int NT, bool kVotes>
__global__ void __launch_bounds__(kFp4Warps * 32, (Fp4Occupancy<T, D, NT>::kCtas)) attention_fp4_kernel(const Fp4AttnParams p) {
    pdl_prologue();
    constexpr int C = 8 * NT;
    using Ring = Fp4Ring<D>;
    extern __shared__ __align__(16) uint8_t smem[];                              // rings; after a segment [warps][C][D] outputs and [warps][C][2] (reference, sum)
    float* smem_f = reinterpret_cast<float*>(smem);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int group = p.hq / p.hkv;
    const Fp4Line line = fp4_line(p, C, lane);
    int at = blockIdx.x * line.per;
    const int stop = min(line.total, at + line.per);
    if (at >= stop) return;
    int seq_start = 0, seq = fp4_locate(p, C, lane, at, seq_start);
    const float base = p.scale * 1.4426950408889634f * p.scales[0];
    const uint32_t ring_at = smem_u32(smem) + warp * Ring::kStages * Ring::kBytes;
    const uint8_t* ring_ptr = smem + warp * Ring::kStages * Ring::kBytes;

    while (at < stop) {
        const int ql = p.q_len[seq], past = p.past_len[seq], columns = ql * group;
        const int tiles = fp4_tiles(past, ql, p.window), items = fp4_items(ql, group, p.hkv, C);
        if (at >= seq_start + tiles * items) {                                   // on to the next sequence
            seq_start += tiles * items;
            ++seq;
            continue;
        }
        const int item = (at - seq_start) / tiles, off = (at - seq_start) - item * tiles;
        const int count = min(tiles - off, stop - at);
        const int chunk = item / p.hkv, kvh = item - chunk * p.hkv;
        const int tile0 = fp4_first_tile(past, p.window) + off, tile1 = tile0 + count;
        const int q0 = p.q_start[seq];
        float o[NT][D / 16][4], ref[NT][2], sum[NT][2];
        fp4_keys<T, D, NT, kVotes>(p, seq, kvh, chunk, q0, past, columns, tile0, tile1, fp4_first_ids(p, seq), ring_at, ring_ptr, base, o, ref, sum);
        const bool whole = count == tiles;
        const size_t slot = (size_t)blockIdx.x * 2 + (off == 0);                 // parts: [0] what began in an earlier CTA, [1] what goes on in a later one
        if (threadIdx.x == 0 && off == 0 && item < p.max_items)
            p.spans[(size_t)seq * p.max_items + item] = make_int2(blockIdx.x, (at + tiles - 1) / line.per);
        fp4_join<D, NT>(smem_f, min(C, columns - chunk * C), o, ref, sum, [&](int col, int d, float4 acc, float top, float l) {
            if (!whole) {
                *reinterpret_cast<float4*>(p.part_o + (slot * C + col) * D + d) = acc;
                if (d == 0) *reinterpret_cast<float2*>(p.part_ml + (slot * C + col) * 2) = make_float2(top, l);
            } else {
                const int c = chunk * C + col, r = c / group, h = kvh * group + c - r * group;
                fp4_finish<T, D>(p, (size_t)(q0 + r) * p.hq + h, h, d, acc, top, l);
            }
        });
        at += count;
        if (at < stop) __syncthreads();                                          // the next segment's tiles go where the results were
    }
}

// grid (items of a sequence, sequences, columns of an item): the parts of a column joined in their order, every 16th of them a warp's.
template <typename T, int D, int NT>
__global__ void __launch_bounds__(512) attention_fp4_merge_kernel(const Fp4AttnParams p) {
    constexpr int C = 8 * NT, W = 16, E = D / 32;
    __shared__ __align__(16) float s_o[W][D];
    __shared__ float s_l[W], s_top[W];
    const int item = blockIdx.x, seq = blockIdx.y, col = blockIdx.z, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    pdl_prologue();
    const int group = p.hq / p.hkv, chunk = item / p.hkv, kvh = item - chunk * p.hkv;
    const int c = chunk * C + col, ql = p.q_len[seq];
    if (c >= ql * group) return;
    const int2 span = p.spans[(size_t)seq * p.max_items + item];
    if (span.x >= span.y) return;                                                // whole: written already
    const int parts = span.y - span.x + 1;
    // the first part is slot 1 of its CTA, the others slot 0
    auto slot_of = [&](int i) { return ((size_t)(span.x + i) * 2 + (i == 0)) * C + col; };
    float top = kRefStart, l = 0.f, acc[E];
#pragma unroll
    for (int i = 0; i < E; ++i) acc[i] = 0.f;
    for (int i0 = warp; i0 < parts; i0 += 8 * W) {
        float2 ml[8];
        float v[8][E], next = top;
#pragma unroll
        for (int u = 0; u < 8; ++u) {                                            // eight parts on their way
            const int i = i0 + u * W;
            ml[u] = make_float2(kRefStart, 0.f);
#pragma unroll
            for (int k = 0; k < E; ++k) v[u][k] = 0.f;
            if (i < parts) {
                ml[u] = *reinterpret_cast<const float2*>(p.part_ml + slot_of(i) * 2);
                const float* src = p.part_o + slot_of(i) * D + lane * E;
                if constexpr (E == 2) *reinterpret_cast<float2*>(v[u]) = *reinterpret_cast<const float2*>(src);
                else
#pragma unroll
                    for (int k = 0; k < E; k += 4) *reinterpret_cast<float4*>(v[u] + k) = *reinterpret_cast<const float4*>(src + k);
            }
            next = fmaxf(next, ml[u].x);
        }
        const float keep = exp2_approx(top - next);
        top = next;
        l *= keep;
#pragma unroll
        for (int k = 0; k < E; ++k) acc[k] *= keep;
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const float f = exp2_approx(ml[u].x - top);
            l += f * ml[u].y;
#pragma unroll
            for (int k = 0; k < E; ++k) acc[k] += f * v[u][k];
        }
    }
#pragma unroll
    for (int k = 0; k < E; ++k) s_o[warp][lane * E + k] = acc[k];
    if (lane == 0) s_top[warp] = top, s_l[warp] = l;
    __syncthreads();
    if (threadIdx.x >= D / 4) return;
    const int d = threadIdx.x * 4, r = c / group, h = kvh * group + c - r * group;
    top = kRefStart;
#pragma unroll
    for (int w = 0; w < W; ++w) top = fmaxf(top, s_top[w]);
    float4 out = make_float4(0.f, 0.f, 0.f, 0.f);
    l = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) {
        const float f = exp2_approx(s_top[w] - top);
        const float4 v = *reinterpret_cast<const float4*>(&s_o[w][d]);
        out.x += f * v.x, out.y += f * v.y, out.z += f * v.z, out.w += f * v.w;
        l += f * s_l[w];
    }
    fp4_finish<T, D>(p, (size_t)(p.q_start[seq] + r) * p.hq + h, h, d, out, top, l);
}

// The weights where the attention kernel could not add them itself.  grid (groups of 4 tiles, KV heads, sequences)
__global__ void __launch_bounds__(128) attention_fp4_weights_kernel(const Fp4AttnParams p) {
    pdl_prologue();
    const int seq = blockIdx.z, kvh = blockIdx.y, ql = p.q_len[seq], past = p.past_len[seq], group = p.hq / p.hkv, q0 = p.q_start[seq];
    fp4_weigh<1>(p, seq, kvh, ql, past, blockIdx.x * 4 + (threadIdx.x >> 5), 1, min(fp4_tiles(past, ql, p.window), p.tiles), [&](int col) {
        const int r = col / group;
        return *reinterpret_cast<const float2*>(p.stat + ((size_t)(q0 + r) * p.hq + kvh * group + col - r * group) * 2);
    });
}

template <typename T, int D, int NT, bool kVotes>
int launch_attention_fp4_nt(const Fp4AttnParams& p, int columns, cudaStream_t stream) {
    constexpr int C = 8 * NT;
    constexpr int kSmem = kFp4Warps * Fp4Ring<D>::kStages * Fp4Ring<D>::kBytes;
    static_assert(kSmem >= kFp4Warps * C * (D + 2) * 4 + C * 24, "the warps' results fit where their rings were");
    static int most_ranks[64] = {};                                              // clusters of 16 where the device places them
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64) return fail("telb_paged_attention_fp4: device index above 63");
    if (!most_ranks[dev]) {
        cudaError_t e = cudaFuncSetAttribute(attention_fp4_kernel<T, D, NT, kVotes>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
        if (e == cudaSuccess) e = cudaFuncSetAttribute(attention_fp4_cluster_kernel<T, D, NT, kVotes>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
        if (e == cudaSuccess) e = cudaFuncSetAttribute(attention_fp4_cluster_kernel<T, D, NT, kVotes>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (e != cudaSuccess) return fail("cudaFuncSetAttribute(attention_fp4)", e);
        cudaLaunchConfig_t c{};
        c.gridDim = dim3(16);
        c.blockDim = dim3(kFp4Warps * 32);
        c.dynamicSmemBytes = kSmem;
        cudaLaunchAttribute a;
        a.id = cudaLaunchAttributeClusterDimension;
        a.val.clusterDim.x = 16;
        a.val.clusterDim.y = a.val.clusterDim.z = 1;
        c.attrs = &a;
        c.numAttrs = 1;
        int clusters = 0;
        const bool placed = cudaOccupancyMaxActiveClusters(&clusters, attention_fp4_cluster_kernel<T, D, NT, kVotes>, &c) == cudaSuccess && clusters > 0;
        cudaGetLastError();
        most_ranks[dev] = placed ? 16 : 8;
    }
    if (p.ranks > 0) {
        const int ranks = min(p.ranks, most_ranks[dev]);
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3(ranks, p.max_items, p.num_seqs);
        cfg.blockDim = dim3(kFp4Warps * 32);
        cfg.dynamicSmemBytes = kSmem;
        cfg.stream = stream;
        cudaLaunchAttribute attr[2];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = ranks;
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[1].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = attr;
        cfg.numAttrs = pdl_enabled() ? 2 : 1;
        cudaError_t e = cudaLaunchKernelEx(&cfg, attention_fp4_cluster_kernel<T, D, NT, kVotes>, p);
        return e == cudaSuccess ? 0 : fail("attention_fp4_cluster_kernel", e);
    }
    TELB_LAUNCH("attention_fp4_kernel", (attention_fp4_kernel<T, D, NT, kVotes>), dim3(p.ctas), dim3(kFp4Warps * 32), kSmem, stream, p);
    TELB_LAUNCH("attention_fp4_merge_kernel", (attention_fp4_merge_kernel<T, D, NT>), dim3(p.max_items, p.num_seqs, min(columns, C)), dim3(512), 0, stream, p);
    return 0;
}

template <typename T, int D>
int launch_attention_fp4(const Fp4AttnParams& p, int cols, cudaStream_t stream) {
    const int columns = p.max_q_len * (p.hq / p.hkv);
    constexpr int kMost = D == 256 ? 1 : 2;
    if (!p.weights)
        return cols == 8 ? launch_attention_fp4_nt<T, D, 1, false>(p, columns, stream) : launch_attention_fp4_nt<T, D, kMost, false>(p, columns, stream);
    const int rc = cols == 8 ? launch_attention_fp4_nt<T, D, 1, true>(p, columns, stream) : launch_attention_fp4_nt<T, D, kMost, true>(p, columns, stream);
    if (rc || (p.ranks > 0 && p.max_items == p.hkv)) return rc;     // a cluster has all columns of its keys: it adds the weights itself
    TELB_LAUNCH("attention_fp4_weights_kernel", attention_fp4_weights_kernel, dim3((p.tiles + 3) / 4, p.hkv, p.num_seqs), dim3(128), 0, stream, p);
    return 0;
}

}  // namespace telb

using namespace telb;

// CTAs that run at once, with items of `cols` columns.
extern "C" int telb_attention_fp4_ctas(int cols, int d) {
    const int nt = cols / 8;
    return sm_count() * (d * nt <= 128 ? 4 : d * nt <= 256 && d < 256 ? 3 : 2);
}

// ranks > 0: clusters of so many CTAs per item (sequence, KV head, C columns; 8 in place of 16 where the device places none of 16); 0: the line of all items' tiles cut into `ctas` parts, with
// part_o [2 ctas, C, d], part_ml [2 ctas, C, 2] and spans [num_seqs, max_items] (C = cols: 8, or 16 of at most 128 features; max_items = KV heads x chunks of the longest
// sequence's columns): scratch.  `weights` null: outputs only; else `stat` [tokens, hq, 2]
// and `scores` [num_seqs, hkv, columns / 8, tiles, 2, 8, pairs] float4 are scratch: `tiles` of 32 keys hold every sequence's, `pairs` columns of 8 (at most 4).
extern "C" int telb_paged_attention_fp4(const Fp4AttnParams* params, int cols, int d, int is_bf16, cudaStream_t stream) {
    const Fp4AttnParams& p = *params;
    if (p.tokens <= 0 || p.num_seqs <= 0) return 0;
    if (d != 64 && d != 128 && d != 256) return fail("telb_paged_attention_fp4: head_dim must be 64, 128 or 256");
    if (p.page_size < 16 || p.page_size != 1 << p.page_shift) return fail("telb_paged_attention_fp4: the page size must be a power of two, at least 16");
    if (p.hkv <= 0 || p.hq % p.hkv) return fail("telb_paged_attention_fp4: query heads must be a multiple of the KV heads");
    if (p.ranks < 0 || p.ranks > 16) return fail("telb_paged_attention_fp4: clusters of at most 16 CTAs");
    if (p.ranks == 0 && (p.ctas < 1 || !p.part_o || !p.part_ml || !p.spans)) return fail("telb_paged_attention_fp4: no room for the parts");
    const int columns = p.max_q_len * (p.hq / p.hkv);
    if (cols != 8 && (cols != 16 || d == 256)) return fail("telb_paged_attention_fp4: items of 8 columns, or 16 of at most 128 features");
    if (p.max_items != p.hkv * ((columns + cols - 1) / cols)) return fail("telb_paged_attention_fp4: items of another size");
    if (p.max_items > 65535) return fail("telb_paged_attention_fp4: too many rows x heads");
    if (2LL * p.hkv * p.page_size * (d / 2 + d / 16) >= 1LL << 31) return fail("telb_paged_attention_fp4: pages of less than 2 GB");
    if (p.num_seqs > 65535) return fail("telb_paged_attention_fp4: more than 65535 sequences");
    if (p.weights && (!p.stat || !p.scores || p.tiles < 1 || p.pairs < 1 || p.pairs > 4 || p.hkv > 65535)) return fail("telb_paged_attention_fp4: weights without room for the scores");
    if (!p.weights && p.scores) return fail("telb_paged_attention_fp4: scores are kept for weights");
    if (is_bf16) {
        if (d == 128) return launch_attention_fp4<__nv_bfloat16, 128>(p, cols, stream);
        if (d == 64) return launch_attention_fp4<__nv_bfloat16, 64>(p, cols, stream);
        return launch_attention_fp4<__nv_bfloat16, 256>(p, cols, stream);
    }
    if (d == 128) return launch_attention_fp4<__half, 128>(p, cols, stream);
    if (d == 64) return launch_attention_fp4<__half, 64>(p, cols, stream);
    return launch_attention_fp4<__half, 256>(p, cols, stream);
}
