// Attention of few query rows a sequence over four-bit cache pages (layout: kv_fp4_common.cuh), read in place.
//
// The rows of a sequence and the query heads of a KV head make `columns`; 16 keys, 16 features and 8 columns make one fp16 matrix instruction.
//   scores  S[key, column] = sum over d of K[key, d] q[column, d]       A = keys, 16 bytes a lane from a key's row, B = queries in registers
//   output  O[d, column]  += sum over keys of V[key, d] P[key, column]  A = values, the nibbles of two keys joined before they become half2
// Features and keys may come in any order inside a sum, so both operands are taken from the pages in the order in which they lie there; no
// data crosses lanes but the probabilities (one 8 x 8 transposition per 8 keys).  code * block scale is exact in fp16; scales[] and the softmax scale
// multiply the 32-bit sums.  Probabilities are exp2(score - reference), the reference 8 to 16 below the maximum: fp16 keeps eleven bits of
// those down to 2^-22 of the largest, and the accumulators are rescaled only when a score outgrows the reference by 2^15.
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
    int num_seqs, tokens, max_q_len, num_pages, max_pages, page_size, hq, hkv, window, splits;
    float scale, decay;
};

constexpr int kFp4Warps = 4, kFp4Tile = 32;               // warps of a CTA; keys that a warp takes at a time
constexpr float kRefStart = -1e30f;

__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
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
        // bf16 queries enter as fp16, divided by the power of two below their column's largest: exact for all that is above 2^-25 of it
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
    template <int NT>
    __device__ __forceinline__ void scores(const uint32_t (&b)[NT][D / 16][2], float (&acc)[NT][4]) const {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[n][i] = 0.f;
#pragma unroll
        for (int j2 = 0; j2 < D / 32; ++j2) {                                   // a word: eight features, two steps
            uint32_t a[2][4], sc[2];
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                e2m1x8_to_half(w[r][j2], a[r][0], a[r][1], a[r][2], a[r][3]);
                const uint32_t two = e4m3x2_to_half(s[r][j2 / 4]);                // the blocks of 16 features: two words each
                sc[r] = __byte_perm(two, two, (j2 / 2) % 2 ? 0x3232 : 0x1010);
#pragma unroll
                for (int i = 0; i < 4; ++i) a[r][i] = hmul2u(a[r][i], sc[r]);
            }
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const uint32_t lo[4] = {a[0][0], a[1][0], a[0][1], a[1][1]}, hi[4] = {a[0][2], a[1][2], a[0][3], a[1][3]};
                mma_f16(acc[n], lo, b[n][2 * j2][0], b[n][2 * j2][1]);
                mma_f16(acc[n], hi, b[n][2 * j2 + 1][0], b[n][2 * j2 + 1][1]);
            }
        }
    }
};

// A 16-key tile of values: of the keys key_place(2t), (2t + 1), (2t + 8), (2t + 9), features g * D/8 ...
template <int D>
struct ValueTile {
    uint32_t w[4][D / 64];
    uint16_t s[4];
    __device__ __forceinline__ static int place(int i, int t) { return key_place(2 * t + (i & 1) + 8 * (i >> 1)); }
    __device__ __forceinline__ void load(const uint8_t* codes, const uint8_t* sf, int g, int t, int live) {
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
            if (at >= live) s[i] = 0;                                             // what lies behind the last key may be anything, NaN scales too
        }
    }
    template <int NT>
    __device__ __forceinline__ void add(const uint32_t (&pb)[NT][2], float (&o)[NT][D / 16][4]) const {
#pragma unroll
        for (int half = 0; half < (D == 256 ? 2 : 1); ++half) {                  // D = 256: two blocks of 16 features a lane
            const uint32_t s01 = e4m3x2_to_half((uint16_t)(((s[0] >> (8 * half)) & 0xff) | ((s[1] >> (8 * half)) << 8)));
            const uint32_t s23 = e4m3x2_to_half((uint16_t)(((s[2] >> (8 * half)) & 0xff) | ((s[3] >> (8 * half)) << 8)));
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

// grid (splits, KV heads x chunks of 8 NT columns, sequences).  Every split takes a contiguous part of the sequence's own keys, its warps every fourth tile.
template <typename T, int D, int NT>
__global__ void __launch_bounds__(kFp4Warps * 32) attention_fp4_kernel(const Fp4AttnParams p) {
    pdl_prologue();
    constexpr int C = 8 * NT;
    extern __shared__ float smem[];                                              // [warps][C][D] outputs, then [warps][C][2] (reference, sum)
    const int seq = blockIdx.z, kvh = blockIdx.y % p.hkv, chunk = blockIdx.y / p.hkv;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int group = p.hq / p.hkv, ql = p.q_len[seq], past = p.past_len[seq], columns = ql * group;
    if (chunk * C >= columns) return;
    const int q0 = p.q_start[seq];
    const int* table = p.page_table + (size_t)seq * p.max_pages;
    const size_t slab = fp4_slab_bytes(p.page_size, D);

    uint32_t qb[NT][D / 16][2];
    float factor[NT][2];
    int low[NT][2], high[NT][2];
    const float base = p.scale * 1.4426950408889634f * p.scales[0];
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
    const int r_first = chunk * C / group, r_last = (min(columns, chunk * C + C) - 1) / group;
    const int first = p.window > 0 ? max(0, past + r_first + 1 - p.window) : 0, end = past + r_last + 1;
    const int all_low = p.window > 0 ? max(0, past + r_last + 1 - p.window) : 0, all_high = past + r_first + 1;      // visible to every column
    const int tile0 = first / kFp4Tile, tiles = (end + kFp4Tile - 1) / kFp4Tile - tile0;
    const int t_begin = tile0 + (int)((long long)tiles * blockIdx.x / p.splits), t_end = tile0 + (int)((long long)tiles * (blockIdx.x + 1) / p.splits);

    float o[NT][D / 16][4], ref[NT][2], sum[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int i = 0; i < D / 16; ++i)
#pragma unroll
            for (int k = 0; k < 4; ++k) o[n][i][k] = 0.f;
        ref[n][0] = ref[n][1] = kRefStart;
        sum[n][0] = sum[n][1] = 0.f;
    }
    for (int tile = t_begin + warp; tile < t_end; tile += kFp4Warps) {
        const int kb = tile * kFp4Tile;
        float s[2][NT][4];
        KeyTile<D> kt[2];
        ValueTile<D> vt[2];
        bool there[2];
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            const int k0 = kb + 16 * m, lp = k0 / p.page_size, at = k0 - lp * p.page_size;
            const int page = k0 < end && lp < p.max_pages ? table[lp] : -1;
            there[m] = (unsigned)page < (unsigned)p.num_pages;
            const uint8_t* ks = p.pool + ((size_t)(there[m] ? page : 0) * 2 * p.hkv + kvh) * slab;
            const uint8_t* vs = ks + (size_t)p.hkv * slab;
            kt[m].load(ks + (size_t)at * (D / 2), ks + (size_t)p.page_size * (D / 2) + (size_t)at * (D / 16), g, t);
            vt[m].load(vs + (size_t)at * (D / 2), vs + (size_t)p.page_size * (D / 2) + (size_t)at * (D / 16), g, t, there[m] ? end - k0 : 0);
        }
#pragma unroll
        for (int m = 0; m < 2; ++m) kt[m].template scores<NT>(qb, s[m]);
        const bool open = kb >= all_low && kb + kFp4Tile <= all_high && there[0] && there[1];
        uint32_t pb[2][NT][2];
        float x[2][NT][4];
        auto shifted = [&]() {
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        x[m][n][i] = fmaf(s[m][n][i], factor[n][i & 1], -ref[n][i & 1]);
                        if (!open) {
                            const int key = kb + 16 * m + key_place(g) + 8 * (i >> 1);
                            if (!there[m] || key < low[n][i & 1] || key >= high[n][i & 1]) x[m][n][i] = -INFINITY;
                        }
                    }
        };
        shifted();
        bool over = false;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) over = over || x[0][n][i] > 15.f || x[1][n][i] > 15.f;
        if (__any_sync(0xffffffffu, over)) {
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
                    const float next = top - ref[n][c] > 15.f ? top - 8.f : ref[n][c];
                    up[n][c] = exp2_approx(ref[n][c] - next);
                    ref[n][c] = next;
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
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int n = 0; n < NT; ++n) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    x[m][n][i] = exp2_approx(x[m][n][i]);
                    sum[n][i & 1] += x[m][n][i];
                }
                pb[m][n][0] = transpose8(Cvt<__half>::pack2(x[m][n][0], x[m][n][1]));
                pb[m][n][1] = transpose8(Cvt<__half>::pack2(x[m][n][2], x[m][n][3]));
            }
#pragma unroll
        for (int m = 0; m < 2; ++m) vt[m].template add<NT>(pb[m], o);
    }
    // join the warps
    float* so = smem + warp * C * D;
    float* sml = smem + kFp4Warps * C * D;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
#pragma unroll
            for (int d = 4; d < 32; d *= 2) sum[n][c] += __shfl_xor_sync(0xffffffffu, sum[n][c], d);
            const int col = n * 8 + 2 * t + c;
            if (g == 0) {
                sml[(warp * C + col) * 2] = ref[n][c];
                sml[(warp * C + col) * 2 + 1] = sum[n][c];
            }
#pragma unroll
            for (int i = 0; i < D / 16; ++i) *reinterpret_cast<float2*>(so + col * D + g * (D / 8) + 2 * i) = make_float2(o[n][i][c], o[n][i][c + 2]);
        }
    __syncthreads();
    const int live = min(C, columns - chunk * C);
    for (int i = threadIdx.x; i < live * (D / 4); i += blockDim.x) {
        const int col = i / (D / 4), d = (i - col * (D / 4)) * 4;
        float top = kRefStart;
#pragma unroll
        for (int w = 0; w < kFp4Warps; ++w) top = fmaxf(top, sml[(w * C + col) * 2]);
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        float l = 0.f;
#pragma unroll
        for (int w = 0; w < kFp4Warps; ++w) {
            const float f = exp2_approx(sml[(w * C + col) * 2] - top);
            const float4 v = *reinterpret_cast<const float4*>(smem + (w * C + col) * D + d);
            acc.x += f * v.x, acc.y += f * v.y, acc.z += f * v.z, acc.w += f * v.w;
            l += f * sml[(w * C + col) * 2 + 1];
        }
        const int c = chunk * C + col, r = c / group, h = kvh * group + c - r * group;
        const size_t row = (size_t)(q0 + r) * p.hq + h;
        if (p.splits > 1) {
            const size_t at = row * p.splits + blockIdx.x;
            *reinterpret_cast<float4*>(p.part_o + at * D + d) = acc;
            if (d == 0) *reinterpret_cast<float2*>(p.part_ml + at * 2) = make_float2(top, l);
        } else {
            if (p.sinks) {
                const float z = p.sinks[h] * 1.4426950408889634f, m = fmaxf(top, z), f = exp2_approx(top - m);
                acc.x *= f, acc.y *= f, acc.z *= f, acc.w *= f;
                l = l * f + exp2_approx(z - m);
                top = m;
            }
            const float inv = l == 0.f ? 0.f : 1.f / l, f = inv * p.scales[1];                 // a row that sees nothing gives zeros
            *reinterpret_cast<uint2*>(reinterpret_cast<T*>(p.out) + row * D + d) = make_uint2(Cvt<T>::pack2(acc.x * f, acc.y * f), Cvt<T>::pack2(acc.z * f, acc.w * f));
            if (p.stat && d == 0) *reinterpret_cast<float2*>(p.stat + row * 2) = make_float2(top, inv);
        }
    }
}

// One warp per (row, head): the splits' parts joined in their order.
template <typename T, int D>
__global__ void __launch_bounds__(128) attention_fp4_merge_kernel(const Fp4AttnParams p) {
    pdl_prologue();
    const long long row = (blockIdx.x * (long long)blockDim.x + threadIdx.x) >> 5;
    const int lane = threadIdx.x & 31;
    if (row >= (long long)p.tokens * p.hq) return;
    const int h = (int)(row % p.hq);
    const float* ml = p.part_ml + (size_t)row * p.splits * 2;
    const float z = p.sinks ? p.sinks[h] * 1.4426950408889634f : kRefStart;
    float top = z;
    for (int s = lane; s < p.splits; s += 32) top = fmaxf(top, ml[2 * s]);
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
    constexpr int E = D / 32;
    float acc[E], l = p.sinks ? exp2_approx(z - top) : 0.f;
#pragma unroll
    for (int i = 0; i < E; ++i) acc[i] = 0.f;
    for (int s = 0; s < p.splits; ++s) {
        const float f = exp2_approx(ml[2 * s] - top);
        l += f * ml[2 * s + 1];
        const float* src = p.part_o + ((size_t)row * p.splits + s) * D + lane * E;
#pragma unroll
        for (int i = 0; i < E; ++i) acc[i] += f * src[i];
    }
    const float inv = l == 0.f ? 0.f : 1.f / l, f = inv * p.scales[1];
    T* dst = reinterpret_cast<T*>(p.out) + (size_t)row * D + lane * E;
#pragma unroll
    for (int i = 0; i < E; i += 2) *reinterpret_cast<uint32_t*>(dst + i) = Cvt<T>::pack2(acc[i] * f, acc[i + 1] * f);
    if (p.stat && lane == 0) *reinterpret_cast<float2*>(p.stat + (size_t)row * 2) = make_float2(top, inv);
}

// Accumulated attention weights: weights[page, head, slot] = decay * weights + the sum over the step's rows and the group's heads of
// exp2(score - top) / sum, for keys that some row sees; the step's own keys start from zero.  A warp owns its keys, so the sum has one order.
template <typename T, int D>
__global__ void __launch_bounds__(kFp4Warps * 32) attention_fp4_weights_kernel(const Fp4AttnParams p) {
    pdl_prologue();
    const int seq = blockIdx.z, kvh = blockIdx.y;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int group = p.hq / p.hkv, ql = p.q_len[seq], past = p.past_len[seq], columns = ql * group;
    if (columns == 0) return;
    const int q0 = p.q_start[seq];
    const int* table = p.page_table + (size_t)seq * p.max_pages;
    const size_t slab = fp4_slab_bytes(p.page_size, D);
    const int first = p.window > 0 ? max(0, past + 1 - p.window) : 0, end = past + ql;
    const int tile0 = first / kFp4Tile, tiles = (end + kFp4Tile - 1) / kFp4Tile - tile0;
    const int t_begin = tile0 + (int)((long long)tiles * blockIdx.x / p.splits), t_end = tile0 + (int)((long long)tiles * (blockIdx.x + 1) / p.splits);
    const float base = p.scale * 1.4426950408889634f * p.scales[0];
    for (int tile = t_begin + warp; tile < t_end; tile += kFp4Warps) {
        const int kb = tile * kFp4Tile;
        KeyTile<D> kt[2];
        int pages[2];
        float given[2][2] = {{0.f, 0.f}, {0.f, 0.f}};
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            const int k0 = kb + 16 * m, lp = k0 / p.page_size, at = k0 - lp * p.page_size;
            pages[m] = k0 < end && lp < p.max_pages ? table[lp] : -1;
            if ((unsigned)pages[m] >= (unsigned)p.num_pages) pages[m] = -1;
            const uint8_t* ks = p.pool + ((size_t)max(pages[m], 0) * 2 * p.hkv + kvh) * slab;
            kt[m].load(ks + (size_t)at * (D / 2), ks + (size_t)p.page_size * (D / 2) + (size_t)at * (D / 16), g, t);
        }
        for (int c0 = 0; c0 < columns; c0 += 8) {
            uint32_t qb[1][D / 16][2];
            const int c = c0 + g, r = c / group, h = kvh * group + c - r * group;
            const float up = load_query<T, D>(reinterpret_cast<const T*>(p.q) + ((size_t)(q0 + r) * p.hq + h) * D + t * (D / 4), c < columns, qb[0]);
            float factor[2], top[2], inv[2];
            int low[2], high[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                factor[i] = base * __shfl_sync(0xffffffffu, up, (2 * t + i) * 4);
                const int cc = c0 + 2 * t + i, rr = cc / group;
                const ColumnLimits lim(cc, columns, group, past, p.window);
                low[i] = lim.low;
                high[i] = lim.high;
                const float2 st = cc < columns ? *reinterpret_cast<const float2*>(p.stat + ((size_t)(q0 + rr) * p.hq + kvh * group + cc - rr * group) * 2)
                                               : make_float2(0.f, 0.f);
                top[i] = st.x;
                inv[i] = st.y;
            }
#pragma unroll
            for (int m = 0; m < 2; ++m) {
                float s[1][4];
                kt[m].template scores<1>(qb, s);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int key = kb + 16 * m + key_place(g) + 8 * (i >> 1);
                    if (key >= low[i & 1] && key < high[i & 1]) given[m][i >> 1] += exp2_approx(fmaf(s[0][i], factor[i & 1], -top[i & 1])) * inv[i & 1];
                }
            }
        }
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                given[m][r] += __shfl_xor_sync(0xffffffffu, given[m][r], 1);
                given[m][r] += __shfl_xor_sync(0xffffffffu, given[m][r], 2);
                const int key = kb + 16 * m + key_place(g) + 8 * r;
                if (t == 0 && pages[m] >= 0 && key >= first && key < end) {
                    float* w = p.weights + ((size_t)pages[m] * p.hkv + kvh) * p.page_size + key % p.page_size;
                    *w = (key >= past ? 0.f : p.decay * *w) + given[m][r];
                }
            }
    }
}

template <typename T, int D>
int launch_attention_fp4(const Fp4AttnParams& p, cudaStream_t stream) {
    const int columns = p.max_q_len * (p.hq / p.hkv);
    constexpr int kMost = D == 256 ? 1 : 2;
    const int nt = columns > 8 ? kMost : 1;
    const int chunks = (columns + 8 * nt - 1) / (8 * nt);
    if ((long long)chunks * p.hkv > 65535 || p.num_seqs > 65535) return fail("telb_paged_attention_fp4: too many sequences or columns");
    const int smem = kFp4Warps * 8 * nt * (D + 2) * 4;
    const dim3 grid(p.splits, chunks * p.hkv, p.num_seqs), blk(kFp4Warps * 32);
    if (nt == 1) {
        TELB_LAUNCH("attention_fp4_kernel", (attention_fp4_kernel<T, D, 1>), grid, blk, smem, stream, p);
    } else {
        TELB_LAUNCH("attention_fp4_kernel", (attention_fp4_kernel<T, D, kMost>), grid, blk, smem, stream, p);
    }
    if (p.splits > 1) {
        const long long rows = (long long)p.tokens * p.hq;
        TELB_LAUNCH("attention_fp4_merge_kernel", (attention_fp4_merge_kernel<T, D>), dim3((unsigned)((rows + 3) / 4)), dim3(128), 0, stream, p);
    }
    return 0;
}

template <typename T, int D>
int launch_weights_fp4(const Fp4AttnParams& p, cudaStream_t stream) {
    TELB_LAUNCH("attention_fp4_weights_kernel", (attention_fp4_weights_kernel<T, D>), dim3(p.splits, p.hkv, p.num_seqs), dim3(kFp4Warps * 32), 0, stream, p);
    return 0;
}

}  // namespace telb

using namespace telb;

// `weights` null: outputs only; else `stat` [tokens, hq, 2] is scratch and `weight_splits` parts of every sequence's keys run at once.
extern "C" int telb_paged_attention_fp4(const Fp4AttnParams* params, int d, int weight_splits, int is_bf16, cudaStream_t stream) {
    const Fp4AttnParams& p = *params;
    if (p.tokens <= 0 || p.num_seqs <= 0) return 0;
    if (d != 64 && d != 128 && d != 256) return fail("telb_paged_attention_fp4: head_dim must be 64, 128 or 256");
    if (p.page_size <= 0 || p.page_size % 16) return fail("telb_paged_attention_fp4: the page size must be a multiple of 16");
    if (p.hkv <= 0 || p.hq % p.hkv) return fail("telb_paged_attention_fp4: query heads must be a multiple of the KV heads");
    if (p.splits < 1 || (p.splits > 1 && (!p.part_o || !p.part_ml))) return fail("telb_paged_attention_fp4: splits without room for their parts");
    if (p.weights && (!p.stat || weight_splits < 1)) return fail("telb_paged_attention_fp4: weights without room for the softmax statistics");
    int rc;
    Fp4AttnParams w = p;
    w.splits = weight_splits;
#define ATTN_FP4(T, D) rc = launch_attention_fp4<T, D>(p, stream); if (rc == 0 && p.weights) rc = launch_weights_fp4<T, D>(w, stream)
    if (is_bf16) {
        if (d == 128) { ATTN_FP4(__nv_bfloat16, 128); }
        else if (d == 64) { ATTN_FP4(__nv_bfloat16, 64); }
        else { ATTN_FP4(__nv_bfloat16, 256); }
    } else {
        if (d == 128) { ATTN_FP4(__half, 128); }
        else if (d == 64) { ATTN_FP4(__half, 64); }
        else { ATTN_FP4(__half, 256); }
    }
    return rc;
}
