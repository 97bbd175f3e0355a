// Four-bit (NVFP4) cache pages: what writes them and what expands them.  The page layout is in kv_fp4_common.cuh.
//
//   rope_kv_write_fp4  per-head RMS norm and rotation of a step's queries and keys, and the step's keys and values quantised into the pages:
//                      a = max |r| over 16 features, s = e4m3(min(a / 6 / scale, 448)), code = e2m1(r / (s * scale)).  r is the 16-bit value
//                      that a 16-bit cache would hold.  The products of the rotation are rounded one by one and the sum of squares is taken
//                      in 64 bits, so that the codes, which jump at a border, are those of the formula and not of one order of additions.
//   kv_fp4_stage       16-bit pages of the cached rows of a step's sequences, for the prompt kernels.
#include <type_traits>

#include "host_utils.h"
#include "kv_fp4_common.cuh"

namespace telb {

struct Fp4WriteParams {
    const void* qkv;
    void* q_out;
    uint8_t* pool;
    const float* cos_sin;
    const int *positions, *seq_ids, *q_start, *past_len, *page_table, *kv_offsets;
    const void *q_norm, *k_norm;
    const float* scales;
    void* stage;
    const int* stage_table;
    int tokens, hq, hkv, rot, max_pos, page_size, max_pages, num_pages, stage_page, stage_max, stage_pages;
    double eps;                                                  // as the formula has it: in 32 bits it is off by 2^-26 of small rows' mean square
};

// 1 / sqrt(x), rounded to 32 bits from a value that two Newton steps in 64 bits have brought to some 2^-50; the full root where 32 bits cannot hold x.
__device__ __forceinline__ float inverse_root(double x) {
    const float f = (float)x;
    if (!(f > 1e-30f && f < 1e30f)) return (float)(1.0 / sqrt(x));
    double y = (double)rsqrtf(f);
    y = y * (1.5 - 0.5 * x * y * y);
    y = y * (1.5 - 0.5 * x * y * y);
    return (float)y;
}

// Eight values of a block of 16, whose other eight lie in the neighbouring lane: their codes, the block's scale byte and what the codes stand for.
// Quotients by a reciprocal and one correction (Markstein 1990) are rounded as a division rounds them, away from the ends of the range; the
// remainder is taken with the sign that leaves a zero its own.
__device__ __forceinline__ float quotient(float a, float b, float inv_b) {
    const float q = __fmul_rn(a, inv_b);
    return __fmaf_rn(-__fmaf_rn(q, b, -a), inv_b, q);
}
__device__ __forceinline__ bool middling(float x) { return x > 1e-18f && x < 1e18f; }

__device__ __forceinline__ uint32_t fp4_block_half(const float (&v)[8], float scale, float inv_scale, uint8_t& sf, float (&back)[8]) {
    uint32_t m = 0;                                             // the largest magnitude, compared as bit patterns so that a NaN stays one
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
    const float most = __uint_as_float(m);
    const bool plain = middling(most) && middling(scale);
    float want = plain ? quotient(quotient(most, 6.f, 1.f / 6.f), scale, inv_scale) : __fdiv_rn(__fdiv_rn(most, 6.f), scale);
    want = want > 448.f ? 448.f : want;
    sf = __nv_cvt_float_to_fp8(want, __NV_SATFINITE, __NV_E4M3);
    const float step = __fmul_rn(e4m3_to_float(sf), scale);
    float y[8];
    if (plain && middling(step)) {
        const float inv = __frcp_rn(step);
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = quotient(v[i], step, inv);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = step > 0.f ? __fdiv_rn(v[i], step) : v[i] != v[i] ? 0.f : copysignf(0.f, v[i]);
    }
    uint32_t codes = 0;
#pragma unroll
    for (int i = 0; i < 8; i += 2) codes |= e2m1_pair(y[i], y[i + 1]) << (4 * i);
    uint32_t h[4];
    e2m1x8_to_half(codes, h[0], h[1], h[2], h[3]);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
        back[2 * i] = __fmul_rn(f.x, step);
        back[2 * i + 1] = __fmul_rn(f.y, step);
    }
    return codes;
}

template <typename T>
__device__ __forceinline__ uint4 pack8(const float (&v)[8]) {
    return make_uint4(Cvt<T>::pack2(v[0], v[1]), Cvt<T>::pack2(v[2], v[3]), Cvt<T>::pack2(v[4], v[5]), Cvt<T>::pack2(v[6], v[7]));
}
template <typename T>
__device__ __forceinline__ void unpack8(const uint4& u, float (&v)[8]) {
    const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = Cvt<T>::to_f(e[i]);
}

// round(round(v * inv) * w), both to the 16-bit type: the second product of two 16-bit numbers rounds once, as it does from 32 bits.
template <typename T>
__device__ __forceinline__ void scale_rows(float (&v)[8], float inv, const uint4& w) {
    uint4 u = make_uint4(Cvt<T>::pack2(__fmul_rn(v[0], inv), __fmul_rn(v[1], inv)), Cvt<T>::pack2(__fmul_rn(v[2], inv), __fmul_rn(v[3], inv)),
                         Cvt<T>::pack2(__fmul_rn(v[4], inv), __fmul_rn(v[5], inv)), Cvt<T>::pack2(__fmul_rn(v[6], inv), __fmul_rn(v[7], inv)));
    using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
    T2* a = reinterpret_cast<T2*>(&u);
    const T2* b = reinterpret_cast<const T2*>(&w);
#pragma unroll
    for (int i = 0; i < 4; ++i) a[i] = __hmul2_rn(a[i], b[i]);
    unpack8<T>(u, v);
}

// Whole heads turn: D/16 lanes a head, a lane holds features 8 l .. and D/2 + 8 l .., which turn together; a warp takes every `parts`-th group of 512 / D heads
// of a token, whose cos / sin row, norm weights and page look-up it fetches once.  A long prompt is bound by the arithmetic of the exact codes beside the
// traffic: 8129 rows of 32 / 8 heads of 128, 16-bit copies too, 52 us (0.63 of the copy rate); 64 rows take 5.5 us, the latency of one row.
template <typename T, int D>
__global__ void __launch_bounds__(128, 6) rope_kv_write_fp4_kernel(const Fp4WriteParams p, int parts) {
    pdl_prologue();
    constexpr int L = D / 16, H = 32 / L;                       // lanes of a head, heads of a warp
    const int unit = (int)((blockIdx.x * (long long)blockDim.x + threadIdx.x) >> 5);
    const int t = unit / parts, part = unit - t * parts, lane = threadIdx.x & 31, l = lane % L, hh = lane / L;
    if (t >= p.tokens) return;
    const int heads = p.hq + 2 * p.hkv, groups = (heads + H - 1) / H;
    const T* row = reinterpret_cast<const T*>(p.qkv) + (size_t)t * heads * D;
    uint4 next[2];
    auto fetch = [&](int grp) {
        const int h = min(grp * H + hh, heads - 1);
        const T* src = row + (size_t)h * D + 8 * l;
        next[0] = *reinterpret_cast<const uint4*>(src);
        next[1] = *reinterpret_cast<const uint4*>(src + D / 2);
    };
    fetch(part);
    float c[8], sn[8];
    {
        const float* cs = p.cos_sin + (size_t)min(max(p.positions[t], 0), p.max_pos - 1) * D + 8 * l;
        *reinterpret_cast<float4*>(c) = *reinterpret_cast<const float4*>(cs);
        *reinterpret_cast<float4*>(c + 4) = *reinterpret_cast<const float4*>(cs + 4);
        *reinterpret_cast<float4*>(sn) = *reinterpret_cast<const float4*>(cs + D / 2);
        *reinterpret_cast<float4*>(sn + 4) = *reinterpret_cast<const float4*>(cs + D / 2 + 4);
    }
    const int s = p.seq_ids[t];
    const int slot = p.past_len[s] + (p.kv_offsets ? p.kv_offsets[t] : t - p.q_start[s]);
    const int lp = slot / p.page_size, at = slot - lp * p.page_size;
    const int page = slot >= 0 && lp < p.max_pages ? p.page_table[(size_t)s * p.max_pages + lp] : -1;
    int sp = -1, stage_at = 0;
    if (p.stage) {
        const int sl = slot / p.stage_page;
        stage_at = slot - sl * p.stage_page;
        sp = slot >= 0 && sl < p.stage_max ? p.stage_table[(size_t)s * p.stage_max + sl] : -1;
    }
    const float scale_k = p.scales[0], scale_v = p.scales[1], inv_k = __frcp_rn(scale_k), inv_v = __frcp_rn(scale_v);
    for (int grp = part; grp < groups; grp += parts) {
        const int h = grp * H + hh;
        float lo[8], hi[8];
        unpack8<T>(next[0], lo);
        unpack8<T>(next[1], hi);
        if (grp + parts < groups) fetch(grp + parts);
        const bool is_q = h < p.hq, is_v = h >= p.hq + p.hkv;
        const bool norm = is_q ? p.q_norm != nullptr : !is_v && p.k_norm != nullptr;
        if (__any_sync(0xffffffffu, norm)) {
            double ss = 0.0;
#pragma unroll
            for (int i = 0; i < 8; ++i) ss += (double)lo[i] * (double)lo[i] + (double)hi[i] * (double)hi[i];
#pragma unroll
            for (int o = L / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
            if (norm) {
                const float inv = inverse_root(ss / D + p.eps);
                const T* nw = reinterpret_cast<const T*>(is_q ? p.q_norm : p.k_norm) + 8 * l;
                scale_rows<T>(lo, inv, *reinterpret_cast<const uint4*>(nw));
                scale_rows<T>(hi, inv, *reinterpret_cast<const uint4*>(nw + D / 2));
            }
        }
        if (!is_v) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float a = lo[i], b = hi[i];
                lo[i] = __fsub_rn(__fmul_rn(a, c[i]), __fmul_rn(b, sn[i]));
                hi[i] = __fadd_rn(__fmul_rn(b, c[i]), __fmul_rn(a, sn[i]));
            }
        }
        const uint4 plo = pack8<T>(lo), phi = pack8<T>(hi);
        if (is_q) {
            T* dst = reinterpret_cast<T*>(p.q_out) + ((size_t)t * p.hq + h) * D + 8 * l;
            *reinterpret_cast<uint4*>(dst) = plo;
            *reinterpret_cast<uint4*>(dst + D / 2) = phi;
        }
        if (__all_sync(0xffffffffu, is_q)) continue;
        unpack8<T>(plo, lo);                                    // what a 16-bit cache would hold
        unpack8<T>(phi, hi);
        uint8_t sf[2];
        float back[2][8];
        const uint32_t codes_lo = fp4_block_half(lo, is_v ? scale_v : scale_k, is_v ? inv_v : inv_k, sf[0], back[0]);
        const uint32_t codes_hi = fp4_block_half(hi, is_v ? scale_v : scale_k, is_v ? inv_v : inv_k, sf[1], back[1]);
        if (is_q || h >= heads) continue;
        const int head = is_v ? h - p.hq - p.hkv : h - p.hq;
        if ((unsigned)page < (unsigned)p.num_pages) {           // else: a row that has no page is not stored
            uint8_t* slab = p.pool + (((size_t)page * 2 + is_v) * p.hkv + head) * fp4_slab_bytes(p.page_size, D);
            uint8_t* dst = slab + (size_t)at * (D / 2) + 4 * l;
            *reinterpret_cast<uint32_t*>(dst) = codes_lo;
            *reinterpret_cast<uint32_t*>(dst + D / 4) = codes_hi;
            if (!(l & 1)) {
                uint8_t* f = slab + (size_t)p.page_size * (D / 2) + (size_t)at * (D / 16) + l / 2;
                f[0] = sf[0];
                f[D / 32] = sf[1];
            }
        }
        if ((unsigned)sp < (unsigned)p.stage_pages) {
            T* dst = reinterpret_cast<T*>(p.stage) + ((((size_t)sp * 2 + is_v) * p.hkv + head) * p.stage_page + stage_at) * D + 8 * l;
#pragma unroll
            for (int i = 0; i < 8; ++i) back[0][i] = fp4_bound<T>(back[0][i]), back[1][i] = fp4_bound<T>(back[1][i]);
            *reinterpret_cast<uint4*>(dst) = pack8<T>(back[0]);
            *reinterpret_cast<uint4*>(dst + D / 2) = pack8<T>(back[1]);
        }
    }
}

// A part of a head turns: one warp per (token, head); a lane holds E neighbouring features, with true divisions and 64-bit roots for every head.  Rows of 32 / 8 heads
// of 128, half of each turning: 64 rows 3.9 us, 500 10.9, 8129 132 (whole heads 3.5, 6.8, 47): bound by that arithmetic, 2.8 times the form above.
template <typename T, int D>
__global__ void __launch_bounds__(256) rope_part_kv_write_fp4_kernel(const Fp4WriteParams p) {
    pdl_prologue();
    constexpr int E = D / 32, kLanes = 16 / E;                 // lanes of a block of 16 features
    const int heads = p.hq + 2 * p.hkv;
    const long long wid = (blockIdx.x * (long long)blockDim.x + threadIdx.x) >> 5;
    const int lane = threadIdx.x & 31;
    if (wid >= (long long)p.tokens * heads) return;
    const int t = (int)(wid / heads), h = (int)(wid - (long long)t * heads);
    const bool is_q = h < p.hq, is_v = h >= p.hq + p.hkv;
    alignas(16) T x[E];
    {
        const T* src = reinterpret_cast<const T*>(p.qkv) + ((size_t)t * heads + h) * D + lane * E;
        if constexpr (E == 2) *reinterpret_cast<uint32_t*>(x) = *reinterpret_cast<const uint32_t*>(src);
        else if constexpr (E == 4) *reinterpret_cast<uint2*>(x) = *reinterpret_cast<const uint2*>(src);
        else *reinterpret_cast<uint4*>(x) = *reinterpret_cast<const uint4*>(src);
    }
    const T* nw = reinterpret_cast<const T*>(is_q ? p.q_norm : is_v ? nullptr : p.k_norm);
    if (nw) {
        double ss = 0.0;
#pragma unroll
        for (int i = 0; i < E; ++i) ss += (double)Cvt<T>::to_f(x[i]) * (double)Cvt<T>::to_f(x[i]);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        const float inv = (float)(1.0 / sqrt(ss / D + p.eps));
#pragma unroll
        for (int i = 0; i < E; ++i)
            x[i] = Cvt<T>::from_f(__fmul_rn(Cvt<T>::to_f(Cvt<T>::from_f(__fmul_rn(Cvt<T>::to_f(x[i]), inv))), Cvt<T>::to_f(nw[lane * E + i])));
    }
    if (!is_v) {
        // features i and i + rot / 2 turn together; rot is a multiple of 2 E, so the other one is at the same place of another lane
        const int half = p.rot / 2, step = half / E, d0 = lane * E;
        const bool turns = d0 < p.rot, low = d0 < half;
        const int other = !turns ? lane : low ? lane + step : lane - step;
        const float* cs = p.cos_sin + (size_t)min(max(p.positions[t], 0), p.max_pos - 1) * p.rot + (low ? d0 : d0 - half);
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const float a = Cvt<T>::to_f(x[i]);
            const float b = __shfl_sync(0xffffffffu, a, other);
            if (turns) {
                const float c = cs[i], s = cs[half + i];
                x[i] = Cvt<T>::from_f(low ? __fsub_rn(__fmul_rn(a, c), __fmul_rn(b, s)) : __fadd_rn(__fmul_rn(a, c), __fmul_rn(b, s)));
            }
        }
    }
    auto put = [&](T* dst) {
        if constexpr (E == 2) *reinterpret_cast<uint32_t*>(dst) = *reinterpret_cast<const uint32_t*>(x);
        else if constexpr (E == 4) *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<const uint2*>(x);
        else *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(x);
    };
    if (is_q) {
        put(reinterpret_cast<T*>(p.q_out) + ((size_t)t * p.hq + h) * D + lane * E);
        return;
    }
    const int s = p.seq_ids[t];
    const int slot = p.past_len[s] + (p.kv_offsets ? p.kv_offsets[t] : t - p.q_start[s]);
    const int lp = slot / p.page_size, at = slot - lp * p.page_size;
    const int page = slot >= 0 && lp < p.max_pages ? p.page_table[(size_t)s * p.max_pages + lp] : -1;
    const int head = is_v ? h - p.hq - p.hkv : h - p.hq;
    const float scale = p.scales[is_v];
    // the largest magnitude of the block, compared as bit patterns so that a NaN stays one
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < E; ++i) m = max(m, __float_as_uint(Cvt<T>::to_f(x[i])) & 0x7fffffffu);
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    float want = __fdiv_rn(__fdiv_rn(__uint_as_float(m), 6.f), scale);
    want = want > 448.f ? 448.f : want;
    const uint8_t sf = __nv_cvt_float_to_fp8(want, __NV_SATFINITE, __NV_E4M3);
    const float step = __fmul_rn(e4m3_to_float(sf), scale);
    uint32_t codes = 0;
    float back[E];
#pragma unroll
    for (int i = 0; i < E; i += 2) {
        float y[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const float v = Cvt<T>::to_f(x[i + j]);
            y[j] = step > 0.f ? __fdiv_rn(v, step) : v != v ? 0.f : copysignf(0.f, v);
        }
        const uint32_t c = e2m1_pair(y[0], y[1]);
        codes |= c << (4 * i);
        uint32_t hb;
        asm("{\n\t.reg .b8 b, z;\n\tmov.b16 {b, z}, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, b;\n\t}" : "=r"(hb) : "h"((uint16_t)c));
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&hb));
        back[i] = __fmul_rn(f.x, step);
        back[i + 1] = __fmul_rn(f.y, step);
    }
    if ((unsigned)page < (unsigned)p.num_pages) {              // else: a row that has no page is not stored
        uint8_t* slab = p.pool + (((size_t)page * 2 + is_v) * p.hkv + head) * fp4_slab_bytes(p.page_size, D);
        uint8_t* row = slab + (size_t)at * (D / 2) + lane * (E / 2);
        if constexpr (E == 2) *row = (uint8_t)codes;
        else if constexpr (E == 4) *reinterpret_cast<uint16_t*>(row) = (uint16_t)codes;
        else *reinterpret_cast<uint32_t*>(row) = codes;
        if (lane % kLanes == 0) slab[(size_t)p.page_size * (D / 2) + (size_t)at * (D / 16) + lane / kLanes] = sf;
    }
    if (p.stage) {
        const int sl = slot / p.stage_page;
        const int sp = slot >= 0 && sl < p.stage_max ? p.stage_table[(size_t)s * p.stage_max + sl] : -1;
        if ((unsigned)sp >= (unsigned)p.stage_pages) return;
#pragma unroll
        for (int i = 0; i < E; ++i) x[i] = fp4_round<T>(back[i]);
        put(reinterpret_cast<T*>(p.stage) + ((((size_t)sp * 2 + is_v) * p.hkv + head) * p.stage_page + slot - sl * p.stage_page) * D + lane * E);
    }
}

// Pages of 64 rows that a sequence takes in a packed copy: whole 128-key tiles, one at least.
__device__ __forceinline__ int fp4_stage_own(int total, int most) { return min(2 * max(1, (total + 127) / 128), most); }

// A CTA per page of the 16-bit copy (64 rows; page blockIdx.x, plane (K|V, head) blockIdx.y); a thread expands blocks of 16 features.  Packed, the sequences'
// pages follow one another, and the last page of the copy is zeros for what the table has behind a sequence's own pages; else every sequence has
// `stage_pages`, and those behind its last 128-key tile, which no kernel reads, are left as they are.  Bound by the bytes, and the launch where they are few:
// 8 sequences of 1024 rows of 8 heads of 128 10.4 us (43 MB, 0.63 of the copy rate); 63 of 1024 beside one of 32768 109 us (packed; 432 MB written, and the
// search for a page's sequence, which costs 0.5 us of a small step), 2125 with every sequence as long as the longest.  The step's own rows are left out unless `own`; rows behind them, up to the page's end, become zero, and so do those that a window hides from
// every row, whose values enter the product of a tile times a probability of zero.  holes[seq, lp] says which of a page's
// four groups of 16 rows the cache does not have: their zeros must not be taken for keys.
template <typename T, int D>
__global__ void __launch_bounds__(256) kv_fp4_stage_kernel(const uint8_t* __restrict__ pool, T* __restrict__ stage, int* __restrict__ stage_table, uint8_t* __restrict__ holes,
                                                           const int* __restrict__ past_len, const int* __restrict__ q_len, const int* __restrict__ page_table,
                                                           const float* __restrict__ scales, int num_seqs, int max_pages, int num_pages, int page_shift, int stage_pages,
                                                           int packed, int hkv, int window, int own) {
    pdl_prologue();
    const int at_page = blockIdx.x, plane = blockIdx.y, lane = threadIdx.x & 31;
    T* dst = stage + ((size_t)at_page * 2 * hkv + plane) * 64 * D;
    constexpr int B = D / 16;
    int seq = at_page / stage_pages, lp = at_page - seq * stage_pages;
    if (packed) {                                               // every warp finds the page's sequence for itself
        int base = 0;
        seq = -1;
        for (int s0 = 0; s0 < num_seqs && seq < 0; s0 += 32) {
            const int n = s0 + lane < num_seqs ? fp4_stage_own(past_len[s0 + lane] + q_len[s0 + lane], stage_pages) : 0;
            int incl = n;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o) incl += v;
            }
            const unsigned here = __ballot_sync(0xffffffffu, at_page < base + incl);
            if (here) {
                const int l = __ffs(here) - 1;
                seq = s0 + l;
                lp = at_page - base - __shfl_sync(0xffffffffu, incl - n, l);
            }
            base += __shfl_sync(0xffffffffu, incl, 31);
        }
        if (seq < 0) {                                          // behind all sequences
            for (int i = threadIdx.x; i < 64 * D / 8; i += 256) reinterpret_cast<uint4*>(dst)[i] = make_uint4(0, 0, 0, 0);
            return;
        }
        if (lp == 0 && plane == 0)
            for (int i = fp4_stage_own(past_len[seq] + q_len[seq], stage_pages) + threadIdx.x; i < stage_pages; i += 256) {
                stage_table[seq * stage_pages + i] = (int)gridDim.x - 1;
                holes[seq * stage_pages + i] = 0;
            }
    }
    if (plane == 0 && threadIdx.x == 0) stage_table[seq * stage_pages + lp] = at_page;
    const int past = past_len[seq], total = past + q_len[seq], count = own ? total : past;
    if (plane == 0 && threadIdx.x < 32) {
        const int slot = lp * 64 + 16 * threadIdx.x, at = slot >> page_shift;
        const int page = threadIdx.x < 4 && slot < total && at < max_pages ? page_table[(size_t)seq * max_pages + at] : -1;
        const unsigned gone = __ballot_sync(0xffffffffu, threadIdx.x < 4 && slot < total && (unsigned)page >= (unsigned)num_pages);
        if (threadIdx.x == 0) holes[seq * stage_pages + lp] = (uint8_t)gone;
    }
    if (lp >= fp4_stage_own(total, stage_pages)) return;
    if (window > 0 && (lp + 1) * 64 + 2 * 128 <= past - window) return;        // before every tile that the windowed kernels touch
    const int first = window > 0 ? past + 1 - window : 0;
    const size_t slab = fp4_slab_bytes(1 << page_shift, D);
    const float scale = scales ? scales[plane >= hkv] : 1.f;
#pragma unroll
    for (int u = 0; u < 64 * B / 256; ++u) {
        const int i = u * 256 + threadIdx.x, r = i / B, b = i % B, slot = lp * 64 + r;
        if (slot >= count && slot < total) continue;
        const int page = slot >= first && slot < count && slot >> page_shift < max_pages ? page_table[(size_t)seq * max_pages + (slot >> page_shift)] : -1;
        uint4 out[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
        if ((unsigned)page < (unsigned)num_pages) {
            const uint8_t* src = pool + ((size_t)page * 2 * hkv + plane) * slab;
            const int at = slot & ((1 << page_shift) - 1);
            const uint2 w = *reinterpret_cast<const uint2*>(src + (size_t)at * (D / 2) + b * 8);
            const float step = __fmul_rn(e4m3_to_float(src[((size_t)(D / 2) << page_shift) + (size_t)at * B + b]), scale);
            uint32_t h[8];
            e2m1x8_to_half(w.x, h[0], h[1], h[2], h[3]);
            e2m1x8_to_half(w.y, h[4], h[5], h[6], h[7]);
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                float v[8];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[4 * half + j]));
                    v[2 * j] = fp4_bound<T>(__fmul_rn(f.x, step));
                    v[2 * j + 1] = fp4_bound<T>(__fmul_rn(f.y, step));
                }
                out[half] = pack8<T>(v);
            }
        }
        *reinterpret_cast<uint4*>(dst + (size_t)r * D + b * 16) = out[0];
        *reinterpret_cast<uint4*>(dst + (size_t)r * D + b * 16 + 8) = out[1];
    }
}

// Rows of accepted draft tokens move together: the row at slot past + path[j] to past + j, j from 1, of every layer, plane and head.  All words of a row
// (codes, then block scales) are read before any is written.  Four rows of 8 heads of 128 in 36 layers: 8 sequences 12.9 us, 64 90 us (latency of a block's
// look-ups, page table and path, in several waves of blocks).
constexpr int kCommitWords = 12;                                // of a thread
template <int D>
__global__ void __launch_bounds__(256) kv_fp4_commit_path_kernel(uint8_t* __restrict__ pool, const int* __restrict__ page_table, const int* __restrict__ past_len,
                                                                 const int* __restrict__ path, const int* __restrict__ path_len, int max_path, int max_pages,
                                                                 int num_pages, int hkv, int page_size) {
    pdl_prologue();
    constexpr int kCodes = D / 8, kWords = kCodes + D / 64;     // 32-bit words of a row: codes, all
    const int b = blockIdx.x, head = blockIdx.y % hkv, plane = blockIdx.y / hkv;       // plane: layer * 2 + (K|V)
    const int m = min(path_len[b], max_path) - 1;               // rows to move (path[0] is the root and stays)
    if (m <= 0) return;
    const int past = past_len[b];
    const size_t slab = fp4_slab_bytes(page_size, D);
    auto word_at = [&](int slot, int w) -> uint32_t* {
        const int lp = slot / page_size, page = slot >= 0 && lp < max_pages ? page_table[(size_t)b * max_pages + lp] : -1, at = slot - lp * page_size;
        if ((unsigned)page >= (unsigned)num_pages) return nullptr;
        uint8_t* s = pool + ((((size_t)(plane >> 1) * num_pages + page) * 2 + (plane & 1)) * hkv + head) * slab;
        return reinterpret_cast<uint32_t*>(w < kCodes ? s + (size_t)at * (D / 2) + w * 4 : s + (size_t)page_size * (D / 2) + (size_t)at * (D / 16) + (w - kCodes) * 4);
    };
    uint32_t v[kCommitWords];
    const int total = m * kWords;
#pragma unroll
    for (int i = 0; i < kCommitWords; ++i) {
        const int x = threadIdx.x + i * 256, j = x / kWords + 1, w = x % kWords;
        const uint32_t* src = x < total ? word_at(past + path[(size_t)b * max_path + j], w) : nullptr;
        v[i] = src ? *src : 0u;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kCommitWords; ++i) {
        const int x = threadIdx.x + i * 256, j = x / kWords + 1, w = x % kWords;
        uint32_t* dst = x < total ? word_at(past + j, w) : nullptr;
        if (dst) *dst = v[i];
    }
}

}  // namespace telb

using namespace telb;

extern "C" int telb_rope_kv_write_fp4(const Fp4WriteParams* params, int d, int is_bf16, cudaStream_t stream) {
    const Fp4WriteParams& p = *params;
    if (p.tokens <= 0) return 0;
    if (d != 64 && d != 128 && d != 256) return fail("telb_rope_kv_write_fp4: head_dim must be 64, 128 or 256");
    if (p.rot < 0 || p.rot > d || p.rot % (d / 16)) return fail("telb_rope_kv_write_fp4: the rotated part must be a multiple of head_dim / 16");
    if (p.rot == d) {
        // A warp for all heads of a token where that fills the device, else several, up to one for every group of heads.  32 / 8 heads of 128, 1, 2, 4, 12
        // warps a token (us): 64 tokens 11.6, 7.7, 5.9, 4.8; 500: 12.1, 8.7, 8.2, 8.1; 2000: 21, 19, 19, 24; 8129: 51, 52, 59, 85.
        const int groups = (p.hq + 2 * p.hkv + 512 / d - 1) / (512 / d);
        const int parts = (int)min((long long)groups, max(1LL, (16LL * 4 * sm_count() + p.tokens - 1) / p.tokens));
        const long long warps = (long long)p.tokens * parts;
        const dim3 grid((unsigned)((warps + 3) / 4)), blk(128);
#define WRITE_FP4(T, D) TELB_LAUNCH("rope_kv_write_fp4_kernel", (rope_kv_write_fp4_kernel<T, D>), grid, blk, 0, stream, p, parts)
        if (is_bf16) {
            if (d == 128) WRITE_FP4(__nv_bfloat16, 128);
            else if (d == 64) WRITE_FP4(__nv_bfloat16, 64);
            else WRITE_FP4(__nv_bfloat16, 256);
        } else {
            if (d == 128) WRITE_FP4(__half, 128);
            else if (d == 64) WRITE_FP4(__half, 64);
            else WRITE_FP4(__half, 256);
        }
#undef WRITE_FP4
        return 0;
    }
    const long long warps = (long long)p.tokens * (p.hq + 2 * p.hkv);
    const dim3 grid((unsigned)((warps + 7) / 8)), blk(256);
#define WRITE_FP4(T, D) TELB_LAUNCH("rope_part_kv_write_fp4_kernel", (rope_part_kv_write_fp4_kernel<T, D>), grid, blk, 0, stream, p)
    if (is_bf16) {
        if (d == 128) WRITE_FP4(__nv_bfloat16, 128);
        else if (d == 64) WRITE_FP4(__nv_bfloat16, 64);
        else WRITE_FP4(__nv_bfloat16, 256);
    } else {
        if (d == 128) WRITE_FP4(__half, 128);
        else if (d == 64) WRITE_FP4(__half, 64);
        else WRITE_FP4(__half, 256);
    }
#undef WRITE_FP4
    return 0;
}

// pool: one layer; stage_table [num_seqs, stage_pages] is filled in; stage: 16-bit [stage_total, 2, Hkv, 64, d], the sequences' pages of 64 rows packed (`packed`: stage_total
// is one more than the sum of max(1, ceil(rows / 128)) * 2 over the sequences) or num_seqs * stage_pages of them; holes [num_seqs, stage_pages] bytes: bit i is set where the rows 16 i .. 16 i + 15 of a page have no page of the pool.  own: the step's own
// rows too.  `scales` null: code * block scale, which both 16-bit types hold exactly.
extern "C" int telb_kv_fp4_stage(const void* pool, void* stage, int* stage_table, uint8_t* holes, const int* past_len, const int* q_len, const int* page_table, const float* scales,
                                 int num_seqs, int max_pages, int num_pages, int page_size, int stage_pages, int stage_total, int packed, int hkv, int d, int window,
                                 int own, int is_bf16, cudaStream_t stream) {
    if (num_seqs <= 0 || stage_pages <= 0 || stage_total <= 0) return 0;
    if (!packed && (long long)num_seqs * stage_pages != stage_total) return fail("telb_kv_fp4_stage: pages of another number");
    if (d != 64 && d != 128 && d != 256) return fail("telb_kv_fp4_stage: head_dim must be 64, 128 or 256");
    if (page_size < 16 || page_size & (page_size - 1)) return fail("telb_kv_fp4_stage: the page size must be a power of two, at least 16");
    if (2 * hkv > 65535) return fail("telb_kv_fp4_stage: more than 65535 planes");
    int shift = 0;
    while (1 << shift < page_size) ++shift;
    const dim3 grid(stage_total, 2 * hkv), blk(256);
#define STAGE_FP4(T, D) TELB_LAUNCH("kv_fp4_stage_kernel", (kv_fp4_stage_kernel<T, D>), grid, blk, 0, stream, (const uint8_t*)pool, (T*)stage, stage_table, holes, past_len, q_len, \
                                    page_table, scales, num_seqs, max_pages, num_pages, shift, stage_pages, packed, hkv, window, own)
    if (is_bf16) {
        if (d == 128) STAGE_FP4(__nv_bfloat16, 128);
        else if (d == 64) STAGE_FP4(__nv_bfloat16, 64);
        else STAGE_FP4(__nv_bfloat16, 256);
    } else {
        if (d == 128) STAGE_FP4(__half, 128);
        else if (d == 64) STAGE_FP4(__half, 64);
        else STAGE_FP4(__half, 256);
    }
#undef STAGE_FP4
    return 0;
}

// pool: all layers [layers, num_pages, 2, hkv, slab].
extern "C" int telb_kv_fp4_commit_path(void* pool, const int* page_table, const int* past_len, const int* path, const int* path_len, int batch, int max_path,
                                       int max_pages, int layers, int num_pages, int hkv, int page_size, int d, cudaStream_t stream) {
    if (batch <= 0 || layers <= 0) return 0;
    if (d != 64 && d != 128 && d != 256) return fail("telb_kv_fp4_commit_path: head_dim must be 64, 128 or 256");
    if ((max_path - 1) * (d / 8 + d / 64) > 256 * kCommitWords) return fail("telb_kv_fp4_commit_path: accepted path too long for one block");
    if (2LL * layers * hkv > 65535) return fail("telb_kv_fp4_commit_path: more than 65535 planes");
    const dim3 grid(batch, layers * 2 * hkv), blk(256);
#define COMMIT_FP4(D) TELB_LAUNCH("kv_fp4_commit_path_kernel", (kv_fp4_commit_path_kernel<D>), grid, blk, 0, stream, (uint8_t*)pool, page_table, past_len, path, path_len, \
                                  max_path, max_pages, num_pages, hkv, page_size)
    if (d == 128) COMMIT_FP4(128);
    else if (d == 64) COMMIT_FP4(64);
    else COMMIT_FP4(256);
#undef COMMIT_FP4
    return 0;
}
