// i4d_kv8_attn.cuh -- attention over the cache of 8-bit codes.
//
// k_kv8_attn: eight (or sixteen) query rows of one cache head against a chunk
// of its tokens.  Each warp takes tiles of 16 tokens, which tensor copies
// bring into a ring of its own in shared memory, two tiles ahead, so no warp
// waits for another before the end (2 KB tensor copies stream at 6.7 TB/s
// where 16-byte asynchronous copies stopped at 5.1; 812 MB of codes).  The
// order of the summation index of a matrix instruction is free, so a thread's
// 16 contiguous codes of a token serve as its part of four steps of K q, and a
// V^T tile takes the codes of the four tokens whose probabilities the thread
// holds: codes go from shared memory to registers in 16-byte pieces without a
// transposition, and the copies' 128-byte swizzle keeps the banks apart.  The
// products are transposed (tokens x rows, then dims x rows), which wastes half
// as much of a 16 x 8 tile on few rows.
//   scores   S^T [16 tokens x 8 rows] = K [16 x dim] Q^T     (m16n8k16, FP16 in, FP32 sums)
//   output   O^T [16 dims x 8 rows]  += V^T [16 x 16 tokens] P^T
// Every code is exact in FP16.  A query row is scaled by a power of two into
// FP16's range, which is exact for BF16 and FP16 rows up to 2^-39 of the row's
// largest value; FP32 rows are split in two FP16 parts (2^-22).  A weight goes to
// FP16 in one part (2^-11 of it at most, an eighth of a BF16 output's rounding);
// for FP16 outputs in two (2^-22, but not less than 2^-34 of the row's greatest
// weight), for FP32 outputs in two of which the second is scaled (2^-22).
// Weights under 2^-23 of the greatest go in again, 2^24 times, so that they are
// right where the greatest ones meet codes of 0; under 2^-95 they are 0.
//
// One pass over the tokens: M is a bound of the scores so far (in powers of
// two), l the sum of 2^(x - M), R a bound of x + log2(v_scale): the values
// that enter the second product are 2^(x - R) v_scale, so a block whose scale
// is far above the others' costs the others no bits unless it outweighs them.
// M and R are raised only when a score passes them by more than 2^6 (R lies 2^9
// under the greatest, FP16 holds 2^15), so most tiles do without the reduction
// over lanes; the vote that asks for it asks for small weights too (which
// costs 24 ragged contexts 3 %, three rows a sequence 6 %, FP32 rows of 256
// 10 %).
// Bound: the codes of K and V, read once (24 contexts of 301 to 32749 tokens,
// 8 heads of 128, 812 MB of INT8 codes: 173 to 178 us, 4.7 TB/s; the same copies
// without arithmetic 133 us).
#pragma once

#include <cuda.h>

#include "i4d_kv8_cache.cuh"
#include "i4d_ring.h"

namespace i4d_ops {

constexpr int kAttnThreads = 128;
constexpr int kAttnWarps = 4;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kSlack = 6.f;
// R lies this far under the greatest x + log2(v_scale): a weight is at most
// 2^(kHead + kSlack) in FP16, which keeps its precision down to 2^-14.
constexpr float kHead = 9.f;
constexpr float kSmallWeight = 0x1p-14f;
constexpr float kSmallStep = 0x1p24f, kSmallMost = 0x1p72f;  // (sums reach 2^54: 2^28 tokens a warp, weights under 2^16, codes under 2^9)
// R stays above M - 126, so 2^(M - R) and 2^(R - M) are normal numbers.  Less
// would be needed only where a row has seen nothing but value scales under
// 2^-126, or of 0.
constexpr float kFarScales = 126.f;

struct AttnDev {
    CUtensorMap maps[2];  // K, V codes as rows of dim bytes; boxes of 16 rows x 128 (dim <= 64: 64) bytes
    Kv8Dev cache;
    SeqArrays seq;
    const void* q;
    void* out;
    float* lse;
    float* weights;
    int64_t q_tok, q_head, out_tok, out_head, weights_stride;
    int heads, group, window, dtype, max_length, wide_q, wide_out;
    float scale_log2;  // softmax scale * log2(e)
    int batch, row_tiles;  // row tiles of a (sequence, cache head), at most
    int even;              // CTAs that share the tokens evenly, or 0: a cluster for each (sequence, cache head, row tile)
    int cluster;           // its CTAs, which share the segment's tokens and join through distributed shared memory
    float* part;       // workspace: [even][2][rows][dim]: O of a CTA's pieces that are not whole
    float4* stats;     // workspace: [even][2][rows]: M, l, R
    float* lse2;       // workspace: [tokens][heads], log2 of the softmax sum (with weights)
    int4* segments;    // workspace: [segment]: first and last CTA of its pieces, slot of the first
    float* scores;     // workspace (few rows, with weights): [segment][rows][score_stride], log2 scale
    int64_t score_stride;  // a multiple of 4
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ uint32_t pack_h2(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// Codes to halves.  INT8 with BIAS: byte v + 128 as the low byte of a half, a
// subnormal worth (v + 128) 2^-24, which the tensor cores take exactly; the
// 128 leaves again as 128 times the sum of the query row.  That is half the
// instructions of an exact conversion, for a sum whose terms are up to 255
// codes large in place of 127: used for the scores of 16-bit rows.  INT8
// without: 1024 + 128 + v, minus 1152.  E4M3: exact.
template <int CODE, bool BIAS>
constexpr bool kBiased = CODE == I4D_CODE_INT8 && BIAS;
template <int CODE, bool BIAS>
constexpr float kCodeUnit = kBiased<CODE, BIAS> ? 0x1p24f : 1.f;  // what a product of such halves is multiplied by

// Codes 0 and 2 (PAIR 0) or 1 and 3 of a word.
template <int CODE, bool BIAS, int PAIR>
__device__ __forceinline__ uint32_t halves(uint32_t w) {
    if constexpr (kBiased<CODE, BIAS>) {
        return ((PAIR ? w >> 8 : w) ^ 0x00800080u) & 0x00ff00ffu;
    } else if constexpr (CODE == I4D_CODE_INT8) {
        const uint32_t m = __byte_perm(w ^ 0x80808080u, 0x64646464u, PAIR ? 0x4341 : 0x4240);
        const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&m), __half2half2(__ushort_as_half(0x6480)));
        return *reinterpret_cast<const uint32_t*>(&h);
    } else {
        uint32_t h;
        const uint16_t p = static_cast<uint16_t>(__byte_perm(w, 0, PAIR ? 0x4431 : 0x4420));
        asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(p));
        return h;
    }
}

// Codes 0, 1 (PAIR 0) or 2, 3 (PAIR 1) of words a and b (INT8: with their top
// bits flipped): out[0] the first code of both, out[1] the second.
template <int CODE, int PAIR>
__device__ __forceinline__ void halves2(uint32_t a, uint32_t b, uint32_t out[2]) {
    const uint32_t x = __byte_perm(a, b, PAIR ? 0x7362 : 0x5140);  // a0 b0 a1 b1
    if constexpr (CODE == I4D_CODE_INT8) {
        const uint32_t m0 = __byte_perm(x, 0x64646464u, 0x4140), m1 = __byte_perm(x, 0x64646464u, 0x4342);
        const __half2 bias = __half2half2(__ushort_as_half(0x6480));
        const __half2 h0 = __hsub2(*reinterpret_cast<const __half2*>(&m0), bias), h1 = __hsub2(*reinterpret_cast<const __half2*>(&m1), bias);
        out[0] = *reinterpret_cast<const uint32_t*>(&h0);
        out[1] = *reinterpret_cast<const uint32_t*>(&h1);
    } else {
        const uint16_t lo = static_cast<uint16_t>(x), hi = static_cast<uint16_t>(x >> 16);
        asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(out[0]) : "h"(lo));
        asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(out[1]) : "h"(hi));
    }
}

template <int CODE>
__device__ __forceinline__ uint32_t flip(uint32_t w) {
    return CODE == I4D_CODE_INT8 ? w ^ 0x80808080u : w;
}

__device__ __forceinline__ void mma(float c[4], const uint32_t a[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

// 16 elements of q from element i (wide: 16-byte aligned rows).
__device__ __forceinline__ void load_q16(const AttnDev& a, int64_t i, float out[16]) {
    if (a.dtype == I4D_F32) {
        const float* p = static_cast<const float*>(a.q) + i;
        if (a.wide_q) {
#pragma unroll
            for (int k = 0; k < 4; ++k) *reinterpret_cast<float4*>(out + 4 * k) = fetch(reinterpret_cast<const float4*>(p) + k);
        } else {
#pragma unroll
            for (int k = 0; k < 16; ++k) out[k] = fetch(p + k);
        }
        return;
    }
    const unsigned short* p = static_cast<const unsigned short*>(a.q) + i;
    union {
        uint4 v[2];
        unsigned short h[16];
    } x;
    if (a.wide_q) {
        x.v[0] = fetch(reinterpret_cast<const uint4*>(p));
        x.v[1] = fetch(reinterpret_cast<const uint4*>(p) + 1);
    } else {
#pragma unroll
        for (int k = 0; k < 16; ++k) x.h[k] = fetch(p + k);
    }
#pragma unroll
    for (int k = 0; k < 16; ++k)
        out[k] = a.dtype == I4D_BF16 ? __uint_as_float(static_cast<uint32_t>(x.h[k]) << 16) : __half2float(__ushort_as_half(x.h[k]));
}

__device__ __forceinline__ void store_out(const AttnDev& a, int64_t i, float v) {
    if (a.dtype == I4D_F32) static_cast<float*>(a.out)[i] = v;
    else if (a.dtype == I4D_BF16) static_cast<__nv_bfloat16*>(a.out)[i] = __float2bfloat16_rn(v);
    else static_cast<__half*>(a.out)[i] = __float2half_rn(v);
}

// Four neighbouring values from a multiple of four on.
__device__ __forceinline__ void store_out4(const AttnDev& a, int64_t i, float4 v) {
    if (!a.wide_out) {
        store_out(a, i, v.x);
        store_out(a, i + 1, v.y);
        store_out(a, i + 2, v.z);
        store_out(a, i + 3, v.w);
    } else if (a.dtype == I4D_F32) {
        *reinterpret_cast<float4*>(static_cast<float*>(a.out) + i) = v;
    } else {
        union {
            __nv_bfloat162 b[2];
            __half2 h[2];
            uint2 w;
        } u;
        if (a.dtype == I4D_BF16) {
            u.b[0] = __floats2bfloat162_rn(v.x, v.y);
            u.b[1] = __floats2bfloat162_rn(v.z, v.w);
        } else {
            u.h[0] = __floats2half2_rn(v.x, v.y);
            u.h[1] = __floats2half2_rn(v.z, v.w);
        }
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + i) = u.w;
    }
}

// First of the 16 dims of lane t's piece c of a token's codes: neighbouring
// pieces, so that two rows of an access phase take the even and the odd pieces
// of a swizzled row and hit all banks.
template <int DT>
__device__ __forceinline__ int k_dim(int t, int c) {
    return DT == 64 ? 16 * t : (c >> 1) * 128 + (2 * t + (c & 1)) * 16;
}

// The query rows of a tile as B operands: row `nt * 8 + lane / 4`, the codes'
// order of the summation index (elements 0 and 2, 1 and 3 of four).  Score
// sums of row nt * 8 + 2 (lane % 4) + j are multiplied by factor[nt][j] (and
// the block's scale) after offset[nt][j] has been taken off.
template <int DT, int NT, bool HL>
struct QTile {
    static constexpr int KS = DT / 16;
    uint32_t hi[NT][KS][2];
    uint32_t lo[HL ? NT : 1][HL ? KS : 1][2];
    float factor[NT][2], offset[NT][2];
};

template <int DT, int CODE, int NT, bool HL>
__device__ __forceinline__ void load_qtile(const AttnDev& a, const Seq& s, int h, int row0, QTile<DT, NT, HL>& q) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, dim = a.cache.dim;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const int row = row0 + nt * 8 + g;
        const bool live = row < s.n * a.group;
        const int64_t base = live ? (s.first + row / a.group) * a.q_tok + (h * a.group + row % a.group) * a.q_head : 0;
        float top = 0.f, x[DT / 64][16];
#pragma unroll
        for (int c = 0; c < DT / 64; ++c) {
            const int d0 = k_dim<DT>(t, c);
            if (live && d0 < dim) {
                load_q16(a, base + d0, x[c]);
            } else {
#pragma unroll
                for (int i = 0; i < 16; ++i) x[c][i] = 0.f;
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) top = fmaxf(top, fabsf(x[c][i]));
        }
        top = fmaxf(top, __shfl_xor_sync(~0u, top, 1));
        top = fmaxf(top, __shfl_xor_sync(~0u, top, 2));
        // 2^e with the row's largest value in [2^13, 2^14)
        const int e = max(-115, min(126, 13 - ((__float_as_int(top) >> 23) - 127)));
        const float up = __int_as_float((e + 127) << 23), down = __int_as_float((127 - e) << 23);
        float total = 0.f;
#pragma unroll
        for (int c = 0; c < DT / 64; ++c)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int e = i / 2 * 4 + (i & 1);
                const float u = x[c][e] * up, v = x[c][e + 2] * up;
                const uint32_t w = pack_h2(u, v);
                q.hi[nt][c * 4 + i / 2][i & 1] = w;
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
                total += f.x + f.y;
                if constexpr (HL) q.lo[nt][c * 4 + i / 2][i & 1] = pack_h2(u - f.x, v - f.y);
            }
        total += __shfl_xor_sync(~0u, total, 1);
        total += __shfl_xor_sync(~0u, total, 2);
        constexpr float unit = kCodeUnit<CODE, !HL>;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            q.factor[nt][j] = __shfl_sync(~0u, down, (2 * t + j) * 4) * a.scale_log2 * unit;
            q.offset[nt][j] = kBiased<CODE, !HL> ? __shfl_sync(~0u, total, (2 * t + j) * 4) * (128.f / unit) : 0.f;
        }
    }
}

// K codes of 16 tokens: the thread's 16-byte pieces of tokens g and g + 8.
template <int DT>
struct KTile {
    uint4 w[2][DT / 64];
};

template <int DT>
__device__ __forceinline__ void load_ktile(const uint8_t* k, int dim, int n, KTile<DT>& kt) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int c = 0; c < DT / 64; ++c) {
            const int d0 = k_dim<DT>(t, c);
            kt.w[r][c] = (g + 8 * r < n && d0 < dim) ? fetch(reinterpret_cast<const uint4*>(k + (g + 8 * r) * dim + d0)) : make_uint4(0, 0, 0, 0);
        }
}

// A ring slot: 16 rows of K, then of V, in boxes of 128 (64) bytes a row with
// the copies' swizzle: the 16-byte pieces of a row are exchanged by the row's
// place in the pattern.
template <int DT>
__device__ __forceinline__ uint32_t slot_at(uint32_t slot, int which, int row, int d) {
    if constexpr (DT == 64) return slot + which * 1024 + row * 64 + (d ^ ((row >> 1 & 3) << 4));
    return slot + which * 16 * DT + (d >> 7) * 2048 + row * 128 + ((d & 127) ^ ((row & 7) << 4));
}

__device__ __forceinline__ void bar_init(uint32_t bar, int count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}

// False if the barrier's phase did not end within the limit (about a second).
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity) {
    for (int i = 0; i < (1 << 20); ++i) {
        uint32_t ok;
        asm volatile("{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
                     : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
        if (ok) return true;
    }
    return false;
}

// One lane: the 16 rows from `row` of K and V into a slot.
template <int DT>
__device__ __forceinline__ void copy_tile(const AttnDev& a, uint32_t slot, uint32_t bar, int row) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(32 * DT) : "memory");
#pragma unroll
    for (int which = 0; which < 2; ++which)
#pragma unroll
        for (int x = 0; x < (DT + 127) / 128; ++x)
            asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
                             slot + which * 16 * DT + x * 2048),
                         "l"(&a.maps[which]), "r"(x * 128), "r"(row), "r"(bar)
                         : "memory");
}

__device__ __forceinline__ uint4 lds16(uint32_t at) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
    return v;
}

template <int DT>
__device__ __forceinline__ void read_ktile(uint32_t slot, KTile<DT>& kt) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int c = 0; c < DT / 64; ++c) kt.w[r][c] = lds16(slot_at<DT>(slot, 0, g + 8 * r, k_dim<DT>(t, c)));
}

template <int DT, int CODE, int NT, bool HL>
__device__ __forceinline__ void score_tile(const KTile<DT>& kt, const QTile<DT, NT, HL>& q, float s[NT][4]) {
    float odd[NT][4];  // two chains of dependent sums
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[nt][i] = odd[nt][i] = 0.f;
#pragma unroll
    for (int c = 0; c < DT / 64; ++c) {
        const uint32_t* w0 = reinterpret_cast<const uint32_t*>(&kt.w[0][c]);
        const uint32_t* w1 = reinterpret_cast<const uint32_t*>(&kt.w[1][c]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t f[4] = {halves<CODE, !HL, 0>(w0[i]), halves<CODE, !HL, 0>(w1[i]), halves<CODE, !HL, 1>(w0[i]), halves<CODE, !HL, 1>(w1[i])};
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                float* sum = i & 1 ? odd[nt] : s[nt];
                mma(sum, f, q.hi[nt][c * 4 + i][0], q.hi[nt][c * 4 + i][1]);
                if constexpr (HL) mma(sum, f, q.lo[nt][c * 4 + i][0], q.lo[nt][c * 4 + i][1]);
            }
        }
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[nt][i] += odd[nt][i];
}

// V codes of 16 tokens: of tokens 2t, 2t + 1, 2t + 8, 2t + 9, the dims
// v_dim(lane / 4, word) and the three after it.
template <int DT>
__device__ __forceinline__ int v_dim(int g, int w) {
    return DT == 64 ? g * 8 + w * 4 : (w >> 2) * 128 + g * 16 + (w & 3) * 4;
}

template <int DT>
struct VTile {
    uint32_t w[4][DT / 32];
};

template <int DT>
__device__ __forceinline__ void read_vtile(uint32_t slot, VTile<DT>& vt) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const int tok = 2 * t + (r & 1) + (r >> 1) * 8;
        if constexpr (DT == 64) {
            const uint32_t at = slot_at<DT>(slot, 1, tok, g >> 1 << 4) + (g & 1) * 8;
            asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(vt.w[r][0]), "=r"(vt.w[r][1]) : "r"(at) : "memory");
        } else {
#pragma unroll
            for (int c = 0; c < DT / 128; ++c) {
                const uint4 x = lds16(slot_at<DT>(slot, 1, tok, c * 128 + g * 16));
                vt.w[r][4 * c] = x.x;
                vt.w[r][4 * c + 1] = x.y;
                vt.w[r][4 * c + 2] = x.z;
                vt.w[r][4 * c + 3] = x.w;
            }
        }
    }
}

// Zeros in place of the tokens from `live` on: their bytes may be anything.
template <int DT>
__device__ __forceinline__ void clear_vtile(int live, VTile<DT>& vt) {
    const int t = threadIdx.x & 3;
#pragma unroll
    for (int r = 0; r < 4; ++r)
        if (2 * t + (r & 1) + (r >> 1) * 8 >= live) {
#pragma unroll
            for (int w = 0; w < DT / 32; ++w) vt.w[r][w] = 0;
        }
}

// How a weight goes to FP16: in one part, in two, or in two of which the second
// is 2^11 times what the first leaves (it meets codes times 2^-11, which are
// exact too), so that it has its eleven bits wherever the first has.
enum { kOnePart, kTwoParts, kTwoPartsFar };

template <int PARTS>
__device__ __forceinline__ uint32_t second_part(float lo, float hi, uint32_t first) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&first));
    constexpr float up = PARTS == kTwoPartsFar ? 2048.f : 1.f;
    return pack_h2((lo - f.x) * up, (hi - f.y) * up);
}

// The weights of a tile as operands: w[nt][k] of row 2t + k % 2 and token
// g + k / 2 * 8.
template <int NT, int PARTS>
__device__ __forceinline__ void pack_weights(const float (&w)[NT][4], uint32_t (&p)[NT][2], uint32_t (&pl)[NT][2]) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const uint32_t hi = pack_h2(w[nt][2 * r], w[nt][2 * r + 1]);
            p[nt][r] = transpose8(hi);
            pl[nt][r] = 0;
            if constexpr (PARTS != kOnePart) pl[nt][r] = transpose8(second_part<PARTS>(w[nt][2 * r], w[nt][2 * r + 1], hi));
        }
}

// The codes as if they had just been read: what is made of them is made here, not
// ahead of a loop, where it would take the registers of twice the codes.
template <int DT>
__device__ __forceinline__ void fresh_vtile(VTile<DT>& vt) {
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int w = 0; w < DT / 32; ++w) asm volatile("" : "+r"(vt.w[r][w]));
}

// Takes the weights that are too small for FP16 out of w, kSmallStep times into
// `kept`; whether any lane has one.
template <int NT>
__device__ __forceinline__ bool split_small(float (&w)[NT][4], volatile float (&kept)[NT][4]) {
    bool any = false;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int k = 0; k < 4; ++k) any |= w[nt][k] > 0.f && w[nt][k] < kSmallWeight;
    if (!__any_sync(~0u, any)) return false;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const bool small = w[nt][k] < kSmallWeight;
            kept[nt][k] = small ? w[nt][k] * kSmallStep : 0.f;
            if (small) w[nt][k] = 0.f;
        }
    return true;
}

template <int DT, int NT>
__device__ __forceinline__ void scale_sums(float acc[DT / 16][NT][4], float by) {
#pragma unroll
    for (int i = 0; i < DT / 16; ++i)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int k = 0; k < 4; ++k) acc[i][nt][k] *= by;
}

// acc[i]: dims v_dim(lane / 4, i / 2) + 2 (i % 2) and the next, rows 2t and
// 2t + 1 of each tile.
template <int DT, int CODE, int NT, int PARTS>
__device__ __forceinline__ void value_tile(const VTile<DT>& vt, const uint32_t (&p)[NT][2], const uint32_t (&pl)[NT][2], float acc[DT / 16][NT][4]) {
#pragma unroll
    for (int w = 0; w < DT / 32; ++w) {
        const uint32_t w0 = flip<CODE>(vt.w[0][w]), w1 = flip<CODE>(vt.w[1][w]), w2 = flip<CODE>(vt.w[2][w]), w3 = flip<CODE>(vt.w[3][w]);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            uint32_t x[2], y[2];
            if (half) {
                halves2<CODE, 1>(w0, w1, x);
                halves2<CODE, 1>(w2, w3, y);
            } else {
                halves2<CODE, 0>(w0, w1, x);
                halves2<CODE, 0>(w2, w3, y);
            }
            uint32_t f[4] = {x[0], x[1], y[0], y[1]};
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma(acc[2 * w + half][nt], f, p[nt][0], p[nt][1]);
            if constexpr (PARTS == kTwoPartsFar) {
#pragma unroll
                for (int i = 0; i < 4; ++i)  // times 2^-11
                    asm volatile("mul.rn.f16x2 %0, %0, %1;" : "+r"(f[i]) : "r"(0x10001000u));
            }
            if constexpr (PARTS != kOnePart) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) mma(acc[2 * w + half][nt], f, pl[nt][0], pl[nt][1]);
            }
        }
    }
}

// 2^(M - R) v_scale.  It passes FP32's range only for a block that the row sees
// nothing of (0 times it must be 0), or nothing but tokens 2^-113 of the
// greatest.
__device__ __forceinline__ float weight_unit(float to_r, float v_scale) { return fminf(to_r * v_scale, 0x1.fffffep127f); }

// First and one past the last token that a row at cache index pos sees.
__device__ __forceinline__ int2 row_span(const AttnDev& a, int pos) {
    return make_int2(a.window > 0 ? max(0, pos - a.window + 1) : 0, pos + 1);
}

template <int DT>
constexpr int kAttnSlots = DT == 256 ? 3 : DT == 128 ? 3 : 6;  // ring slots of a warp
constexpr int kAttnBlocks = 256; // blocks whose ids and scales are held at a time

template <int DT, int NT>
constexpr size_t attn_smem() {
    const size_t ring = static_cast<size_t>(kAttnWarps) * kAttnSlots<DT> * 32 * DT;
    const size_t merge = static_cast<size_t>(kAttnWarps) * 8 * NT * (DT + 4) * sizeof(float);
    return (ring > merge ? ring : merge) + 1024;
}

// CTAs an SM: by shared memory and by registers (8 rows of up to 128 values in
// 128 registers, FP32 ones in two parts in 168).
constexpr int attn_places(int dt, int nt, bool hlq) { return dt == 256 || nt == 2 ? 2 : dt == 128 && hlq ? 3 : 4; }

// The work of a call in units of 16 tokens: sequence by sequence, its row
// tiles of each head, the tokens that any row of the sequence sees.
struct Units {
    int tiles;     // token tiles of one (head, row tile)
    int segments;  // heads * row tiles of the sequence
};
__device__ __forceinline__ Units seq_units(const AttnDev& a, const Seq& s, int rows_per_tile) {
    if (s.n == 0 || s.len > a.max_length) return {0, 0};
    const int lo = row_span(a, s.len - s.n).x & ~15;
    return {(s.len - lo + 15) >> 4, a.cache.heads * ((s.n * a.group + rows_per_tile - 1) / rows_per_tile)};
}

struct Place {
    int64_t before;  // units of the sequences before `seq`
    int seq;
};

// Units of the whole batch and, in *at, the sequence in which unit u(total)
// lies.  The CTA's threads take consecutive sequences each.
template <typename U>
__device__ __forceinline__ int64_t find_units(const AttnDev& a, int rows_per_tile, U&& unit, bool report, Place* at) {
    __shared__ int64_t s_sum[kAttnWarps];
    __shared__ Place s_place;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int per = (a.batch + kAttnThreads - 1) / kAttnThreads, b0 = min(a.batch, static_cast<int>(threadIdx.x) * per), b1 = min(a.batch, b0 + per);
    auto size = [&](int b, bool tell) {
        const Seq s = load_seq(a.seq, b, tell);
        if (tell && s.len > a.max_length) atomicOr(a.seq.err, kBadSequence);
        const Units n = seq_units(a, s, rows_per_tile);
        return static_cast<int64_t>(n.tiles) * n.segments;
    };
    int64_t mine = 0, last = 0;
    for (int b = b0; b < b1; ++b) mine += last = size(b, report);
    int64_t upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t x = __shfl_up_sync(~0u, upto, o);
        if (lane >= o) upto += x;
    }
    if (lane == 31) s_sum[warp] = upto;
    __syncthreads();
    int64_t total = 0;
#pragma unroll
    for (int w = 0; w < kAttnWarps; ++w) {
        if (w < warp) upto += s_sum[w];
        total += s_sum[w];
    }
    const int64_t u = unit(total);
    int64_t before = upto - mine;
    if (u >= before && u < upto) {
        for (int b = b0; b < b1; ++b) {
            const int64_t next = before + (b1 - b0 == 1 ? last : size(b, false));
            if (u < next) {
                s_place = {before, b};
                break;
            }
            before = next;
        }
    }
    __syncthreads();
    *at = s_place;
    return total;
}

// One piece of work of a CTA: token tiles [t0, t1) of a segment, whose first
// tile begins at token lo.
struct Piece {
    int b, h, rt;
    int begin, end;  // tokens, begin a multiple of 16
    bool whole;      // the segment's only piece (of the cluster, if there is one)
    int slot;        // where its partial sums go otherwise: 0 the CTA's first piece, 1 its last
};

// Four values of a finished row from dim d on.
__device__ __forceinline__ void store_row(const AttnDev& a, const Seq& s, int h, int row, int d, float4 o) {
    const int64_t at = (s.first + row / a.group) * a.out_tok + (h * a.group + row % a.group) * a.out_head + d;
    store_out4(a, at, o);
}

// stats: M, l of a finished row.
__device__ __forceinline__ void store_lse(const AttnDev& a, const Seq& s, int h, int row, float4 stats) {
    const int64_t at = (s.first + row / a.group) * static_cast<int64_t>(a.heads) + h * a.group + row % a.group;
    const float l2 = stats.y == 0.f ? -INFINITY : stats.x + log2f(stats.y);
    if (a.lse) a.lse[at] = l2 * kLn2;
    if (a.weights) a.lse2[at] = l2 == -INFINITY ? INFINITY : l2;  // a row that saw nothing weighs nothing: 2^(x - inf)
}

// HLQ: FP32 query rows in two parts; HLP: probabilities in two parts.
template <int DT, int CODE, int NT, bool HLQ, bool HLP>
__device__ __forceinline__ void attend(const AttnDev& a, const Seq& s, const Piece& pc, unsigned char* attn_ring, float4* s_block, uint64_t* s_bar, Ring& copies) {
    constexpr int kRows = 8 * NT, kSlots = kAttnSlots<DT>, kParts = !HLP ? kOnePart : HLQ ? kTwoPartsFar : kTwoParts;
    float (*merge)[kRows][DT + 4] = reinterpret_cast<float (*)[kRows][DT + 4]>(attn_ring);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const int b = pc.b, h = pc.h, row0 = pc.rt * kRows;
    const int first = s.len - s.n;  // cache index of row 0's query
    const int last_row = min(row0 + kRows, s.n * a.group) - 1;
    // tokens that any row of the tile sees, and that all of them see
    const int2 lo_span = row_span(a, first + row0 / a.group), hi_span = row_span(a, first + last_row / a.group);
    const int begin = max(lo_span.x & ~15, pc.begin), end = min(hi_span.y, pc.end);
    const int all_from = hi_span.x, all_to = lo_span.y;

    float M[NT][2], R[NT][2], l[NT][2], to_r[NT][2], from[NT][2], acc[DT / 16][NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            M[nt][j] = R[nt][j] = -INFINITY;
            l[nt][j] = to_r[nt][j] = from[nt][j] = 0.f;
        }
#pragma unroll
    for (int i = 0; i < DT / 16; ++i)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[i][nt][j] = 0.f;

    if (begin < end) {
        const int bs = a.cache.block_tokens, shift = 31 - __clz(bs);
        const uint32_t ring = static_cast<uint32_t>(__cvta_generic_to_shared(attn_ring)) + warp * kSlots * 32 * DT;
        const uint32_t bars = static_cast<uint32_t>(__cvta_generic_to_shared(s_bar)) + warp * kSlots * 8;
        QTile<DT, NT, HLQ> q;
        const int span = kAttnBlocks << shift;  // tokens whose blocks the table holds
        for (int from_tok = begin; from_tok < end;) {
            // [from_tok, to_tok): up to a block's end, so that the table's entries do
            const int blk0 = from_tok >> shift, to_tok = static_cast<int>(min(static_cast<int64_t>(end), (static_cast<int64_t>(blk0) << shift) + span));
            if (from_tok != begin) __syncthreads();  // the table is free
            for (int i = threadIdx.x; i <= ((to_tok - 1) >> shift) - blk0; i += kAttnThreads) {
                const int id = load_block(a.seq, b, blk0 + i, true);
                float4 x = make_float4(__int_as_float(id), 0.f, 0.f, 0.f);
                if (id >= 0) {
                    const int64_t at = static_cast<int64_t>(id) * a.cache.heads + h;
                    x.y = fetch(a.cache.scale[0] + at);
                    x.z = fetch(a.cache.scale[1] + at);
                    x.w = __log2f(x.z);  // only a bound: its rounding cancels
                }
                s_block[i] = x;
            }
            __syncthreads();
            const int tiles = (to_tok - from_tok + 15) >> 4;
            auto issue = [&](int i, int slot) {
                if (lane != 0 || i >= tiles) return;
                const int at = from_tok + 16 * i, id = __float_as_int(s_block[(at >> shift) - blk0].x);
                if (id >= 0) copy_tile<DT>(a, ring + slot * 32 * DT, bars + slot * 8, (id * a.cache.heads + h) * bs + (at & (bs - 1)));
                else asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bars + slot * 8) : "memory");
            };
            ring_fill<kSlots>(copies, warp, kAttnWarps, issue);
            if (from_tok == begin) load_qtile<DT, CODE, NT, HLQ>(a, s, h, row0, q);
            const auto wait = [&](int slot, uint32_t parity) { return bar_wait(bars + slot * 8, parity); };
            const auto any_late = [&](bool landed) {  // (the whole warp)
                if (__all_sync(~0u, landed)) return false;
                if (lane == 0) atomicOr(a.seq.err, kTimeout);
                return true;
            };
            // (free: all lanes are done with the slot to fill)
            ring_walk<kSlots>(copies, warp, kAttnWarps, tiles, issue, wait, [] { __syncwarp(); }, [&](int i, int slot, bool landed) {
                const uint32_t at_slot = ring + slot * 32 * DT;
                const int at = from_tok + 16 * i;
                const float4 block = s_block[(at >> shift) - blk0];
                const float lvs = block.w;
                const int live = __float_as_int(block.x) < 0 ? 0 : min(16, to_tok - at);
                if (live == 0 && !a.scores) return !any_late(landed);  // (the kept scores of a bad block are -inf)
                float x[NT][4];
                {
                    KTile<DT> kt;
                    read_ktile<DT>(at_slot, kt);
                    score_tile<DT, CODE, NT, HLQ>(kt, q, x);
                }
                VTile<DT> vt;
                // FP32 rows read V's codes late, for their registers (24 contexts, dim
                // 256: 214 us, 276 with the codes read here).
                constexpr bool kLate = HLQ;
                if constexpr (!kLate) {
                    read_vtile<DT>(at_slot, vt);
                    if (live < 16) clear_vtile<DT>(live, vt);
                }
                float top[NT][2];
                const bool whole = live == 16 && at >= all_from && at + 16 <= all_to;
                bool raise = !landed;  // one vote a tile answers both
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const float f = q.factor[nt][j] * block.y, off = q.offset[nt][j] * f;
                        float y0 = fmaf(x[nt][j], f, -off), y1 = fmaf(x[nt][j + 2], f, -off);
                        if (!whole) {
                            const int2 span = row_span(a, first + (row0 + nt * 8 + 2 * t + j) / a.group);
                            if (!(g < live && at + g >= span.x && at + g < span.y)) y0 = -INFINITY;
                            if (!(g + 8 < live && at + g + 8 >= span.x && at + g + 8 < span.y)) y1 = -INFINITY;
                        }
                        x[nt][j] = y0;
                        x[nt][j + 2] = y1;
                        top[nt][j] = fmaxf(y0, y1);
                        raise |= top[nt][j] > M[nt][j] + kSlack || top[nt][j] + lvs > R[nt][j] + (kSlack + kHead);
                        raise |= fminf(y0, y1) + lvs < R[nt][j] - 14.f;  // small weights, and tokens that are not seen
                    }
                const bool voted = __any_sync(~0u, raise);
                if (voted) {
                    if (any_late(landed)) return false;
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            float m = top[nt][j];
#pragma unroll
                            for (int o = 4; o < 32; o <<= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
                            const float mr = fmaxf(m + lvs - kHead, R[nt][j]);
                            m = fmaxf(m, M[nt][j]);
                            const float r = fmaxf(mr, m - kFarScales);
                            const float fm = M[nt][j] == m ? 1.f : ex2(M[nt][j] - m), fr = R[nt][j] == r ? 1.f : ex2(R[nt][j] - r);
                            l[nt][j] *= fm;
#pragma unroll
                            for (int i2 = 0; i2 < DT / 16; ++i2) {
                                acc[i2][nt][j] *= fr;
                                acc[i2][nt][j + 2] *= fr;
                            }
                            M[nt][j] = m;
                            R[nt][j] = r;
                            from[nt][j] = m == -INFINITY ? 0.f : m;
                            to_r[nt][j] = r == -INFINITY ? 0.f : ex2(m - r);
                        }
                }
                if (a.scores) {
                    const int64_t tile = (static_cast<int64_t>(b) * a.cache.heads + h) * a.row_tiles + pc.rt;
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const int r = nt * 8 + 2 * t + (k & 1), n = g + (k >> 1) * 8;
                            if (at + n < to_tok && row0 + r <= last_row) a.scores[(tile * kRows + r) * a.score_stride + at + n] = x[nt][k];
                        }
                }
                float w[NT][4];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const int j = k & 1;
                        const float e = ex2(x[nt][k] - from[nt][j]);
                        l[nt][j] += e;
                        w[nt][k] = e * weight_unit(to_r[nt][j], block.z);
                    }
                // Weights under FP16's range count where the greatest ones' codes
                // are 0: they go in 2^24 times, to 2^24 times the sums, and so on.
                volatile float kept[NT][4];  // (in memory: most tiles have none)
                bool more = voted && split_small<NT>(w, kept);
                float down = 1.f;
#pragma unroll 1
                for (;;) {
                    uint32_t p[NT][2], pl[NT][2];
                    pack_weights<NT, kParts>(w, p, pl);
                    if constexpr (kLate) {
                        read_vtile<DT>(at_slot, vt);
                        if (live < 16) clear_vtile<DT>(live, vt);
                    } else {
                        fresh_vtile<DT>(vt);
                    }
                    value_tile<DT, CODE, NT, kParts>(vt, p, pl, acc);
                    if (!more) break;
                    down *= 1.f / kSmallStep;
                    scale_sums<DT, NT>(acc, kSmallStep);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int k = 0; k < 4; ++k) w[nt][k] = kept[nt][k];
                    more = split_small<NT>(w, kept) && down > 1.f / kSmallMost;
                }
                if (down != 1.f) scale_sums<DT, NT>(acc, down);
                return true;
            });
            from_tok = to_tok;
        }
        __syncthreads();  // the ring is free for the join
    }

    // Join the four warps.
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) l[nt][j] += __shfl_xor_sync(~0u, l[nt][j], o);
            float* m = merge[warp][nt * 8 + 2 * t + j];
#pragma unroll
            for (int i = 0; i < DT / 16; ++i) {
                const int d = v_dim<DT>(g, i >> 1) + 2 * (i & 1);
                m[d] = acc[i][nt][j];
                m[d + 1] = acc[i][nt][j + 2];
            }
            if (g == 0) {
                m[DT] = M[nt][j];
                m[DT + 1] = l[nt][j];
                m[DT + 2] = R[nt][j];
            }
        }
    __syncthreads();
    const int dim = a.cache.dim, rows = last_row - row0 + 1;
    if (threadIdx.x < rows) {  // a row's statistics, and what its warps' sums are multiplied by
        const int r = threadIdx.x, row = row0 + r;
        float m = -INFINITY, rr = -INFINITY, sum = 0.f;
#pragma unroll
        for (int w = 0; w < kAttnWarps; ++w) {
            m = fmaxf(m, merge[w][r][DT]);
            rr = fmaxf(rr, merge[w][r][DT + 2]);
        }
#pragma unroll
        for (int w = 0; w < kAttnWarps; ++w)  // (a warp that saw nothing of the row: its sums are 0, or NaN with the row's)
            sum += merge[w][r][DT + 1] * (merge[w][r][DT] == -INFINITY ? 1.f : ex2(merge[w][r][DT] - m));
        const bool done = pc.whole && a.cluster <= 1;
        const float back = !done ? 1.f : sum == 0.f || rr == -INFINITY ? 0.f : ex2(rr - m) / sum;
#pragma unroll
        for (int w = 0; w < kAttnWarps; ++w)
            merge[w][r][DT + 3] = (merge[w][r][DT + 2] == -INFINITY ? 1.f : ex2(merge[w][r][DT + 2] - rr)) * back;
        const float4 stats = make_float4(m, sum, rr, 0.f);
        if (done) store_lse(a, s, h, row, stats);
        else if (pc.whole) s_block[r] = stats;
        else a.stats[(static_cast<int64_t>(blockIdx.x) * 2 + pc.slot) * kRows + r] = stats;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < rows * (DT / 4); i += kAttnThreads) {
        const int r = i / (DT / 4), d = i % (DT / 4) * 4, row = row0 + r;
        if (d >= dim) continue;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kAttnWarps; ++w) {
            const float4 x = *reinterpret_cast<const float4*>(&merge[w][r][d]);
            const float f = merge[w][r][DT + 3];
            o.x += x.x * f;
            o.y += x.y * f;
            o.z += x.z * f;
            o.w += x.w * f;
        }
        if (!pc.whole) *reinterpret_cast<float4*>(a.part + ((static_cast<int64_t>(blockIdx.x) * 2 + pc.slot) * kRows + r) * dim + d) = o;
        else if (a.cluster > 1) *reinterpret_cast<float4*>(&merge[0][r][d]) = o;  // (only this thread reads it above)
        else store_row(a, s, h, row, d, o);
    }
    if (pc.whole && a.cluster > 1) {
        cooperative_groups::cluster_group cl = cooperative_groups::this_cluster();
        const int ctas = a.cluster, rank = blockIdx.x % ctas;
        cl.sync();
        for (int i = rank * kAttnThreads + threadIdx.x; i < rows * (DT / 4); i += ctas * kAttnThreads) {
            const int r = i / (DT / 4), d = i % (DT / 4) * 4, row = row0 + r;
            float4 stats[8];
            float m = -INFINITY, rr = -INFINITY, sum = 0.f;
#pragma unroll
            for (int c = 0; c < 8; ++c) {
                stats[c] = make_float4(-INFINITY, 0.f, -INFINITY, 0.f);
                if (c < ctas) stats[c] = cl.map_shared_rank(s_block, c)[r];
                m = fmaxf(m, stats[c].x);
                rr = fmaxf(rr, stats[c].z);
            }
            float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int c = 0; c < 8; ++c) {
                if (c >= ctas) break;
                sum += stats[c].y * (stats[c].x == -INFINITY ? 1.f : ex2(stats[c].x - m));
                if (d >= dim) continue;
                const float4 x = *reinterpret_cast<const float4*>(&cl.map_shared_rank(&merge[0][0][0], c)[r * (DT + 4) + d]);
                const float f = stats[c].z == -INFINITY ? 1.f : ex2(stats[c].z - rr);
                o.x += x.x * f;
                o.y += x.y * f;
                o.z += x.z * f;
                o.w += x.w * f;
            }
            const float back = sum == 0.f || rr == -INFINITY ? 0.f : ex2(rr - m) / sum;
            if (d < dim) store_row(a, s, h, row, d, make_float4(o.x * back, o.y * back, o.z * back, o.w * back));
            if (d == 0) store_lse(a, s, h, row, make_float4(m, sum, rr, 0.f));
        }
        cl.sync();  // no CTA leaves while another reads its memory
    }
}

template <int DT, int CODE, int NT, bool HLQ, bool HLP>
__global__ void __launch_bounds__(kAttnThreads, attn_places(DT, NT, HLQ)) k_kv8_attn(const __grid_constant__ AttnDev a) {
    op_begin();
    constexpr int kRows = 8 * NT;
    extern __shared__ unsigned char attn_smem_base[];
    // the copies' swizzle counts from 1024-byte boundaries
    unsigned char* attn_ring = attn_smem_base + (-static_cast<uint32_t>(__cvta_generic_to_shared(attn_smem_base)) & 1023u);
    __shared__ uint64_t s_bar[kAttnWarps * kAttnSlots<DT>];
    Ring copies;
    if (threadIdx.x < kAttnWarps * kAttnSlots<DT>) bar_init(static_cast<uint32_t>(__cvta_generic_to_shared(s_bar + threadIdx.x)), 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    __syncthreads();
    __shared__ float4 s_block[kAttnBlocks];  // id, scale of K, of V, log2 of the latter
    if (!a.even) {
        const int segment = blockIdx.x / a.cluster, rank = blockIdx.x % a.cluster;
        const int rt = segment % a.row_tiles, h = segment / a.row_tiles % a.cache.heads, b = segment / a.row_tiles / a.cache.heads;
        const bool report = rt == 0 && h == 0 && rank == 0 && threadIdx.x == 0;
        const Seq s = load_seq(a.seq, b, report);
        if (report && s.len > a.max_length) atomicOr(a.seq.err, kBadSequence);
        if (s.len > a.max_length || rt * kRows >= s.n * a.group) return;  // the whole cluster
        const int first = s.len - s.n, lo = row_span(a, first + rt * kRows / a.group).x & ~15;
        const int share = ((s.len - lo + 15) / 16 + a.cluster - 1) / a.cluster * 16;
        attend<DT, CODE, NT, HLQ, HLP>(a, s, {b, h, rt, lo + rank * share, min(s.len, lo + (rank + 1) * share), true, 0}, attn_ring, s_block, s_bar, copies);
        return;
    }
    Place at;
    int64_t share = 0;
    const int64_t total = find_units(a, kRows, [&](int64_t n) {
        share = (n + a.even - 1) / a.even;
        return share * blockIdx.x;
    }, blockIdx.x == 0, &at);
    int64_t u = share * blockIdx.x;
    const int64_t u_end = min(total, u + share), u0 = u;
    if (u >= u_end) return;
    while (u < u_end) {
        const Seq s = load_seq(a.seq, at.seq, false);
        const Units n = seq_units(a, s, kRows);
        const int64_t size = static_cast<int64_t>(n.tiles) * n.segments;
        if (u >= at.before + size) {
            at.before += size;
            ++at.seq;
            continue;
        }
        const int seg = static_cast<int>((u - at.before) / n.tiles), row_tiles = n.segments / a.cache.heads;
        const int64_t seg0 = at.before + static_cast<int64_t>(seg) * n.tiles;
        const int t0 = static_cast<int>(u - seg0), t1 = static_cast<int>(min(static_cast<int64_t>(n.tiles), u_end - seg0));
        const int lo = row_span(a, s.len - s.n).x & ~15;
        if (t0 == 0 && threadIdx.x == 0)
            a.segments[(static_cast<int64_t>(at.seq) * a.cache.heads + seg / row_tiles) * a.row_tiles + seg % row_tiles] =
                make_int4(blockIdx.x, static_cast<int>((seg0 + n.tiles - 1) / share), u == u0 ? 0 : 1, 0);
        if (u != u0) {
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // the join wrote where the next copies go
            __syncthreads();
        }
        attend<DT, CODE, NT, HLQ, HLP>(a, s, {at.seq, seg / row_tiles, seg % row_tiles, lo + 16 * t0, min(s.len, lo + 16 * t1), t0 == 0 && t1 == n.tiles, u == u0 ? 0 : 1},
                                       attn_ring, s_block, s_bar, copies);
        u = seg0 + t1;
    }
}

constexpr int kJoinThreads = 512;

// Joins the pieces of the segments that several CTAs shared: one CTA for a
// segment, whose warps take rows and, if there are fewer rows than warps,
// every so-manieth piece of one, so that the pieces are read at once.
__global__ void __launch_bounds__(kJoinThreads) k_kv8_join(AttnDev a, int rows_per_tile) {
    op_begin();
    constexpr int kWarps = kJoinThreads / 32;
    __shared__ float4 s_o[kWarps][64];
    __shared__ float s_sum[kWarps];
    const int4 segment = a.segments[blockIdx.x];
    const int rt = blockIdx.x % a.row_tiles, h = blockIdx.x / a.row_tiles % a.cache.heads, b = blockIdx.x / a.row_tiles / a.cache.heads;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, dim = a.cache.dim;
    const Seq s = load_seq(a.seq, b, false);
    const Units n = seq_units(a, s, rows_per_tile);
    if (rt >= n.segments / a.cache.heads) return;  // (its entry in the table was not written)
    const int c0 = segment.x, c1 = segment.y;
    if (c0 == c1) return;  // whole
    const int rows = min(rows_per_tile, s.n * a.group - rt * rows_per_tile), parts = kWarps / rows;
    const int r = warp / parts, part = warp % parts;  // rows <= 16
    float m = -INFINITY, rr = -INFINITY, sum = 0.f;
    float4 o[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};  // dims 4 lane and 128 + 4 lane
    const bool low = 4 * lane < dim, high = 128 + 4 * lane < dim;
    // the first CTA's piece may be its last, those of the others are their first
    auto index = [&](int c) { return (static_cast<int64_t>(c) * 2 + (c == c0 ? segment.z : 0)) * rows_per_tile + r; };
    if (r < rows) {
        for (int c = c0 + lane; c <= c1; c += 32) {
            const float4 x = a.stats[index(c)];
            m = fmaxf(m, x.x);
            rr = fmaxf(rr, x.z);
        }
        m = warp_max(m);
        rr = warp_max(rr);
#pragma unroll 4
        for (int c = c0 + part; c <= c1; c += parts) {
            const float4 x = a.stats[index(c)];
            const float* p = a.part + index(c) * dim + 4 * lane;
            const float4 y = low ? *reinterpret_cast<const float4*>(p) : make_float4(0.f, 0.f, 0.f, 0.f);
            const float4 z = high ? *reinterpret_cast<const float4*>(p + 128) : make_float4(0.f, 0.f, 0.f, 0.f);
            const float f = x.z == -INFINITY ? 1.f : ex2(x.z - rr);
            sum += x.y * (x.x == -INFINITY ? 1.f : ex2(x.x - m));
            o[0].x += y.x * f;
            o[0].y += y.y * f;
            o[0].z += y.z * f;
            o[0].w += y.w * f;
            o[1].x += z.x * f;
            o[1].y += z.y * f;
            o[1].z += z.z * f;
            o[1].w += z.w * f;
        }
    }
    s_o[warp][lane] = o[0];
    s_o[warp][32 + lane] = o[1];
    if (lane == 0) s_sum[warp] = sum;
    __syncthreads();
    if (part || r >= rows) return;
    for (int k = 1; k < parts; ++k) {
        sum += s_sum[warp + k];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const float4 x = s_o[warp + k][32 * i + lane];
            o[i].x += x.x;
            o[i].y += x.y;
            o[i].z += x.z;
            o[i].w += x.w;
        }
    }
    const float back = sum == 0.f || rr == -INFINITY ? 0.f : ex2(rr - m) / sum;
    const int row = rt * rows_per_tile + r;
#pragma unroll
    for (int i = 0; i < 2; ++i)
        if (i ? high : low) store_row(a, s, h, row, 128 * i + 4 * lane, make_float4(o[i].x * back, o[i].y * back, o[i].z * back, o[i].w * back));
    if (lane == 0) store_lse(a, s, h, row, make_float4(m, sum, rr, 0.f));
}

// Probabilities summed over a head's few rows for each token, from the scores
// that k_kv8_attn kept: four tokens a thread, rows in order.
__global__ void __launch_bounds__(128) k_kv8_weights_kept(AttnDev a, int rows_per_tile, int chunks) {
    op_begin();
    const int64_t bh = blockIdx.x / chunks;
    const int n = ((blockIdx.x % chunks) * 128 + threadIdx.x) * 4, h = bh % a.cache.heads, b = bh / a.cache.heads;
    const Seq s = load_seq(a.seq, b, false);
    if (s.len > a.max_length || s.n == 0 || n >= s.len) return;
    const int rows = s.n * a.group, first = s.len - s.n;
    float* to = a.weights + bh * a.weights_stride + n;
    float w[4], sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = n + i < s.len ? to[i] : 0.f;
#pragma unroll 4
    for (int row = 0; row < rows; ++row) {
        const int2 sp = row_span(a, first + row / a.group);
        const int64_t at = (bh * a.row_tiles + row / rows_per_tile) * rows_per_tile + row % rows_per_tile;
        const float l2 = a.lse2[(s.first + row / a.group) * static_cast<int64_t>(a.heads) + h * a.group + row % a.group];
        const float4 x = *reinterpret_cast<const float4*>(a.scores + at * a.score_stride + n);
        const float y[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int i = 0; i < 4; ++i)  // (scores outside the row's span may not have been written)
            sum[i] += n + i >= sp.x && n + i < sp.y ? ex2(y[i] - l2) : 0.f;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (n + i < s.len) to[i] = w[i] + sum[i];
}

// Probabilities summed over a head's rows for each token: the scores again,
// 2^(x - lse2), a warp for 16 tokens, rows in order.
template <int DT, int CODE, bool HL>
__global__ void __launch_bounds__(kAttnThreads) k_kv8_weights(AttnDev a, int tiles) {
    op_begin();
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int tile = blockIdx.x % tiles, bh = blockIdx.x / tiles, h = bh % a.cache.heads, b = bh / a.cache.heads;
    const Seq s = load_seq(a.seq, b, false);
    const int at = (tile * kAttnWarps + (threadIdx.x >> 5)) * 16;
    if (s.len > a.max_length || s.n == 0 || at >= s.len) return;
    const int bs = a.cache.block_tokens, dim = a.cache.dim, first = s.len - s.n;
    const int id = load_block(a.seq, b, at / bs, false);
    if (id < 0) return;
    const int live = min(16, s.len - at);
    KTile<DT> kt;
    load_ktile<DT>(a.cache.codes[0] + code_offset(a.cache, id, h) + static_cast<int64_t>(at % bs) * dim, dim, live, kt);
    const float ks = fetch(a.cache.scale[0] + static_cast<int64_t>(id) * a.cache.heads + h);
    float sum[2] = {0.f, 0.f};
    // rows whose query stands at or behind the first token and, with a window, not past the last one's
    const int rows = s.n * a.group;
    const int from = max(0, at - first) * a.group & ~7;
    const int to = a.window > 0 ? static_cast<int>(min(static_cast<int64_t>(rows), max(int64_t{0}, (static_cast<int64_t>(at) + 15 + a.window - first)) * a.group)) : rows;
    for (int row0 = from; row0 < to; row0 += 8) {
        QTile<DT, 1, HL> q;
        load_qtile<DT, CODE, 1, HL>(a, s, h, row0, q);
        float x[1][4];
        score_tile<DT, CODE, 1, HL>(kt, q, x);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int row = row0 + 2 * t + j;
            if (row >= rows) continue;
            const float l2 = a.lse2[(s.first + row / a.group) * static_cast<int64_t>(a.heads) + h * a.group + row % a.group];
            const int2 sp = row_span(a, first + row / a.group);
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const int n = at + g + 8 * r;
                if (n < s.len && n >= sp.x && n < sp.y) sum[r] += ex2(fmaf(x[0][j + 2 * r] - q.offset[0][j], q.factor[0][j] * ks, -l2));
            }
        }
    }
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        sum[r] += __shfl_xor_sync(~0u, sum[r], 1);
        sum[r] += __shfl_xor_sync(~0u, sum[r], 2);
        const int n = at + g + 8 * r;
        if (t == 0 && n < s.len) a.weights[(static_cast<int64_t>(b) * a.cache.heads + h) * a.weights_stride + n] += sum[r];
    }
}

}  // namespace i4d_ops
