// i4d_ops_common.cuh -- helpers of the long-context serving operators.
//
// Unlike the decode path these translation units are compiled with
// multiply-add contraction; where a rounding order is part of an operator's
// definition it is written with explicit intrinsics.
#pragma once

#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include "i4d.h"
#include "i4d_seq.h"

namespace i4d_ops {

// Bits of the operators' device error word.
constexpr unsigned kBadSequence = 1u;  // q_start or lengths outside what the call's arguments allow
constexpr unsigned kBadBlock = 2u;     // a block id outside the pool
constexpr unsigned kTimeout = 4u;      // a bounded wait gave up

template <int DT>
struct ElemOf;
template <>
struct ElemOf<I4D_F32> { using T = float; };
template <>
struct ElemOf<I4D_BF16> { using T = __nv_bfloat16; };
template <>
struct ElemOf<I4D_F16> { using T = __half; };

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }

// A load of what a kernel before this one may have written, or this one writes in
// place.  A plain one, not of the read-only path (__ldg): the launches overlap,
// so that memory is not constant while the kernel lives, and nothing would keep
// such a load behind op_begin()'s wait.
template <typename T>
__device__ __forceinline__ T fetch(const T* p) {
    return *p;
}

// Loads from the L2 of what other CTAs of the cluster write between barriers.
// (volatile: they stay between the barriers where they stand)
__device__ __forceinline__ float fetch_l2(const float* p) {
    float x;
    asm volatile("ld.global.cg.f32 %0, [%1];" : "=f"(x) : "l"(p));
    return x;
}
__device__ __forceinline__ uint4 fetch_l2(const uint4* p) {
    uint4 x;
    asm volatile("ld.global.cg.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w) : "l"(p));
    return x;
}

// N elements by 16-byte accesses (N * sizeof(T) a multiple of 16, aligned).
template <typename T, int N>
struct alignas(16) Vec {
    T v[N];
};

template <typename T, int N>
__device__ __forceinline__ Vec<T, N> load_vec(const T* p) {
    Vec<T, N> r;
    if constexpr (N * sizeof(T) % 16 == 0) {
#pragma unroll
        for (int i = 0; i < static_cast<int>(N * sizeof(T) / 16); ++i)
            reinterpret_cast<uint4*>(&r)[i] = fetch(reinterpret_cast<const uint4*>(p) + i);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) r.v[i] = p[i];
    }
    return r;
}

template <typename T, int N>
__device__ __forceinline__ void store_vec(T* p, const Vec<T, N>& r) {
    if constexpr (N * sizeof(T) % 16 == 0) {
#pragma unroll
        for (int i = 0; i < static_cast<int>(N * sizeof(T) / 16); ++i)
            reinterpret_cast<uint4*>(p)[i] = reinterpret_cast<const uint4*>(&r)[i];
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) p[i] = r.v[i];
    }
}

// First of all in every kernel of the operators: waits for what the stream
// holds before it, whose end its launch may overlap, then lets the next one's
// launch overlap its own.
__device__ __forceinline__ void op_begin() {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

// The arrays that say where the tokens of a batch are.
struct SeqArrays {
    const int32_t* q_start;
    const int32_t* lengths;
    const int32_t* table;
    int64_t table_stride;
    int tokens, max_q, block_tokens, blocks, table_blocks;
    unsigned* err;
};

struct Seq {
    int first, n, len;  // first row, rows, tokens in the cache
};

// A sequence whose arrays contradict the call's bounds is skipped (n = 0).
__device__ __forceinline__ Seq load_seq(const SeqArrays& a, int b, bool report) {
    const int q0 = fetch(a.q_start + b), q1 = fetch(a.q_start + b + 1), len = fetch(a.lengths + b);
    const bool ok = seq_ok(q0, q1, len, a.tokens, a.max_q, a.table_blocks, a.block_tokens);
    if (!ok && report) atomicOr(a.err, kBadSequence);
    return {q0, ok ? q1 - q0 : 0, ok ? len : 0};
}

// Block id of a table entry, or -1 for one outside the pool.
__device__ __forceinline__ int load_block(const SeqArrays& a, int b, int j, bool report) {
    const int id = fetch(a.table + static_cast<int64_t>(b) * a.table_stride + j);
    if (block_ok(id, a.blocks)) return id;
    if (report) atomicOr(a.err, kBadBlock);
    return -1;
}

// ------------------------------------------------------------- 8-bit codes

// Least power of two s >= 2^-126 with amax <= 127 s (INT8) or 448 s (E4M3):
// amax = f 2^e with f in [1, 2), 127 = 1.984375 * 2^6, 448 = 1.75 * 2^8.
__device__ __forceinline__ float power_scale(float amax, int code) {
    const int bits = __float_as_int(amax);
    const int e = (bits >> 23) - 127, frac = bits & 0x7fffff;
    int es = code == I4D_CODE_INT8 ? e - 6 + (frac > 0x7e0000) : e - 8 + (frac > 0x600000);
    es = max(es, -126);
    return __int_as_float((es + 127) << 23);
}

// Four codes of y (already divided by the scale): NaN 0, beyond the range the
// largest code, else the nearest with ties to even.
template <int CODE>
__device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d) {
    if constexpr (CODE == I4D_CODE_INT8) {
        // (a conversion to an integer saturates and makes 0 of NaN)
        const int ia = max(min(__float2int_rn(a), 127), -127), ib = max(min(__float2int_rn(b), 127), -127);
        const int ic = max(min(__float2int_rn(c), 127), -127), id = max(min(__float2int_rn(d), 127), -127);
        return __byte_perm(__byte_perm(ia, ib, 0x0040), __byte_perm(ic, id, 0x0040), 0x5410);
    } else {
        uint16_t lo, hi;
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
        const uint32_t w = lo | static_cast<uint32_t>(hi) << 16;
        // NaN alone becomes 0x7f or 0xff
        const uint32_t nan = (w & 0x7f7f7f7fu) + 0x01010101u & 0x80808080u;
        return nan ? w & ~((nan >> 7) * 255u) : w;
    }
}

// The four code values of a word.
template <int CODE>
__device__ __forceinline__ void decode4(uint32_t w, float out[4]) {
    if constexpr (CODE == I4D_CODE_INT8) {
#pragma unroll
        for (int i = 0; i < 4; ++i) out[i] = static_cast<float>(static_cast<int8_t>(w >> (8 * i)));
    } else {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            uint32_t h;
            const uint16_t p = static_cast<uint16_t>(w >> (16 * i));
            asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(p));
            const float2 f = __half22float2(*reinterpret_cast<__half2*>(&h));
            out[2 * i] = f.x;
            out[2 * i + 1] = f.y;
        }
    }
}

// round(code * ratio) of a word's codes, 0 <= ratio <= 1.  Powers of two down to
// 2^-14 keep every product exact in FP16, where an INT8 code is rounded by the
// sum with 1536 (whose steps are 1): a third of the instructions of FP32.
struct Rescale {
    float ratio;
    __half2 half;
    bool fast;
};
__device__ __forceinline__ Rescale make_rescale(float r) { return {r, __float2half2_rn(r), (__float_as_int(r) & 0x7fffff) == 0 && r >= 0x1p-14f}; }

template <int CODE>
__device__ __forceinline__ uint32_t rescale4(uint32_t w, const Rescale& r) {
    if (r.fast) {
        if constexpr (CODE == I4D_CODE_INT8) {
            const uint32_t x = w ^ 0x80808080u, m0 = __byte_perm(x, 0x64646464u, 0x4140), m1 = __byte_perm(x, 0x64646464u, 0x4342);
            const __half2 bias = __half2half2(__ushort_as_half(0x6480)), whole = __half2half2(__ushort_as_half(0x6600));
            const __half2 h0 = __hfma2(__hsub2(*reinterpret_cast<const __half2*>(&m0), bias), r.half, whole);
            const __half2 h1 = __hfma2(__hsub2(*reinterpret_cast<const __half2*>(&m1), bias), r.half, whole);
            return __byte_perm(*reinterpret_cast<const uint32_t*>(&h0), *reinterpret_cast<const uint32_t*>(&h1), 0x6420);
        } else {
            uint32_t h[2];
            uint16_t e[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h[i]) : "h"(static_cast<uint16_t>(w >> (16 * i))));
                const __half2 y = __hmul2(*reinterpret_cast<const __half2*>(&h[i]), r.half);
                asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(e[i]) : "r"(*reinterpret_cast<const uint32_t*>(&y)));
            }
            return e[0] | static_cast<uint32_t>(e[1]) << 16;
        }
    }
    float f[4];
    decode4<CODE>(w, f);
    return encode4<CODE>(__fmul_rn(f[0], r.ratio), __fmul_rn(f[1], r.ratio), __fmul_rn(f[2], r.ratio), __fmul_rn(f[3], r.ratio));
}

__device__ __forceinline__ float warp_max(float x) {
#pragma unroll
    for (int o = 16; o; o >>= 1) x = fmaxf(x, __shfl_xor_sync(~0u, x, o));
    return x;
}

__device__ __forceinline__ float warp_sum(float x) {
#pragma unroll
    for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(~0u, x, o);
    return x;
}

}  // namespace i4d_ops
