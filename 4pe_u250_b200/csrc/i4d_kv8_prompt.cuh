// i4d_kv8_prompt.cuh -- attention of many query rows over the cache of 8-bit
// codes on the fifth-generation tensor cores.
//
// A CTA takes up to 256 rows (query, head of the group) of one cache head at a
// time: two tiles of 128 rows take turns, so that one tile's products run under the
// other's softmax.  Tiles of 128 tokens go through
//   producer (1 warp)      codes of 16 tokens a tensor copy, scales of 16 tokens into a table
//   converters (4 warps)   codes -> FP16 operands in the 128-byte swizzle, a token row a thread
//   products (2 threads)   a row tile each: S = Q K^T (128 x 128), O += P V, both into tensor memory
//   softmax (2 x 4 warps)  a row a thread: bounds M and R, P = 2^(x - M) v_scale 2^(M - R) in FP16 over S
// K is the second operand of S with its dims contiguous, V that of O with its
// dims contiguous too (the transposed form), so both convert alike; P is the
// first operand straight from tensor memory.  The arithmetic is
// i4d_kv8_attn.cuh's: exact codes and query rows, FP32 sums, probabilities in
// one FP16 part for BF16 outputs (2^-11), in two for FP16 ones (2^-22, twice the
// second products), but not less than 2^-31 of the row's greatest: the few-row
// kernel's second look at small weights has no tensor memory left for its sums
// here.  A row's statistics stay in its thread, and O is rescaled
// only where a score passes the bound by more than 2^6.
// Bound: 4 dim products a visible (row, token) at the tensor rate, and one
// exponential for each at the rate of the special-function units, which for
// dim 128 takes as long (16 a cycle and SM against 8192 products).  Two chunks
// of 1537 to 2048 rows over 6151 to 8192 tokens, 32 heads of 128: 569 us with the
// join, 661 TFLOP/s (FP16 outputs 15 % more); tensor pipe 50 %, exponentials 36 %,
// issue slots 43 % busy: the softmax threads wait for tensor memory.
#pragma once

#include "i4d_kv8_attn.cuh"

namespace i4d_ops {

constexpr int kPrThreads = 480;
constexpr int kPrRows = 256;
constexpr int kPrTokens = 128;

template <int DT>
struct PromptSmem {
    static constexpr int kBlock = 16384;                  // 128 rows of 64 halves
    static constexpr int kOperand = DT / 64 * kBlock;     // 128 rows of DT halves
    static constexpr int kRaw = kPrTokens * DT;           // codes of a tile
    static constexpr int q = 0;
    static constexpr int k = q + 2 * kOperand;            // two buffers
    static constexpr int v = k + 2 * kOperand;
    static constexpr int raw = v + kOperand;              // two stages of K, V
    static constexpr int total = raw + 4 * kRaw;
};

// Barriers.
enum {
    kRawKFull = 0, kRawVFull = 2, kRawKEmpty = 4, kRawVEmpty = 6, kKFull = 8, kKEmpty = 10,
    kVFull = 12, kVEmpty, kSFull, kPFull = kSFull + 4, kPvDone = kPFull + 4, kQFull = kPvDone + 4, kODone = kQFull + 2,
    kFirstP = kODone + 2,  // completes once: tile 0's first probabilities of the CTA
    kPrBars
};

constexpr int kPrWarps = kPrThreads / 32;

struct PrShared {
    uint64_t bar[kPrBars];
    int64_t sums[kPrWarps], before;  // units of work (find_prompt)
    int pair;
    float4 table[4][8];  // of 16 tokens: scale of K, of V, log2 of it
    int missing[4];      // bit g: the table's 16 tokens g are not there
    uint32_t tmem;
    int abort;
};

__device__ __forceinline__ uint32_t bar_at(const PrShared& sh, int i) { return static_cast<uint32_t>(__cvta_generic_to_shared(&sh.bar[i])); }

// False once the wait, or another one of the CTA, has given up.
__device__ __forceinline__ bool pr_wait(PrShared& sh, int i, uint32_t parity) {
    const uint32_t bar = bar_at(sh, i);
    for (int n = 0; n < (1 << 16); ++n) {
        uint32_t ok;
        asm volatile("{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
                     : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
        if (ok) return true;
        if ((n & 63) == 63 && *reinterpret_cast<volatile int*>(&sh.abort)) return false;
    }
    *reinterpret_cast<volatile int*>(&sh.abort) = 1;
    return false;
}

__device__ __forceinline__ void pr_arrive(const PrShared& sh, int i) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar_at(sh, i)) : "memory");
}

// The issuing thread's products so far arrive on a barrier when they are done.
__device__ __forceinline__ void pr_commit(const PrShared& sh, int i) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar_at(sh, i)) : "memory");
}

// Shared-memory operands in the 128-byte swizzle, 1024 bytes between groups of
// eight rows; `lead` bytes between blocks of 64 along a contiguous non-summed
// dimension (unused where the summed one is contiguous).
__device__ __forceinline__ uint64_t operand_desc(uint32_t addr, uint32_t lead) {
    return static_cast<uint64_t>((addr & 0x3ffff) >> 4) | static_cast<uint64_t>(lead >> 4) << 16 | static_cast<uint64_t>(1024 >> 4) << 32 |
           1ull << 46 | 2ull << 61;
}

// FP16 operands, FP32 sums, 128 rows, n columns.
__host__ __device__ constexpr uint32_t product_desc(int n, bool b_transposed) {
    return 1u << 4 | (b_transposed ? 1u << 16 : 0u) | static_cast<uint32_t>(n >> 3) << 17 | (128u >> 4) << 24;
}

__device__ __forceinline__ void product_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t desc, bool add) {
    asm volatile("{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d), "l"(a), "l"(b),
                 "r"(desc), "r"(static_cast<uint32_t>(add)) : "memory");
}

__device__ __forceinline__ void product_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t desc, bool add) {
    asm volatile("{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d), "r"(a), "l"(b),
                 "r"(desc), "r"(static_cast<uint32_t>(add)) : "memory");
}

#define I4D_R8(x, i) "=r"(x[i]), "=r"(x[i + 1]), "=r"(x[i + 2]), "=r"(x[i + 3]), "=r"(x[i + 4]), "=r"(x[i + 5]), "=r"(x[i + 6]), "=r"(x[i + 7])
#define I4D_W8(x, i) "r"(x[i]), "r"(x[i + 1]), "r"(x[i + 2]), "r"(x[i + 3]), "r"(x[i + 4]), "r"(x[i + 5]), "r"(x[i + 6]), "r"(x[i + 7])

// 32 columns of the warp's 32 lanes of tensor memory, a lane a thread.
__device__ __forceinline__ void tmem_load32(uint32_t at, uint32_t x[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,"
        "%28,%29,%30,%31}, [%32];"
        : I4D_R8(x, 0), I4D_R8(x, 8), I4D_R8(x, 16), I4D_R8(x, 24)
        : "r"(at));
}
__device__ __forceinline__ void tmem_store32(uint32_t at, const uint32_t x[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,"
        "%27,%28,%29,%30,%31,%32};" ::"r"(at),
        I4D_W8(x, 0), I4D_W8(x, 8), I4D_W8(x, 16), I4D_W8(x, 24)
        : "memory");
}
__device__ __forceinline__ void tmem_store16(uint32_t at, const uint32_t x[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(at), I4D_W8(x, 0),
                 I4D_W8(x, 8)
                 : "memory");
}
// The loaded registers hold their values behind this point.
__device__ __forceinline__ void tmem_wait_load(uint32_t x[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(x[0]), "+r"(x[1]), "+r"(x[2]), "+r"(x[3]), "+r"(x[4]), "+r"(x[5]), "+r"(x[6]), "+r"(x[7]), "+r"(x[8]), "+r"(x[9]), "+r"(x[10]),
                   "+r"(x[11]), "+r"(x[12]), "+r"(x[13]), "+r"(x[14]), "+r"(x[15]), "+r"(x[16]), "+r"(x[17]), "+r"(x[18]), "+r"(x[19]), "+r"(x[20]),
                   "+r"(x[21]), "+r"(x[22]), "+r"(x[23]), "+r"(x[24]), "+r"(x[25]), "+r"(x[26]), "+r"(x[27]), "+r"(x[28]), "+r"(x[29]), "+r"(x[30]),
                   "+r"(x[31])::"memory");
}
__device__ __forceinline__ void tmem_load16(uint32_t at, uint32_t x[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];" : I4D_R8(x, 0), I4D_R8(x, 8) : "r"(at));
}
__device__ __forceinline__ void tmem_wait_load16(uint32_t x[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(x[0]), "+r"(x[1]), "+r"(x[2]), "+r"(x[3]), "+r"(x[4]), "+r"(x[5]), "+r"(x[6]), "+r"(x[7]), "+r"(x[8]), "+r"(x[9]), "+r"(x[10]),
                   "+r"(x[11]), "+r"(x[12]), "+r"(x[13]), "+r"(x[14]), "+r"(x[15])::"memory");
}
// 2^x for a whole x <= 0; -inf and NaN (of two -inf) 0.
__device__ __forceinline__ float whole_ex2(float x) { return x >= -126.f ? __int_as_float((static_cast<int>(x) + 127) << 23) : 0.f; }
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ float max16(const uint32_t* x) {
    const float* y = reinterpret_cast<const float*>(x);
    const float a = max3(y[0], y[1], y[2]), b = max3(y[3], y[4], y[5]), c = max3(y[6], y[7], y[8]), d = max3(y[9], y[10], y[11]), e = max3(y[12], y[13], y[14]);
    return max3(max3(a, b, c), max3(d, e, y[15]), c);
}
// Two FP32 operations an instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{\n .reg .b64 a, b, c, d;\n mov.b64 a, {%2, %3};\n mov.b64 b, {%4, %5};\n mov.b64 c, {%6, %7};\n fma.rn.f32x2 d, a, b, c;\n mov.b64 {%0, %1}, d;\n}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 d;
    asm("{\n .reg .b64 a, b, d;\n mov.b64 a, {%2, %3};\n mov.b64 b, {%4, %5};\n mul.rn.f32x2 d, a, b;\n mov.b64 {%0, %1}, d;\n}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("{\n .reg .b64 a, b, d;\n mov.b64 a, {%2, %3};\n mov.b64 b, {%4, %5};\n add.rn.f32x2 d, a, b;\n mov.b64 {%0, %1}, d;\n}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ void tmem_wait_store() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// One token row of codes (128 or 64 bytes with the copy's swizzle) to halves
// in an operand's row; zeros for a row that is not there.
template <int DT, int CODE>
__device__ __forceinline__ void convert_row(uint32_t raw, uint32_t to, int row, bool there) {
    uint4 w[DT / 16];
#pragma unroll
    for (int c = 0; c < DT / 16; ++c) {
        const uint32_t from = DT == 64 ? raw + row * 64 + ((c ^ (row >> 1 & 3)) << 4) : raw + row * 128 + ((c ^ (row & 7)) << 4);
        w[c] = lds16(from);
    }
#pragma unroll
    for (int c = 0; c < DT / 16; ++c) {
        if (!there) w[c] = make_uint4(0, 0, 0, 0);
        const uint32_t ws[4] = {w[c].x, w[c].y, w[c].z, w[c].w};
        uint32_t h[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (CODE == I4D_CODE_INT8) {
                const uint32_t x = ws[i] ^ 0x80808080u;
                const __half2 bias = __half2half2(__ushort_as_half(0x6480));
                const uint32_t m0 = __byte_perm(x, 0x64646464u, 0x4140), m1 = __byte_perm(x, 0x64646464u, 0x4342);
                const __half2 h0 = __hsub2(*reinterpret_cast<const __half2*>(&m0), bias), h1 = __hsub2(*reinterpret_cast<const __half2*>(&m1), bias);
                h[2 * i] = *reinterpret_cast<const uint32_t*>(&h0);
                h[2 * i + 1] = *reinterpret_cast<const uint32_t*>(&h1);
            } else {
                const uint16_t lo = static_cast<uint16_t>(ws[i]), hi = static_cast<uint16_t>(ws[i] >> 16);
                asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h[2 * i]) : "h"(lo));
                asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h[2 * i + 1]) : "h"(hi));
            }
        }
        const uint32_t line = to + (c >> 2) * 16384 + row * 128;
#pragma unroll
        for (int p = 0; p < 2; ++p)
            asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(line + ((((c & 3) * 2 + p) ^ (row & 7)) << 4)), "r"(h[4 * p]), "r"(h[4 * p + 1]),
                         "r"(h[4 * p + 2]), "r"(h[4 * p + 3])
                         : "memory");
    }
}

__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// Token tiles of row tile rt of a sequence, from token `begin`.
struct PrSpan {
    int tiles, begin, end, live;  // live rows
};
__device__ __forceinline__ PrSpan prompt_span(const AttnDev& a, const Seq& s, int rt) {
    const int rows = s.n * a.group, row0 = rt * kPrRows, first = s.len - s.n;
    if (s.len > a.max_length || row0 >= rows) return {0, 0, 0, 0};
    const int live = min(kPrRows, rows - row0);
    const int begin = row_span(a, first + row0 / a.group).x & ~15, end = row_span(a, first + (row0 + live - 1) / a.group).y;
    return {(end - begin + kPrTokens - 1) / kPrTokens, begin, end, live};
}

// Units of the batch (token tiles of 128 for each sequence, row tile, head, in
// this order) and the pair (sequence * row tiles + row tile) in which unit
// u(total) lies, with the units before it.  WARPS warps take consecutive pairs.
template <int WARPS, typename U>
__device__ __forceinline__ int64_t find_prompt(const AttnDev& a, U&& unit, bool report, int64_t* sums, int64_t* before_out, int* pair_out) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t pairs = static_cast<int64_t>(a.batch) * a.row_tiles, per = (pairs + WARPS * 32 - 1) / (WARPS * 32);
    const int64_t p0 = min(pairs, threadIdx.x * per), p1 = min(pairs, p0 + per);
    auto size = [&](int64_t p, bool tell) {
        const int b = static_cast<int>(p / a.row_tiles), rt = static_cast<int>(p % a.row_tiles);
        const Seq s = load_seq(a.seq, b, tell && rt == 0);
        if (tell && rt == 0 && s.len > a.max_length) atomicOr(a.seq.err, kBadSequence);
        return static_cast<int64_t>(prompt_span(a, s, rt).tiles) * a.cache.heads;
    };
    int64_t mine = 0;
    for (int64_t p = p0; p < p1; ++p) mine += size(p, report);
    int64_t upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t x = __shfl_up_sync(~0u, upto, o);
        if (lane >= o) upto += x;
    }
    if (lane == 31) sums[warp] = upto;
    __syncthreads();
    int64_t total = 0;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
        if (w < warp) upto += sums[w];
        total += sums[w];
    }
    const int64_t u = unit(total);
    int64_t before = upto - mine;
    if (u >= before && u < upto)
        for (int64_t p = p0; p < p1; ++p) {
            const int64_t next = before + size(p, false);
            if (u < next) {
                *before_out = before;
                *pair_out = static_cast<int>(p);
                break;
            }
            before = next;
        }
    __syncthreads();
    return total;
}

// Calls f for each of a CTA's pieces in turn until it returns false: token
// tiles [j0, j1) of a (sequence, row tile, head).
struct PrPiece {
    Seq s;
    PrSpan span;
    int b, rt, h, j0, j1, slot;  // slot: where partial sums go, 0 the CTA's first piece, 1 its last
    bool whole;
};
template <typename F>
__device__ __forceinline__ void each_piece(const AttnDev& a, int64_t u, int64_t u_end, int64_t before, int pair, F&& f) {
    const int64_t u0 = u;
    while (u < u_end) {
        PrPiece p;
        p.b = pair / a.row_tiles;
        p.rt = pair % a.row_tiles;
        p.s = load_seq(a.seq, p.b, false);
        p.span = prompt_span(a, p.s, p.rt);
        const int64_t next = before + static_cast<int64_t>(p.span.tiles) * a.cache.heads;
        if (u >= next) {
            before = next;
            ++pair;
            continue;
        }
        p.h = static_cast<int>((u - before) / p.span.tiles);
        const int64_t first = before + static_cast<int64_t>(p.h) * p.span.tiles;
        p.j0 = static_cast<int>(u - first);
        p.j1 = static_cast<int>(min(static_cast<int64_t>(p.span.tiles), u_end - first));
        p.whole = p.j0 == 0 && p.j1 == p.span.tiles;
        p.slot = u == u0 ? 0 : 1;
        if (!f(p)) return;
        u = first + p.j1;
    }
}

// HLP: probabilities in two parts, which both lie in place of their own scores.
template <int DT, int CODE, bool HLP>
__global__ void __launch_bounds__(kPrThreads, 1) k_kv8_prompt(const __grid_constant__ AttnDev a) {
    op_begin();
    using L = PromptSmem<DT>;
    extern __shared__ unsigned char pr_base[];
    __shared__ PrShared sh;
    const uint32_t base_raw = static_cast<uint32_t>(__cvta_generic_to_shared(pr_base));
    const uint32_t base = (base_raw + 1023u) & ~1023u;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int bs = a.cache.block_tokens, shift = 31 - __clz(bs), dim = a.cache.dim;
    // The CTA's even share of the units.
    int64_t u, u_end;
    {
        int64_t share = 0;
        const int64_t total = find_prompt<kPrWarps>(a, [&](int64_t n) {
            share = (n + gridDim.x - 1) / gridDim.x;
            return share * blockIdx.x;
        }, blockIdx.x == 0, sh.sums, &sh.before, &sh.pair);
        u = share * blockIdx.x;
        u_end = min(total, u + share);
    }
    if (u >= u_end) return;
    const int64_t before = sh.before;
    const int pair = sh.pair;

    if (threadIdx.x == 0) {
        for (int i = 0; i < kPrBars; ++i) {
            const bool warps = (i >= kRawKEmpty && i < kKEmpty) || i == kVFull || (i >= kPFull && i < kPvDone) || i == kQFull || i == kQFull + 1 || i == kFirstP;
            const int count = warps ? 4 : (i >= kKEmpty && i < kVFull) || i == kVEmpty ? 2 : 1;
            bar_init(bar_at(sh, i), count);
        }
        sh.abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 13) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(&sh.tmem))) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        fence_before();
    }
    __syncthreads();
    fence_after();
    const uint32_t tmem = sh.tmem;

    if (warp == 12) {  // ------------------------------------------- producer
        constexpr int kBoxBytes = 16 * DT;
        int n = 0;  // tiles so far, over all pieces
        int sent[2] = {0, 0};  // of K, of V
        each_piece(a, u, u_end, before, pair, [&](const PrPiece& p) {
            bool ok = true;
            for (int j = p.j0; ok && j < p.j1; ++j, ++n) {
                const int st = n & 1, at = p.span.begin + kPrTokens * j + 16 * lane;
                int id = -1;
                float4 entry = make_float4(0.f, 0.f, -INFINITY, 0.f);
                if (lane < 8 && at < p.span.end) {
                    id = load_block(a.seq, p.b, at >> shift, true);
                    if (id >= 0) {
                        const int64_t sc = static_cast<int64_t>(id) * a.cache.heads + p.h;
                        entry.x = fetch(a.cache.scale[0] + sc);
                        entry.y = fetch(a.cache.scale[1] + sc);
                        entry.z = __log2f(entry.y);  // only a bound: its rounding cancels
                    }
                }
                const int row = (id * a.cache.heads + p.h) * bs + (at & (bs - 1));
                const unsigned found = __ballot_sync(~0u, id >= 0);
                const int bytes = __popc(found) * kBoxBytes;
#pragma unroll
                for (int which = 0; which < 2; ++which) {
                    ok = __all_sync(~0u, pr_wait(sh, (which ? kRawVEmpty : kRawKEmpty) + st, (n >> 1 & 1) ^ 1));
                    if (!ok) break;
                    if (!which) {
                        if (lane < 8) sh.table[n & 3][lane] = entry;
                        if (lane == 0) sh.missing[n & 3] = ~found & 0xff;
                        __syncwarp();
                    }
                    const uint32_t bar = bar_at(sh, (which ? kRawVFull : kRawKFull) + st);
                    if (lane == 0) asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
                    __syncwarp();
                    if (id >= 0)
                        asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
                                         base + L::raw + (st * 2 + which) * L::kRaw + lane * kBoxBytes),
                                     "l"(&a.maps[which]), "r"(0), "r"(row), "r"(bar)
                                     : "memory");
                    ++sent[which];
                }
            }
            return ok;
        });
        if (sh.abort)  // copies in flight land before the CTA leaves
#pragma unroll
            for (int which = 0; which < 2; ++which)
                for (int j = max(0, sent[which] - 2); j < sent[which]; ++j)
                    bar_wait(bar_at(sh, (which ? kRawVFull : kRawKFull) + (j & 1)), j >> 1 & 1);
    } else if (warp >= 13) {  // ------------------------------------- products
        const int t = warp - 13;  // the row tile
        if (lane == 0) {
            constexpr uint32_t kScores = product_desc(64, false), kValues = product_desc(DT, true);
            const uint32_t s_at = tmem + t * 128, o_at = tmem + 256 + t * 128;
            const uint64_t q_desc = operand_desc(base + L::q + t * L::kOperand, 16), k_desc = operand_desc(base + L::k, 16),
                           v_desc = operand_desc(base + L::v, L::kBlock);
            // Token tiles of all pieces; of those with rows in this row tile,
            // whose barriers count them; pieces with such rows.
            int n = 0, m = 0, pieces = 0;
            bool ok = true;
            each_piece(a, u, u_end, before, pair, [&](const PrPiece& p) {
                const int count = p.j1 - p.j0;
                if (t * 128 >= p.span.live) {  // nothing here for this row tile: it only gives the buffers on
                    for (int j = 0; ok && j < count; ++j, ++n) {
                        ok = pr_wait(sh, kKFull + (n & 1), n >> 1 & 1);
                        if (ok) pr_arrive(sh, kKEmpty + (n & 1));
                        ok = ok && pr_wait(sh, kVFull, n & 1);
                        if (ok) pr_arrive(sh, kVEmpty);
                    }
                    return ok;
                }
                ok = pr_wait(sh, kQFull + t, pieces++ & 1);
                // Tile 1 begins when tile 0 has its first probabilities: the
                // one's products then run under the other's softmax.  (Not by
                // kPFull, whose phases tile 0 goes on through: tile 1, with rows
                // that come late, would find it two on and wait for good.)
                if (t == 1 && n == 0) ok = ok && pr_wait(sh, kFirstP, 0);
                for (int j = 0; ok && j <= count; ++j) {
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        const int at = 2 * t + half;
                        // O takes P of 64 tokens from the tensor memory that the
                        // scores of the next tile's 64 then go to.
                        if (j > 0) {
                            ok = ok && pr_wait(sh, kVFull, (n + j - 1) & 1) && pr_wait(sh, kPFull + at, (m + j - 1) & 1);
                            if (!ok) break;
                            fence_after();
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const uint32_t p = s_at + half * 64 + (HLP ? (i >> 1) * 32 + (i & 1) * 8 : i * 8);
                                const uint64_t vd = v_desc + ((4 * half + i) * 2048 >> 4);
                                product_ts(o_at, p, vd, kValues, j > 1 || half > 0 || i > 0);
                                if constexpr (HLP) product_ts(o_at, p + 16, vd, kValues, true);
                            }
                            pr_commit(sh, kPvDone + at);
                            if (half) pr_commit(sh, kVEmpty);
                            if (j == count) continue;
                            ok = pr_wait(sh, kPvDone + at, (m + j - 1) & 1);
                        }
                        ok = ok && pr_wait(sh, kKFull + ((n + j) & 1), (n + j) >> 1 & 1);
                        if (!ok) break;
                        fence_after();
                        const uint64_t kd = k_desc + ((((n + j) & 1) * L::kOperand + half * 8192) >> 4);
#pragma unroll
                        for (int i = 0; i < DT / 16; ++i) {
                            const int step = ((i >> 2) * L::kBlock + (i & 3) * 32) >> 4;
                            product_ss(s_at + half * 64, q_desc + step, kd + step, kScores, i > 0);
                        }
                        pr_commit(sh, kSFull + at);
                        if (half) pr_commit(sh, kKEmpty + ((n + j) & 1));
                    }
                }
                pr_commit(sh, kODone + t);
                n += count;
                m += count;
                return ok;
            });
            if (!ok && pieces) bar_wait(bar_at(sh, kODone + t), (pieces - 1) & 1);  // products in flight end before the CTA leaves
        }
        __syncwarp();
    } else if (warp >= 8) {  // --------------------------------------- converters
        const int row = threadIdx.x - 256;
        int n = 0;
        each_piece(a, u, u_end, before, pair, [&](const PrPiece& p) {
            for (int j = p.j0; j < p.j1; ++j, ++n) {
                const int st = n & 1;
                if (!__all_sync(~0u, pr_wait(sh, kRawKFull + st, n >> 1 & 1) && pr_wait(sh, kKEmpty + st, (n >> 1 & 1) ^ 1))) return false;
                const bool there = p.span.begin + kPrTokens * j + row < p.s.len && !(sh.missing[n & 3] >> (row >> 4) & 1);
                convert_row<DT, CODE>(base + L::raw + st * 2 * L::kRaw, base + L::k + st * L::kOperand, row, true);
                fence_async();
                __syncwarp();
                if (lane == 0) {
                    pr_arrive(sh, kKFull + st);
                    pr_arrive(sh, kRawKEmpty + st);
                }
                if (!__all_sync(~0u, pr_wait(sh, kRawVFull + st, n >> 1 & 1) && pr_wait(sh, kVEmpty, (n & 1) ^ 1))) return false;
                convert_row<DT, CODE>(base + L::raw + (st * 2 + 1) * L::kRaw, base + L::v, row, there);
                fence_async();
                __syncwarp();
                if (lane == 0) {
                    pr_arrive(sh, kVFull);
                    pr_arrive(sh, kRawVEmpty + st);
                }
            }
            return true;
        });
    } else {  // ------------------------------------------------------- softmax
        const int tile = warp >> 2, r = threadIdx.x & 127;
        int n = 0, m = 0, pieces = 0;  // as in the products' threads
        each_piece(a, u, u_end, before, pair, [&](const PrPiece& piece) {
        const int count = piece.j1 - piece.j0;
        if (tile * 128 >= piece.span.live) {
            n += count;
            return true;
        }
        const Seq& s = piece.s;
        const int first = s.len - s.n, row0 = piece.rt * kPrRows, row = row0 + tile * 128 + r, rows = s.n * a.group, h = piece.h;
        const bool mine = row < rows;
        const int64_t tok = s.first + row / a.group;
        const int head = h * a.group + row % a.group;
        float down = 0.f;
        {  // the row to FP16: two passes over memory, the largest value, then the halves
            const int64_t at = mine ? tok * a.q_tok + head * a.q_head : 0;
            float top = 0.f, x[16];
            for (int c = 0; mine && c < dim / 16; ++c) {
                load_q16(a, at + 16 * c, x);
#pragma unroll
                for (int i = 0; i < 16; ++i) top = fmaxf(top, fabsf(x[i]));
            }
            const int e = max(-115, min(126, 13 - ((__float_as_int(top) >> 23) - 127)));
            float up = __int_as_float((e + 127) << 23);
            down = __int_as_float((127 - e) << 23) * fabsf(a.scale_log2);
            if (a.scale_log2 < 0.f) up = -up;
            for (int c = 0; c < DT / 16; ++c) {
                uint32_t w[8];
                if (mine && 16 * c < dim) {
                    load_q16(a, at + 16 * c, x);
#pragma unroll
                    for (int i = 0; i < 8; ++i) w[i] = pack_h2(x[2 * i] * up, x[2 * i + 1] * up);
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i) w[i] = 0;
                }
                const uint32_t line = base + L::q + tile * L::kOperand + (c >> 2) * L::kBlock + r * 128;
#pragma unroll
                for (int p = 0; p < 2; ++p)
                    asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(line + ((((c & 3) * 2 + p) ^ (r & 7)) << 4)), "r"(w[4 * p]), "r"(w[4 * p + 1]),
                                 "r"(w[4 * p + 2]), "r"(w[4 * p + 3])
                                 : "memory");
            }
            fence_async();
            __syncwarp();
            if (lane == 0) pr_arrive(sh, kQFull + tile);
        }
        const uint32_t quarter = static_cast<uint32_t>(warp & 3) << 21;  // lanes 32 (warp % 4) of tensor memory
        const uint32_t s_at = tmem + quarter + tile * 128, o_at = tmem + quarter + 256 + tile * 128;
        const int2 span = row_span(a, first + row / a.group);
        const int tile_last = min(row0 + tile * 128 + 127, row0 + piece.span.live - 1);
        const int all_from = row_span(a, first + tile_last / a.group).x, all_to = min(s.len, row_span(a, first + (row0 + tile * 128) / a.group).y);
        float M = -INFINITY, R = -INFINITY, to_r = 0.f, off = 0.f;
        float2 sum[2] = {{0.f, 0.f}, {0.f, 0.f}};
        bool ok = true;
        for (int j = 0; ok && j < count; ++j) {
            const int at = piece.span.begin + kPrTokens * (piece.j0 + j), parity = (m + j) & 1;
            int missing = 0;
            bool whole = false;
            const float4* table = sh.table[(n + j) & 3];
            // 32 scores to probabilities, which overlay those of their half of the tile.
            // (HLP: of their own chunk, the second parts 16 columns behind the first)
            auto p_at = [&](int c) { return s_at + (c >> 1) * 64 + (c & 1) * (HLP ? 32 : 16); };
            auto chunk = [&](uint32_t (&x)[32], int c) {
                if (!whole) {  // scores that the row does not see
                    const int lo = min(32, max(0, span.x - at - 32 * c)), hi = min(32, max(lo, min(span.y, s.len) - at - 32 * c));
                    uint32_t seen = static_cast<uint32_t>((1ull << hi) - (1ull << lo));
                    if (missing >> (2 * c) & 1) seen &= 0xffff0000u;
                    if (missing >> (2 * c + 1) & 1) seen &= 0x0000ffffu;
#pragma unroll
                    for (int i = 0; i < 32; ++i)
                        if (!(seen >> i & 1)) x[i] = 0xff800000u;
                }
                const float4 b0 = table[2 * c], b1 = table[2 * c + 1];
                // (a factor of zero would make NaN of what is not seen)
                const float f0 = fmaxf(down * b0.x, 1e-37f), f1 = fmaxf(down * b1.x, 1e-37f);
                const float m0 = max16(x) * f0, m1 = max16(x + 16) * f1;
                const float top = fmaxf(m0, m1), rtop = fmaxf(m0 + b0.z, m1 + b1.z);
                uint32_t p[16], pl[HLP ? 16 : 1];
                float2 part[2];
                for (;;) {
                    // With the bounds as they are; if a score passes them, again with raised ones.
#pragma unroll
                    for (int g = 0; g < 2; ++g) {
                        const float2 f = g ? make_float2(f1, f1) : make_float2(f0, f0), o = make_float2(-off, -off);
                        const float wv = weight_unit(to_r, g ? b1.y : b0.y);
                        const float2 w = make_float2(wv, wv);
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const float2 y = fma2(make_float2(__uint_as_float(x[16 * g + 2 * i]), __uint_as_float(x[16 * g + 2 * i + 1])), f, o);
                            const float2 e = make_float2(ex2(y.x), ex2(y.y));
                            part[g] = i ? add2(part[g], e) : e;
                            const float2 z = mul2(e, w);
                            p[8 * g + i] = pack_h2(z.x, z.y);
                            if constexpr (HLP) pl[8 * g + i] = second_part<kTwoParts>(z.x, z.y, p[8 * g + i]);
                        }
                    }
                    const bool raise = top > M + kSlack || rtop > R + (kSlack + kHead);
                    if (!__any_sync(~0u, raise)) break;
                    // (whole powers of two: the sums and the halves so far are scaled exactly)
                    const float m = raise ? fmaxf(top, M) : M, rr = raise ? ceilf(fmaxf(fmaxf(rtop - kHead, R), m - kFarScales)) : R;
                    const float fm = M == m ? 1.f : ex2(M - m), f = whole_ex2(R - rr);
                    sum[0].x *= fm;
                    sum[0].y *= fm;
                    sum[1].x *= fm;
                    sum[1].y *= fm;
                    M = m;
                    R = rr;
                    off = M == -INFINITY ? 0.f : M;
                    to_r = R == -INFINITY ? 0.f : ex2(M - R);
                    // O so far (with the products before this half of the tile), and the half's P so far
                    tmem_wait_store();
                    const bool any_o = j > 0 || c > 1;
                    if (any_o) {
                        ok = __all_sync(~0u, pr_wait(sh, kPvDone + 2 * tile + (c < 2), c < 2 ? parity ^ 1 : parity)) && ok;
                        fence_after();
                    }
                    uint32_t y[16];
#pragma unroll 1
                    for (int k = 0; any_o && k < DT / 16; ++k) {
                        tmem_load16(o_at + 16 * k, y);
                        tmem_wait_load16(y);
#pragma unroll
                        for (int i = 0; i < 16; ++i) y[i] = __float_as_uint(__uint_as_float(y[i]) * f);
                        tmem_store16(o_at + 16 * k, y);
                    }
#pragma unroll 1
                    for (int k = 0; k < (c & 1) * (HLP ? 2 : 1); ++k) {  // (in FP32: FP16 may not hold the factor where it holds the product)
                        tmem_load16(p_at(c - 1) + 16 * k, y);
                        tmem_wait_load16(y);
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            const float2 z = __half22float2(*reinterpret_cast<const __half2*>(&y[i]));
                            y[i] = pack_h2(z.x * f, z.y * f);
                        }
                        tmem_store16(p_at(c - 1) + 16 * k, y);
                    }
                }
                sum[0] = add2(sum[0], part[0]);
                sum[1] = add2(sum[1], part[1]);
                tmem_store16(p_at(c), p);
                if constexpr (HLP) tmem_store16(p_at(c) + 16, pl);
            };
#pragma unroll 1
            for (int half = 0; half < 2; ++half) {
                ok = ok && __all_sync(~0u, pr_wait(sh, kSFull + 2 * tile + half, parity));
                if (!ok) break;
                fence_after();
                missing = sh.missing[(n + j) & 3];
                whole = at >= all_from && at + kPrTokens <= all_to && !missing;
#pragma unroll 1
                for (int c = 2 * half; c < 2 * half + 2; ++c) {
                    uint32_t x[32];
                    tmem_load32(s_at + 32 * c, x);
                    tmem_wait_load(x);
                    chunk(x, c);
                }
                tmem_wait_store();
                fence_before();
                __syncwarp();
                if (lane == 0) {
                    pr_arrive(sh, kPFull + 2 * tile + half);
                    if (tile + half + n + j == 0) pr_arrive(sh, kFirstP);
                }
            }
        }
        const float l = (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
        if (!ok || !__all_sync(~0u, pr_wait(sh, kODone + tile, pieces & 1))) return false;
        fence_after();
        const float back = !piece.whole ? 1.f : l == 0.f || R == -INFINITY ? 0.f : ex2(R - M) / l;
        const int64_t part = (static_cast<int64_t>(blockIdx.x) * 2 + piece.slot) * kPrRows + tile * 128 + r;
#pragma unroll
        for (int c = 0; c < DT / 32; ++c) {
            uint32_t x[32];
            __syncwarp();
            tmem_load32(o_at + 32 * c, x);
            tmem_wait_load(x);
            if (!mine) continue;
            if (!piece.whole) {
#pragma unroll
                for (int i = 0; i < 32; i += 4)
                    if (32 * c + i < dim) *reinterpret_cast<uint4*>(a.part + part * dim + 32 * c + i) = make_uint4(x[i], x[i + 1], x[i + 2], x[i + 3]);
                continue;
            }
            const int64_t to = tok * a.out_tok + head * a.out_head + 32 * c;
#pragma unroll
            for (int i = 0; i < 32; i += 8) {
                if (32 * c + i >= dim) break;
                uint32_t w[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float y0 = __uint_as_float(x[i + 2 * k]) * back, y1 = __uint_as_float(x[i + 2 * k + 1]) * back;
                    if (a.dtype == I4D_BF16) {
                        const __nv_bfloat162 y = __floats2bfloat162_rn(y0, y1);
                        w[k] = *reinterpret_cast<const uint32_t*>(&y);
                    } else {
                        w[k] = pack_h2(y0, y1);
                    }
                }
                unsigned short* out = static_cast<unsigned short*>(a.out) + to + i;
                if (a.wide_out) {
                    *reinterpret_cast<uint4*>(out) = make_uint4(w[0], w[1], w[2], w[3]);
                } else {
#pragma unroll
                    for (int k = 0; k < 8; ++k) out[k] = static_cast<unsigned short>(w[k / 2] >> (16 * (k & 1)));
                }
            }
        }
        if (mine) {
            if (piece.whole) {
                const float l2 = l == 0.f ? -INFINITY : M + log2f(l);
                if (a.lse) a.lse[tok * a.heads + head] = l2 * kLn2;
                if (a.weights) a.lse2[tok * a.heads + head] = l2 == -INFINITY ? INFINITY : l2;
            } else {
                a.stats[part] = make_float4(M, l, R, 0.f);
            }
        }
        fence_before();
        n += count;
        m += count;
        ++pieces;
        __syncwarp();
        return true;
        });
    }
    fence_before();
    __syncthreads();
    if (warp == 13) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
    if (threadIdx.x == 0 && sh.abort) atomicOr(a.seq.err, kTimeout);
}

// Joins the pieces of a segment that several CTAs of k_kv8_prompt shared:
// blockIdx.x / 8 + 1 is the first CTA whose share begins inside the segment,
// blockIdx.x % 8 the 32 rows.
__global__ void __launch_bounds__(256) k_kv8_prompt_join(AttnDev a) {
    op_begin();
    __shared__ int64_t s_sums[8], s_before;
    __shared__ int s_pair;
    const int c = blockIdx.x / 8 + 1, lane = threadIdx.x & 31, dim = a.cache.dim;
    int64_t share = 0;
    const int64_t total = find_prompt<8>(a, [&](int64_t n) {
        share = (n + a.even - 1) / a.even;
        return share * c;
    }, false, s_sums, &s_before, &s_pair);
    const int64_t u = share * c;
    if (u >= total) return;
    const int b = s_pair / a.row_tiles, rt = s_pair % a.row_tiles;
    const Seq s = load_seq(a.seq, b, false);
    const PrSpan span = prompt_span(a, s, rt);
    const int h = static_cast<int>((u - s_before) / span.tiles);
    const int64_t seg0 = s_before + static_cast<int64_t>(h) * span.tiles, seg1 = seg0 + span.tiles;
    if (u == seg0 || u - share > seg0) return;  // no CTA's share begins inside, or an earlier one's does
    const int c0 = c - 1, c1 = static_cast<int>((seg1 - 1) / share);
    // Four rows a warp, eight lanes each, so that all their loads are on their way at once.
    const int sub = lane & 7, r = (blockIdx.x & 7) * 32 + (threadIdx.x >> 3);
    const bool live = r < span.live;
    // the first CTA's last piece (or its only one), the others' first
    auto index = [&](int k) { return (static_cast<int64_t>(k) * 2 + (k == c0 && share * c0 < seg0 ? 1 : 0)) * kPrRows + (live ? r : 0); };
    float m = -INFINITY, rr = -INFINITY, sum = 0.f;
    for (int k = c0 + sub; k <= c1; k += 8) {
        const float4 x = a.stats[index(k)];
        m = fmaxf(m, x.x);
        rr = fmaxf(rr, x.z);
    }
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) {
        m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
        rr = fmaxf(rr, __shfl_xor_sync(~0u, rr, o));
    }
    float4 acc[4] = {};
#pragma unroll 2
    for (int k = c0; k <= c1; ++k) {
        const float4 x = a.stats[index(k)];
        const float4* part = reinterpret_cast<const float4*>(a.part + index(k) * dim);
        float4 y[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) y[j] = 4 * (8 * j + sub) < dim ? part[8 * j + sub] : make_float4(0.f, 0.f, 0.f, 0.f);
        sum += x.y * (x.x == -INFINITY ? 1.f : ex2(x.x - m));
        const float f = x.z == -INFINITY ? 1.f : ex2(x.z - rr);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            acc[j].x += y[j].x * f;
            acc[j].y += y[j].y * f;
            acc[j].z += y[j].z * f;
            acc[j].w += y[j].w * f;
        }
    }
    if (!live) return;
    const float back = sum == 0.f || rr == -INFINITY ? 0.f : ex2(rr - m) / sum;
    const int row = rt * kPrRows + r;
    const int64_t tok = s.first + row / a.group;
    const int head = h * a.group + row % a.group;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if (4 * (8 * j + sub) >= dim) continue;
        store_out4(a, tok * a.out_tok + head * a.out_head + 4 * (8 * j + sub),
                   make_float4(acc[j].x * back, acc[j].y * back, acc[j].z * back, acc[j].w * back));
    }
    if (sub == 0) {
        const float l2 = sum == 0.f ? -INFINITY : m + log2f(sum);
        if (a.lse) a.lse[tok * a.heads + head] = l2 * kLn2;
        if (a.weights) a.lse2[tok * a.heads + head] = l2 == -INFINITY ? INFINITY : l2;
    }
}

}  // namespace i4d_ops
