// i4d_kv8_cache.cuh -- the paged cache of 8-bit codes: append, read, evict.
//
// A value is code * scale, one scale for each (block of tokens, head) of K and
// of V.  Appended blocks get a scale that is a power of two: divisions by it
// are exact, so a code depends on its value and scale alone, and when a later
// token raises the scale of a partly filled block, rewriting the older codes
// is a shift with one rounding; all such roundings of a code sum to less than
// one step of the last scale (1/2 + 1/4 + ...).
#pragma once

#include "i4d_ops_common.cuh"

namespace i4d_ops {

struct Kv8Dev {
    uint8_t* codes[2];  // K, V: [blocks][heads][block_tokens][dim]
    float* scale[2];    // [blocks][heads]
    int heads, dim, block_tokens;
};

__device__ __forceinline__ int64_t code_offset(const Kv8Dev& c, int block, int head) {
    return (static_cast<int64_t>(block) * c.heads + head) * c.block_tokens * c.dim;
}

// ---------------------------------------------------------------- append

struct AppendDev {
    Kv8Dev cache;
    SeqArrays seq;
    const void* in[2];
    int64_t tok[2], head[2];
    int touched;  // blocks that a sequence of max_q new tokens can touch
};

template <typename T, int V>
__device__ __forceinline__ void load8(const T* p, float out[8]) {
    if constexpr (V == 8) {
        const Vec<T, 8> x = load_vec<T, 8>(p);
#pragma unroll
        for (int i = 0; i < 8; ++i) out[i] = to_f32(x.v[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) out[i] = to_f32(p[i]);
    }
}

// One unit (sequence, touched block, head, K or V) for each group of
// THREADS threads.  Two passes over the new values: the largest, then the
// codes (the second pass reads L1/L2).  Bound: the values in, the codes out.
template <typename T, int V, int CODE, int THREADS>
__global__ void __launch_bounds__(THREADS < 128 ? 128 : THREADS) k_kv8_append(AppendDev a, int units) {
    constexpr int kPerCta = THREADS < 128 ? 128 / THREADS : 1;
    constexpr int kWarps = THREADS / 32;
    const int tid = threadIdx.x % THREADS;
    const int unit = blockIdx.x * kPerCta + threadIdx.x / THREADS;
    if (unit >= units) return;  // whole warps; CTAs of one unit never leave here
    const int which = unit & 1, h = (unit >> 1) % a.cache.heads;
    const int rest = (unit >> 1) / a.cache.heads;
    const int b = rest / a.touched, j = rest % a.touched;
    const bool report = which == 0 && h == 0 && tid == 0;
    const Seq s = load_seq(a.seq, b, report && j == 0);
    if (s.n == 0) return;
    const int bs = a.cache.block_tokens, dim = a.cache.dim;
    const int first = s.len - s.n, blk = first / bs + j;
    if (blk * bs >= s.len) return;
    const int id = load_block(a.seq, b, blk, report);
    if (id < 0) return;
    const int lo = max(first, blk * bs), hi = min(s.len, (blk + 1) * bs), old = lo - blk * bs;
    const T* in = static_cast<const T*>(a.in[which]) + static_cast<int64_t>(s.first + lo - first) * a.tok[which] +
                  h * a.head[which];
    float* scale = a.cache.scale[which] + static_cast<int64_t>(id) * a.cache.heads + h;
    const float had = old ? *scale : 0.f;
    const int per_tok = dim / 8, items = (hi - lo) * per_tok;
    float amax = 0.f;
    for (int i = tid; i < items; i += THREADS) {
        float x[8];
        load8<T, V>(in + static_cast<int64_t>(i / per_tok) * a.tok[which] + i % per_tok * 8, x);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const float m = fabsf(x[k]);
            amax = m < INFINITY ? fmaxf(amax, m) : amax;
        }
    }
    amax = warp_max(amax);
    if constexpr (kWarps > 1) {
        __shared__ float part[kWarps];
        if (threadIdx.x % 32 == 0) part[threadIdx.x / 32] = amax;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kWarps; ++w) amax = fmaxf(amax, part[w]);
    }
    const float now = fmaxf(power_scale(amax, CODE), had);
    if (tid == 0) *scale = now;  // every thread has read `had` (the barrier above, or the shuffles)
    uint8_t* codes = a.cache.codes[which] + code_offset(a.cache, id, h);
    if (old && now > had) {
        const float ratio = __fdiv_rn(had, now);
        uint2* p = reinterpret_cast<uint2*>(codes);
        for (int i = tid; i < old * per_tok; i += THREADS) {
            uint2 w = p[i];
            w.x = rescale4<CODE>(w.x, ratio);
            w.y = rescale4<CODE>(w.y, ratio);
            p[i] = w;
        }
    }
    const bool power = (__float_as_int(now) & 0x7fffff) == 0;
    const float inv = power ? __fdiv_rn(1.f, now) : 0.f;
    uint2* p = reinterpret_cast<uint2*>(codes + static_cast<int64_t>(old) * dim);
    for (int i = tid; i < items; i += THREADS) {
        float x[8];
        load8<T, V>(in + static_cast<int64_t>(i / per_tok) * a.tok[which] + i % per_tok * 8, x);
#pragma unroll
        for (int k = 0; k < 8; ++k) x[k] = power ? __fmul_rn(x[k], inv) : __fdiv_rn(x[k], now);
        p[i] = make_uint2(encode4<CODE>(x[0], x[1], x[2], x[3]), encode4<CODE>(x[4], x[5], x[6], x[7]));
    }
}

// ------------------------------------------------------------------ read

struct ReadDev {
    Kv8Dev cache;
    SeqArrays seq;
    __nv_bfloat16* out[2];
};

constexpr int kReadTokens = 16;

// One CTA for kReadTokens rows of a sequence: 16 codes in, 16 BF16 values out
// an item.  Bound: bytes.
template <int CODE>
__global__ void __launch_bounds__(256) k_kv8_read(ReadDev a, int chunks) {
    const int b = blockIdx.x / chunks, t0 = blockIdx.x % chunks * kReadTokens;
    const Seq s = load_seq(a.seq, b, threadIdx.x == 0 && t0 == 0);
    if (t0 >= s.n) return;
    const int rows = min(kReadTokens, s.n - t0), first = s.len - s.n + t0;
    const int bs = a.cache.block_tokens, per_head = a.cache.dim / 16, per_tok = a.cache.heads * per_head;
    for (int i = threadIdx.x; i < rows * per_tok; i += 256) {
        const int r = i / per_tok, e = i % per_tok, h = e / per_head, c = e % per_head;
        const int p = first + r, id = load_block(a.seq, b, p / bs, true);
        if (id < 0) continue;
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            const float scale = __ldg(a.cache.scale[which] + static_cast<int64_t>(id) * a.cache.heads + h);
            const uint4 w = __ldg(reinterpret_cast<const uint4*>(a.cache.codes[which] + code_offset(a.cache, id, h) +
                                                                 static_cast<int64_t>(p % bs) * a.cache.dim) + c);
            const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
            Vec<__nv_bfloat16, 16> o;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                float f[4];
                decode4<CODE>(ws[k], f);
#pragma unroll
                for (int m = 0; m < 4; ++m) o.v[4 * k + m] = __float2bfloat16_rn(f[m] * scale);
            }
            store_vec<__nv_bfloat16, 16>(a.out[which] + (static_cast<int64_t>(s.first + t0 + r) * a.cache.heads + h) * a.cache.dim + c * 16, o);
        }
    }
}

// ----------------------------------------------------------------- evict

struct EvictDev {
    Kv8Dev cache;
    SeqArrays seq;  // q_start unused
    const float* weights;
    float* weights_out;
    int64_t weights_stride, weights_out_stride;
    int32_t* lengths_out;
    int32_t* keep;
    float* old_scale;  // workspace [batch][heads][2][old_blocks]: scales before the move
    int old_blocks, budget, recent, max_length;
};

// Order of weights as unsigned numbers: greater weight, greater key; NaN 0,
// both zeros alike.
__device__ __forceinline__ uint32_t weight_key(float w) {
    if (!(w == w)) return 0u;
    const uint32_t u = __float_as_uint(w + 0.f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ int evict_length(const EvictDev& a, int b, bool report) {
    const int len = __ldg(a.seq.lengths + b);
    const bool ok = len >= 0 && len <= a.max_length;
    if (!ok && report) atomicOr(a.seq.err, kBadSequence);
    return ok ? len : 0;
}

constexpr int kSelectThreads = 1024;

// Inclusive sum over the CTA of one value a thread; *total receives the sum.
__device__ __forceinline__ int cta_scan(int x, int* warp_sums, int* total) {
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(~0u, x, o);
        if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == 31) warp_sums[w] = x;
    __syncthreads();
    if (w == 0) {
        int y = warp_sums[lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int z = __shfl_up_sync(~0u, y, o);
            if (lane >= o) y += z;
        }
        warp_sums[lane] = y;
    }
    __syncthreads();
    *total = warp_sums[31];
    return x + (w ? warp_sums[w - 1] : 0);
}

// One CTA for each (sequence, head): the key of the (budget - recent)-th
// greatest weight by four passes over 8 bits each, then the kept indices in
// order (of equal keys the first ones), their weights, and a copy of the
// scales, which the move overwrites.
__global__ void __launch_bounds__(kSelectThreads) k_kv8_select(EvictDev a) {
    __shared__ int hist[256];
    __shared__ int sums[32];
    __shared__ int chosen, above;
    const int b = blockIdx.x / a.cache.heads, h = blockIdx.x % a.cache.heads, tid = threadIdx.x;
    const int len = evict_length(a, b, tid == 0 && h == 0);
    const float* w = a.weights + (static_cast<int64_t>(b) * a.cache.heads + h) * a.weights_stride;
    float* wo = a.weights_out + (static_cast<int64_t>(b) * a.cache.heads + h) * a.weights_out_stride;
    int32_t* keep = a.keep + (static_cast<int64_t>(b) * a.cache.heads + h) * a.budget;
    if (h == 0 && tid == 0) a.lengths_out[b] = min(len, a.budget);
    if (len <= a.budget) {
        for (int i = tid; i < a.budget; i += kSelectThreads) keep[i] = i < len ? i : -1;
        if (w != wo)
            for (int i = tid; i < len; i += kSelectThreads) wo[i] = w[i];
        return;
    }
    const int bs = a.cache.block_tokens, nblk = (len + bs - 1) / bs;
    float* old = a.old_scale + (static_cast<int64_t>(b) * a.cache.heads + h) * 2 * a.old_blocks;
    for (int i = tid; i < nblk; i += kSelectThreads) {
        const int id = load_block(a.seq, b, i, h == 0);
        const int64_t at = static_cast<int64_t>(id) * a.cache.heads + h;
        old[i] = id < 0 ? 0.f : a.cache.scale[0][at];
        old[a.old_blocks + i] = id < 0 ? 0.f : a.cache.scale[1][at];
    }
    const int free_len = len - a.recent;
    int want = a.budget - a.recent;  // of the tokens before free_len; want < free_len
    uint32_t key = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
        __syncthreads();
        if (tid < 256) hist[tid] = 0;
        __syncthreads();
        const uint32_t high = shift == 24 ? 0u : ~0u << (shift + 8);
        for (int i = tid; i < free_len; i += kSelectThreads) {
            const uint32_t k = weight_key(w[i]);
            if ((k & high) == (key & high)) atomicAdd(&hist[(k >> shift) & 255u], 1);
        }
        __syncthreads();
        // bins from the greatest: the one in which the want-th falls
        const int mine = tid < 256 ? hist[255 - tid] : 0;
        int total;
        const int upto = cta_scan(mine, sums, &total);
        if (tid < 256 && want > 0 && upto >= want && upto - mine < want) {
            chosen = 255 - tid;
            above = upto - mine;
        }
        __syncthreads();
        if (want > 0) {
            key |= static_cast<uint32_t>(chosen) << shift;
            want -= above;
        }
    }
    // `want` of the weights equal to key are kept, all above it; if nothing
    // but the recent ones is kept, none.
    const bool none = a.budget == a.recent;
    int kept = 0, equal = 0;
    for (int base = 0; base < len; base += kSelectThreads) {
        const int i = base + tid;
        const bool inside = i < len, free_tok = i < free_len;
        const float wi = inside ? w[i] : 0.f;
        const uint32_t k = weight_key(wi);
        const bool same = inside && free_tok && !none && k == key;
        int n_same, n_kept;
        const int rank = equal + cta_scan(same, sums, &n_same);
        const bool take = inside && (!free_tok || (!none && (k > key || (same && rank <= want))));
        const int place = kept + cta_scan(take, sums, &n_kept);
        __syncthreads();  // every weight of this range is read before any is overwritten in place
        if (take) {
            keep[place - 1] = i;
            wo[place - 1] = wi;
        }
        equal += n_same;
        kept += n_kept;
    }
    __syncthreads();
    for (int i = a.budget + tid; i < len; i += kSelectThreads) wo[i] = 0.f;
}

constexpr int kMoveThreads = 256;

// Moves the kept tokens up, in place.  One CTA for each (sequence, head, K or
// V, slice of 32 code bytes) walks its destination tokens in order: a kept
// token's index is never below its destination, so once a group's codes are
// in registers its destinations can be written, and what the next groups read
// lies behind them.  Slices are independent because a block's new scale comes
// from the old scales alone (k_kv8_select copied them).
// Bound: kept codes read and written; 32-byte sectors, one CTA's loads in
// flight at a time.
template <int CODE>
__global__ void __launch_bounds__(kMoveThreads) k_kv8_move(EvictDev a, int slices) {
    constexpr int kRound = kMoveThreads / 2;  // destination tokens a pass: two threads of 16 bytes each
    __shared__ float dst_scale[kRound / 16];
    __shared__ float src_scale[kRound];
    const int slice = blockIdx.x % slices, rest = blockIdx.x / slices;
    const int which = rest & 1, h = (rest >> 1) % a.cache.heads, b = (rest >> 1) / a.cache.heads;
    const int len = evict_length(a, b, false);
    if (len <= a.budget) return;
    const int tid = threadIdx.x, bs = a.cache.block_tokens, dim = a.cache.dim;
    const int32_t* keep = a.keep + (static_cast<int64_t>(b) * a.cache.heads + h) * a.budget;
    const float* old = a.old_scale + ((static_cast<int64_t>(b) * a.cache.heads + h) * 2 + which) * a.old_blocks;
    const int col = slice * 32 + (tid & 1) * 16;
    const int group = max(bs, kRound) / bs * bs;  // whole blocks a pass (bs divides kRound or equals it)
    for (int base = 0; base < a.budget; base += group) {
        const int i = base + tid / 2;
        const bool live = i < a.budget;
        uint4 x = {0, 0, 0, 0};
        float scale = 0.f;
        int to = -1;
        if (live) {
            const int from = keep[i];
            const int src = load_block(a.seq, b, from / bs, false);
            to = load_block(a.seq, b, i / bs, false);
            scale = old[from / bs];
            if (src >= 0 && col < dim)
                x = __ldcg(reinterpret_cast<const uint4*>(a.cache.codes[which] + code_offset(a.cache, src, h) +
                                                          static_cast<int64_t>(from % bs) * dim + col));
        }
        if ((tid & 1) == 0) src_scale[tid / 2] = scale;
        __syncthreads();
        if (tid < kRound / bs) {
            float m = 0.f;
            for (int k = 0; k < bs; ++k) m = fmaxf(m, src_scale[tid * bs + k]);
            dst_scale[tid] = m;
        }
        __syncthreads();
        if (live && to >= 0) {
            const float now = dst_scale[(i - base) / bs];
            if (scale != now) {
                const float ratio = now > 0.f ? __fdiv_rn(scale, now) : 0.f;
                x.x = rescale4<CODE>(x.x, ratio);
                x.y = rescale4<CODE>(x.y, ratio);
                x.z = rescale4<CODE>(x.z, ratio);
                x.w = rescale4<CODE>(x.w, ratio);
            }
            if (col < dim)
                *reinterpret_cast<uint4*>(a.cache.codes[which] + code_offset(a.cache, to, h) +
                                          static_cast<int64_t>(i % bs) * dim + col) = x;
            if (slice == 0 && (tid & 1) == 0 && i % bs == 0)
                a.cache.scale[which][static_cast<int64_t>(to) * a.cache.heads + h] = now;
        }
        __syncthreads();
    }
}

}  // namespace i4d_ops
