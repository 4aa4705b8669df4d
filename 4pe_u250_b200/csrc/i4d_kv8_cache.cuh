// i4d_kv8_cache.cuh -- the paged cache of 8-bit codes: append, read, evict.
//
// A value is code * scale, one scale for each (block of tokens, head) of K and
// of V.  Appended blocks get a scale that is a power of two: divisions by it
// are exact, so a code depends on its value and scale alone, and when a later
// token raises the scale of a partly filled block, rewriting the older codes
// is a shift with one rounding; all such roundings of a code sum to less than
// one step of the last scale (1/2 + 1/4 + ...).
#pragma once

#include <cooperative_groups.h>

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

constexpr int kAppendHeld = 4;  // groups of eight values that a thread holds

struct AppendDev {
    Kv8Dev cache;
    SeqArrays seq;
    const void* in[2];
    int64_t tok[2], head[2];
    int touched;  // blocks that a sequence of max_q new tokens can touch
};

// Eight values as they lie in memory.
template <typename T, int V>
__device__ __forceinline__ Vec<T, 8> load8(const T* p) {
    if constexpr (V == 8) return load_vec<T, 8>(p);
    Vec<T, 8> x;
#pragma unroll
    for (int i = 0; i < 8; ++i) x.v[i] = p[i];
    return x;
}

// One unit (sequence, touched block, head, K or V) for each group of
// THREADS threads.  Two passes over the new values: the largest, then the
// codes.  The first four groups of eight of each thread stay in registers between them, in
// their own type, which covers blocks of 8192 values (64 tokens of 128); the
// rest is read again from L1/L2.  Bound: the values in, the codes out (6 x 501
// to 1531 FP32 rows of 8 heads of 128: 16 us, 60 MB; 48 rows in BF16: 4 us).
template <typename T, int V, int CODE, int THREADS>
__global__ void __launch_bounds__(THREADS < 128 ? 128 : THREADS, 4) k_kv8_append(AppendDev a, int units) {
    op_begin();
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
    const int first = s.len - s.n, blk = touched_block(first, s.len, bs, j);
    if (blk < 0) return;
    const int lo = max(first, blk * bs), hi = min(s.len, (blk + 1) * bs), old = lo - blk * bs;
    const T* in = static_cast<const T*>(a.in[which]) + static_cast<int64_t>(s.first + lo - first) * a.tok[which] +
                  h * a.head[which];
    const int per_tok = dim / 8, items = (hi - lo) * per_tok;
    // item i of eight values: token i / per_tok, values from 8 * (i % per_tok); this thread's lie THREADS apart
    const int step_tok = THREADS / per_tok, step_part = THREADS % per_tok;
    struct Place {
        int tok, part;
    };
    auto start = [&]() -> Place { return {tid / per_tok, tid % per_tok}; };
    auto advance = [&](Place& x) {
        x.tok += step_tok;
        x.part += step_part;
        if (x.part >= per_tok) {
            x.part -= per_tok;
            ++x.tok;
        }
    };
    auto load = [&](const Place& x) { return load8<T, V>(in + static_cast<int64_t>(x.tok) * a.tok[which] + x.part * 8); };
    Vec<T, 8> held[kAppendHeld];  // on their way before the block's id is known
    Place behind = start();
#pragma unroll
    for (int k = 0; k < kAppendHeld; ++k) {
        if (k * THREADS + tid < items) held[k] = load(behind);
        advance(behind);
    }
    const int id = load_block(a.seq, b, blk, report);
    if (id < 0) return;
    float* scale = a.cache.scale[which] + static_cast<int64_t>(id) * a.cache.heads + h;
    const float had = old ? *scale : 0.f;
    // The greatest magnitude (a maximum passes NaN over); only if that is an
    // infinity, again without those.
    auto greatest = [&](auto&& magnitude) {
        float amax = 0.f;
#pragma unroll
        for (int k = 0; k < kAppendHeld; ++k)
            if (k * THREADS + tid < items)
#pragma unroll
                for (int j = 0; j < 8; ++j) amax = fmaxf(amax, magnitude(to_f32(held[k].v[j])));
        Place at = behind;
        for (int i = kAppendHeld * THREADS + tid; i < items; i += THREADS, advance(at)) {
            const Vec<T, 8> x = load(at);
#pragma unroll
            for (int j = 0; j < 8; ++j) amax = fmaxf(amax, magnitude(to_f32(x.v[j])));
        }
        amax = warp_max(amax);
        if constexpr (kWarps > 1) {
            __shared__ float part[kWarps];
            __syncthreads();
            if (threadIdx.x % 32 == 0) part[threadIdx.x / 32] = amax;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < kWarps; ++w) amax = fmaxf(amax, part[w]);
        }
        return amax;
    };
    float amax = greatest([](float x) { return fabsf(x); });
    if (amax == INFINITY) amax = greatest([](float x) { return fabsf(x) < INFINITY ? fabsf(x) : 0.f; });
    const float now = fmaxf(power_scale(amax, CODE), had);
    if (tid == 0) *scale = now;  // every thread has read `had` (the barrier above, or the shuffles)
    uint8_t* codes = a.cache.codes[which] + code_offset(a.cache, id, h);
    if (old && now > had) {
        const Rescale ratio = make_rescale(__fdiv_rn(had, now));
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
    auto put = [&](int i, const Vec<T, 8>& v) {
        float x[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) x[k] = power ? __fmul_rn(to_f32(v.v[k]), inv) : __fdiv_rn(to_f32(v.v[k]), now);
        p[i] = make_uint2(encode4<CODE>(x[0], x[1], x[2], x[3]), encode4<CODE>(x[4], x[5], x[6], x[7]));
    };
#pragma unroll
    for (int k = 0; k < kAppendHeld; ++k)
        if (k * THREADS + tid < items) put(k * THREADS + tid, held[k]);
    for (int i = kAppendHeld * THREADS + tid; i < items; i += THREADS, advance(behind)) put(i, load(behind));
}

// ------------------------------------------------------------------ read

struct ReadDev {
    Kv8Dev cache;
    SeqArrays seq;
    __nv_bfloat16* out[2];
};

constexpr int kReadItems = 512;  // of a CTA of 256 threads

// An item: 16 codes of K and of V in, 16 BF16 values each out.  Bound: bytes;
// two items a thread, so that short reads spread over the GPU (16 tokens a CTA
// took 30 us for 1024 tokens of 32 heads, 8 us so; 200 MB in and out: 34 us).
template <int CODE>
__global__ void __launch_bounds__(256) k_kv8_read(ReadDev a, int chunks) {
    op_begin();
    const int b = blockIdx.x / chunks, i0 = blockIdx.x % chunks * kReadItems;
    const Seq s = load_seq(a.seq, b, threadIdx.x == 0 && i0 == 0);
    const int bs = a.cache.block_tokens, shift = 31 - __clz(bs), per_head = a.cache.dim / 16, per_tok = a.cache.heads * per_head;
    // (all loads before the first store)
    constexpr int kItems = kReadItems / 256;
    uint4 codes[kItems][2];
    float scale[kItems][2];
    int64_t to[kItems];
#pragma unroll
    for (int u = 0; u < kItems; ++u) {
        const int i = i0 + u * 256 + threadIdx.x;
        const int r = i / per_tok, e = i - r * per_tok, h = e / per_head, c = e - h * per_head;
        to[u] = -1;
        if (r >= s.n) continue;
        const int p = s.len - s.n + r, id = load_block(a.seq, b, p >> shift, true);
        if (id < 0) continue;
        to[u] = (static_cast<int64_t>(s.first + r) * a.cache.heads + h) * a.cache.dim + c * 16;
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            scale[u][which] = fetch(a.cache.scale[which] + static_cast<int64_t>(id) * a.cache.heads + h);
            codes[u][which] = fetch(reinterpret_cast<const uint4*>(a.cache.codes[which] + code_offset(a.cache, id, h) +
                                                                   static_cast<int64_t>(p & (bs - 1)) * a.cache.dim) + c);
        }
    }
#pragma unroll
    for (int u = 0; u < kItems; ++u) {
        if (to[u] < 0) continue;
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            const uint32_t ws[4] = {codes[u][which].x, codes[u][which].y, codes[u][which].z, codes[u][which].w};
            Vec<__nv_bfloat16, 16> o;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                float f[4];
                decode4<CODE>(ws[k], f);
#pragma unroll
                for (int m = 0; m < 4; ++m) o.v[4 * k + m] = __float2bfloat16_rn(f[m] * scale[u][which]);
            }
            store_vec<__nv_bfloat16, 16>(a.out[which] + to[u], o);
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
    const int len = fetch(a.seq.lengths + b);
    const bool ok = length_ok(len, a.max_length);
    if (!ok && report) atomicOr(a.seq.err, kBadSequence);
    return ok ? len : 0;
}

constexpr int kSelectThreads = 512;
constexpr int kSelectWarps = kSelectThreads / 32;

// Inclusive sum over the warp.
__device__ __forceinline__ int warp_scan(int x) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(~0u, x, o);
        if ((threadIdx.x & 31) >= o) x += y;
    }
    return x;
}

// Inclusive sum over the CTA of one value a thread; *total receives the sum.
__device__ __forceinline__ int cta_scan(int x, int* warp_sums, int* total) {
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    x = warp_scan(x);
    __syncthreads();
    if (lane == 31) warp_sums[w] = x;
    __syncthreads();
    if (w == 0) {
        const int y = warp_scan(lane < kSelectWarps ? warp_sums[lane] : 0);
        if (lane < kSelectWarps) warp_sums[lane] = y;
    }
    __syncthreads();
    *total = warp_sums[kSelectWarps - 1];
    return x + (w ? warp_sums[w - 1] : 0);
}

constexpr int kSelectBits = 11;  // 11 + 11 + 10 bits of a key
constexpr int kSelectBins = 1 << kSelectBits;
constexpr int kSelectHeld = 16;  // weights that a thread holds in registers

// One cluster for each (sequence, head), whose CTAs take consecutive parts of
// the weights and their threads consecutive weights: the key of the (budget -
// recent)-th greatest weight in three passes over its digits, each a histogram
// that the cluster adds up through distributed shared memory, then the kept
// indices in order (of equal keys the first ones), their weights, and a copy
// of the scales, which the move overwrites.  Rows of up to 65536 weights are
// read once into registers.  Bound: the chain of cluster barriers (8 heads of 4
// rows of up to 40009 weights: 23 us; one row of 2047, 32 heads: 12 us).
__global__ void __launch_bounds__(kSelectThreads, 2) k_kv8_select(EvictDev a, int ctas) {
    op_begin();
    __shared__ __align__(16) int hist[kSelectBins];
    __shared__ __align__(8) int groups[kSelectBins / 32];
    __shared__ int sums[32];
    __shared__ int chosen, above;
    __shared__ __align__(8) int counts[2];
    cooperative_groups::cluster_group cl = cooperative_groups::this_cluster();
    const int row = blockIdx.x / ctas, rank = blockIdx.x % ctas;
    const int b = row / a.cache.heads, h = row % a.cache.heads, tid = threadIdx.x, lane = tid & 31;
    const int len = evict_length(a, b, tid == 0 && h == 0 && rank == 0);
    const float* w = a.weights + row * a.weights_stride;
    float* wo = a.weights_out + row * a.weights_out_stride;
    int32_t* keep = a.keep + static_cast<int64_t>(row) * a.budget;
    if (h == 0 && rank == 0 && tid == 0) a.lengths_out[b] = min(len, a.budget);
    const int first = rank * kSelectThreads + tid, stride = ctas * kSelectThreads;
    if (len <= a.budget) {  // the whole cluster leaves
        for (int i = first; i < a.budget; i += stride) keep[i] = i < len ? i : -1;
        if (w != wo)
            for (int i = first; i < len; i += stride) wo[i] = w[i];
        return;
    }
    // This thread's weights [lo, lo + n).
    const int per = (len + stride - 1) / stride, lo = min(len, first * per), n = min(len, lo + per) - lo;
    float held[kSelectHeld];
#pragma unroll
    for (int k = 0; k < kSelectHeld; ++k) held[k] = k < n ? w[lo + k] : 0.f;
    auto each = [&](auto&& f) {
#pragma unroll
        for (int k = 0; k < kSelectHeld; ++k)
            if (k < n) f(lo + k, held[k]);
        for (int k = kSelectHeld; k < n; ++k) f(lo + k, w[lo + k]);
    };
    const int free_len = len - a.recent;
    int want = a.budget - a.recent;  // of the tokens before free_len; want < free_len
    const bool none = want == 0;
    uint32_t key = 0, high = 0;
    for (int shift = 21; !none; shift = max(0, shift - kSelectBits)) {
        const int bits = shift == 0 ? 10 : kSelectBits;
        for (int i = tid; i < kSelectBins; i += kSelectThreads) hist[i] = 0;
        __syncthreads();
        each([&](int i, float x) {
            const uint32_t k = weight_key(x);
            if (i < free_len && (k & high) == key) atomicAdd(&hist[(k >> shift) & ((1 << bits) - 1)], 1);
        });
        __syncthreads();
        // Sums of 32 bins each, so that the search reads these of all CTAs and
        // then one group of their bins, not every bin (5 us a pass with all).
#pragma unroll
        for (int k = 0; k < kSelectBins / 32 / kSelectWarps; ++k) {
            const int g = (tid >> 5) * (kSelectBins / 32 / kSelectWarps) + k;
            const int sum = __reduce_add_sync(~0u, hist[g * 32 + lane]);
            if (lane == 0) groups[g] = sum;
        }
        cl.sync();
        if (tid < 32) {
            // groups 63 - 2 lane and 62 - 2 lane, from the greatest on
            int2 n = make_int2(0, 0);
#pragma unroll
            for (int c = 0; c < 8; ++c) {
                if (c >= ctas) break;
                const int2 x = reinterpret_cast<const int2*>(cl.map_shared_rank(groups, c))[31 - lane];
                n.x += x.x;
                n.y += x.y;
            }
            const int before = warp_scan(n.x + n.y) - n.x - n.y;
            const bool upper = before + n.y >= want;
            const unsigned here = __ballot_sync(~0u, before < want && before + n.x + n.y >= want);
            const int at = __shfl_sync(~0u, upper ? before : before + n.y, __ffs(here) - 1);
            const int group = __shfl_sync(~0u, 63 - 2 * lane - !upper, __ffs(here) - 1);
            const int bin = group * 32 + 31 - lane;
            int m = 0;
#pragma unroll
            for (int c = 0; c < 8; ++c) {
                if (c >= ctas) break;
                m += cl.map_shared_rank(hist, c)[bin];
            }
            const int upto = at + warp_scan(m);
            if (upto >= want && upto - m < want) {
                chosen = bin;
                above = upto - m;
            }
        }
        cl.sync();  // hist is read, chosen is written
        key |= static_cast<uint32_t>(chosen) << shift;
        high |= static_cast<uint32_t>((1 << bits) - 1) << shift;
        want -= above;
        if (shift == 0) break;
    }
    // `want` of the weights equal to key are kept and all above it.  A
    // thread's places follow those of the threads and CTAs before it.
    int same = 0, more = 0;
    each([&](int i, float x) {
        const uint32_t k = weight_key(x);
        same += i < free_len && !none && k == key;
        more += i >= free_len || (!none && k > key);
    });
    int all_same, all_more;
    const int same_upto = cta_scan(same, sums, &all_same);
    const int more_upto = cta_scan(more, sums, &all_more);
    if (tid == 0) {
        counts[0] = all_same;
        counts[1] = all_more;
    }
    cl.sync();
    int equal = same_upto - same, larger = more_upto - more;
#pragma unroll
    for (int c = 0; c < 7; ++c) {
        if (c >= rank) break;
        const int2 other = *reinterpret_cast<const int2*>(cl.map_shared_rank(counts, c));
        equal += other.x;
        larger += other.y;
    }
    int place = larger + min(equal, want);
    // In place and more than the registers hold: the weights move after the
    // indices are known (below); otherwise every weight has been read by now.
    const bool late = w == wo && per > kSelectHeld;
    each([&](int i, float x) {
        const uint32_t k = weight_key(x);
        const bool is_same = i < free_len && !none && k == key;
        if (i >= free_len || (!none && k > key) || (is_same && equal < want)) {
            keep[place] = i;
            if (!late) wo[place] = x;
            ++place;
        }
        equal += is_same;
    });
    const int nblk = (len + a.cache.block_tokens - 1) / a.cache.block_tokens;
    float* old = a.old_scale + static_cast<int64_t>(row) * 2 * a.old_blocks;
    for (int i = first; i < nblk; i += stride) {
        const int id = load_block(a.seq, b, i, h == 0);
        const int64_t at = static_cast<int64_t>(id) * a.cache.heads + h;
        old[i] = id < 0 ? 0.f : a.cache.scale[0][at];
        old[a.old_blocks + i] = id < 0 ? 0.f : a.cache.scale[1][at];
    }
    if (late) {
        cl.sync();  // keep is written; no CTA reads its part of w in the loop above any more
        for (int base = 0; base < a.budget; base += stride * 8) {
            float x[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const int i = base + u * stride + first;
                x[u] = i < a.budget ? fetch_l2(w + keep[i]) : 0.f;
            }
            cl.sync();  // the sources of this round are read; those of later rounds lie behind its destinations
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const int i = base + u * stride + first;
                if (i < a.budget) wo[i] = x[u];
            }
        }
    }
    cl.sync();
    for (int i = a.budget + first; i < len; i += stride) wo[i] = 0.f;
}

constexpr int kMoveThreads = 512;

// 16-byte pieces that a thread holds, all of one column, and destination
// tokens of a CTA in a round: whole blocks.
constexpr int kMovePieces = 4;
__host__ __device__ constexpr int move_tokens(int dim) { return kMovePieces * (kMoveThreads / (dim / 16)) / 128 * 128; }

// Moves the kept tokens up, in place.  One cluster for each (sequence, head, K
// or V) walks its destination tokens in order, a round of all its CTAs at a
// time: a kept token's index is never below its destination, so a round's
// destinations can be written once all of the round's codes are in registers
// (the cluster's barrier), and what later rounds read lies behind them, so
// their loads start before; a round's loads and scales run between its arrival
// and its wait (4 contexts of 8192 kept tokens, 8 heads of 128: 49.8 us, 50.5
// with both at once; the gathers' latency is what is left).  A block's new
// scale comes from the old scales, which k_kv8_select copied.
// Bound: kept codes read and written in whole rows.
template <int CODE>
__global__ void __launch_bounds__(kMoveThreads, 2) k_kv8_move(EvictDev a, int ctas) {
    op_begin();
    constexpr int VECS = kMovePieces;
    __shared__ float token_scale[2][kMoveThreads * VECS];
    __shared__ float block_scale[2][kMoveThreads * VECS / 16];
    const int rank = blockIdx.x % ctas, rest = blockIdx.x / ctas;
    const int which = rest & 1, h = (rest >> 1) % a.cache.heads, b = (rest >> 1) / a.cache.heads;
    const int len = evict_length(a, b, false);
    if (len <= a.budget) return;  // the whole cluster leaves
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, bs = a.cache.block_tokens, shift = 31 - __clz(bs), dim = a.cache.dim;
    const int pieces = dim / 16, per = kMoveThreads / pieces, tokens = move_tokens(dim), round = ctas * tokens;
    const int32_t* keep = a.keep + (static_cast<int64_t>(b) * a.cache.heads + h) * a.budget + rank * tokens;
    const float* old = a.old_scale + ((static_cast<int64_t>(b) * a.cache.heads + h) * 2 + which) * a.old_blocks;
    uint8_t* codes = a.cache.codes[which];
    // piece u of a round: this CTA's token tok + u * per, 16 codes from col
    const int tok = tid < per * pieces ? tid / pieces : tokens, col = tid % pieces * 16;
    auto live = [&](int base, int u) { return tok + u * per < tokens && base + rank * tokens + tok + u * per < a.budget; };
    // kept index of a piece's token (-1: none), its codes, its scale
    auto kept = [&](int base, int u) { return live(base, u) ? fetch(keep + base + tok + u * per) : -1; };
    auto piece = [&](int from, float& scale) {
        uint4 x = make_uint4(0, 0, 0, 0);
        scale = 0.f;
        if (from >= 0) {
            const int id = load_block(a.seq, b, from >> shift, false);
            scale = fetch(old + (from >> shift));
            if (id >= 0) x = fetch_l2(reinterpret_cast<const uint4*>(codes + code_offset(a.cache, id, h) + static_cast<int64_t>(from & (bs - 1)) * dim + col));
        }
        return x;
    };
    uint4 x[VECS];
    float scale[VECS];
    int next[VECS];
#pragma unroll
    for (int u = 0; u < VECS; ++u) {
        x[u] = piece(kept(0, u), scale[u]);
        next[u] = kept(round, u);
    }
    int half = 0;
    for (int base = 0; base < a.budget; base += round, half ^= 1) {
        const int mine = base + rank * tokens;
        // (a release: this round's codes, loaded a round ago, have been read)
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
        uint4 ahead[VECS];
        float ahead_scale[VECS];
        int to[VECS];
#pragma unroll
        for (int u = 0; u < VECS; ++u) {
            ahead[u] = piece(next[u], ahead_scale[u]);
            next[u] = kept(base + 2 * round, u);
            to[u] = live(base, u) ? load_block(a.seq, b, (mine + tok + u * per) >> shift, false) : -1;
            if (tok + u * per < tokens && col == 0) token_scale[half][tok + u * per] = scale[u];
        }
        __syncthreads();
        for (int k = warp; k < tokens >> shift; k += kMoveThreads / 32) {
            float m = 0.f;
            for (int i = lane; i < bs; i += 32) m = fmaxf(m, token_scale[half][(k << shift) + i]);
            m = warp_max(m);
            if (lane == 0) block_scale[half][k] = m;
        }
        __syncthreads();
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
#pragma unroll
        for (int u = 0; u < VECS; ++u) {
            if (to[u] >= 0) {
                const int at = (mine + tok + u * per) & (bs - 1);
                const float now = block_scale[half][(tok + u * per) >> shift];
                uint4 v = x[u];
                if (scale[u] != now) {
                    const Rescale ratio = make_rescale(__fdiv_rn(scale[u], now));
                    v.x = rescale4<CODE>(v.x, ratio);
                    v.y = rescale4<CODE>(v.y, ratio);
                    v.z = rescale4<CODE>(v.z, ratio);
                    v.w = rescale4<CODE>(v.w, ratio);
                }
                *reinterpret_cast<uint4*>(codes + code_offset(a.cache, to[u], h) + static_cast<int64_t>(at) * dim + col) = v;
                if (col == 0 && at == 0) a.cache.scale[which][static_cast<int64_t>(to[u]) * a.cache.heads + h] = now;
            }
            x[u] = ahead[u];
            scale[u] = ahead_scale[u];
        }
    }
}

}  // namespace i4d_ops
