// i4d_logits.cuh -- penalties, biases and masks on rows of logits.
//
// One cluster of CTAs for a row, each with a part of it.  The tokens that the
// history or the biases touch are few, so a CTA marks them in a bitmap, gives
// each a place by counting bits, and gathers counts (integer atomics, whose sum
// does not depend on the order) and biases there.  Then it streams its part,
// where an untouched logit only meets the mask, and last works out the touched
// ones, a thread each, so that no warp runs the penalties' division for one
// lane.  The row's best index is joined over the cluster through distributed
// shared memory; nothing is kept in global memory between launches.
// Bound: the logits in and out; for one row the chain of barriers.
#pragma once

#include <cooperative_groups.h>

#include "i4d_ops_common.cuh"

namespace i4d_ops {

constexpr int kLogitsThreads = 512;
constexpr int kLogitsTouched = 8192;  // touched tokens that a CTA can hold
constexpr int kLogitsPart = 65536;    // logits of a part, with no more than that many ids in the lists
// Shared memory for `places` touched tokens (a multiple of 8) of parts of `words` words (a multiple of 4).
__host__ __device__ constexpr int logits_smem_bytes(int places, int words) { return places * (4 + 4 + 2) + words * (4 + 2); }

struct LogitsDev {
    const void* in;
    void* out;
    int32_t* best;
    const int32_t* history;
    const int32_t* history_len;
    const int32_t* prompt_len;
    const float* repetition;
    const float* frequency;
    const float* presence;
    const int32_t* bias_ids;
    const float* bias_values;
    const int32_t* bias_len;
    const uint32_t* mask;
    int64_t stride, out_stride, history_stride, bias_stride, mask_stride;
    int vocab, history_max, bias_max;
    int places, words;  // touched tokens and bitmap words that the launch has shared memory for
};

// Greater value, greater key; of equal values the lower index.  0: none.
__device__ __forceinline__ unsigned long long logit_key(float x, int index) {
    if (!(x > -INFINITY)) return 0ull;  // NaN and -inf
    const uint32_t u = __float_as_uint(x + 0.f);
    const uint32_t k = u & 0x80000000u ? ~u : u | 0x80000000u;
    return static_cast<unsigned long long>(k) << 32 | (0xffffffffu - index);
}

// Marks, places and values of the touched tokens of a part.
struct Touched {
    int* counts;          // [place] bit 0: in the prompt, above: 2 * occurrences after it
    float* bias;          // [place]
    uint32_t* bits;       // [part / 32]
    uint16_t* ids;        // [place] id - first
    uint16_t* before;     // [part / 32] places before a word
    int first, span;      // ids [first, first + span), span <= kLogitsPart
    __device__ __forceinline__ bool holds(int id) const { return static_cast<unsigned>(id - first) < static_cast<unsigned>(span); }
    // (Few tokens are most of a text: a mark that stands is not written again.)
    __device__ __forceinline__ void mark(int id) const {
        const int at = id - first;
        const uint32_t bit = 1u << (at & 31);
        if (!(*static_cast<volatile uint32_t*>(bits + (at >> 5)) & bit)) atomicOr(bits + (at >> 5), bit);
    }
    __device__ __forceinline__ int place(int id) const {
        const int at = id - first;
        return before[at >> 5] + __popc(bits[at >> 5] & ((1u << (at & 31)) - 1));
    }
};

template <typename T>
__global__ void __launch_bounds__(kLogitsThreads, 3) k_logits(LogitsDev a, int ctas) {
    extern __shared__ __align__(16) unsigned char logits_smem[];
    constexpr int V = 16 / sizeof(T);
    Touched t;
    t.counts = reinterpret_cast<int*>(logits_smem);
    t.bias = reinterpret_cast<float*>(t.counts + a.places);
    t.bits = reinterpret_cast<uint32_t*>(t.bias + a.places);
    t.ids = reinterpret_cast<uint16_t*>(t.bits + a.words);
    t.before = t.ids + a.places;
    __shared__ int found[kLogitsThreads / 32];
    __shared__ float2 entries[kLogitsThreads];
    __shared__ unsigned long long keys[kLogitsThreads / 32];
    __shared__ unsigned long long cta_key[16];
    cooperative_groups::cluster_group cl = cooperative_groups::this_cluster();
    if (a.best) cl.barrier_arrive();  // the wait stands before the first access to another CTA's memory
    const int row = blockIdx.x / ctas, rank = blockIdx.x % ctas, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const T* in = static_cast<const T*>(a.in) + row * a.stride;
    T* out = static_cast<T*>(a.out) + row * a.out_stride;
    const int32_t* hist = a.history ? a.history + row * a.history_stride : nullptr;
    const int n_hist = hist ? min(max(__ldg(a.history_len + row), 0), a.history_max) : 0;
    const int n_prompt = hist && a.prompt_len ? __ldg(a.prompt_len + row) : 0;
    const int32_t* bias_ids = a.bias_ids ? a.bias_ids + row * a.bias_stride : nullptr;
    const int n_bias = bias_ids ? min(max(__ldg(a.bias_len + row), 0), a.bias_max) : 0;
    const float rep = a.repetition ? __ldg(a.repetition + row) : 1.f;
    const float freq = a.frequency ? __ldg(a.frequency + row) : 0.f;
    const float pres = a.presence ? __ldg(a.presence + row) : 0.f;
    const uint32_t* mask = a.mask ? a.mask + row * a.mask_stride : nullptr;
    // Vector j holds entries [V j - skew, V j - skew + V): 16-byte aligned in
    // the input, and in the output if its rows have the same alignment.
    const int skew = static_cast<int>(reinterpret_cast<uintptr_t>(in) / sizeof(T) % V);
    const bool aligned_out = static_cast<int>(reinterpret_cast<uintptr_t>(out) / sizeof(T) % V) == skew;
    const int vecs = (a.vocab + skew + V - 1) / V;
    const int per_cta = (vecs + ctas - 1) / ctas;
    const int v_end = min(vecs, (rank + 1) * per_cta);
    // More ids than places: parts of so many logits that no more can be touched.
    const int part = (n_hist + n_bias <= a.places ? a.words * 32 : min(a.places, a.words * 32)) / V;
    constexpr int kAhead = 2;  // vectors that a thread loads before it works on them
    unsigned long long key = 0;
    float best = -INFINITY;  // of this thread's streamed logits, whose ids only grow
    int best_id = -1;
    for (int v0 = rank * per_cta; v0 < v_end; v0 += part) {
        const int v1 = min(v_end, v0 + part);
        // the stream's cache lines, on their way while the tokens are counted
        for (int v = v0 + tid * (128 / 16); v < v1; v += kLogitsThreads * (128 / 16))
            asm volatile("prefetch.global.L2 [%0];" ::"l"(in + max(v * V - skew, 0)));
        t.first = max(0, v0 * V - skew);
        t.span = min(a.vocab, v1 * V - skew) - t.first;
        const int words = (t.span + 31) / 32;
        int touched = 0;
        if (n_hist | n_bias) {
            __syncthreads();
            for (int i = tid; i < words; i += kLogitsThreads) t.bits[i] = 0;
            __syncthreads();
#pragma unroll 4
            for (int i = tid; i < n_hist; i += kLogitsThreads) {
                const int id = __ldg(hist + i);
                if (t.holds(id)) t.mark(id);
            }
            for (int i = tid; i < n_bias; i += kLogitsThreads) {
                const int id = __ldg(bias_ids + i);
                if (t.holds(id)) t.mark(id);
            }
            __syncthreads();
            // places: each thread's words follow those of the threads before it
            const int per = (words + kLogitsThreads - 1) / kLogitsThreads, w0 = min(words, tid * per), w1 = min(words, w0 + per);
            int mine = 0;
            for (int w = w0; w < w1; ++w) mine += __popc(t.bits[w]);
            int upto = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int x = __shfl_up_sync(~0u, upto, o);
                if (lane >= o) upto += x;
            }
            if (lane == 31) found[warp] = upto;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < kLogitsThreads / 32; ++w) {
                if (w < warp) upto += found[w];
                touched += found[w];
            }
            int at = upto - mine;
            for (int w = w0; w < w1; ++w) {
                t.before[w] = static_cast<uint16_t>(at);
                for (uint32_t x = t.bits[w]; x; x &= x - 1) {
                    t.ids[at] = static_cast<uint16_t>(w * 32 + __ffs(x) - 1);
                    t.counts[at] = 0;
                    t.bias[at++] = 0.f;
                }
            }
            __syncthreads();
#pragma unroll 4
            for (int i = tid; i < n_hist; i += kLogitsThreads) {
                const int id = __ldg(hist + i);
                if (t.holds(id)) {
                    int* count = &t.counts[t.place(id)];
                    if (i < n_prompt) {
                        if (!(*static_cast<volatile int*>(count) & 1)) atomicOr(count, 1);
                    } else {  // one lane adds for all lanes with its token
                        const unsigned peers = __match_any_sync(__activemask(), id);
                        if (__ffs(peers) - 1 == lane) atomicAdd(count, 2 * __popc(peers));
                    }
                }
            }
            // Biases: the part's entries of a round in their order, then the
            // first of each id adds up the values of that id.
            for (int i = 0; i < n_bias; i += kLogitsThreads) {
                const int id = i + tid < n_bias ? __ldg(bias_ids + i + tid) : -1;
                const bool in_part = t.holds(id);
                const unsigned votes = __ballot_sync(~0u, in_part);
                __syncthreads();
                if (lane == 0) found[warp] = __popc(votes);
                __syncthreads();
                int to = __popc(votes & ((1u << lane) - 1)), total = 0;
#pragma unroll
                for (int w = 0; w < kLogitsThreads / 32; ++w) {
                    to += w < warp ? found[w] : 0;
                    total += found[w];
                }
                if (in_part) entries[to] = make_float2(__int_as_float(t.place(id)), __ldg(a.bias_values + row * a.bias_stride + i + tid));
                __syncthreads();
                if (tid < total) {
                    const int slot = __float_as_int(entries[tid].x);
                    bool leads = true;
                    for (int k = 0; k < tid; ++k) leads &= __float_as_int(entries[k].x) != slot;
                    if (leads) {
                        float sum = t.bias[slot];
                        for (int k = tid; k < total; ++k)
                            if (__float_as_int(entries[k].x) == slot) sum = __fadd_rn(sum, entries[k].y);
                        t.bias[slot] = sum;
                    }
                }
            }
        }
        // The stream: touched logits go out as they came.
        for (int vb = v0; vb < v1; vb += kLogitsThreads * kAhead) {
        Vec<T, V> ahead[kAhead];
        uint2 words_ahead[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int v = vb + u * kLogitsThreads + tid, e = v * V - skew;
            words_ahead[u] = make_uint2(~0u, ~0u);
            if (v < v1 && e >= 0 && e + V <= a.vocab) {
                ahead[u] = *reinterpret_cast<const Vec<T, V>*>(in + e);
                if (mask) words_ahead[u] = make_uint2(__ldg(mask + (e >> 5)), __ldg(mask + ((e + V - 1) >> 5)));
            }
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int v = vb + u * kLogitsThreads + tid, e = v * V - skew;
            if (v >= v1) continue;
            if (e >= 0 && e + V <= a.vocab) {
                Vec<T, V> x = ahead[u];
                uint32_t skip = 0;
                const uint32_t seen = __funnelshift_r(words_ahead[u].x, words_ahead[u].y, e & 31);
                if (touched) {
                    const int at = e - t.first, w = at >> 5;
                    skip = __funnelshift_r(t.bits[w], w + 1 < words ? t.bits[w + 1] : 0u, at & 31);
                }
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float y = to_f32(x.v[i]);
                    const bool gone = !(seen >> i & 1), raw = skip >> i & 1;
                    if (gone && !raw) x.v[i] = from_f32<T>(-INFINITY);
                    if (y > best && !gone && !raw) {
                        best = y;
                        best_id = e + i;
                    }
                }
                if (aligned_out) {
                    *reinterpret_cast<Vec<T, V>*>(out + e) = x;
                } else {
#pragma unroll
                    for (int i = 0; i < V; ++i) out[e + i] = x.v[i];
                }
            } else {
                for (int id = max(e, 0); id < min(e + V, a.vocab); ++id) {
                    const T x = in[id];
                    const int at = id - t.first;
                    const bool raw = touched && (t.bits[at >> 5] >> (at & 31) & 1);
                    const bool gone = mask && !(__ldg(mask + (id >> 5)) >> (id & 31) & 1);
                    out[id] = gone && !raw ? from_f32<T>(-INFINITY) : x;
                    if (to_f32(x) > best && !gone && !raw) {
                        best = to_f32(x);
                        best_id = id;
                    }
                }
            }
        }
        }
        if (touched) {
            __syncthreads();  // counts and biases are complete, the touched logits lie in `out`
            for (int k = tid; k < touched; k += kLogitsThreads) {
                const int id = t.first + t.ids[k], c = t.counts[k], n = c >> 1;
                float y = to_f32(out[id]);
                if (c && a.repetition) y = y > 0.f ? __fdiv_rn(y, rep) : __fmul_rn(y, rep);
                if (n) y = __fsub_rn(__fsub_rn(y, __fmul_rn(freq, static_cast<float>(n))), pres);
                y = __fadd_rn(y, t.bias[k]);
                if (mask && !(__ldg(mask + (id >> 5)) >> (id & 31) & 1)) y = -INFINITY;
                const T z = from_f32<T>(y);
                out[id] = z;
                key = max(key, logit_key(to_f32(z), id));
            }
        }
    }
    if (!a.best) return;
    key = max(key, logit_key(best, best_id));
#pragma unroll
    for (int o = 16; o; o >>= 1) key = max(key, __shfl_xor_sync(~0u, key, o));
    if (lane == 0) keys[warp] = key;
    __syncthreads();
    cl.barrier_wait();
    if (tid == 0) {
        for (int w = 1; w < kLogitsThreads / 32; ++w) key = max(key, keys[w]);
        *cl.map_shared_rank(&cta_key[rank], 0) = key;
    }
    cl.sync();
    if (rank == 0 && tid == 0) {
        for (int c = 0; c < ctas; ++c) key = max(key, cta_key[c]);
        a.best[row] = key ? static_cast<int>(0xffffffffu - static_cast<uint32_t>(key)) : -1;
    }
}

}  // namespace i4d_ops
