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
// Bound: the logits in and out; but a list of thousands of ids costs a CTA's
// phases, each with its barriers, as much again (192 rows of 128001 in bf16:
// 32 us without lists, 60 with histories and biases, 15 at the copy's rate),
// and one row the chain of those phases (7 us for 32000 in FP32).
#pragma once

#include <cooperative_groups.h>

#include <type_traits>

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

// Puts -inf in place of the logits whose bit in `seen` is 0, but for those
// whose bit in `raw` is 1, which stay; returns the greatest of those that are
// seen and not raw (-inf: none; NaN passed over).
__device__ __forceinline__ float mask_vec(Vec<float, 4>& x, uint32_t seen, uint32_t raw) {
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (seen & ~raw & 1u << i) top = fmaxf(top, x.v[i]);
        if (!((seen | raw) & 1u << i)) x.v[i] = -INFINITY;
    }
    return top;
}
// 16-bit logits two at a time.
template <typename T>
__device__ __forceinline__ float mask_vec(Vec<T, 8>& x, uint32_t seen, uint32_t raw) {
    constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
    constexpr uint32_t kNone = kBf16 ? 0xff80ff80u : 0xfc00fc00u;  // two of -inf
    // bit 2 i and bit 2 i + 1 to two masks of 16
    auto both = [](uint32_t bits, int i) {
        return __byte_perm(static_cast<int>(bits << (31 - 2 * i)) >> 31, static_cast<int>(bits << (30 - 2 * i)) >> 31, 0x5410);
    };
    uint32_t* w = reinterpret_cast<uint32_t*>(&x);
    uint32_t top = kNone;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t counts = both(seen & ~raw, i), stays = both(raw, i);
        const uint32_t y = (w[i] & counts) | (kNone & ~counts);
        w[i] = (w[i] & stays) | (y & ~stays);
        if constexpr (kBf16) {
            const __nv_bfloat162 z = __hmax2(*reinterpret_cast<const __nv_bfloat162*>(&top), *reinterpret_cast<const __nv_bfloat162*>(&y));
            top = *reinterpret_cast<const uint32_t*>(&z);
        } else {
            const __half2 z = __hmax2(*reinterpret_cast<const __half2*>(&top), *reinterpret_cast<const __half2*>(&y));
            top = *reinterpret_cast<const uint32_t*>(&z);
        }
    }
    const T* y = reinterpret_cast<const T*>(&top);
    return fmaxf(to_f32(y[0]), to_f32(y[1]));
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
    __device__ __forceinline__ void mark(int id) const {
        const int at = id - first;
        atomicOr(bits + (at >> 5), 1u << (at & 31));
    }
    __device__ __forceinline__ int place(int id) const {
        const int at = id - first;
        return before[at >> 5] + __popc(bits[at >> 5] & ((1u << (at & 31)) - 1));
    }
};

template <typename T>
__global__ void __launch_bounds__(kLogitsThreads, 2) k_logits(LogitsDev a, int ctas) {
    op_begin();
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
    const int n_hist = hist ? min(max(fetch(a.history_len + row), 0), a.history_max) : 0;
    const int n_prompt = hist && a.prompt_len ? fetch(a.prompt_len + row) : 0;
    const int32_t* bias_ids = a.bias_ids ? a.bias_ids + row * a.bias_stride : nullptr;
    const int n_bias = bias_ids ? min(max(fetch(a.bias_len + row), 0), a.bias_max) : 0;
    const float rep = a.repetition ? fetch(a.repetition + row) : 1.f;
    const float freq = a.frequency ? fetch(a.frequency + row) : 0.f;
    const float pres = a.presence ? fetch(a.presence + row) : 0.f;
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
    // The lists' ids, read once into registers as far as they hold them; each is
    // looked at twice for every part.
    constexpr int kHeld = 6;
    constexpr int kFew = 8;  // bits of a word that one thread takes
    int held[kHeld], held_bias = -1;
    float held_value = 0.f;
#pragma unroll
    for (int k = 0; k < kHeld; ++k) held[k] = k * kLogitsThreads + tid < n_hist ? fetch(hist + k * kLogitsThreads + tid) : -1;
    if (tid < n_bias) {
        held_bias = fetch(bias_ids + tid);
        held_value = fetch(a.bias_values + row * a.bias_stride + tid);
    }
    auto each_id = [&](auto&& f) {
#pragma unroll
        for (int k = 0; k < kHeld; ++k) f(k * kLogitsThreads + tid, held[k]);
        for (int i = kHeld * kLogitsThreads + tid; i < n_hist; i += kLogitsThreads) f(i, fetch(hist + i));
    };
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
            each_id([&](int, int id) {
                if (t.holds(id)) t.mark(id);
            });
            if (t.holds(held_bias)) t.mark(held_bias);
            for (int i = kLogitsThreads + tid; i < n_bias; i += kLogitsThreads) {
                const int id = fetch(bias_ids + i);
                if (t.holds(id)) t.mark(id);
            }
            __syncthreads();
            // places: each thread's words follow those of the threads before it.  A
            // warp's words lie 33 apart: the full ones, of frequent tokens, are
            // neighbours (and an odd distance reaches every bank).
            const int w0 = tid * 33 % kLogitsThreads;
            int mine = 0;
            for (int w = w0; w < words; w += kLogitsThreads) mine += __popc(t.bits[w]);
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
            for (int wb = 0; wb < words; wb += kLogitsThreads) {
                const int w = wb + w0;
                const uint32_t x = w < words ? t.bits[w] : 0u;
                if (w < words) t.before[w] = static_cast<uint16_t>(at);
                const bool full = __popc(x) > kFew;
                if (!full)
                    for (uint32_t y = x, to = at; y; y &= y - 1) t.ids[to++] = static_cast<uint16_t>(w * 32 + __ffs(y) - 1);
                for (unsigned todo = __ballot_sync(~0u, full); todo; todo &= todo - 1) {  // a lane for each bit
                    const int from = __ffs(todo) - 1;
                    const uint32_t y = __shfl_sync(~0u, x, from);
                    const int to = __shfl_sync(~0u, at, from) + __popc(y & ((1u << lane) - 1)), word = __shfl_sync(~0u, w, from);
                    if (y >> lane & 1) t.ids[to] = static_cast<uint16_t>(word * 32 + lane);
                }
                at += __popc(x);
            }
            for (int k = tid; k < touched; k += kLogitsThreads) {
                t.counts[k] = 0;
                t.bias[k] = 0.f;
            }
            __syncthreads();
            each_id([&](int i, int id) {
                if (t.holds(id)) {
                    int* count = &t.counts[t.place(id)];
                    if (i < n_prompt) atomicOr(count, 1);
                    else atomicAdd(count, 2);
                }
            });
            // Biases, a thread for each.  A thread that finds its own mark in its
            // place adds alone; else the part's entries of the round are listed in
            // their order, and the first of each id adds up the values of that id.
            for (int i = 0; i < n_bias; i += kLogitsThreads) {
                const int id = i == 0 ? held_bias : i + tid < n_bias ? fetch(bias_ids + i + tid) : -1;
                const float value = i == 0 ? held_value : i + tid < n_bias ? fetch(a.bias_values + row * a.bias_stride + i + tid) : 0.f;
                const bool in_part = t.holds(id);
                float* sum_of = &t.bias[in_part ? t.place(id) : 0];
                float prior = 0.f;
                if (i) {
                    __syncthreads();
                    if (in_part) prior = *sum_of;
                    __syncthreads();
                }
                if (in_part) *sum_of = __int_as_float(tid);
                __syncthreads();
                const bool shared = in_part && __float_as_int(*sum_of) != tid;
                const int several = __syncthreads_or(shared);
                if (in_part) *sum_of = several ? prior : __fadd_rn(prior, value);
                if (!several) continue;
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
                if (in_part) entries[to] = make_float2(__int_as_float(t.place(id)), value);
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
                if (mask) words_ahead[u] = make_uint2(fetch(mask + (e >> 5)), fetch(mask + ((e + V - 1) >> 5)));
            }
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int v = vb + u * kLogitsThreads + tid, e = v * V - skew;
            if (v >= v1) continue;
            if (e >= 0 && e + V <= a.vocab) {
                Vec<T, V> x = ahead[u];
                uint32_t raw = 0;
                const uint32_t seen = __funnelshift_r(words_ahead[u].x, words_ahead[u].y, e & 31);
                if (touched) {
                    const int at = e - t.first, w = at >> 5;
                    raw = __funnelshift_r(t.bits[w], w + 1 < words ? t.bits[w + 1] : 0u, at & 31);
                }
                const float top = mask_vec(x, seen, raw);
                if (top > best) {
                    best = top;
#pragma unroll
                    for (int i = V - 1; i >= 0; --i)
                        if ((seen & ~raw) >> i & 1 && to_f32(x.v[i]) == top) best_id = e + i;
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
                    const bool gone = mask && !(fetch(mask + (id >> 5)) >> (id & 31) & 1);
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
            constexpr int kLate = 4;  // logits that a thread loads before it works on them
            for (int kb = tid; kb < touched; kb += kLogitsThreads * kLate) {
                float ys[kLate];
                int ids[kLate];
                uint32_t seen[kLate];
#pragma unroll
                for (int u = 0; u < kLate; ++u) {
                    const int k = kb + u * kLogitsThreads;
                    ids[u] = k < touched ? t.first + t.ids[k] : t.first;
                    ys[u] = k < touched ? to_f32(out[ids[u]]) : 0.f;
                    seen[u] = mask ? fetch(mask + (ids[u] >> 5)) >> (ids[u] & 31) & 1 : 1;
                }
#pragma unroll
                for (int u = 0; u < kLate; ++u) {
                    const int k = kb + u * kLogitsThreads;
                    if (k >= touched) break;
                    const int c = t.counts[k], n = c >> 1;
                    float y = ys[u];
                    if (c && a.repetition) y = y > 0.f ? __fdiv_rn(y, rep) : __fmul_rn(y, rep);
                    if (n) y = __fsub_rn(__fsub_rn(y, __fmul_rn(freq, static_cast<float>(n))), pres);
                    y = __fadd_rn(y, t.bias[k]);
                    if (!seen[u]) y = -INFINITY;
                    const T z = from_f32<T>(y);
                    out[ids[u]] = z;
                    key = max(key, logit_key(to_f32(z), ids[u]));
                }
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
