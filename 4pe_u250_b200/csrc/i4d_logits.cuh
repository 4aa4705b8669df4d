// i4d_logits.cuh -- penalties, biases and masks on rows of logits.
//
// One cluster of CTAs for a row.  A CTA walks slices of the row: the counts of
// the history's tokens that fall in the slice are gathered in shared memory
// with integer atomics (their sum does not depend on the order), the biases
// beside them, then each logit is read, changed and written once.  The row's
// best index is joined over the cluster through distributed shared memory, so
// nothing is kept in global memory between launches.
// Bound: the logits in and out; for one row the chain of barriers.
#pragma once

#include <cooperative_groups.h>

#include "i4d_ops_common.cuh"

namespace i4d_ops {

constexpr int kLogitsThreads = 512;
constexpr int kLogitsSlice = 8192;  // entries: 32 KB of counts and 32 KB of biases

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
};

// Greater value, greater key; of equal values the lower index.  0: none.
__device__ __forceinline__ unsigned long long logit_key(float x, int index) {
    if (!(x > -INFINITY)) return 0ull;  // NaN and -inf
    const uint32_t u = __float_as_uint(x + 0.f);
    const uint32_t k = u & 0x80000000u ? ~u : u | 0x80000000u;
    return static_cast<unsigned long long>(k) << 32 | (0xffffffffu - index);
}

template <typename T>
__global__ void __launch_bounds__(kLogitsThreads, 2) k_logits(LogitsDev a, int ctas) {
    extern __shared__ __align__(16) unsigned char logits_smem[];
    constexpr int V = 16 / sizeof(T);
    int* counts = reinterpret_cast<int*>(logits_smem);                  // bit 0: seen in the prompt, above: 2 * occurrences after it
    float* bias = reinterpret_cast<float*>(counts + kLogitsSlice);
    __shared__ int found[kLogitsThreads / 32];
    __shared__ float2 entries[kLogitsThreads];
    __shared__ unsigned long long keys[kLogitsThreads / 32];
    __shared__ unsigned long long cta_key[16];
    cooperative_groups::cluster_group cl = cooperative_groups::this_cluster();
    if (a.best) cl.barrier_arrive();  // the wait stands before the first access to another CTA's memory
    const int row = blockIdx.x / ctas, rank = blockIdx.x % ctas, tid = threadIdx.x;
    const T* in = static_cast<const T*>(a.in) + row * a.stride;
    T* out = static_cast<T*>(a.out) + row * a.out_stride;
    const int32_t* hist = a.history ? a.history + row * a.history_stride : nullptr;
    const int n_hist = hist ? min(max(__ldg(a.history_len + row), 0), a.history_max) : 0;
    const int n_prompt = hist && a.prompt_len ? __ldg(a.prompt_len + row) : 0;
    const int n_bias = a.bias_ids ? min(max(__ldg(a.bias_len + row), 0), a.bias_max) : 0;
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
    unsigned long long key = 0;
    // A thread's vectors of the next slice are loaded before the counting of
    // its tokens, which hides the wait for them.
    constexpr int kVecs = kLogitsSlice / V / kLogitsThreads;
    for (int v0 = rank * per_cta; v0 < v_end; v0 += kLogitsSlice / V) {
        const int v1 = min(v_end, v0 + kLogitsSlice / V);
        const int e0 = v0 * V - skew, span = (v1 - v0) * V;
        Vec<T, V> x[kVecs];
        uint2 words[kVecs];
#pragma unroll
        for (int u = 0; u < kVecs; ++u) {
            const int v = v0 + u * kLogitsThreads + tid, e = v * V - skew;
            words[u] = make_uint2(~0u, ~0u);
            if (v >= v1) continue;
            if (e >= 0 && e + V <= a.vocab) {
                x[u] = *reinterpret_cast<const Vec<T, V>*>(in + e);
            } else {
#pragma unroll
                for (int i = 0; i < V; ++i)
                    if (e + i >= 0 && e + i < a.vocab) x[u].v[i] = in[e + i];
            }
            if (mask) words[u] = make_uint2(__ldg(mask + max(e, 0) / 32), __ldg(mask + min(e + V - 1, a.vocab - 1) / 32));
        }
        __syncthreads();
        if (n_hist)
            for (int i = tid; i < kLogitsSlice / 4; i += kLogitsThreads) reinterpret_cast<int4*>(counts)[i] = make_int4(0, 0, 0, 0);
        if (n_bias)
            for (int i = tid; i < kLogitsSlice / 4; i += kLogitsThreads) reinterpret_cast<int4*>(bias)[i] = make_int4(0, 0, 0, 0);
        __syncthreads();
#pragma unroll 4
        for (int i = tid; i < n_hist; i += kLogitsThreads) {
            const int id = __ldg(hist + i);
            if (id >= max(e0, 0) && id < a.vocab && id - e0 < span) {
                if (i < n_prompt) atomicOr(&counts[id - e0], 1);
                else atomicAdd(&counts[id - e0], 2);
            }
        }
        // Biases: the slice's entries of a round in their order, then the first
        // of each id adds up the values of that id.
        for (int i = 0; i < n_bias; i += kLogitsThreads) {
            const bool live = i + tid < n_bias;
            const int id = live ? __ldg(a.bias_ids + row * a.bias_stride + i + tid) : -1;
            const bool mine = live && id >= max(e0, 0) && id < a.vocab && id - e0 < span;
            const unsigned votes = __ballot_sync(~0u, mine);
            if ((tid & 31) == 0) found[tid >> 5] = __popc(votes);
            __syncthreads();
            int at = __popc(votes & ((1u << (tid & 31)) - 1)), total = 0;
#pragma unroll
            for (int w = 0; w < kLogitsThreads / 32; ++w) {
                at += w < tid >> 5 ? found[w] : 0;
                total += found[w];
            }
            if (mine) entries[at] = make_float2(__int_as_float(id - e0), __ldg(a.bias_values + row * a.bias_stride + i + tid));
            __syncthreads();
            if (tid < total) {
                const int slot = __float_as_int(entries[tid].x);
                bool leads = true;
                for (int k = 0; k < tid; ++k) leads &= __float_as_int(entries[k].x) != slot;
                if (leads) {
                    float sum = bias[slot];
                    for (int k = tid; k < total; ++k)
                        if (__float_as_int(entries[k].x) == slot) sum = __fadd_rn(sum, entries[k].y);
                    bias[slot] = sum;
                }
            }
        }
        __syncthreads();
#pragma unroll
        for (int u = 0; u < kVecs; ++u) {
            const int v = v0 + u * kLogitsThreads + tid, e = v * V - skew, at = (v - v0) * V;
            if (v >= v1) continue;
            const bool whole = e >= 0 && e + V <= a.vocab;
#pragma unroll
            for (int i0 = 0; i0 < V; i0 += 4) {
                int c[4];
                float add[4];
                *reinterpret_cast<int4*>(c) = n_hist ? *reinterpret_cast<const int4*>(counts + at + i0) : make_int4(0, 0, 0, 0);
                if (n_bias) *reinterpret_cast<float4*>(add) = *reinterpret_cast<const float4*>(bias + at + i0);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int i = i0 + k, id = e + i;
                    if (!whole && (id < 0 || id >= a.vocab)) continue;
                    float y = to_f32(x[u].v[i]);
                    if (c[k]) {
                        const int n = c[k] >> 1;
                        if (a.repetition) y = y > 0.f ? __fdiv_rn(y, rep) : __fmul_rn(y, rep);
                        if (n) y = __fsub_rn(__fsub_rn(y, __fmul_rn(freq, static_cast<float>(n))), pres);
                    }
                    if (n_bias) y = __fadd_rn(y, add[k]);
                    const uint32_t w = (id >> 5) == (max(e, 0) >> 5) ? words[u].x : words[u].y;
                    if (!(w >> (id & 31) & 1)) y = -INFINITY;
                    x[u].v[i] = from_f32<T>(y);
                    key = max(key, logit_key(to_f32(x[u].v[i]), id));
                }
            }
            if (whole && aligned_out) {
                *reinterpret_cast<Vec<T, V>*>(out + e) = x[u];
            } else {
#pragma unroll
                for (int i = 0; i < V; ++i)
                    if (e + i >= 0 && e + i < a.vocab) out[e + i] = x[u].v[i];
            }
        }
    }
    if (!a.best) return;
#pragma unroll
    for (int o = 16; o; o >>= 1) key = max(key, __shfl_xor_sync(~0u, key, o));
    if ((tid & 31) == 0) keys[tid >> 5] = key;
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
