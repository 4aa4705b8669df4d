// i4d_rope.cuh -- rotary positions of query and key heads.
//
// Angle = position * frequency, kept as a 64-bit fraction of a turn: the
// frequency is a fraction of a turn in units of 2^-64, so the integer product
// modulo 2^64 is the exact angle of the rounded frequency at any position, and
// the top bits give the octant.  What is left for the sine is within an eighth
// of a turn, so FP32 holds it to 2^-27 turns; no FP64 and no range reduction.
// Bound: q and k are read and written once; a token's angles are computed once
// in shared memory and used by all of its heads (8191 tokens of 40 heads of 128
// in BF16: 30.7 us, 5.5 TB/s).
#pragma once

#include "i4d_ops_common.cuh"

namespace i4d_ops {

constexpr int kRopeThreads = 256;

struct RopeDev {
    const void* in[2];
    void* out[2];
    int64_t in_tok[2], in_head[2], out_tok[2], out_head[2];
    const int32_t* positions;
    const uint64_t* turns;
    int heads[2];
    int tokens, dim, rot, inverse;
    int copy_tail;  // 0: in place, elements behind rot stay where they are
    float magnitude;
};

__device__ __forceinline__ float2 turn_cos_sin(uint64_t turn, float magnitude) {
    // quarter q and remainder r in [-1/8, 1/8) turns
    const uint64_t shifted = turn + (1ull << 61);
    const int quarter = static_cast<int>(shifted >> 62);
    const int64_t rem = static_cast<int64_t>(turn - (static_cast<uint64_t>(quarter) << 62));
    float s, c;
    sincospif(static_cast<float>(rem) * 0x1p-63f, &s, &c);
    const float cc = quarter & 1 ? s : c, ss = quarter & 1 ? c : s;
    return make_float2((quarter == 1 || quarter == 2) ? -cc * magnitude : cc * magnitude,
                       quarter >= 2 ? -ss * magnitude : ss * magnitude);
}

// (cos, sin) * magnitude of pair i's angle at token t.
__device__ __forceinline__ float2 rope_angle(const RopeDev& a, int t, int i) {
    const uint64_t turn = static_cast<uint64_t>(static_cast<int64_t>(fetch(a.positions + t))) * fetch(a.turns + i);
    return turn_cos_sin(a.inverse ? 0 - turn : turn, a.magnitude);
}

// One item: V elements of interleaved pairs, or V elements and their partners
// rot/2 away, or V elements that are copied.
template <typename T, int V, bool INTERLEAVED>
struct RopeItem {
    Vec<T, V> x, y;
    T* out;
    int slot;  // -1: none

    __device__ __forceinline__ void load(const RopeDev& a, int64_t t, int it, int total, int per_head, int rot_items) {
        slot = -1;
        if (it >= total) return;
        int h = it / per_head;
        slot = it - h * per_head;
        const int which = h >= a.heads[0];
        if (which) h -= a.heads[0];
        const T* in = static_cast<const T*>(a.in[which]) + t * a.in_tok[which] + h * a.in_head[which];
        out = static_cast<T*>(a.out[which]) + t * a.out_tok[which] + h * a.out_head[which];
        if (slot >= rot_items) {
            x = load_vec<T, V>(in + a.rot + (slot - rot_items) * V);
        } else {
            x = load_vec<T, V>(in + slot * V);
            if constexpr (!INTERLEAVED) y = load_vec<T, V>(in + slot * V + a.rot / 2);
        }
    }

    __device__ __forceinline__ void finish(const RopeDev& a, const float2* cs, int rot_items) {
        if (slot < 0) return;
        if (slot >= rot_items) {
            store_vec<T, V>(out + a.rot + (slot - rot_items) * V, x);
        } else if constexpr (INTERLEAVED) {
#pragma unroll
            for (int i = 0; i < V; i += 2) {
                const float2 c = cs[(slot * V + i) / 2];
                const float u = to_f32(x.v[i]), w = to_f32(x.v[i + 1]);
                x.v[i] = from_f32<T>(u * c.x - w * c.y);
                x.v[i + 1] = from_f32<T>(w * c.x + u * c.y);
            }
            store_vec<T, V>(out + slot * V, x);
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float2 c = cs[slot * V + i];
                const float u = to_f32(x.v[i]), w = to_f32(y.v[i]);
                x.v[i] = from_f32<T>(u * c.x - w * c.y);
                y.v[i] = from_f32<T>(w * c.x + u * c.y);
            }
            store_vec<T, V>(out + slot * V, x);
            store_vec<T, V>(out + slot * V + a.rot / 2, y);
        }
    }
};

// Few tokens: `groups` CTAs for each.
template <typename T, int V, bool INTERLEAVED>
__global__ void __launch_bounds__(kRopeThreads) k_rope(RopeDev a, int groups) {
    op_begin();
    __shared__ float2 cs[128];
    const int t = blockIdx.x / groups, part = blockIdx.x % groups;
    const int rot_items = (INTERLEAVED ? a.rot : a.rot / 2) / V;
    const int per_head = rot_items + (a.copy_tail ? (a.dim - a.rot) / V : 0);
    const int total = (a.heads[0] + a.heads[1]) * per_head;
    for (int i = threadIdx.x; i < a.rot / 2; i += kRopeThreads) cs[i] = rope_angle(a, t, i);
    __syncthreads();
    for (int it = part * kRopeThreads + threadIdx.x; it < total; it += groups * kRopeThreads) {
        RopeItem<T, V, INTERLEAVED> item;
        item.load(a, t, it, total, per_head, rot_items);
        item.finish(a, cs, rot_items);
    }
}

constexpr int kRopeWarps = 4;

// Many tokens: a warp for each, no barrier of the CTA.  A lane keeps one place
// of a head, and so its pairs' cosines and sines, in registers and walks the
// heads; the elements that are copied go in a walk of their own.  (With a
// division and the angles from shared memory for every item it was bound by
// 195 instructions an item: 8191 tokens of 40 heads, half rotated, 41 us.)
template <typename T, int V, bool INTERLEAVED>
__global__ void __launch_bounds__(32 * kRopeWarps) k_rope_many(RopeDev a) {
    op_begin();
    constexpr int kPairs = INTERLEAVED ? V / 2 : V;
    constexpr int kAhead = 4;
    __shared__ float2 angles[kRopeWarps][128];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, t = blockIdx.x * kRopeWarps + warp;
    if (t >= a.tokens) return;
    for (int i = lane; i < a.rot / 2; i += 32) angles[warp][i] = rope_angle(a, t, i);
    __syncwarp();
    const int places[2] = {(INTERLEAVED ? a.rot : a.rot / 2) / V, a.copy_tail ? (a.dim - a.rot) / V : 0};
#pragma unroll
    for (int copy = 0; copy < 2; ++copy) {
        // 2^log places of a head side by side, the heads of a step after them
        const int n = places[copy], log = n >= 32 ? 5 : n <= 1 ? 0 : 32 - __clz(n - 1), step = 32 >> log;
        for (int place = lane & ((1 << log) - 1); place < n; place += 32) {
            float2 c[kPairs];
            if (!copy) {
#pragma unroll
                for (int i = 0; i < kPairs; ++i) c[i] = angles[warp][place * kPairs + i];
            }
            const int at = copy ? a.rot + place * V : place * V;
#pragma unroll
            for (int which = 0; which < 2; ++which) {
                const T* in = static_cast<const T*>(a.in[which]) + t * a.in_tok[which] + at;
                T* out = static_cast<T*>(a.out[which]) + t * a.out_tok[which] + at;
                const int64_t in_head = a.in_head[which], out_head = a.out_head[which];
                const int heads = a.heads[which];
                for (int h0 = lane >> log; h0 < heads; h0 += step * kAhead) {
                    Vec<T, V> x[kAhead], y[kAhead];
#pragma unroll
                    for (int u = 0; u < kAhead; ++u) {
                        const int h = h0 + u * step;
                        if (h < heads) {
                            x[u] = load_vec<T, V>(in + h * in_head);
                            if (!copy && !INTERLEAVED) y[u] = load_vec<T, V>(in + h * in_head + a.rot / 2);
                        }
                    }
#pragma unroll
                    for (int u = 0; u < kAhead; ++u) {
                        const int h = h0 + u * step;
                        if (h >= heads) break;
                        if (!copy) {
#pragma unroll
                            for (int i = 0; i < kPairs; ++i) {
                                T& first = x[u].v[INTERLEAVED ? 2 * i : i];
                                T& second = INTERLEAVED ? x[u].v[INTERLEAVED ? 2 * i + 1 : 0] : y[u].v[INTERLEAVED ? 0 : i];
                                const float p = to_f32(first), q = to_f32(second);
                                first = from_f32<T>(p * c[i].x - q * c[i].y);
                                second = from_f32<T>(q * c[i].x + p * c[i].y);
                            }
                        }
                        store_vec<T, V>(out + h * out_head, x[u]);
                        if (!copy && !INTERLEAVED) store_vec<T, V>(out + h * out_head + a.rot / 2, y[u]);
                    }
                }
            }
        }
    }
}

}  // namespace i4d_ops
