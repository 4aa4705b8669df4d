// i4d_rope.cuh -- rotary positions of query and key heads.
//
// Angle = position * frequency, kept as a 64-bit fraction of a turn: the
// frequency is a fraction of a turn in units of 2^-64, so the integer product
// modulo 2^64 is the exact angle of the rounded frequency at any position, and
// the top bits give the octant.  What is left for the sine is within an eighth
// of a turn, so FP32 holds it to 2^-27 turns; no FP64 and no range reduction.
// Bound: q and k are read and written once; the angles are computed once for
// a token in shared memory and used by all of its heads.
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

// V elements per access.  An item is V elements of interleaved pairs, or V
// elements and their partners rot/2 away, or V elements that are copied.
template <typename T, int V, bool INTERLEAVED>
__global__ void __launch_bounds__(kRopeThreads) k_rope(RopeDev a, int groups) {
    __shared__ float2 cs[128];
    const int t = blockIdx.x / groups, part = blockIdx.x % groups;
    const int64_t pos = __ldg(a.positions + t);
    for (int i = threadIdx.x; i < a.rot / 2; i += kRopeThreads) {
        uint64_t turn = static_cast<uint64_t>(pos) * __ldg(a.turns + i);
        if (a.inverse) turn = 0 - turn;
        cs[i] = turn_cos_sin(turn, a.magnitude);
    }
    __syncthreads();
    const int rot_items = (INTERLEAVED ? a.rot : a.rot / 2) / V;
    const int per_head = rot_items + (a.copy_tail ? (a.dim - a.rot) / V : 0);
    const int total = (a.heads[0] + a.heads[1]) * per_head;
    for (int it = part * kRopeThreads + threadIdx.x; it < total; it += groups * kRopeThreads) {
        int h = it / per_head;
        const int slot = it - h * per_head;
        const int which = h >= a.heads[0];
        if (which) h -= a.heads[0];
        const T* in = static_cast<const T*>(a.in[which]) + t * a.in_tok[which] + h * a.in_head[which];
        T* out = static_cast<T*>(a.out[which]) + t * a.out_tok[which] + h * a.out_head[which];
        if (slot >= rot_items) {
            const int e = a.rot + (slot - rot_items) * V;
            store_vec<T, V>(out + e, load_vec<T, V>(in + e));
        } else if constexpr (INTERLEAVED) {
            Vec<T, V> x = load_vec<T, V>(in + slot * V);
#pragma unroll
            for (int i = 0; i < V; i += 2) {
                const float2 c = cs[(slot * V + i) / 2];
                const float u = to_f32(x.v[i]), w = to_f32(x.v[i + 1]);
                x.v[i] = from_f32<T>(u * c.x - w * c.y);
                x.v[i + 1] = from_f32<T>(w * c.x + u * c.y);
            }
            store_vec<T, V>(out + slot * V, x);
        } else {
            const int e = slot * V;
            Vec<T, V> x = load_vec<T, V>(in + e), y = load_vec<T, V>(in + e + a.rot / 2);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float2 c = cs[e + i];
                const float u = to_f32(x.v[i]), w = to_f32(y.v[i]);
                x.v[i] = from_f32<T>(u * c.x - w * c.y);
                y.v[i] = from_f32<T>(w * c.x + u * c.y);
            }
            store_vec<T, V>(out + e, x);
            store_vec<T, V>(out + e + a.rot / 2, y);
        }
    }
}

}  // namespace i4d_ops
