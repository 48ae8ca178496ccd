// rope.cuh — rotary positions of query and key heads on device tensors:
// half or interleaved pairs, the first `rot` of a head's dims, any table of
// angles per position (scaled ones included).
//
//   half:         (x_i, x_{i+rot/2}),  interleaved: (x_{2i}, x_{2i+1})
//   y_a = f (x_a cos t - x_b sin t),   y_b = f (x_b cos t + x_a sin t),   t = pos * freq_i
//
// The angle is formed in 64 bits as turns, pos * (freq_i / 2 pi), and reduced
// to [-1/2, 1/2] there: in 32 bits pos * freq alone is off by 0.06 rad at
// position 10^6.  cos and sin of the reduced angle, the products and the sums
// are 32-bit; the result is rounded once to the tensor's type.
#pragma once
#include <cuda_bf16.h>

#include "common.cuh"

namespace qtts {

struct RopeArgs {
    const void * q, * k;              // k may be null
    void * q_out, * k_out;            // may be the inputs themselves
    int64_t qs_row, qs_head, ks_row, ks_head, qo_row, qo_head, ko_row, ko_head;   // strides in elements
    const int * pos;                  // [rows]
    const double * freq;              // [rot/2] radians per position
    float factor;                     // on the rotated dims
    int rows, q_heads, k_heads, dim, rot, interleaved;
    int heads_per_warp, chunks;       // chunks = warps per row
};

__device__ __forceinline__ float2 rope_unit(int pos, double freq, float factor) {
    const double turns = (double) pos * (freq * 0.15915494309189533577);   // 1 / (2 pi)
    const float r = (float)(turns - rint(turns));
    float s, c;
    sincospif(2.0f * r, &s, &c);
    return make_float2(c * factor, s * factor);
}

// One warp per (row, run of heads).  A lane owns V consecutive dims of every
// head, so it holds their cos / sin in registers for all heads of the run; the
// partner values of a head go through shared memory, which serves every layout,
// pair distance and rotated part alike.
constexpr int ROPE_WARPS = 8;
template <class T, int V>
__global__ void __launch_bounds__(ROPE_WARPS * 32) k_rope(RopeArgs a) {
    constexpr int D = V * 32;
    __shared__ float2 s_cs[ROPE_WARPS][D / 2];
    __shared__ __align__(16) T s_x[ROPE_WARPS][D];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t unit = (int64_t) blockIdx.x * ROPE_WARPS + warp;
    const int64_t row = unit / a.chunks;
    if (row >= a.rows) return;
    const int h0 = (int)(unit % a.chunks) * a.heads_per_warp;
    const int h1 = min(a.q_heads + a.k_heads, h0 + a.heads_per_warp);
    const int half = a.rot >> 1, pos = a.pos[row];
    for (int i = lane; i < half; i += 32) s_cs[warp][i] = rope_unit(pos, a.freq[i], a.factor);
    __syncwarp();
    float c[V], s[V];
    int partner[V];
#pragma unroll
    for (int e = 0; e < V; ++e) {
        const int d = lane * V + e;
        c[e] = 1.0f; s[e] = 0.0f; partner[e] = d;
        if (d < a.rot) {
            const int i = a.interleaved ? d >> 1 : (d < half ? d : d - half);
            const bool first = a.interleaved ? !(d & 1) : d < half;
            const float2 u = s_cs[warp][i];
            c[e] = u.x;
            s[e] = first ? -u.y : u.y;
            partner[e] = a.interleaved ? d ^ 1 : (first ? d + half : d - half);
        }
    }
    struct alignas(sizeof(T) * V) Vec { T x[V]; };
    for (int h = h0; h < h1; ++h) {
        const bool is_q = h < a.q_heads;
        const int hh = is_q ? h : h - a.q_heads;
        const T * src = static_cast<const T *>(is_q ? a.q : a.k) + row * (is_q ? a.qs_row : a.ks_row) + hh * (is_q ? a.qs_head : a.ks_head);
        T * dst = static_cast<T *>(is_q ? a.q_out : a.k_out) + row * (is_q ? a.qo_row : a.ko_row) + hh * (is_q ? a.qo_head : a.ko_head);
        const Vec x = *reinterpret_cast<const Vec *>(src + lane * V);
        *reinterpret_cast<Vec *>(&s_x[warp][lane * V]) = x;
        __syncwarp();
        Vec y;
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const float o = (float) s_x[warp][partner[e]];
            y.x[e] = lane * V + e < a.rot ? T(__fmaf_rn((float) x.x[e], c[e], __fmul_rn(o, s[e]))) : x.x[e];
        }
        *reinterpret_cast<Vec *>(dst + lane * V) = y;
        __syncwarp();
    }
}

// Any head size and any alignment: one thread per (row, head, pair or unrotated dim).
template <class T>
__global__ void __launch_bounds__(256) k_rope_any(RopeArgs a) {
    const int half = a.rot >> 1, units = a.dim - half, heads = a.q_heads + a.k_heads;
    const int64_t total = (int64_t) a.rows * heads * units;
    for (int64_t t = (int64_t) blockIdx.x * blockDim.x + threadIdx.x; t < total; t += (int64_t) gridDim.x * blockDim.x) {
        const int u = (int)(t % units), h = (int)(t / units % heads);
        const int64_t row = t / units / heads;
        const bool is_q = h < a.q_heads;
        const int hh = is_q ? h : h - a.q_heads;
        const T * src = static_cast<const T *>(is_q ? a.q : a.k) + row * (is_q ? a.qs_row : a.ks_row) + hh * (is_q ? a.qs_head : a.ks_head);
        T * dst = static_cast<T *>(is_q ? a.q_out : a.k_out) + row * (is_q ? a.qo_row : a.ko_row) + hh * (is_q ? a.qo_head : a.ko_head);
        if (u >= half) { dst[half + u] = src[half + u]; continue; }
        const float2 cs = rope_unit(a.pos[row], a.freq[u], a.factor);
        const int ia = a.interleaved ? 2 * u : u, ib = a.interleaved ? 2 * u + 1 : u + half;
        const float xa = (float) src[ia], xb = (float) src[ib];
        dst[ia] = T(__fmaf_rn(xa, cs.x, __fmul_rn(xb, -cs.y)));
        dst[ib] = T(__fmaf_rn(xb, cs.x, __fmul_rn(xa, cs.y)));
    }
}

}  // namespace qtts
