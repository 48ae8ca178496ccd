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

// Two 16-bit values of a word as floats, and back (one rounding each).
template <class T> __device__ __forceinline__ float2 rope_up(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2 *>(&w)); }
template <> __device__ __forceinline__ float2 rope_up<__nv_bfloat16>(uint32_t w) { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }
template <class T> __device__ __forceinline__ uint32_t rope_down(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
template <> __device__ __forceinline__ uint32_t rope_down<__nv_bfloat16>(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
// 16 bytes as floats.
template <class T> struct RopeWord {
    static constexpr int V = 16 / sizeof(T);
    float x[V];
    __device__ __forceinline__ explicit RopeWord(const uint4 & u) {
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (sizeof(T) == 4) x[i] = __uint_as_float(w[i]);
            else { const float2 f = rope_up<T>(w[i]); x[2 * i] = f.x; x[2 * i + 1] = f.y; }
        }
    }
    __device__ __forceinline__ uint4 pack() const {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (sizeof(T) == 4) w[i] = __float_as_uint(x[i]);
            else w[i] = rope_down<T>(x[2 * i], x[2 * i + 1]);
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
};

// One warp per (row, run of heads).  A lane owns the same 16 bytes of every head it
// sees (L lanes a head, 32 / L heads at a time), so it holds their cos / sin in
// registers for the whole run; the next heads' loads are in flight while these are
// turned.  Partners: in the lane's own word (interleaved), 16 bytes of another lane
// through shared memory (half), or, where the rotated part does not end or split at a
// word, single values of shared memory.  Bound by memory: every value is read and
// written once.
constexpr int ROPE_WARPS = 8, ROPE_DEEP = 2;
enum : int { ROPE_PAIR = 0, ROPE_WORD = 1, ROPE_VALUE = 2 };
template <class T, int L, int MODE>
__global__ void __launch_bounds__(ROPE_WARPS * 32) k_rope(RopeArgs a) {
    constexpr int V = 16 / sizeof(T), D = L * V, HPW = 32 / L;
    __shared__ float2 s_cs[ROPE_WARPS][D / 2];
    __shared__ uint4 s_x[MODE == ROPE_PAIR ? 1 : ROPE_WARPS][ROPE_DEEP][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = lane / L, d0 = lane % L * V;
    const int64_t unit = (int64_t) blockIdx.x * ROPE_WARPS + warp;
    const int64_t row = unit / a.chunks;
    pdl_trigger();
    pdl_wait();
    if (row >= a.rows) return;
    const int h0 = (int)(unit % a.chunks) * a.heads_per_warp, heads = a.q_heads + a.k_heads, h1 = min(heads, h0 + a.heads_per_warp);
    const int half = a.rot >> 1;
    // key heads follow the query heads: head h of k at k + (h - q_heads) * stride
    const T * qi = static_cast<const T *>(a.q) + row * a.qs_row + d0, * ki = static_cast<const T *>(a.k) + row * a.ks_row - a.q_heads * a.ks_head + d0;
    T * qo = static_cast<T *>(a.q_out) + row * a.qo_row + d0, * ko = static_cast<T *>(a.k_out) + row * a.ko_row - a.q_heads * a.ko_head + d0;
    uint4 x[ROPE_DEEP];
    auto load = [&](int hb) {
#pragma unroll
        for (int i = 0; i < ROPE_DEEP; ++i) {
            const int h = hb + i * HPW + sub;
            if (h < h1) x[i] = *reinterpret_cast<const uint4 *>(h < a.q_heads ? qi + h * a.qs_head : ki + h * a.ks_head);
        }
    };
#pragma unroll
    for (int i = 0; i < ROPE_DEEP; ++i) x[i] = make_uint4(0, 0, 0, 0);
    load(h0);
    const int pos = a.pos[row];
    for (int i = lane; i < half; i += 32) s_cs[warp][i] = rope_unit(pos, a.freq[i], a.factor);
    __syncwarp();
    float c[V], s[V];
    int partner[V];
    bool turned[V];
#pragma unroll
    for (int e = 0; e < V; ++e) {
        const int d = d0 + e;
        turned[e] = MODE == ROPE_VALUE ? d < a.rot : d0 < a.rot;
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
    for (int hb = h0; hb < h1; hb += ROPE_DEEP * HPW) {
        uint4 now[ROPE_DEEP];
#pragma unroll
        for (int i = 0; i < ROPE_DEEP; ++i) now[i] = x[i];
        if (hb + ROPE_DEEP * HPW < h1) load(hb + ROPE_DEEP * HPW);
        if (MODE != ROPE_PAIR) {
            __syncwarp();
#pragma unroll
            for (int i = 0; i < ROPE_DEEP; ++i) s_x[warp][i][lane] = now[i];
            __syncwarp();
        }
#pragma unroll
        for (int i = 0; i < ROPE_DEEP; ++i) {
            const int h = hb + i * HPW + sub;
            uint4 y = now[i];
            if (turned[0]) {
                RopeWord<T> v(now[i]), o(MODE == ROPE_WORD ? s_x[warp][i][sub * L + partner[0] / V] : now[i]), r(now[i]);
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const float p = MODE == ROPE_PAIR ? v.x[e ^ 1]
                                  : MODE == ROPE_WORD ? o.x[e] : (float) reinterpret_cast<const T *>(&s_x[warp][i][sub * L])[partner[e]];
                    if (MODE != ROPE_VALUE || turned[e]) r.x[e] = __fmaf_rn(v.x[e], c[e], __fmul_rn(p, s[e]));
                }
                y = r.pack();                         // values that do not turn come back as they were: the conversions are exact
            }
            if (h < h1) *reinterpret_cast<uint4 *>(h < a.q_heads ? qo + h * a.qo_head : ko + h * a.ko_head) = y;
        }
    }
}

// Any head size and any alignment: one thread per (row, head, pair or unrotated dim).
template <class T>
__global__ void __launch_bounds__(256) k_rope_any(RopeArgs a) {
    const int half = a.rot >> 1, units = a.dim - half, heads = a.q_heads + a.k_heads;
    const int64_t total = (int64_t) a.rows * heads * units;
    pdl_trigger();
    pdl_wait();
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
