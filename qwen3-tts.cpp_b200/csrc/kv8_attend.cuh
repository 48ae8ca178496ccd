// kv8_attend.cuh — attention over the 8-bit paged cache (kv8.cuh).
//
//   s_j = scale * k_scale(j) * sum_d q_d ck_jd            (codes ck, cv)
//   p_j = exp(s_j - m) / l,   o_d = sum_j p_j v_scale(j) cv_jd
//
// over the keys j that a row sees: j <= p and, with a window w, j > p - w, where
// p = len - n + i is the position of row i of the n rows that a sequence brings.
// A row that sees nothing gives zeros and lse = -inf.
#pragma once
#include "kv8.cuh"

namespace qtts {

struct K8AttendArgs {
    qtts_kv8 c;
    const int32_t * table, * lens, * cu;
    const void * q;
    void * out;
    int64_t q_row, q_head, o_row, o_head;      // strides in elements
    int n_rows, max_q, n_heads, window;
    float scale;
    float * lse;                               // [n_rows][n_heads] or null
    const float * w_in;                        // [n_seqs][H][w_stride] or null
    float * w_out;
    int64_t w_stride;
};

// Keys [lo, hi) of row i of a sequence.
__device__ __forceinline__ void k8_span(const K8Seq & s, int i, int window, int & lo, int & hi) {
    const int p = s.len - s.n + i;
    hi = p + 1 > 0 ? p + 1 : 0;
    lo = window > 0 && p - window + 1 > 0 ? p - window + 1 : 0;
}

// The plain kernel: one warp per (row, query head), a lane owns D / 32 dims, one
// key at a time with the running maximum and sum.  Right for every case; bound by
// the five shuffles of each key.
template <class T, bool E4M3, int D>
__global__ void __launch_bounds__(128) k_kv8_attend_plain(K8AttendArgs a, float * lse_ws) {
    constexpr int V = D / 32;
    const int lane = threadIdx.x & 31, H = a.c.n_kv_heads, G = a.n_heads / H;
    const int64_t unit = (int64_t) blockIdx.x * 4 + (threadIdx.x >> 5);
    const int hq = (int)(unit % a.n_heads), i = (int)(unit / a.n_heads % a.max_q);
    const int64_t b = unit / a.n_heads / a.max_q;
    if (b >= a.c.n_seqs) return;
    const K8Seq s = k8_seq((int) b, a.lens, a.cu, a.c.max_pages, a.n_rows, a.max_q, false);
    if (s.status && lane == 0) k8_flag(a.c.status, s.status);
    if (i >= s.n) return;
    const int h = hq / G, row = s.row0 + i;
    int lo, hi;
    k8_span(s, i, a.window, lo, hi);
    const T * q = static_cast<const T *>(a.q) + row * a.q_row + hq * a.q_head + lane * V;
    float qv[V], o[V];
#pragma unroll
    for (int e = 0; e < V; ++e) { qv[e] = (float) q[e]; o[e] = 0.0f; }
    float m = -INFINITY, l = 0.0f;
    for (int j = lo; j < hi; ++j) {
        const int page = k8_page(a.table + b * a.c.max_pages, j / K8_PAGE, a.c.n_pages);
        if (page < 0) { if (lane == 0) k8_flag(a.c.status, K8_BAD_PAGE); continue; }
        const int64_t at = k8_code_off(page, h, j % K8_PAGE, H, D) + lane * V, sa = k8_scale_off(page, h, j % K8_PAGE / K8_BLOCK, H);
        float d = 0.0f;
#pragma unroll
        for (int e = 0; e < V; ++e) d = fmaf(qv[e], Code8<E4M3>::value(static_cast<const uint8_t *>(a.c.k)[at + e]), d);
        d = warp_sum(d) * a.c.k_scale[sa] * a.scale;
        const float m2 = fmaxf(m, d);
        const float f = expf(m - m2), p = expf(d - m2), ps = p * a.c.v_scale[sa];
        l = l * f + p;
#pragma unroll
        for (int e = 0; e < V; ++e) o[e] = fmaf(ps, Code8<E4M3>::value(static_cast<const uint8_t *>(a.c.v)[at + e]), o[e] * f);
        m = m2;
    }
    T * out = static_cast<T *>(a.out) + row * a.o_row + hq * a.o_head + lane * V;
    const float inv = l > 0.0f ? 1.0f / l : (l == 0.0f ? 0.0f : l);
#pragma unroll
    for (int e = 0; e < V; ++e) out[e] = T(l == 0.0f ? 0.0f : o[e] * inv);
    if (lane == 0) {
        const float L = l == 0.0f ? -INFINITY : m + logf(l);
        if (a.lse) a.lse[(int64_t) row * a.n_heads + hq] = L;
        if (lse_ws) lse_ws[(int64_t) row * a.n_heads + hq] = L;
    }
}

// Accumulated weights, plain: one warp per (sequence, kv head, key), rows and heads in order.
template <class T, bool E4M3, int D>
__global__ void __launch_bounds__(128) k_kv8_weigh_plain(K8AttendArgs a, const float * lse) {
    constexpr int V = D / 32;
    const int lane = threadIdx.x & 31, H = a.c.n_kv_heads, G = a.n_heads / H, cap = a.c.max_pages * K8_PAGE;
    const int64_t unit = (int64_t) blockIdx.x * 4 + (threadIdx.x >> 5);
    const int j = (int)(unit % cap), h = (int)(unit / cap % H);
    const int64_t b = unit / cap / H;
    if (b >= a.c.n_seqs) return;
    const K8Seq s = k8_seq((int) b, a.lens, a.cu, a.c.max_pages, a.n_rows, a.max_q, false);
    if (j >= s.len) return;
    const int page = k8_page(a.table + b * a.c.max_pages, j / K8_PAGE, a.c.n_pages);
    const int64_t wa = (b * H + h) * a.w_stride + j;
    float w = 0.0f;
    if (page >= 0) {
        const int64_t at = k8_code_off(page, h, j % K8_PAGE, H, D) + lane * V;
        const float sc = a.c.k_scale[k8_scale_off(page, h, j % K8_PAGE / K8_BLOCK, H)];
        for (int i = 0; i < s.n; ++i) {
            int lo, hi;
            k8_span(s, i, a.window, lo, hi);
            if (j < lo || j >= hi) continue;
            for (int g = 0; g < G; ++g) {
                const int row = s.row0 + i, hq = h * G + g;
                const T * q = static_cast<const T *>(a.q) + row * a.q_row + hq * a.q_head + lane * V;
                float d = 0.0f;
#pragma unroll
                for (int e = 0; e < V; ++e) d = fmaf((float) q[e], Code8<E4M3>::value(static_cast<const uint8_t *>(a.c.k)[at + e]), d);
                d = warp_sum(d) * sc * a.scale;
                w += expf(d - lse[(int64_t) row * a.n_heads + hq]);
            }
        }
    }
    if (lane == 0) a.w_out[wa] = a.w_in[wa] + w;
}

}  // namespace qtts
