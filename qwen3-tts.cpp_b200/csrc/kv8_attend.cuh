// kv8_attend.cuh — attention over the 8-bit paged cache (kv8.cuh).
//
//   s_j = scale * k_scale(j) * sum_d q_d ck_jd            (codes ck, cv)
//   p_j = exp(s_j - m) / l,   o_d = sum_j p_j v_scale(j) cv_jd
//
// over the keys j that a row sees: j <= p and, with a window w, j > p - w, where
// p = len - n + i is the position of row i of the n rows that a sequence brings.
// A row that sees nothing gives zeros and lse = -inf.
//
// The products run on the tensor cores in F16 with F32 sums: codes of both kinds
// are exact in F16, the scales stay outside in F32.  Bound by memory for few rows: at
// 32 sequences of 4,400 (287 MB) 59 us, 4.85 TB/s, 75% of the measured copy rate; 12 us of
// it are fixed latency, beyond which it runs at 6.2 TB/s.
#pragma once
#include <cuda.h>
#include <type_traits>

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
    int * line;                                // split kernel: [n_seqs + 1] pages of work before each sequence
    float * part;                              // and its partial results
    int tiles;                                 // row tiles of one (sequence, kv head)
    int ctas;                                  // CTAs of the split kernel
    int part_rows;                             // rows of a partial result
};

// Keys [lo, hi) of row i of a sequence.
__device__ __forceinline__ void k8_span(const K8Seq & s, int i, int window, int & lo, int & hi) {
    const int p = s.len - s.n + i;
    hi = p + 1 > 0 ? p + 1 : 0;
    lo = window > 0 && p - window + 1 > 0 ? p - window + 1 : 0;
}

// ---- fragments ---------------------------------------------------------------
// The scores are formed transposed, S^T = K Q^T (16 keys x 8 rows per MMA), and so
// is the output, O^T = V^T P^T (16 dims x 8 rows): with one query token a group of
// G <= 8 heads fills one MMA column tile, where the usual orientation would pad it
// to 16.  An MMA's inner index may be permuted freely if both operands agree, so a
// lane reads what it needs from a block's rows as 16-byte words:
//   K: lane (g, t) = (lane / 4, lane % 4) holds 16 consecutive dims (chunk t of each 64)
//      of keys k8_key(g) and k8_key(g) + 8; word w of them is one k-step (4 dims a lane).
//   V: the lane holds D / 8 dims (chunk g of each 128) of the keys of MMA rows 2t, 2t+1
//      and those + 8; dims 2j and 2j+1 of them are rows g and g + 8 of output tile j.
// Nothing is exchanged or transposed between the page and the MMA.  The rows lie in
// shared memory as TMA's 128-byte swizzle leaves them (16-byte chunk ^= row % 8), and
// k8_key's order spreads both patterns over all banks: eight lanes read chunks t of two
// keys that differ in bit 2 (K), and chunks g, g ^ 1 of four keys that differ in bits
// 1 and 2 (V).
__device__ __forceinline__ void k8_mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float k8_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t k8_pack(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ uint32_t k8_transpose(uint32_t x) {   // an 8 x 8 matrix of 16-bit values over the warp
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ int k8_key(int g) { return g ^ (g & 1) << 2; }   // the key of MMA row g

struct K8Maps { CUtensorMap k, v; };             // the pools as [pages * kv heads * 64][D] bytes, boxes of a step's rows x min(D, 128)

// A slot of a warp's ring in shared memory: the K and the V rows of U blocks (D = 256: in
// two halves of 128 dims), swizzled.  Beside the ring: the page's scales and a barrier
// for each slot.
template <int D, int U> struct K8Slot {
    static constexpr int rows = U * K8_BLOCK, row_bytes = D < 128 ? D : 128, half = rows * row_bytes, side = D < 256 ? half : 2 * half, bytes = 2 * side;
};
__device__ __forceinline__ void k8_tma(uint32_t dst, const CUtensorMap * map, int x, int y, uint64_t * bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                 ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(smem_u32(bar)) : "memory");
}
// One lane: a step's rows and its page's scales into a slot.
template <int D, int U>
__device__ __forceinline__ void k8_fetch(uint32_t slot, float * scales, uint64_t * bar, const K8AttendArgs & a, const K8Maps & maps, int page, int h, int block) {
    using Slot = K8Slot<D, U>;
    const int H = a.c.n_kv_heads, y = (page * H + h) * K8_PAGE + block * K8_BLOCK;
    mbar_expect_tx(bar, Slot::bytes + 32);
#pragma unroll
    for (int x = 0; x < D; x += 128) {
        k8_tma(slot + x / 128 * Slot::half, &maps.k, x, y, bar);
        k8_tma(slot + Slot::side + x / 128 * Slot::half, &maps.v, x, y, bar);
    }
    bulk_g2s(scales, a.c.k_scale + k8_scale_off(page, h, 0, H), 16, bar);
    bulk_g2s(scales + 4, a.c.v_scale + k8_scale_off(page, h, 0, H), 16, bar);
}
__device__ __forceinline__ uint4 k8_lds16(uint32_t p) {
    uint4 r;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(p) : "memory");
    return r;
}
__device__ __forceinline__ uint2 k8_lds8(uint32_t p) {
    uint2 r;
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(r.x), "=r"(r.y) : "r"(p) : "memory");
    return r;
}
// The first dim of output tile j of a lane (its second one follows).
template <int D> __device__ __forceinline__ int k8_dim(int j, int lane) {
    const int g = lane >> 2;
    if constexpr (D == 64) return g * 8 + 2 * j;
    else return (j >> 3) * 128 + g * 16 + 2 * (j & 7);
}

// The query rows of a tile as MMA column fragments: row g (+ 8 nt) of a lane, dims as
// in K.  BF16 rows are scaled by a power of two to a largest magnitude in [1, 2)
// first (F16 has their precision but not their range; what falls below F16's
// smallest step is 2^-25 of the row's largest value); `back` undoes it.
template <class T, int D> struct K8Q { uint32_t x[D / 16][2]; };
template <class T, int D>
__device__ __forceinline__ float k8_load_q(K8Q<T, D> & q, const T * row, int lane, bool real) {
    const uint16_t * p = reinterpret_cast<const uint16_t *>(row) + (lane & 3) * 16;
    uint32_t most = 0;
    const bool vec = (reinterpret_cast<uintptr_t>(row) & 15) == 0;
#pragma unroll
    for (int c = 0; c < D / 64; ++c) {
        uint32_t w[8];
        if (!real) {
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i] = 0;
        } else if (vec) {
            const uint4 x = *reinterpret_cast<const uint4 *>(p + c * 64), y = *reinterpret_cast<const uint4 *>(p + c * 64 + 8);
            w[0] = x.x; w[1] = x.y; w[2] = x.z; w[3] = x.w; w[4] = y.x; w[5] = y.y; w[6] = y.z; w[7] = y.w;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i] = p[c * 64 + 2 * i] | (uint32_t) p[c * 64 + 2 * i + 1] << 16;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            q.x[4 * c + (i >> 1)][i & 1] = w[i];
            most = max(most, max(w[i] & 0x7fffu, (w[i] >> 16) & 0x7fffu));
        }
    }
    if constexpr (sizeof(T) == 2 && Row16<T>::inf == 0x7c00u) return 1.0f;
    most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
    most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
    // 2^-e and 2^e of the largest magnitude's exponent, kept within F32
    int e = (int)(most >> 7) - 127;
    e = most == 0 || most >= Row16<T>::inf ? 0 : max(-120, min(120, e));
    const float down = __int_as_float((127 - e) << 23), back = __int_as_float((127 + e) << 23);
#pragma unroll
    for (int i = 0; i < D / 16; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const uint32_t w = q.x[i][j];
            q.x[i][j] = k8_pack(__uint_as_float(w << 16) * down, __uint_as_float(w & 0xffff0000u) * down);
        }
    return back;
}

// ---- few rows ----------------------------------------------------------------
// One warp's running state over its blocks: per row a reference value m (log2 units)
// and the sum of the weights 2^(s - m + 8), and the output in units of `unit`, a V
// scale.  References move only when a score passes m by more than 4, or a block's V
// scale passes `unit` more than 8 times: most blocks need a vote and no reduction over
// lanes.  A weight times its block's V scale over `unit`, at most 2^15, is rounded to
// F16 for the product with V: half a step is 2^-12 relative, independent from key to
// key, or 2^-33 of the largest weight times the largest V scale.  That is well under
// the rounding of a BF16 output; for an F16 output, where it is as large (1.45 times the
// plain form's error), the rest of the weight takes a second product with up to 8 rows
// (the plain form's error, no time: 57.8 us against 59 at 32 sequences of 4,400).  The sum
// of the weights is taken before that, in F32.
constexpr float K8_LIFT = 8.0f, K8_SLACK = 4.0f, K8_UNIT_SLACK = 8.0f, K8_UNIT_MIN = 7.8886090522101181e-31f;   // 2^-100
template <int D, int NT> struct K8State {
    float m[NT][2], l[NT][2], o[NT][D / 16][4];   // rows 8 nt + 2t, + 1
    float unit;
};
struct K8Rows { int lo[2], hi[2]; };              // keys of the lane's rows 8 nt + 2t + {0, 1}

// Blocks that a warp works on together (independent chains of MMAs), and its ring's
// slots: enough bytes in flight to cover the latency of HBM (148 SMs at 6.4 TB/s need
// some 45 KB each).
template <int D, int NT> constexpr int K8_U = D * NT <= 128 ? 2 : 1;
template <int D, int NT> constexpr int K8_SLOTS = D == 64 ? (NT == 1 ? 3 : 6) : (D == 128 ? (NT == 1 ? 2 : 4) : 2);

struct K8Ring { uint32_t ring; float * scales; uint64_t * bar; };   // a warp's own: slots, 8 scales and a barrier for each

// Steps first, first + step, .. < last of U blocks each.  `phase`: each slot's next parity.
template <bool E4M3, class T, int D, int NT>
__device__ __forceinline__ void k8_blocks(K8State<D, NT> & st, const K8Q<T, D> (&q)[NT], const float (&fac)[NT][2], const K8Rows (&rows)[NT],
                                          const K8AttendArgs & a, const int32_t * table, int h, int first, int last, int step, int all_lo, int all_hi,
                                          int any_hi, const K8Maps & maps, const K8Ring & R, uint32_t & phase, int lane) {
    constexpr int S = K8_SLOTS<D, NT>, U = K8_U<D, NT>, KEYS = U * K8_BLOCK, SPP = K8_PAGE / KEYS;
    constexpr bool LOW = Row16<T>::inf == 0x7c00u && NT == 1;   // F16 rows: the weights' low halves too
    using Slot = K8Slot<D, U>;
    // a lane's places in a block: K chunk t of key kr (chunk 4 + t: ^ 64 bytes), V chunk g of keys 2t and vr
    const int g = lane >> 2, t = lane & 3, kr = k8_key(g), vr = k8_key(2 * t + 1);
    uint32_t k_at, v_at0, v_at1;
    if constexpr (D == 64) {   // 64-byte rows, swizzle of 64 bytes: chunk ^= row / 2 % 4
        k_at = kr * 64 + ((t ^ (kr >> 1 & 3)) << 4);
        v_at0 = 2 * t * 64 + (((g >> 1) ^ t) << 4) + (g & 1) * 8;
        v_at1 = vr * 64 + (((g >> 1) ^ (vr >> 1 & 3)) << 4) + (g & 1) * 8;
    } else {
        k_at = kr * 128 + ((t ^ kr) << 4);
        v_at0 = 2 * t * 128 + ((g ^ (2 * t)) << 4);
        v_at1 = vr * 128 + ((g ^ vr) << 4);
    }
    const int count = first < last ? (last - first + step - 1) / step : 0;
    // page numbers of the next 64 steps, two to a lane
    auto page_of = [&](int i) { return i < count ? k8_page(table, (first + i * step) / SPP, a.c.n_pages) : -1; };
    int pg0 = page_of(lane), pg1 = page_of(lane + 32);
    uint32_t good = 0;                              // slots that hold a step
    auto fetch = [&](int i, int slot) {             // step i into its slot
        good &= ~(1u << slot);
        if (i < count) {
            if (i && i % 32 == 0) { pg0 = pg1; pg1 = page_of(i + 32 + lane); }
            const int page = __shfl_sync(0xffffffffu, pg0, i & 31);
            if (page >= 0) {
                good |= 1u << slot;
                if (lane == 0) k8_fetch<D, U>(R.ring + slot * Slot::bytes, R.scales + slot * 8, R.bar + slot, a, maps, page, h, (first + i * step) % SPP * U);
            } else if (lane == 0) k8_flag(a.c.status, K8_BAD_PAGE);
        }
    };
#pragma unroll
    for (int i = 0; i < S; ++i) fetch(i, i);
    int slot = 0;
    for (int i = 0; i < count; ++i) {
        const int j0 = (first + i * step) * KEYS;   // the step's first key
        const uint32_t at = R.ring + slot * Slot::bytes;
        bool have = good >> slot & 1;
        if (have) {
            have = __all_sync(0xffffffffu, mbar_wait(R.bar + slot, phase >> slot & 1));
            phase ^= 1u << slot;
            if (!have && lane == 0) k8_flag(a.c.status, K8_STUCK);
        }
        if (have) {
            float ks[U], vs[U], s[U][NT][4];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int block = (first + i * step) % SPP * U + u;
                ks[u] = R.scales[slot * 8 + block];
                vs[u] = R.scales[slot * 8 + 4 + block];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[u][nt][e] = 0.0f;
            }
#pragma unroll
            for (int c = 0; c < D / 64; ++c)
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const uint32_t kp = at + (c >> 1) * Slot::half + u * K8_BLOCK * Slot::row_bytes + (c & 1 ? k_at ^ 64 : k_at);
                    const uint4 x = k8_lds16(kp), y = k8_lds16(kp + 8 * Slot::row_bytes);
                    const uint32_t xw[4] = {x.x, x.y, x.z, x.w}, yw[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        uint32_t a0, a1, a2, a3;
                        k8_f16x4<E4M3>(xw[w], a0, a2);
                        k8_f16x4<E4M3>(yw[w], a1, a3);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) k8_mma(s[u][nt], a0, a1, a2, a3, q[nt].x[4 * c + w][0], q[nt].x[4 * c + w][1]);
                    }
                }
            // The rest of the step, twice: `whole` where every row sees every key, else with masks.
            auto finish = [&](auto whole_c) {
                constexpr bool whole = decltype(whole_c)::value;
                bool up = false;
#pragma unroll
                for (int u = 0; u < U; ++u)
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            s[u][nt][e] *= fac[nt][e & 1] * ks[u];
                            if constexpr (!whole) {
                                const int j = j0 + u * K8_BLOCK + kr + (e >> 1) * 8;
                                if (j < rows[nt].lo[e & 1] || j >= rows[nt].hi[e & 1]) s[u][nt][e] = -INFINITY;
                            }
                        }
                        up |= fmaxf(s[u][nt][0], s[u][nt][2]) > st.m[nt][0] + K8_SLACK || fmaxf(s[u][nt][1], s[u][nt][3]) > st.m[nt][1] + K8_SLACK;
                    }
                if (__any_sync(0xffffffffu, up)) {
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int r = 0; r < 2; ++r) {
                            float m = fmaxf(s[0][nt][r], s[0][nt][r + 2]);
#pragma unroll
                            for (int u = 1; u < U; ++u) m = fmaxf(m, fmaxf(s[u][nt][r], s[u][nt][r + 2]));
                            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 4));
                            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
                            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
                            m = fmaxf(m, st.m[nt][r]);
                            const float f = m == st.m[nt][r] ? 1.0f : k8_exp2(st.m[nt][r] - m);
                            st.m[nt][r] = m;
                            st.l[nt][r] *= f;
#pragma unroll
                            for (int j = 0; j < D / 16; ++j) { st.o[nt][j][r] *= f; st.o[nt][j][r + 2] *= f; }
                        }
                }
                float top = vs[0];
#pragma unroll
                for (int u = 1; u < U; ++u) top = fmaxf(top, vs[u]);
                if (top > st.unit * K8_UNIT_SLACK) {    // the same for the whole warp
                    const float f = st.unit / top;
                    st.unit = top;
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int j = 0; j < D / 16; ++j)
#pragma unroll
                            for (int e = 0; e < 4; ++e) st.o[nt][j][e] *= f;
                }
                const float inv = __fdividef(1.0f, st.unit);
                uint32_t p[U][NT][2];
                [[maybe_unused]] uint32_t p_lo[U][NT][2];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const float rv = vs[u] * inv;
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        float e[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const float x = k8_exp2(s[u][nt][i] - (st.m[nt][i & 1] - K8_LIFT));
                            // a key that a row does not see adds nothing, even before the row has seen any or if a scale is NaN
                            const bool hidden = !whole && s[u][nt][i] == -INFINITY;
                            st.l[nt][i & 1] += hidden ? 0.0f : x;
                            e[i] = hidden ? 0.0f : x * rv;
                        }
                        // rows of the transpose: keys 2t, 2t + 1 in MMA order
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            const uint32_t hi = k8_pack(e[2 * i], e[2 * i + 1]);
                            p[u][nt][i] = k8_transpose(hi);
                            if constexpr (LOW) {
                                const float2 f = k8_f32x2(hi);
                                p_lo[u][nt][i] = k8_transpose(k8_pack(e[2 * i] - f.x, e[2 * i + 1] - f.y));
                            }
                        }
                    }
                }
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    // rows of the page past the sequence's end may hold anything
                    const int beyond = any_hi - j0 - u * K8_BLOCK;
                    const uint32_t vp = at + Slot::side + u * K8_BLOCK * Slot::row_bytes;
#pragma unroll
                    for (int c = 0; c < (D + 127) / 128; ++c) {
                        uint32_t v[4][4];
                        constexpr int W = D == 64 ? 2 : 4;
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const uint32_t p = vp + c * Slot::half + (i & 1 ? v_at1 : v_at0) + (i >> 1) * 8 * Slot::row_bytes;
                            if constexpr (D == 64) {
                                const uint2 x = k8_lds8(p);
                                v[i][0] = x.x; v[i][1] = x.y;
                            } else {
                                const uint4 x = k8_lds16(p);
                                v[i][0] = x.x; v[i][1] = x.y; v[i][2] = x.z; v[i][3] = x.w;
                            }
                            if (!whole && (i & 1 ? vr : 2 * t) + (i >> 1) * 8 >= beyond)
#pragma unroll
                                for (int w = 0; w < W; ++w) v[i][w] = 0;
                        }
#pragma unroll
                        for (int w = 0; w < W; ++w) {
                            uint32_t a0[2], a1[2], a2[2], a3[2];
                            // tokens' bytes side by side: [x0 y0 x1 y1], [x2 y2 x3 y3]
                            k8_f16x4<E4M3>(k8_prmt(v[0][w], v[1][w], 0x5140), a0[0], a1[0]);
                            k8_f16x4<E4M3>(k8_prmt(v[0][w], v[1][w], 0x7362), a0[1], a1[1]);
                            k8_f16x4<E4M3>(k8_prmt(v[2][w], v[3][w], 0x5140), a2[0], a3[0]);
                            k8_f16x4<E4M3>(k8_prmt(v[2][w], v[3][w], 0x7362), a2[1], a3[1]);
#pragma unroll
                            for (int o = 0; o < 2; ++o)
#pragma unroll
                                for (int nt = 0; nt < NT; ++nt)
                                    {
                                    k8_mma(st.o[nt][c * 8 + 2 * w + o], a0[o], a1[o], a2[o], a3[o], p[u][nt][0], p[u][nt][1]);
                                    if constexpr (LOW) k8_mma(st.o[nt][c * 8 + 2 * w + o], a0[o], a1[o], a2[o], a3[o], p_lo[u][nt][0], p_lo[u][nt][1]);
                                }
                        }
                    }
                }
            };
            if (j0 >= all_lo && j0 + KEYS <= all_hi) finish(std::true_type{});
            else finish(std::false_type{});
        }
        __syncwarp();                               // the slot has been read
        if (!have && (good >> slot & 1)) {          // a copy that never came: no more of them, and none in flight at the end
            for (int o = 1; o < S; ++o) {
                const int other = (slot + o) % S;
                if (good >> other & 1) { mbar_wait(R.bar + other, phase >> other & 1); phase ^= 1u << other; }
            }
            break;
        }
        fetch(i + S, slot);
        slot = slot + 1 == S ? 0 : slot + 1;
    }
}

// Pages [pg0, pg1) of a sequence that any of its rows sees.
__device__ __forceinline__ void k8_pages(const K8Seq & s, int window, int & pg0, int & pg1) {
    int lo, hi;
    k8_span(s, 0, window, lo, hi);
    pg0 = lo / K8_PAGE;
    pg1 = s.n > 0 ? (s.len + K8_PAGE - 1) / K8_PAGE : 0;
    if (pg1 < pg0) pg1 = pg0;
}

template <class T> __device__ __forceinline__ void k8_write_row(const K8AttendArgs & a, int row, int hq, int d, float o, float inv) {
    static_cast<T *>(a.out)[row * a.o_row + hq * a.o_head + d] = T(o * inv);
}

// One warp: its share (steps first, first + step, ..) of pages [pg0, pg1) of one
// (sequence, kv head, row tile).
template <class T, bool E4M3, int D, int NT>
__device__ __forceinline__ void k8_run(K8State<D, NT> & st, const K8AttendArgs & a, const K8Maps & maps, const K8Seq & s, int b, int h, int tile, int pg0, int pg1,
                                       int first, int step, const K8Ring & ring, uint32_t & phase) {
    const int lane = threadIdx.x & 31, t = lane & 3;
    const int G = a.n_heads / a.c.n_kv_heads, R = s.n * G, r0 = tile * 8 * NT;
    K8Q<T, D> q[NT];
    float fac[NT][2];
    K8Rows rows[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const int r = r0 + nt * 8 + (lane >> 2);
        const bool real = r < R;
        const T * src = static_cast<const T *>(a.q) + (real ? (s.row0 + r / G) * a.q_row + (h * G + r % G) * a.q_head : 0);
        const float back = k8_load_q<T, D>(q[nt], src, lane, real) * (a.scale * 1.44269504088896340736f);   // log2 e
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            fac[nt][i] = __shfl_sync(0xffffffffu, back, 8 * t + 4 * i);
            const int rr = r0 + nt * 8 + 2 * t + i;
            // rows of padding see what the last one sees, so that they force no masking
            k8_span(s, min(rr, R - 1) / G, a.window, rows[nt].lo[i], rows[nt].hi[i]);
        }
    }
    int lo, hi, lo1, hi1;
    k8_span(s, r0 / G, a.window, lo, hi);
    k8_span(s, min(r0 + 8 * NT - 1, R - 1) / G, a.window, lo1, hi1);
    st.unit = K8_UNIT_MIN;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            st.m[nt][i] = -INFINITY;
            st.l[nt][i] = 0.0f;
#pragma unroll
            for (int j = 0; j < D / 16; ++j) st.o[nt][j][i] = st.o[nt][j][i + 2] = 0.0f;
        }
    constexpr int KEYS = K8_U<D, NT> * K8_BLOCK;
    const int X0 = max(pg0 * (K8_PAGE / KEYS), lo / KEYS), X1 = min(pg1 * (K8_PAGE / KEYS), (hi1 + KEYS - 1) / KEYS);
    k8_blocks<E4M3, T, D, NT>(st, q, fac, rows, a, a.table + (int64_t) b * a.c.max_pages, h, X0 + first, X1, step, lo1, hi, hi1,
                              maps, ring, phase, lane);
}
// The sum of a row's weights over the lanes that hold its keys.
__device__ __forceinline__ float k8_row_sum(float l) {
    l += __shfl_xor_sync(0xffffffffu, l, 4);
    l += __shfl_xor_sync(0xffffffffu, l, 8);
    return l + __shfl_xor_sync(0xffffffffu, l, 16);
}
__device__ __forceinline__ float k8_lse(float m, float l) { return l == 0.0f ? -INFINITY : (m - K8_LIFT + log2f(l)) * 0.693147180559945309417f; }

// The warps' states of a CTA that shared an item or a part of it, joined in warp order
// through the shared memory that held the rings: to out and lse (part null), or
// unnormalised to part [part_rows][D + 4] (o, m, l).
template <class T, int D, int NT, int NW>
__device__ __forceinline__ void k8_join_warps(const K8State<D, NT> & st, const K8AttendArgs & a, const K8Seq & s, int h, int tile, float * part, float * smem) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, t = lane & 3;
    const int G = a.n_heads / a.c.n_kv_heads, R = s.n * G, r0 = tile * 8 * NT;
    __syncthreads();
    float * sm = smem, * sl = smem + NW * 8 * NT, * so = smem + 2 * NW * 8 * NT;   // [NW][8 NT] twice, [NW][8 NT][D + 4]
    constexpr int LD = D + 4;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const float l = k8_row_sum(st.l[nt][i]);
            const int r = nt * 8 + 2 * t + i;
            if (r0 + r >= R) continue;
            if (lane < 4) { sm[warp * 8 * NT + r] = st.m[nt][i]; sl[warp * 8 * NT + r] = l; }
#pragma unroll
            for (int j = 0; j < D / 16; ++j)
                *reinterpret_cast<float2 *>(so + (warp * 8 * NT + r) * LD + k8_dim<D>(j, lane)) = make_float2(st.o[nt][j][i] * st.unit, st.o[nt][j][i + 2] * st.unit);
        }
    __syncthreads();
    for (int e = threadIdx.x; e < 8 * NT * D; e += NW * 32) {
        const int r = e / D, d = e % D, rr = r0 + r;
        if (rr >= R) break;
        float m = -INFINITY, l = 0.0f, o = 0.0f;
#pragma unroll
        for (int w = 0; w < NW; ++w) m = fmaxf(m, sm[w * 8 * NT + r]);
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const float mw = sm[w * 8 * NT + r], f = mw == m ? 1.0f : k8_exp2(mw - m);
            l = fmaf(sl[w * 8 * NT + r], f, l);
            o = fmaf(so[(w * 8 * NT + r) * LD + d], f, o);
        }
        if (part) {
            part[r * (D + 4) + d] = o;
            if (d == 0) { part[r * (D + 4) + D] = m; part[r * (D + 4) + D + 1] = l; }
        } else {
            const int row = s.row0 + rr / G, hq = h * G + rr % G;
            k8_write_row<T>(a, row, hq, d, o, l == 0.0f ? 0.0f : 1.0f / l);
            if (d == 0 && a.lse) a.lse[(int64_t) row * a.n_heads + hq] = k8_lse(m, l);
        }
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // the next segment's copies write where the join wrote
    __syncthreads();
}
// Shared memory: the warps' rings, which the join uses too (a multiple of 1 KB, on a 1 KB
// boundary for the swizzle), their slots' scales and barriers.
template <int D, int NT, int NW> __host__ __device__ constexpr int k8_ring_bytes() {
    const int rings = NW * K8_SLOTS<D, NT> * K8Slot<D, K8_U<D, NT>>::bytes, join = (2 * NW * 8 * NT + NW * 8 * NT * (D + 4)) * 4;
    return ((rings > join ? rings : join) + 1023) / 1024 * 1024;
}
template <int D, int NT, int NW> __host__ __device__ constexpr int k8_smem_bytes() {
    return 1024 + k8_ring_bytes<D, NT, NW>() + NW * K8_SLOTS<D, NT> * (32 + 8);
}
extern __shared__ __align__(1024) uint8_t k8_dyn[];
template <int D, int NT, int NW> __device__ __forceinline__ uint8_t * k8_ring(K8Ring & r) {
    constexpr int S = K8_SLOTS<D, NT>;
    const int warp = threadIdx.x >> 5;
    uint8_t * base = k8_dyn + (-(int) smem_u32(k8_dyn) & 1023);
    r.ring = smem_u32(base) + warp * S * K8Slot<D, K8_U<D, NT>>::bytes;
    r.scales = reinterpret_cast<float *>(base + k8_ring_bytes<D, NT, NW>()) + warp * S * 8;
    r.bar = reinterpret_cast<uint64_t *>(base + k8_ring_bytes<D, NT, NW>() + NW * S * 32) + warp * S;
    if ((threadIdx.x & 31) == 0) {
        for (int i = 0; i < S; ++i) mbar_init(r.bar + i, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    __syncwarp();
    return base;
}

// CTAs of 4 warps that are resident together, by their registers.
__host__ __device__ constexpr int k8_ctas_per_sm(int dim, int nt) { return dim * nt <= 64 ? 4 : (dim * nt <= 128 ? 3 : 2); }

// One CTA per (sequence, kv head, row tile).
template <class T, bool E4M3, int D, int NT, int NW>
__global__ void __launch_bounds__(NW * 32, k8_ctas_per_sm(D, NT)) k_kv8_attend_whole(K8AttendArgs a, const __grid_constant__ K8Maps maps) {
    const int H = a.c.n_kv_heads, G = a.n_heads / H;
    const int tile = blockIdx.x % a.tiles, h = blockIdx.x / a.tiles % H, b = blockIdx.x / a.tiles / H;
    pdl_trigger();
    pdl_wait();
    const K8Seq s = k8_seq(b, a.lens, a.cu, a.c.max_pages, a.n_rows, a.max_q, false);
    if (threadIdx.x == 0 && h == 0 && tile == 0) k8_flag(a.c.status, s.status);
    if (tile * 8 * NT >= s.n * G) return;
    int pg0, pg1;
    k8_pages(s, a.window, pg0, pg1);
    K8Ring ring;
    float * smem = reinterpret_cast<float *>(k8_ring<D, NT, NW>(ring));
    uint32_t phase = 0;
    K8State<D, NT> st;
    k8_run<T, E4M3, D, NT>(st, a, maps, s, b, h, tile, pg0, pg1, threadIdx.x >> 5, NW, ring, phase);
    k8_join_warps<T, D, NT, NW>(st, a, s, h, tile, nullptr, smem);
}

// Split along the cache.  All (sequence, kv head, row tile) items laid end to end are
// a line of pages; CTA c takes pages [c * chunk, (c + 1) * chunk) of it, so ragged
// lengths balance to a page whatever they are.  An item that a CTA holds whole is
// finished there; parts (a CTA's first and last segment at most) go to `part` and are
// joined by k_kv8_join.  (A range for each warp of its own measured 61 and 72 us where
// this takes 59 and 60, at 32 sequences of 4,400 and two of 131,072: four times the
// parts to join.)
constexpr int K8_MAX_SPLIT_SEQS = 1024;
// Prefix sums over the sequences of their pages of work in `at` [n_seqs + 1].
template <int NT, int THREADS>
__device__ __forceinline__ void k8_line(const K8AttendArgs & a, int * at, int * s_carry) {
    const int H = a.c.n_kv_heads, G = a.n_heads / H, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (threadIdx.x == 0) { at[0] = 0; }
    int base = 0;
    for (int b0 = 0; b0 < a.c.n_seqs; b0 += THREADS) {
        const int b = b0 + threadIdx.x;
        int w = 0;
        if (b < a.c.n_seqs) {
            const K8Seq s = k8_seq(b, a.lens, a.cu, a.c.max_pages, a.n_rows, a.max_q, false);
            if (blockIdx.x == 0) k8_flag(a.c.status, s.status);
            int pg0, pg1;
            k8_pages(s, a.window, pg0, pg1);
            w = (pg1 - pg0) * H * ((s.n * G + 8 * NT - 1) / (8 * NT));
        }
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) { const int y = __shfl_up_sync(0xffffffffu, w, o); if (lane >= o) w += y; }
        __syncthreads();
        if (lane == 31) s_carry[warp] = w;
        __syncthreads();
        int before = base;
        for (int i = 0; i < warp; ++i) before += s_carry[i];
        if (b < a.c.n_seqs) at[b + 1] = before + w;
        for (int i = 0; i < THREADS / 32; ++i) base += s_carry[i];
    }
    __syncthreads();
}
// Pages of a CTA: at least 4, so that each warp has some.
__device__ __forceinline__ int k8_chunk(int total, int ctas) {
    const int c = (total + ctas - 1) / ctas;
    return c < 4 ? 4 : c;
}

template <class T, bool E4M3, int D, int NT, int NW>
__global__ void __launch_bounds__(NW * 32, k8_ctas_per_sm(D, NT)) k_kv8_attend_split(K8AttendArgs a, const __grid_constant__ K8Maps maps) {
    __shared__ int s_carry[NW];
    pdl_trigger();
    pdl_wait();
    K8Ring ring;
    uint8_t * base = k8_ring<D, NT, NW>(ring);
    uint32_t phase = 0;
    int * at = reinterpret_cast<int *>(base + k8_smem_bytes<D, NT, NW>() - 1024);
    k8_line<NT, NW * 32>(a, at, s_carry);
    if (blockIdx.x == 0)
        for (int i = threadIdx.x; i <= a.c.n_seqs; i += NW * 32) a.line[i] = at[i];
    const int total = at[a.c.n_seqs], chunk = k8_chunk(total, a.ctas);
    int pos = min(total, (int) blockIdx.x * chunk);
    const int end = min(total, pos + chunk);
    const int G = a.n_heads / a.c.n_kv_heads;
    bool first = true;
    while (pos < end) {
        int lo = 0, hi = a.c.n_seqs - 1;            // the last sequence that begins at or before pos
        while (lo < hi) { const int mid = (lo + hi + 1) / 2; if (at[mid] <= pos) lo = mid; else hi = mid - 1; }
        const K8Seq s = k8_seq(lo, a.lens, a.cu, a.c.max_pages, a.n_rows, a.max_q, false);
        int pg0, pg1;
        k8_pages(s, a.window, pg0, pg1);
        const int np = pg1 - pg0, tiles = (s.n * G + 8 * NT - 1) / (8 * NT);
        const int item = (pos - at[lo]) / np, p0 = (pos - at[lo]) % np, p1 = min(np, p0 + end - pos);
        float * part = p0 == 0 && p1 == np ? nullptr : a.part + ((int64_t) blockIdx.x * 2 + (first ? 0 : 1)) * a.part_rows * (D + 4);
        K8State<D, NT> st;
        k8_run<T, E4M3, D, NT>(st, a, maps, s, lo, item / tiles, item % tiles, pg0 + p0, pg0 + p1, threadIdx.x >> 5, NW, ring, phase);
        k8_join_warps<T, D, NT, NW>(st, a, s, item / tiles, item % tiles, part, reinterpret_cast<float *>(base));
        pos += p1 - p0;
        first = false;
    }
}

// Joins the parts of an item: one CTA per (sequence, kv head, row of the tile), its
// warps take the parts in turn (a lane holds D / 32 dims) and are joined in warp
// order, so the order of the sums is fixed.  Rows of items without pages become zeros.
constexpr int K8_JOIN_WARPS = 8;
template <class T, int D, int NT>
__global__ void __launch_bounds__(K8_JOIN_WARPS * 32) k_kv8_join(K8AttendArgs a) {
    __shared__ float s_m[K8_JOIN_WARPS], s_l[K8_JOIN_WARPS], s_o[K8_JOIN_WARPS][D];
    constexpr int V = D / 32;
    const int H = a.c.n_kv_heads, G = a.n_heads / H, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int rr = blockIdx.x % (a.max_q * G), h = blockIdx.x / (a.max_q * G) % H, b = blockIdx.x / (a.max_q * G) / H;
    pdl_trigger();
    pdl_wait();                                     // every CTA, so that the join does not end before the split kernel
    const K8Seq s = k8_seq(b, a.lens, a.cu, a.c.max_pages, a.n_rows, a.max_q, false);
    int pg0, pg1;
    k8_pages(s, a.window, pg0, pg1);
    if (rr >= s.n * G) return;
    const int total = a.line[a.c.n_seqs], chunk = k8_chunk(total, a.ctas);
    const int np = pg1 - pg0, tiles = (s.n * G + 8 * NT - 1) / (8 * NT), tile = rr / (8 * NT), r = rr % (8 * NT);
    const int p0 = a.line[b] + (h * tiles + tile) * np, p1 = p0 + np;
    const int c0 = p0 / chunk, c1 = np ? (p1 - 1) / chunk : c0 - 1;
    if (c0 == c1) return;                           // one CTA had all of it
    float m = -INFINITY, l = 0.0f, o[V];
#pragma unroll
    for (int e = 0; e < V; ++e) o[e] = 0.0f;
#pragma unroll 4
    for (int c = c0 + warp; c <= c1; c += K8_JOIN_WARPS) {
        const float * p = a.part + ((int64_t)(c * 2 + (c == c0 && p0 > c * chunk ? 1 : 0)) * a.part_rows + r) * (D + 4);
        struct alignas(V * 4 > 16 ? 16 : V * 4) Vec { float x[V]; };
        const Vec x = *reinterpret_cast<const Vec *>(p + lane * V);
        const float mc = p[D], lc = p[D + 1], mn = fmaxf(m, mc);
        const float f = m == mn ? 1.0f : k8_exp2(m - mn), fc = mc == mn ? 1.0f : k8_exp2(mc - mn);
        m = mn;
        l = l * f + lc * fc;
#pragma unroll
        for (int e = 0; e < V; ++e) o[e] = o[e] * f + x.x[e] * fc;
    }
    if (lane == 0) { s_m[warp] = m; s_l[warp] = l; }
#pragma unroll
    for (int e = 0; e < V; ++e) s_o[warp][lane * V + e] = o[e];
    __syncthreads();
    if (threadIdx.x >= D) return;
    const int d = threadIdx.x;
    float M = -INFINITY, L = 0.0f, O = 0.0f;
#pragma unroll
    for (int w = 0; w < K8_JOIN_WARPS; ++w) M = fmaxf(M, s_m[w]);
#pragma unroll
    for (int w = 0; w < K8_JOIN_WARPS; ++w) {
        const float f = s_m[w] == M ? 1.0f : k8_exp2(s_m[w] - M);
        L = fmaf(s_l[w], f, L);
        O = fmaf(s_o[w][d], f, O);
    }
    const int row = s.row0 + rr / G, hq = h * G + rr % G;
    k8_write_row<T>(a, row, hq, d, O, L == 0.0f ? 0.0f : 1.0f / L);
    if (d == 0 && a.lse) a.lse[(int64_t) row * a.n_heads + hq] = k8_lse(M, L);
}

// ---- accumulated weights -----------------------------------------------------
// weight_out = weight_in + each key's weights over the rows and the head group.  A warp
// owns W blocks of keys of one (sequence, kv head): their K rows as F16 fragments in
// registers, straight from the page; it goes over the rows eight at a time, recomputes
// the scores as the attention does and adds exp(s - lse) in row order, so the sum's
// order is fixed and nothing is exchanged but four lanes at the end.  Reads K (D bytes
// a key) and 8 bytes of weights; bound by memory for single tokens.
template <int D> constexpr int K8_WEIGH_W = D == 256 ? 1 : 2;
constexpr int K8_WEIGH_WARPS = 4;
template <class T, bool E4M3, int D>
__global__ void __launch_bounds__(K8_WEIGH_WARPS * 32) k_kv8_weigh(K8AttendArgs a) {
    constexpr int W = K8_WEIGH_W<D>, KEYS = W * K8_BLOCK;
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, H = a.c.n_kv_heads, G = a.n_heads / H;
    const int h = blockIdx.y, b = blockIdx.z, j0 = (blockIdx.x * K8_WEIGH_WARPS + (threadIdx.x >> 5)) * KEYS;
    pdl_trigger();
    pdl_wait();
    const K8Seq s = k8_seq(b, a.lens, a.cu, a.c.max_pages, a.n_rows, a.max_q, false);
    if (j0 >= s.len) return;
    const int page = k8_page(a.table + (int64_t) b * a.c.max_pages, j0 / K8_PAGE, a.c.n_pages);
    const float * wi = a.w_in + ((int64_t) b * H + h) * a.w_stride + j0;
    float * wo = a.w_out + ((int64_t) b * H + h) * a.w_stride + j0;
    float w[W][2], old[W][2];
#pragma unroll
    for (int u = 0; u < W; ++u)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int j = u * K8_BLOCK + i * 8 + g;
            w[u][i] = 0.0f;
            old[u][i] = t == 0 && j0 + j < s.len ? wi[j] : 0.0f;
        }
    if (page >= 0 && s.n > 0) {
        uint4 raw[W][2][D / 64];
        float ks[W];
#pragma unroll
        for (int u = 0; u < W; ++u) {
            const int block = j0 % K8_PAGE / K8_BLOCK + u;
            const uint8_t * k = static_cast<const uint8_t *>(a.c.k) + k8_code_off(page, h, block * K8_BLOCK + g, H, D) + t * 16;
#pragma unroll
            for (int c = 0; c < D / 64; ++c) {
                raw[u][0][c] = ld_stream(k + c * 64);
                raw[u][1][c] = ld_stream(k + 8 * D + c * 64);
            }
            ks[u] = a.c.k_scale[k8_scale_off(page, h, block, H)];
        }
        const int R = s.n * G;
        for (int r0 = 0; r0 < R; r0 += 8) {
            int lo[2], hi[2], lo0, hi0, lo1, hi1;
            k8_span(s, r0 / G, a.window, lo0, hi0);
            k8_span(s, min(r0 + 7, R - 1) / G, a.window, lo1, hi1);
            if (hi1 <= j0 || lo0 >= j0 + KEYS) continue;         // no row of these sees a key of ours
            K8Q<T, D> q;
            const int r = r0 + g;
            const bool real = r < R;
            const float back = k8_load_q<T, D>(q, static_cast<const T *>(a.q) + (real ? (s.row0 + r / G) * a.q_row + (h * G + r % G) * a.q_head : 0), lane, real) *
                               (a.scale * 1.44269504088896340736f);
            float fac[2], lse[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                fac[i] = __shfl_sync(0xffffffffu, back, 8 * t + 4 * i);
                const int rr = r0 + 2 * t + i;
                k8_span(s, min(rr, R - 1) / G, a.window, lo[i], hi[i]);
                if (rr >= R) hi[i] = 0;                           // rows of padding see nothing
                lse[i] = rr < R ? a.lse[(int64_t)(s.row0 + rr / G) * a.n_heads + h * G + rr % G] * 1.44269504088896340736f : 0.0f;
            }
#pragma unroll
            for (int u = 0; u < W; ++u) {
                float c4[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int c = 0; c < D / 64; ++c) {
                    const uint32_t xw[4] = {raw[u][0][c].x, raw[u][0][c].y, raw[u][0][c].z, raw[u][0][c].w};
                    const uint32_t yw[4] = {raw[u][1][c].x, raw[u][1][c].y, raw[u][1][c].z, raw[u][1][c].w};
#pragma unroll
                    for (int v = 0; v < 4; ++v) {
                        uint32_t a0, a1, a2, a3;
                        k8_f16x4<E4M3>(xw[v], a0, a2);
                        k8_f16x4<E4M3>(yw[v], a1, a3);
                        k8_mma(c4, a0, a1, a2, a3, q.x[4 * c + v][0], q.x[4 * c + v][1]);
                    }
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int j = j0 + u * K8_BLOCK + (e >> 1) * 8 + g;
                    const float p = k8_exp2(c4[e] * (fac[e & 1] * ks[u]) - lse[e & 1]);
                    w[u][e >> 1] += j >= lo[e & 1] && j < hi[e & 1] ? p : 0.0f;
                }
            }
        }
    } else if (page < 0 && lane == 0) k8_flag(a.c.status, K8_BAD_PAGE);
#pragma unroll
    for (int u = 0; u < W; ++u)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            float x = w[u][i];
            x += __shfl_xor_sync(0xffffffffu, x, 1);
            x += __shfl_xor_sync(0xffffffffu, x, 2);
            const int j = u * K8_BLOCK + i * 8 + g;
            if (t == 0 && j0 + j < s.len) wo[j] = old[u][i] + x;
        }
}

}  // namespace qtts
