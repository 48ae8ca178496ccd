// kv8_tile.cuh — attention of many rows (chunks of prompts) over the 8-bit cache, on
// tcgen05 with accumulators in tensor memory.
//
// A CTA takes 256 rows (two tiles of 128; row r = token r / G, head r % G of the group,
// so that a group's heads share every key) of one (sequence, kv head) over the pages
// that they see, 64 keys at a time:
//   warp 12     copies a page's codes (TMA, swizzled) and scales into a ring;
//   warps 8-11  turn codes into F16 (exact; K a page ahead of V) in the core-matrix order of the MMA's B
//               operands; K is read K-major, V MN-major, so neither is transposed;
//   warp 13     issues S = Q K^T of the next page before O += P V of this one, so that
//               the tensor core works while the softmax does;
//   warps 0-3, 4-7 (a thread a row of its tile) scale and mask the scores, keep the
//               running maximum and sum, and write the weights P as F16.
// As in kv8_attend.cuh, the reference of the maximum moves only when a score passes it by
// more than 4, and V's scales ride on the weights, so O in tensor memory is rarely
// rescaled.  Codes are scaled after the products in F32: the scores per 16 keys, V through
// the weights.
//
// Bound per 64 keys and 256 rows at D = 128: 1,020 cycles of MMA (4,108 F16 FMA a cycle
// and SM at the nominal peak), 1,024 of exponentials (16 a cycle), some 1,000 issue slots a
// scheduler for the scores' arithmetic and the conversion.  Measured: 0.84 ms for 2,048
// tokens of 32 heads over 16,384 keys (613 TFLOP/s, 36% of the measured GEMM rate), some
// 3,000 cycles a page: the hand-offs softmax -> MMA -> softmax are what is left (without
// conversion and exponentials they took 70% of an earlier version's time).  P
// in tensor memory over the scores (its A operand) measured 0.91 ms: the scores two pages
// on then have to wait for the product.
#pragma once
#include "kv8_attend.cuh"
#include "tcgen05.cuh"

namespace qtts {

constexpr int KT_ROWS = 256, KT_THREADS = 448, KT_RAW = 3;
template <int D> struct KtSmem {
    static constexpr int raw_side = K8_PAGE * D, raw = 2 * raw_side;                 // a ring stage: K codes, V codes
    static constexpr int f16_side = K8_PAGE * D * 2, kv = 2 * f16_side;              // a converted stage
    static constexpr int q = 128 * D * 2, p = 128 * K8_PAGE * 2;                     // per row tile
    static constexpr int raw_at = 0, kv_at = raw_at + KT_RAW * raw, q_at = kv_at + 2 * kv, p_at = q_at + 2 * q, scale_at = p_at + 2 * p;
    static constexpr int bar_at = scale_at + (KT_RAW + 4) * 48, bytes = bar_at + 32 * 8 + 16, total = bytes + 1024;
};
// Barriers: raw stages filled / read (3 each); converted K and V stages filled / used (2 each); scales published (4);
// query rows written; scores ready (tile, buffer); weights written, their product done (per tile); all MMAs done.
enum : int { KT_RAW_FULL = 0, KT_RAW_EMPTY = 3, KT_K_FULL = 6, KT_V_FULL = 8, KT_K_EMPTY = 10, KT_V_EMPTY = 12, KT_SC = 14, KT_Q = 18, KT_S = 19, KT_P = 23,
             KT_PV = 25, KT_DONE = 27, KT_BARS = 28 };

__device__ __forceinline__ bool kt_wait(uint64_t * bar, int phase) { return __all_sync(0xffffffffu, mbar_wait(bar, phase & 1)); }
__device__ __forceinline__ void kt_arrive(uint64_t * bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void kt_sts(uint32_t p, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(p), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}

// Two F32 operations in one instruction.
__device__ __forceinline__ float2 kt_fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(reinterpret_cast<uint64_t &>(d))
        : "l"(reinterpret_cast<const uint64_t &>(a)), "l"(reinterpret_cast<const uint64_t &>(b)), "l"(reinterpret_cast<const uint64_t &>(c)));
    return d;
}
__device__ __forceinline__ float2 kt_add2(float2 a, float2 b) {
    float2 d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(reinterpret_cast<uint64_t &>(d)) : "l"(reinterpret_cast<const uint64_t &>(a)), "l"(reinterpret_cast<const uint64_t &>(b)));
    return d;
}

template <class T, bool E4M3, int D>
__global__ void __launch_bounds__(KT_THREADS, 1) k_kv8_attend_tile(K8AttendArgs a, const __grid_constant__ K8Maps maps) {
    using M = KtSmem<D>;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, H = a.c.n_kv_heads, G = a.n_heads / H;
    // the last tiles see the most keys: they begin first
    const int tile = a.tiles - 1 - blockIdx.x / (H * a.c.n_seqs), hb = blockIdx.x % (H * a.c.n_seqs), h = hb % H, b = hb / H;
    pdl_trigger();
    pdl_wait();
    const K8Seq s = k8_seq(b, a.lens, a.cu, a.c.max_pages, a.n_rows, a.max_q, false);
    if (threadIdx.x == 0 && h == 0 && tile == 0) k8_flag(a.c.status, s.status);
    const int R = s.n * G, r0 = tile * KT_ROWS;
    if (r0 >= R) return;
    uint8_t * base = k8_dyn + (-(int) smem_u32(k8_dyn) & 1023);
    const uint32_t sb = smem_u32(base);
    uint64_t * bar = reinterpret_cast<uint64_t *>(base + M::bar_at);
    uint32_t * s_tmem = reinterpret_cast<uint32_t *>(base + M::bar_at + 32 * 8);
    volatile int * s_fail = reinterpret_cast<volatile int *>(s_tmem + 1);
    // scales of a ring stage (0 ..) or published (KT_RAW ..): 4 of K, 4 of V, then whether the page is none
    auto scales = [&](int stage) { return reinterpret_cast<float *>(base + M::scale_at + stage * 48); };

    // pages [t0, t0 + nt[w]) for each tile of 128 rows
    int lo_first, hi_first, t0, nt[2], any_hi;
    k8_span(s, r0 / G, a.window, lo_first, hi_first);
    t0 = lo_first / K8_PAGE;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        int lo, hi;
        k8_span(s, min(r0 + 128 * w + 127, R - 1) / G, a.window, lo, hi);
        nt[w] = r0 + 128 * w < R ? max(0, (hi + K8_PAGE - 1) / K8_PAGE - t0) : 0;
        any_hi = hi;
    }
    const int n = max(nt[0], nt[1]);

    if (threadIdx.x == 0) {
        for (int i = 0; i < KT_BARS; ++i) {
            int count = 1;
            if ((i >= KT_RAW_EMPTY && i < KT_K_EMPTY) || (i >= KT_P && i < KT_PV)) count = 128;
            if (i == KT_Q) count = 256;
            mbar_init(bar + i, count);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        *s_fail = 0;
    }
    if (warp == 13) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(s_tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *s_tmem;

    if (warp == 12) {
        // ---- copies
        if (lane == 0) {
            const int32_t * table = a.table + (int64_t) b * a.c.max_pages + t0;
            int page = n > 0 ? k8_page(table, 0, a.c.n_pages) : -1, issued = 0;
            for (int j = 0; j < n; ++j) {
                const int st = j % KT_RAW, next = j + 1 < n ? k8_page(table, j + 1, a.c.n_pages) : -1;
                if (j >= KT_RAW && !mbar_wait(bar + KT_RAW_EMPTY + st, (j / KT_RAW - 1) & 1)) { *s_fail = 1; break; }
                float * sc = scales(st);
                reinterpret_cast<int *>(sc)[8] = page < 0;
                if (page >= 0) {
                    const uint32_t dst = sb + M::raw_at + st * M::raw;
                    const int y = (page * H + h) * K8_PAGE;
                    mbar_expect_tx(bar + KT_RAW_FULL + st, M::raw + 32);
                    k8_tma(dst, &maps.k, 0, y, bar + KT_RAW_FULL + st);
                    k8_tma(dst + M::raw_side, &maps.v, 0, y, bar + KT_RAW_FULL + st);
                    bulk_g2s(sc, a.c.k_scale + k8_scale_off(page, h, 0, H), 16, bar + KT_RAW_FULL + st);
                    bulk_g2s(sc + 4, a.c.v_scale + k8_scale_off(page, h, 0, H), 16, bar + KT_RAW_FULL + st);
                } else {
                    k8_flag(a.c.status, K8_BAD_PAGE);
                    kt_arrive(bar + KT_RAW_FULL + st);
                }
                issued = j + 1;
                page = next;
            }
            for (int j = max(0, issued - KT_RAW); j < issued; ++j) mbar_wait(bar + KT_RAW_FULL + j % KT_RAW, (j / KT_RAW) & 1);   // none in flight at the end
        }
    } else if (warp == 13) {
        // ---- MMAs
        if (lane == 0 && n > 0) {
            const uint32_t id_s = tc_idesc_f16(K8_PAGE, false), id_o = tc_idesc_f16(D, true);
            bool ok = mbar_wait(bar + KT_Q, 0);
            // descriptors: low words stepped in units of 16 bytes
            const uint64_t dq = tc_desc(sb + M::q_at, 128, 1024), dk = tc_desc(sb + M::kv_at, 128, 1024), dp = tc_desc(sb + M::p_at, 128, 1024),
                           dv = tc_desc(sb + M::kv_at + M::f16_side, D * 16, 128);
            const uint32_t k_hi = (uint32_t)(dk >> 32), v_hi = (uint32_t)(dv >> 32);   // (those of q and p are k's)
            auto scores = [&](int w, int j) {
                ok = ok && mbar_wait(bar + KT_K_FULL + (j & 1), (j >> 1) & 1);
                if (!ok) return;
                tc_fence_after();
                const uint32_t q = (uint32_t) dq + w * (M::q >> 4), k = (uint32_t) dk + (j & 1) * (M::kv >> 4), d = tmem + 2 * D + (w * 2 + (j & 1)) * K8_PAGE;
#pragma unroll
                for (int i = 0; i < D / 16; ++i)
                    tc_mma_lo(d, q + (i >> 2) * 1024 + (i & 3) * 16, k_hi, k + (i >> 2) * 512 + (i & 3) * 16, k_hi, id_s, i > 0);
                tc_commit(bar + KT_S + w * 2 + (j & 1));
            };
            auto both = [&](int j) {
                for (int w = 0; w < 2; ++w)
                    if (j < nt[w]) scores(w, j);
                tc_commit(bar + KT_K_EMPTY + (j & 1));
            };
            both(0);
            for (int j = 0; j < n && ok; ++j) {
                if (j + 1 < n) both(j + 1);
                for (int w = 0; w < 2 && ok; ++w) {
                    if (j >= nt[w]) continue;
                    ok = mbar_wait(bar + KT_P + w, j & 1) && mbar_wait(bar + KT_V_FULL + (j & 1), (j >> 1) & 1);
                    if (!ok) break;
                    tc_fence_after();
                    const uint32_t p = (uint32_t) dp + w * (M::p >> 4), v = (uint32_t) dv + (j & 1) * (M::kv >> 4);
#pragma unroll
                    for (int i = 0; i < K8_PAGE / 16; ++i) tc_mma_lo(tmem + w * D, p + i * 16, k_hi, v + i * 2 * D, v_hi, id_o, j > 0 || i > 0);
                    tc_commit(bar + KT_PV + w);
                }
                tc_commit(bar + KT_V_EMPTY + (j & 1));
            }
            if (!ok) *s_fail = 1;
            tc_commit(bar + KT_DONE);
            if (!mbar_wait(bar + KT_DONE, 0)) *s_fail = 1;      // no MMA in flight at the end
        }
    } else if (warp >= 8) {
        // ---- codes to F16: a lane takes 16 dims of a key; eight lanes the eight keys of a core matrix row group
        // K of the next page before V of this one: K's stage is free when the scores are done, V's a whole softmax later
        const int key_lo = lane & 7, c_lo = lane >> 3;
        auto convert = [&](int side, int j) {
            const int st = j % KT_RAW;
            const bool none = reinterpret_cast<const int *>(scales(st))[8] != 0;
            const int beyond = none ? 0 : any_hi - (t0 + j) * K8_PAGE;      // keys from here on may hold anything
            const uint32_t raw = sb + M::raw_at + st * M::raw + side * M::raw_side, out = sb + M::kv_at + (j & 1) * M::kv + side * M::f16_side;
            constexpr int UNITS = 8 * (D / 64);                             // (key group, chunk group) pairs of a side
            uint4 x[UNITS / 4];
#pragma unroll
            for (int u0 = 0; u0 < UNITS / 4; ++u0) {
                // unit u0 * 4 + (warp - 8): key group u % 8, chunk group u / 8
                const int key = ((u0 & 1) * 4 + (warp - 8)) * 8 + key_lo, chunk = (u0 >> 1) * 4 + c_lo, sw = D == 64 ? chunk ^ (key_lo >> 1) : chunk ^ key_lo;
                x[u0] = k8_lds16(raw + key * D + sw * 16);
            }
            if (beyond < K8_PAGE)
#pragma unroll
                for (int u0 = 0; u0 < UNITS / 4; ++u0)
                    if (((u0 & 1) * 4 + (warp - 8)) * 8 + key_lo >= beyond) x[u0] = make_uint4(0, 0, 0, 0);
#pragma unroll
            for (int u0 = 0; u0 < UNITS / 4; ++u0) {
                const int kg = (u0 & 1) * 4 + (warp - 8), c4 = u0 >> 1;
                uint32_t f[8];
                k8_f16x4<E4M3>(x[u0].x, f[0], f[1]);
                k8_f16x4<E4M3>(x[u0].y, f[2], f[3]);
                k8_f16x4<E4M3>(x[u0].z, f[4], f[5]);
                k8_f16x4<E4M3>(x[u0].w, f[6], f[7]);
                // K: [k tile of 64 dims][key group][8 dims][key], V: [key group][8 dims][key], 16 bytes each
                const uint32_t p = out + key_lo * 16 + (side == 0 ? c4 * 8192 + kg * 1024 + c_lo * 256 : kg * (D * 16) + (c4 * 4 + c_lo) * 256);
                kt_sts(p, f[0], f[1], f[2], f[3]);
                kt_sts(p + 128, f[4], f[5], f[6], f[7]);
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            kt_arrive(bar + (side == 0 ? KT_K_FULL : KT_V_FULL) + (j & 1));
        };
        bool ok = true;
        for (int i = 0; i <= n && n > 0 && ok; ++i) {
            if (i < n) {                                                    // K of page i
                ok = kt_wait(bar + KT_RAW_FULL + i % KT_RAW, i / KT_RAW) && (i < 2 || kt_wait(bar + KT_K_EMPTY + (i & 1), i / 2 - 1));
                if (!ok) break;
                if (warp == 8) {
                    if (lane < 9) scales(KT_RAW + (i & 3))[lane] = scales(i % KT_RAW)[lane];
                    __syncwarp();
                    if (lane == 0) kt_arrive(bar + KT_SC + (i & 3));
                }
                convert(0, i);
            }
            if (i > 0) {                                                    // V of the page before
                const int j = i - 1;
                ok = j < 2 || kt_wait(bar + KT_V_EMPTY + (j & 1), j / 2 - 1);
                if (!ok) break;
                convert(1, j);
                kt_arrive(bar + KT_RAW_EMPTY + j % KT_RAW);
            }
        }
        if (!ok && lane == 0) *s_fail = 1;
    } else {
        // ---- softmax: a thread a row
        const int w = warp >> 2, r = (warp & 3) * 32 + lane, rr = r0 + w * 128 + r;
        const bool real = rr < R;
        const int row = s.row0 + min(rr, R - 1) / G, hq = h * G + min(rr, R - 1) % G;
        float fac = a.scale * 1.44269504088896340736f;                      // log2 e
        {
            const uint16_t * src = static_cast<const uint16_t *>(a.q) + row * a.q_row + hq * a.q_head;
            const bool vec = (reinterpret_cast<uintptr_t>(src) & 15) == 0;
            uint4 x[D / 8];
            uint32_t most = 0;
#pragma unroll
            for (int c = 0; c < D / 8; ++c) {
                x[c] = make_uint4(0, 0, 0, 0);
                if (real) x[c] = vec ? k8_ld8<true>(src + c * 8) : k8_ld8<false>(src + c * 8);
                most = __vmaxu2(most, __vmaxu2(__vmaxu2(x[c].x & 0x7fff7fffu, x[c].y & 0x7fff7fffu), __vmaxu2(x[c].z & 0x7fff7fffu, x[c].w & 0x7fff7fffu)));
            }
            most = max(most & 0xffffu, most >> 16);
            float down = 1.0f;
            if constexpr (Row16<T>::inf == 0x7f80u) {                       // BF16: a power of two brings the row into F16 (kv8_attend.cuh)
                int e = (int)(most >> 7) - 127;
                e = most == 0 || most >= Row16<T>::inf ? 0 : max(-120, min(120, e));
                down = __int_as_float((127 - e) << 23);
                fac *= __int_as_float((127 + e) << 23);
            }
            const uint32_t q = sb + M::q_at + w * M::q + (r >> 3) * 1024 + (r & 7) * 16;
#pragma unroll
            for (int c = 0; c < D / 8; ++c) {
                uint32_t y[4] = {x[c].x, x[c].y, x[c].z, x[c].w};
                if constexpr (Row16<T>::inf == 0x7f80u)
#pragma unroll
                    for (int i = 0; i < 4; ++i) y[i] = k8_pack(__uint_as_float(y[i] << 16) * down, __uint_as_float(y[i] & 0xffff0000u) * down);
                kt_sts(q + (c >> 3) * 16384 + (c & 7) * 128, y[0], y[1], y[2], y[3]);
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            kt_arrive(bar + KT_Q);
        }
        int lo, hi, all_lo, all_hi, x0;
        k8_span(s, min(rr, R - 1) / G, a.window, lo, hi);
        k8_span(s, min(r0 + w * 128, R - 1) / G, a.window, x0, all_hi);
        k8_span(s, min(r0 + w * 128 + 127, R - 1) / G, a.window, all_lo, x0);
        float m = -INFINITY, l = 0.0f, unit = K8_UNIT_MIN;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16, tm_s = tmem + lanes + 2 * D + w * 2 * K8_PAGE, tm_o = tmem + lanes + w * D;
        const uint32_t pw = sb + M::p_at + w * M::p + (r >> 3) * 1024 + (r & 7) * 16;
        const int mine = w == 0 ? nt[0] : nt[1];
        bool ok = true;
        for (int j = 0; j < mine && ok; ++j) {
            ok = kt_wait(bar + KT_SC + (j & 3), j >> 2) && kt_wait(bar + KT_S + w * 2 + (j & 1), j >> 1);
            if (!ok) break;
            tc_fence_after();
            float sv[K8_PAGE];
            tc_ld_wait<K8_PAGE>(tm_s + (j & 1) * K8_PAGE, sv);
            const float * sc = scales(KT_RAW + (j & 3));
            const int kb = (t0 + j) * K8_PAGE;
            const bool none = reinterpret_cast<const int *>(sc)[8] != 0;
            const bool whole = !none && kb >= all_lo && kb + K8_PAGE <= all_hi;
            float ks[4], vs[4], mx = -INFINITY;
            bool plain = whole;                                             // every row sees every key, and no scale of V is NaN
#pragma unroll
            for (int u = 0; u < 4; ++u) { ks[u] = sc[u] * fac; vs[u] = sc[4 + u]; plain = plain && vs[u] == vs[u]; }
            if (!whole) {
#pragma unroll
                for (int i = 0; i < K8_PAGE; ++i)
                    if (none || kb + i < lo || kb + i >= hi) sv[i] = -INFINITY;
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) {                                   // scales are not negative: the largest score of 16 keys is the largest product's
                float x = sv[16 * u];
#pragma unroll
                for (int i = 1; i < 16; ++i) x = fmaxf(x, sv[16 * u + i]);
                mx = fmaxf(mx, x == -INFINITY ? x : x * ks[u]);
            }
            const float top = none ? 0.0f : fmaxf(fmaxf(vs[0], vs[1]), fmaxf(vs[2], vs[3]));
            const bool up = __any_sync(0xffffffffu, mx > m + K8_SLACK || top > unit * K8_UNIT_SLACK);
            if (j > 0 && !(ok = kt_wait(bar + KT_PV + w, j - 1))) break;    // O and P are ours again
            if (up) {
                const float m2 = fmaxf(m, mx);
                float f = m2 == m ? 1.0f : k8_exp2(m - m2);
                l *= f;
                m = m2;
                if (top > unit * K8_UNIT_SLACK) { f *= unit / top; unit = top; }
                if (j > 0) {
                    tc_fence_after();
#pragma unroll
                    for (int c = 0; c < D; c += 32) {
                        float o[32];
                        tc_ld_wait<32>(tm_o + c, o);
#pragma unroll
                        for (int i = 0; i < 32; ++i) o[i] *= f;
                        tc_st16(tm_o + c, o);
                        tc_st16(tm_o + c + 16, o + 16);
                    }
                    tc_wait_st();
                }
            }
            const float inv = __fdividef(1.0f, unit), ref = m - K8_LIFT;
            if (plain) {
                // 2^(s - ref) times a block's V scale over `unit` as one exponential; the sum takes the factor back.  A
                // block of zeros (scale 0) keeps the factor 1, and below 2^-60 nothing is left of it in F16 either way.
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const float rv = vs[u] == 0.0f ? 1.0f : fmaxf(vs[u] * inv, 8.6736173798840355e-19f);
                    const float off = __log2f(rv) - ref;
                    const float2 k2 = make_float2(ks[u], ks[u]), o2 = make_float2(off, off);
                    float2 sum = make_float2(0.0f, 0.0f);
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        uint32_t pk[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            float2 x = kt_fma2(make_float2(sv[16 * u + 8 * c + 2 * i], sv[16 * u + 8 * c + 2 * i + 1]), k2, o2);
                            x.x = k8_exp2(x.x);
                            x.y = k8_exp2(x.y);
                            sum = kt_add2(sum, x);
                            pk[i] = k8_pack(x.x, x.y);
                        }
                        kt_sts(pw + (2 * u + c) * 128, pk[0], pk[1], pk[2], pk[3]);
                    }
                    l += __fdividef(sum.x + sum.y, rv);
                }
            } else {
#pragma unroll
                for (int c = 0; c < K8_PAGE / 8; ++c) {
                    const float rv = vs[c >> 1] * inv;
                    float e[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const float x = k8_exp2(fmaf(sv[c * 8 + i], ks[c >> 1], -ref));
                        const bool hidden = sv[c * 8 + i] == -INFINITY;
                        e[i] = hidden ? 0.0f : x * rv;
                        l += hidden ? 0.0f : x;
                    }
                    kt_sts(pw + c * 128, k8_pack(e[0], e[1]), k8_pack(e[2], e[3]), k8_pack(e[4], e[5]), k8_pack(e[6], e[7]));
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            tc_fence_before();
            kt_arrive(bar + KT_P + w);
        }
        if (ok && mine > 0) ok = kt_wait(bar + KT_PV + w, mine - 1);
        if (!ok && lane == 0) *s_fail = 1;
        if (ok) {
            tc_fence_after();
            const float f = l == 0.0f ? 0.0f : unit / l;
            T * out = static_cast<T *>(a.out) + row * a.o_row + hq * a.o_head;
            const bool vec = (reinterpret_cast<uintptr_t>(out) & 15) == 0;
#pragma unroll
            for (int c = 0; c < D; c += 16) {
                float o[16];
                if (mine > 0) tc_ld_wait<16>(tm_o + c, o);                  // the same for the whole warp
#pragma unroll
                for (int i = 0; i < 16; ++i) o[i] = mine > 0 && l != 0.0f ? o[i] * f : 0.0f;
                if (real) {
                    if (vec) { k8_store8(out + c, o); k8_store8(out + c + 8, o + 8); }
                    else
#pragma unroll
                        for (int i = 0; i < 16; ++i) out[c + i] = T(o[i]);
                }
            }
            if (real && a.lse) a.lse[(int64_t) row * a.n_heads + hq] = k8_lse(m, l);
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 13) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
    if (threadIdx.x == 0 && *s_fail) k8_flag(a.c.status, K8_STUCK);
}

}  // namespace qtts
