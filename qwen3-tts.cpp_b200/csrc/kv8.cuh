// kv8.cuh — the 8-bit paged key/value cache: layout, bounds and the kernels
// that write it (append, evict) and read it back.
//
// A page holds 64 tokens: for every kv head 64 rows of 8-bit codes for K and for
// V, and one F32 scale per block of 16 tokens (value = code * scale).  A block
// is quantised from 16-bit rows,
//     scale = amax / top,   code = rn(x / scale),   top = 127 (int8) or 448 (e4m3),
// with IEEE F32 division, so it is the same bits however its rows arrived.
// For that the rows of a sequence's last two blocks are also kept in 16 bits,
// in a ring of 32 rows per (sequence, kv head): a block that is still filling up
// is requantised from its 16-bit rows at every append, never from codes, and up
// to 16 rows may be taken back (a smaller length) without loss.  A block that
// holds a value that is not finite reads back as NaN (its scale is NaN).
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp8.h>

#include "common.cuh"
#include "qwen3tts_b200.h"

namespace qtts {

constexpr int K8_PAGE = 64, K8_BLOCK = 16, K8_RING = 32;
constexpr int K8_BPP = K8_PAGE / K8_BLOCK;      // blocks per page
enum : int { K8_BAD_PAGE = 1, K8_BAD_LEN = 2, K8_BAD_ROWS = 4, K8_SHARED_PAGE = 8, K8_STUCK = 16 };   // status bits

// A sequence's share of a call, checked against the cache: rows [row0, row0 + n)
// of the packed tensors, its length after them.  Numbers that do not fit set a
// status bit and leave nothing to do for the sequence.
struct K8Seq { int len, row0, n, status; };
__host__ __device__ inline K8Seq k8_seq(int b, const int32_t * lens, const int32_t * cu, int max_pages, int n_rows, int max_n,
                                        bool rows_within) {
    const int64_t len = lens ? lens[b] : 0, row0 = cu ? cu[b] : b, n = cu ? (int64_t) cu[b + 1] - cu[b] : 1;
    K8Seq s{(int) len, (int) row0, 0, 0};
    if (len < 0 || len > (int64_t) max_pages * K8_PAGE) s.status |= K8_BAD_LEN;
    if (n < 0 || n > max_n || row0 < 0 || row0 + n > n_rows || (rows_within && !s.status && n > len)) s.status |= K8_BAD_ROWS;
    s.n = (int) n;
    if (s.status) { s.len = 0; s.n = 0; s.row0 = 0; }
    return s;
}
// The pool index of page p of a sequence, -1 if the table's entry is no page of the pool.
__host__ __device__ inline int k8_page(const int32_t * table_row, int p, int n_pages) {
    const int id = table_row[p];
    return id >= 0 && id < n_pages ? id : -1;
}
// Offsets in the pool, in 64 bits: a long cache passes 2^31 codes.
__host__ __device__ inline int64_t k8_code_off(int64_t page, int head, int row, int heads, int dim) {
    return ((page * heads + head) * K8_PAGE + row) * dim;
}
__host__ __device__ inline int64_t k8_scale_off(int64_t page, int head, int block, int heads) {
    return (page * heads + head) * K8_BPP + block;
}

__device__ __forceinline__ void k8_flag(int32_t * status, int bits) {
    if (status && bits) atomicOr(status, bits);
}

// ---- types -----------------------------------------------------------------
template <class T> struct Row16;
template <> struct Row16<__half> { static constexpr uint32_t inf = 0x7c00u; };
template <> struct Row16<__nv_bfloat16> { static constexpr uint32_t inf = 0x7f80u; };
template <class T> __device__ __forceinline__ float k8_bits_f(uint32_t b) {
    return (float) __ushort_as_half((unsigned short) b);
}
template <> __device__ __forceinline__ float k8_bits_f<__nv_bfloat16>(uint32_t b) { return __uint_as_float(b << 16); }

template <bool E4M3> struct Code8;
template <> struct Code8<false> {
    static constexpr float top = 127.0f;
    static __device__ __forceinline__ uint32_t code(float r) {      // r within +-top
        return (uint32_t)(__float2int_rn(r) & 0xff);
    }
    static __device__ __forceinline__ float value(uint32_t c) { return (float)(int8_t) c; }
};
template <> struct Code8<true> {
    static constexpr float top = 448.0f;
    static __device__ __forceinline__ uint32_t code(float r) { return __nv_cvt_float_to_fp8(r, __NV_SATFINITE, __NV_E4M3); }
    static __device__ __forceinline__ float value(uint32_t c) {
        __half_raw h = __nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t) c, __NV_E4M3);
        return __half2float(__half(h));
    }
};
__device__ __forceinline__ float k8_clamp(float r, float top) { return fminf(fmaxf(r, -top), top); }

// 8 elements of 16 bits at p; VEC: p is 16-byte aligned.
template <bool VEC>
__device__ __forceinline__ uint4 k8_ld8(const uint16_t * p) {
    if constexpr (VEC) return *reinterpret_cast<const uint4 *>(p);
    else {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = p[2 * i] | (uint32_t) p[2 * i + 1] << 16;
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
}

struct K8Args {
    qtts_kv8 c;
    const int32_t * table, * lens, * cu;
    const uint16_t * src[2];          // new K, V rows
    int64_t s_row[2], s_head[2];      // their strides in elements
    int n_rows, max_n, blocks;        // blocks: 16-row blocks per sequence in the grid
};

// ---- append ----------------------------------------------------------------
// One warp per (sequence, touched block, kv head, K or V): 16 rows x D values in
// registers (a lane holds 8 consecutive dims of D / 16 rows), the block's largest
// magnitude as an integer maximum over the sign-less 16-bit patterns (which also
// finds infinities and NaN), then the codes.  Bound by memory: 2 D bytes read and
// D written per row, kv head and side.
constexpr int K8_WARPS = 4;
template <class T, bool E4M3, int D, bool VEC>
__global__ void __launch_bounds__(K8_WARPS * 32) k_kv8_append(K8Args a) {
    constexpr int LPR = D / 8, RPS = 32 / LPR, STEPS = K8_BLOCK / RPS;   // lanes per row, rows per step
    const int lane = threadIdx.x & 31;
    const int H = a.c.n_kv_heads;
    const int64_t unit = (int64_t) blockIdx.x * K8_WARPS + (threadIdx.x >> 5);
    const int kv = (int)(unit & 1), h = (int)((unit >> 1) % H);
    const int nb = (int)((unit >> 1) / H % a.blocks);
    const int64_t b64 = (unit >> 1) / H / a.blocks;
    if (b64 >= a.c.n_seqs) return;
    const int b = (int) b64;
    const K8Seq s = k8_seq(b, a.lens, a.cu, a.c.max_pages, a.n_rows, a.max_n, true);
    if (s.status && lane == 0 && nb == 0) k8_flag(a.c.status, s.status);
    if (s.n == 0) return;
    const int start = s.len - s.n, first = start / K8_BLOCK, last = (s.len - 1) / K8_BLOCK, X = first + nb;
    if (X > last) return;
    const int page = k8_page(a.table + (int64_t) b * a.c.max_pages, X / K8_BPP, a.c.n_pages);
    const uint16_t * src = a.src[kv] + (int64_t) h * a.s_head[kv];
    uint16_t * ring = static_cast<uint16_t *>(kv ? a.c.v_open : a.c.k_open) + ((int64_t) b * H + h) * K8_RING * D;
    const int r0 = lane / LPR, d0 = lane % LPR * 8;
    uint4 x[STEPS];
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
        const int pos = X * K8_BLOCK + i * RPS + r0;
        x[i] = make_uint4(0, 0, 0, 0);
        if (pos < start) x[i] = *reinterpret_cast<const uint4 *>(ring + (pos % K8_RING) * D + d0);
        else if (pos < s.len) x[i] = k8_ld8<VEC>(src + (int64_t)(s.row0 + pos - start) * a.s_row[kv] + d0);
        const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) most = __vmaxu2(most, w[j] & 0x7fff7fffu);
    }
    most = max(most & 0xffffu, most >> 16);
    most = __reduce_max_sync(0xffffffffu, most);
    const bool fine = most < Row16<T>::inf;
    const float top = Code8<E4M3>::top;
    const float scale = fine ? __fdiv_rn(k8_bits_f<T>(most), top) : __int_as_float(0x7fffffff);
    if (page >= 0) {
        uint8_t * dst = static_cast<uint8_t *>(kv ? a.c.v : a.c.k) + k8_code_off(page, h, X % K8_BPP * K8_BLOCK, H, D);
#pragma unroll
        for (int i = 0; i < STEPS; ++i) {
            const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
            uint32_t o[2] = {0, 0};
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float f = k8_bits_f<T>((w[j >> 1] >> (j & 1) * 16) & 0xffffu);
                const uint32_t c = fine && most ? Code8<E4M3>::code(k8_clamp(__fdiv_rn(f, scale), top)) : 0u;
                o[j >> 2] |= c << (j & 3) * 8;
            }
            *reinterpret_cast<uint2 *>(dst + (i * RPS + r0) * D + d0) = make_uint2(o[0], o[1]);
        }
        if (lane == 0) (kv ? a.c.v_scale : a.c.k_scale)[k8_scale_off(page, h, X % K8_BPP, H)] = scale;
    } else if (lane == 0) k8_flag(a.c.status, K8_BAD_PAGE);
    // The ring: the new rows of the last two blocks.  Block Y's half may still hold
    // rows that the first block's warp has to read (the same half, start inside a
    // block): then that warp writes Y's rows, after its reads.
    __syncwarp();
#pragma unroll
    for (int back = 0; back < 2; ++back) {
        const int Y = last - back;
        if (Y < first) break;
        const bool by_first = Y != first && (Y & 1) == (first & 1) && start % K8_BLOCK != 0;
        if ((by_first ? first : Y) != X) continue;
#pragma unroll
        for (int i = 0; i < STEPS; ++i) {
            const int pos = Y * K8_BLOCK + i * RPS + r0;
            if (pos < start || pos >= s.len) continue;
            const uint4 w = Y == X ? x[i] : k8_ld8<VEC>(src + (int64_t)(s.row0 + pos - start) * a.s_row[kv] + d0);
            *reinterpret_cast<uint4 *>(ring + (pos % K8_RING) * D + d0) = w;
        }
    }
}

// ---- read ------------------------------------------------------------------
// Rows begin .. of each sequence as 16- or 32-bit values, packed.  One thread per
// 8 dims of a (row, kv head), both sides.  Rows of pages that are none read as zero.
struct K8ReadArgs {
    qtts_kv8 c;
    const int32_t * table, * begin, * cu;
    int n_rows, max_n, out_type;      // out_type: 0 F32, 1 F16, 30 BF16
    void * k, * v;                    // [n_rows][H][D]
};
template <class T> __device__ __forceinline__ void k8_store8(T * p, const float * f) {
    struct alignas(16) Vec { T x[8]; } y;
#pragma unroll
    for (int j = 0; j < 8; ++j) y.x[j] = T(f[j]);
    *reinterpret_cast<Vec *>(p) = y;
}
template <> __device__ __forceinline__ void k8_store8<float>(float * p, const float * f) {
    *reinterpret_cast<float4 *>(p) = make_float4(f[0], f[1], f[2], f[3]);
    *reinterpret_cast<float4 *>(p + 4) = make_float4(f[4], f[5], f[6], f[7]);
}
template <class T, bool E4M3>
__global__ void __launch_bounds__(256) k_kv8_read(K8ReadArgs a) {
    const int H = a.c.n_kv_heads, D = a.c.head_dim, cpr = H * D / 8, b = blockIdx.y;
    const K8Seq s = k8_seq(b, nullptr, a.cu, a.c.max_pages, a.n_rows, a.max_n, false);
    const int begin = a.begin ? a.begin[b] : 0;
    int bad = s.status;
    if (begin < 0 || (int64_t) begin + s.n > (int64_t) a.c.max_pages * K8_PAGE) bad |= K8_BAD_LEN;
    if (bad) {
        if (blockIdx.x == 0 && threadIdx.x == 0) k8_flag(a.c.status, bad);
        return;
    }
    for (int64_t t = (int64_t) blockIdx.x * 256 + threadIdx.x; t < (int64_t) s.n * cpr; t += (int64_t) gridDim.x * 256) {
        const int i = (int)(t / cpr), c8 = (int)(t % cpr), h = c8 / (D / 8), d0 = c8 % (D / 8) * 8, pos = begin + i;
        const int page = k8_page(a.table + (int64_t) b * a.c.max_pages, pos / K8_PAGE, a.c.n_pages);
        if (page < 0) k8_flag(a.c.status, K8_BAD_PAGE);
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
            float f[8] = {0, 0, 0, 0, 0, 0, 0, 0};
            if (page >= 0) {
                const uint2 w = *reinterpret_cast<const uint2 *>(static_cast<const uint8_t *>(kv ? a.c.v : a.c.k) +
                                                                 k8_code_off(page, h, pos % K8_PAGE, H, D) + d0);
                const float sc = (kv ? a.c.v_scale : a.c.k_scale)[k8_scale_off(page, h, pos % K8_PAGE / K8_BLOCK, H)];
#pragma unroll
                for (int j = 0; j < 8; ++j) f[j] = __fmul_rn(Code8<E4M3>::value(((j < 4 ? w.x : w.y) >> (j & 3) * 8) & 0xffu), sc);
            }
            k8_store8(static_cast<T *>(kv ? a.v : a.k) + ((int64_t)(s.row0 + i) * H + h) * D + d0, f);
        }
    }
}

// ---- eviction --------------------------------------------------------------
// Sequences longer than `budget` keep, per kv head, their first `sinks` and last
// `recent` positions and the heaviest of the others by accumulated weight (ties
// to the lower position; NaN counts as the heaviest), in their order.  Shorter
// sequences keep everything.  The kept rows move to the pages of dst_table.
struct K8EvictArgs {
    qtts_kv8 c;
    const int32_t * table, * lens, * dst_table;   // dst_table [n_seqs][dst_pages]
    int dst_pages;
    const float * weight;             // [n_seqs][H][w_stride]
    int64_t w_stride;
    int budget, sinks, recent;        // budget % 16 == 0
    int32_t * lens_out, * keep;       // [n_seqs], [n_seqs][H][budget] (-1 past the end)
    float * weight_out;               // [n_seqs][H][budget] (0 past the end)
};

__device__ __forceinline__ uint32_t k8_weight_key(float w) {
    if (w != w) return 0xffffffffu;
    return f2key(w == 0.0f ? 0.0f : w);   // -0 and +0 are equal
}

// Exclusive sum of v over the block (1024 threads), total in *total.
__device__ __forceinline__ int k8_scan(int v, int * s_warp, int * total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const int y = __shfl_up_sync(0xffffffffu, x, o); if (lane >= o) x += y; }
    __syncthreads();
    if (lane == 31) s_warp[warp] = x;
    __syncthreads();
    int w = s_warp[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const int y = __shfl_up_sync(0xffffffffu, w, o); if (lane >= o) w += y; }
    *total = __shfl_sync(0xffffffffu, w, 31);
    const int before = __shfl_sync(0xffffffffu, w, warp > 0 ? warp - 1 : 0);
    return x - v + (warp > 0 ? before : 0);
}

// One CTA per (sequence, kv head): radix selection of the k-th largest weight
// (four passes of 8 bits over a shared-memory histogram), then the positions in
// order by block scans: all above it, and the first of those equal to it.
__global__ void __launch_bounds__(1024) k_kv8_select(K8EvictArgs a) {
    __shared__ int hist[256], s_warp[32], s_sel[2];
    const int H = a.c.n_kv_heads, b = blockIdx.x / H, h = blockIdx.x % H, tid = threadIdx.x;
    int n = a.lens[b];
    if (n < 0 || (int64_t) n > (int64_t) a.c.max_pages * K8_PAGE) {
        if (tid == 0 && h == 0) k8_flag(a.c.status, K8_BAD_LEN);
        n = 0;
    }
    const int kept = min(n, a.budget);
    if (h == 0 && tid == 0) a.lens_out[b] = kept;
    // the new pages have to be others than the old ones
    if (h == 0) {
        const int np = (n + K8_PAGE - 1) / K8_PAGE, nd = (kept + K8_PAGE - 1) / K8_PAGE;
        for (int64_t t = tid; t < (int64_t) np * nd; t += 1024)
            if (a.table[(int64_t) b * a.c.max_pages + t / nd] == a.dst_table[(int64_t) b * a.dst_pages + t % nd])
                k8_flag(a.c.status, K8_SHARED_PAGE);
    }
    const float * w = a.weight + ((int64_t) b * H + h) * a.w_stride;
    int32_t * keep = a.keep + ((int64_t) b * H + h) * a.budget;
    float * wo = a.weight_out + ((int64_t) b * H + h) * a.budget;
    for (int i = kept + tid; i < a.budget; i += 1024) { keep[i] = -1; wo[i] = 0.0f; }
    if (n <= a.budget) {
        for (int i = tid; i < n; i += 1024) { keep[i] = i; wo[i] = w[i]; }
        return;
    }
    const int lo = a.sinks, hi = n - a.recent;
    int want = a.budget - a.sinks - a.recent;     // of positions lo .. hi - 1
    uint32_t prefix = 0, mask = 0;
    if (want > 0) {
        for (int shift = 24; shift >= 0; shift -= 8) {
            for (int i = tid; i < 256; i += 1024) hist[i] = 0;
            __syncthreads();
            for (int i = lo + tid; i < hi; i += 1024) {
                const uint32_t k = k8_weight_key(w[i]);
                if ((k & mask) == prefix) atomicAdd(&hist[(k >> shift) & 255], 1);
            }
            __syncthreads();
            if (tid == 0) {
                int left = want, d = 255;
                while (d > 0 && hist[d] < left) { left -= hist[d]; --d; }
                s_sel[0] = d; s_sel[1] = left;
            }
            __syncthreads();
            prefix |= (uint32_t) s_sel[0] << shift;
            mask |= 255u << shift;
            want = s_sel[1];
            __syncthreads();
        }
    }
    // want: how many of those equal to `prefix` stay
    const int total_want = a.budget - a.sinks - a.recent;
    int out = 0, equal_seen = 0;
    for (int base = 0; base < n; base += 1024) {
        const int i = base + tid;
        const float wi = i < n ? w[i] : 0.0f;
        const uint32_t k = k8_weight_key(wi);
        const bool mid = i >= lo && i < hi && total_want > 0, eq = mid && k == prefix;
        int n_eq, n_out;
        const int e = k8_scan(eq ? 1 : 0, s_warp, &n_eq);
        const bool take = i < n && (i < lo || i >= hi || (mid && k > prefix) || (eq && equal_seen + e < want));
        const int o = k8_scan(take ? 1 : 0, s_warp, &n_out);
        if (take) { keep[out + o] = i; wo[out + o] = wi; }
        out += n_out;
        equal_seen += n_eq;
    }
}

// One warp per (sequence, new block, kv head, K or V): gathers the block's 16 rows
// and requantises them from their codes,
//     scale' = max_r scale_r * (max |code_r| / top),  code' = rn(code_r * (scale_r / scale')),
// so rows whose scale is the block's new one keep their codes, and a block that
// moves whole keeps its values.  Rows past the new length are zero codes.
template <bool E4M3, int D>
__global__ void __launch_bounds__(K8_WARPS * 32) k_kv8_move(K8EvictArgs a) {
    constexpr int LPR = D / 8, RPS = 32 / LPR, STEPS = K8_BLOCK / RPS;
    const int lane = threadIdx.x & 31, H = a.c.n_kv_heads, nblk = a.budget / K8_BLOCK;
    const int64_t unit = (int64_t) blockIdx.x * K8_WARPS + (threadIdx.x >> 5);
    const int kv = (int)(unit & 1), h = (int)((unit >> 1) % H), X = (int)((unit >> 1) / H % nblk);
    const int64_t b = (unit >> 1) / H / nblk;
    if (b >= a.c.n_seqs) return;
    const int kept = a.lens_out[b];
    if (X * K8_BLOCK >= kept) return;
    const int dst_page = k8_page(a.dst_table + b * a.dst_pages, X / K8_BPP, a.c.n_pages);
    const int32_t * keep = a.keep + (b * H + h) * a.budget + X * K8_BLOCK;
    const uint8_t * codes = static_cast<const uint8_t *>(kv ? a.c.v : a.c.k);
    const float * scales = kv ? a.c.v_scale : a.c.k_scale;
    const int r0 = lane / LPR, d0 = lane % LPR * 8;
    const float top = Code8<E4M3>::top;
    uint2 x[STEPS];
    float sc[STEPS];
    float best = 0.0f;
    bool nan = false, bad = dst_page < 0;
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
        const int r = i * RPS + r0, pos = keep[r];
        x[i] = make_uint2(0, 0);
        sc[i] = 0.0f;
        if (pos >= 0) {
            const int page = k8_page(a.table + b * a.c.max_pages, pos / K8_PAGE, a.c.n_pages);
            if (page >= 0) {
                x[i] = *reinterpret_cast<const uint2 *>(codes + k8_code_off(page, h, pos % K8_PAGE, H, D) + d0);
                sc[i] = scales[k8_scale_off(page, h, pos % K8_PAGE / K8_BLOCK, H)];
            } else bad = true;
        }
        float m = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) m = fmaxf(m, fabsf(Code8<E4M3>::value(((j < 4 ? x[i].x : x[i].y) >> (j & 3) * 8) & 0xffu)));
#pragma unroll
        for (int o = 1; o < LPR; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        const float s = __fmul_rn(sc[i], __fdiv_rn(m, top));
        nan |= s != s;
        best = fmaxf(best, s);
    }
    best = warp_max(best);
    nan = __any_sync(0xffffffffu, nan);
    bad = __any_sync(0xffffffffu, bad);
    if (bad && lane == 0) k8_flag(a.c.status, K8_BAD_PAGE);
    if (dst_page < 0) return;
    uint8_t * dst = static_cast<uint8_t *>(kv ? a.c.v : a.c.k) + k8_code_off(dst_page, h, X % K8_BPP * K8_BLOCK, H, D);
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
        const float ratio = !nan && best > 0.0f ? __fdiv_rn(sc[i], best) : 0.0f;
        uint32_t o[2] = {0, 0};
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float f = Code8<E4M3>::value(((j < 4 ? x[i].x : x[i].y) >> (j & 3) * 8) & 0xffu);
            o[j >> 2] |= Code8<E4M3>::code(k8_clamp(__fmul_rn(f, ratio), top)) << (j & 3) * 8;
        }
        *reinterpret_cast<uint2 *>(dst + (i * RPS + r0) * D + d0) = make_uint2(o[0], o[1]);
    }
    if (lane == 0) (kv ? a.c.v_scale : a.c.k_scale)[k8_scale_off(dst_page, h, X % K8_BPP, H)] = nan ? __int_as_float(0x7fffffff) : best;
}

}  // namespace qtts
