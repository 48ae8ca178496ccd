// kv8.cuh — the 8-bit paged key/value cache: layout, bounds and the kernels
// that write it (append, evict) and read it back.
//
// A page holds 64 tokens: for every kv head 64 rows of 8-bit codes for K and for
// V, and one F32 scale per block of 16 tokens (value = code * scale).  A block
// is quantised from 16-bit rows,
//     scale = fl(amax / top),   code = rn(x * top / amax),   top = 127 (int8) or 448 (e4m3),
// each code the correct rounding of the exact quotient, so a block is the same bits
// however its rows arrived.
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

__device__ __forceinline__ uint32_t k8_prmt(uint32_t a, uint32_t b, uint32_t s) { return __byte_perm(a, b, s); }
// Four codes -> two F16 pairs (bytes 0, 1 and 2, 3), exactly.
template <bool E4M3> __device__ __forceinline__ void k8_f16x4(uint32_t w, uint32_t & lo, uint32_t & hi);
template <> __device__ __forceinline__ void k8_f16x4<false>(uint32_t w, uint32_t & lo, uint32_t & hi) {
    // byte u = code + 128 as the low mantissa bits of 1024: 1024 + u - 1152 = code
    w ^= 0x80808080u;
    lo = k8_prmt(w, 0x64646464u, 0x4140);
    hi = k8_prmt(w, 0x64646464u, 0x4342);
    const __half2 off = __half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));
    __half2 a = __hsub2(*reinterpret_cast<__half2 *>(&lo), off), b = __hsub2(*reinterpret_cast<__half2 *>(&hi), off);
    lo = *reinterpret_cast<uint32_t *>(&a);
    hi = *reinterpret_cast<uint32_t *>(&b);
}
template <> __device__ __forceinline__ void k8_f16x4<true>(uint32_t w, uint32_t & lo, uint32_t & hi) {
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
        : "=r"(lo), "=r"(hi) : "r"(w));
}
__device__ __forceinline__ float2 k8_f32x2(uint32_t h) { return __half22float2(*reinterpret_cast<const __half2 *>(&h)); }

template <bool E4M3> struct Code8;
template <> struct Code8<false> {
    static constexpr float top = 127.0f;
    // four values within +-top -> four codes: adding 1.5 * 2^23 rounds to an integer (to even) in the low mantissa bits
    static __device__ __forceinline__ uint32_t pack(float a, float b, float c, float d) {
        const float m = 12582912.0f;
        const uint32_t ab = k8_prmt(__float_as_uint(a + m), __float_as_uint(b + m), 0x0040), cd = k8_prmt(__float_as_uint(c + m), __float_as_uint(d + m), 0x0040);
        return k8_prmt(ab, cd, 0x5410);
    }
};
template <> struct Code8<true> {
    static constexpr float top = 448.0f;
    static __device__ __forceinline__ uint32_t pack(float a, float b, float c, float d) {
        uint32_t r;
        asm("{\n\t.reg .b16 x, y;\n\tcvt.rn.satfinite.e4m3x2.f32 x, %2, %1;\n\tcvt.rn.satfinite.e4m3x2.f32 y, %4, %3;\n\tmov.b32 %0, {x, y};\n\t}"
            : "=r"(r) : "f"(a), "f"(b), "f"(c), "f"(d));
        return r;
    }
};
__device__ __forceinline__ float k8_clamp(float r, float top) { return fminf(fmaxf(r, -top), top); }

// fl(x top / amax) for the entries x of a block (|x| <= amax): the product is exact
// (at most 11 + 9 bits), and a quotient q0 by the rounded reciprocal corrected by its
// exact residual is the correctly rounded one (Markstein 1990).  A power of two keeps
// BF16's whole range away from F32's ends.  The result is within +-top.
struct K8Quot {
    float b, y, up;
    __device__ __forceinline__ K8Quot(float amax, float top) {
        const float p = amax > 1.8446744073709552e19f ? 5.421010862427522e-20f : (amax < 5.421010862427522e-20f ? 1.8446744073709552e19f : 1.0f);   // 2^-64, 2^64
        b = amax * p;
        y = amax > 0.0f ? __frcp_rn(b) : 0.0f;
        up = p * top;
    }
    __device__ __forceinline__ float operator()(float x) const {
        const float n = __fmul_rn(x, up), q0 = __fmul_rn(n, y);
        return __fmaf_rn(__fmaf_rn(-q0, b, n), y, q0);
    }
};

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
// registers (a lane holds 16 consecutive dims of D / 32 rows), the block's largest
// magnitude as an integer maximum over the sign-less 16-bit patterns (which also
// finds infinities and NaN), then the codes.  Bound by memory: 2 D bytes read and
// D written per row, kv head and side.
constexpr int K8_WARPS = 4;
template <class T, bool E4M3, int D, bool VEC>
__global__ void __launch_bounds__(K8_WARPS * 32) k_kv8_append(K8Args a) {
    constexpr int LPR = D / 16, RPS = 32 / LPR, STEPS = K8_BLOCK / RPS;   // lanes per row, rows per step
    const int lane = threadIdx.x & 31, H = a.c.n_kv_heads, b = blockIdx.y;
    const int unit = blockIdx.x * K8_WARPS + (threadIdx.x >> 5);
    const int kv = unit & 1, h = (unit >> 1) % H, nb = (unit >> 1) / H;
    pdl_trigger();
    pdl_wait();
    const K8Seq s = k8_seq(b, a.lens, a.cu, a.c.max_pages, a.n_rows, a.max_n, true);
    if (s.status && lane == 0 && nb == 0) k8_flag(a.c.status, s.status);
    if (s.n == 0) return;
    const int start = s.len - s.n, first = start / K8_BLOCK, last = (s.len - 1) / K8_BLOCK, X = first + nb;
    if (X > last || nb >= a.blocks) return;
    const int page = k8_page(a.table + (int64_t) b * a.c.max_pages, X / K8_BPP, a.c.n_pages);
    const uint16_t * src = a.src[kv] + (int64_t) h * a.s_head[kv];
    uint16_t * ring = static_cast<uint16_t *>(kv ? a.c.v_open : a.c.k_open) + ((int64_t) b * H + h) * K8_RING * D;
    const int r0 = lane / LPR, d0 = lane % LPR * 16;
    uint32_t x[STEPS][8];
    uint32_t most = 0;
    auto load = [&](uint32_t (&w)[8], int pos) {     // row `pos` of the sequence: new, or of the ring, or none yet
        const uint16_t * p = pos < start ? ring + (pos % K8_RING) * D + d0 : src + (int64_t)(s.row0 + pos - start) * a.s_row[kv] + d0;
        uint4 u = make_uint4(0, 0, 0, 0), v = u;
        if (pos < start) { u = k8_ld8<true>(p); v = k8_ld8<true>(p + 8); }
        else if (pos < s.len) { u = k8_ld8<VEC>(p); v = k8_ld8<VEC>(p + 8); }
        w[0] = u.x; w[1] = u.y; w[2] = u.z; w[3] = u.w; w[4] = v.x; w[5] = v.y; w[6] = v.z; w[7] = v.w;
    };
#pragma unroll
    for (int i = 0; i < STEPS; ++i) load(x[i], X * K8_BLOCK + i * RPS + r0);
#pragma unroll
    for (int i = 0; i < STEPS; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) most = __vmaxu2(most, x[i][j] & 0x7fff7fffu);
    most = max(most & 0xffffu, most >> 16);
    most = __reduce_max_sync(0xffffffffu, most);
    const bool fine = most < Row16<T>::inf;
    const float top = Code8<E4M3>::top, amax = fine ? k8_bits_f<T>(most) : 0.0f;   // zero codes if not fine
    const float scale = fine ? __fdiv_rn(amax, top) : __int_as_float(0x7fffffff);
    const K8Quot quot(amax, top);
    if (page >= 0) {
        uint8_t * dst = static_cast<uint8_t *>(kv ? a.c.v : a.c.k) + k8_code_off(page, h, X % K8_BPP * K8_BLOCK, H, D);
#pragma unroll
        for (int i = 0; i < STEPS; ++i) {
            uint32_t o[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t u = fine ? x[i][2 * j] : 0u, v = fine ? x[i][2 * j + 1] : 0u;
                o[j] = Code8<E4M3>::pack(quot(k8_bits_f<T>(u & 0xffffu)), quot(k8_bits_f<T>(u >> 16)), quot(k8_bits_f<T>(v & 0xffffu)), quot(k8_bits_f<T>(v >> 16)));
            }
            *reinterpret_cast<uint4 *>(dst + (i * RPS + r0) * D + d0) = make_uint4(o[0], o[1], o[2], o[3]);
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
            if (Y != X) load(x[i], pos);
            uint4 * p = reinterpret_cast<uint4 *>(ring + (pos % K8_RING) * D + d0);
            p[0] = make_uint4(x[i][0], x[i][1], x[i][2], x[i][3]);
            p[1] = make_uint4(x[i][4], x[i][5], x[i][6], x[i][7]);
        }
    }
}

// ---- read ------------------------------------------------------------------
// Rows begin .. of each sequence as 16- or 32-bit values, packed.  One thread per 16
// dims of a (row, kv head), both sides.  Rows of pages that are none read as zero.
struct K8ReadArgs {
    qtts_kv8 c;
    const int32_t * table, * begin, * cu;
    int n_rows, max_n, rows_per_cta;
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
    const int H = a.c.n_kv_heads, D = a.c.head_dim, cph = D / 16, cpr = H * cph, b = blockIdx.y;
    pdl_trigger();
    pdl_wait();
    const K8Seq s = k8_seq(b, nullptr, a.cu, a.c.max_pages, a.n_rows, a.max_n, false);
    const int begin = a.begin ? a.begin[b] : 0;
    int bad = s.status;
    if (begin < 0 || (int64_t) begin + s.n > (int64_t) a.c.max_pages * K8_PAGE) bad |= K8_BAD_LEN;
    if (bad) {
        if (blockIdx.x == 0 && threadIdx.x == 0) k8_flag(a.c.status, bad);
        return;
    }
    for (int c = threadIdx.x; c < a.rows_per_cta * cpr; c += 256) {
        const int i = blockIdx.x * a.rows_per_cta + c / cpr, h = c % cpr / cph, d0 = c % cph * 16, pos = begin + i;
        if (i >= s.n) break;
        const int page = k8_page(a.table + (int64_t) b * a.c.max_pages, pos / K8_PAGE, a.c.n_pages);
        if (page < 0) k8_flag(a.c.status, K8_BAD_PAGE);
        uint4 w[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
        float sc[2] = {0.0f, 0.0f};
        if (page >= 0) {
            const int64_t at = k8_code_off(page, h, pos % K8_PAGE, H, D) + d0, sa = k8_scale_off(page, h, pos % K8_PAGE / K8_BLOCK, H);
            w[0] = *reinterpret_cast<const uint4 *>(static_cast<const uint8_t *>(a.c.k) + at);
            w[1] = *reinterpret_cast<const uint4 *>(static_cast<const uint8_t *>(a.c.v) + at);
            sc[0] = a.c.k_scale[sa];
            sc[1] = a.c.v_scale[sa];
        }
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
            const uint32_t x[4] = {w[kv].x, w[kv].y, w[kv].z, w[kv].w};
            float f[16];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                uint32_t lo, hi;
                k8_f16x4<E4M3>(x[j], lo, hi);
                const float2 u = k8_f32x2(lo), v = k8_f32x2(hi);
                f[4 * j] = __fmul_rn(u.x, sc[kv]); f[4 * j + 1] = __fmul_rn(u.y, sc[kv]);
                f[4 * j + 2] = __fmul_rn(v.x, sc[kv]); f[4 * j + 3] = __fmul_rn(v.y, sc[kv]);
            }
            T * o = static_cast<T *>(kv ? a.v : a.k) + ((int64_t)(s.row0 + i) * H + h) * D + d0;
            k8_store8(o, f);
            k8_store8(o + 8, f + 8);
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

// One CTA per (sequence, kv head).  The k-th largest weight by radix selection: three
// passes (11, 11 and 10 bits) over a shared-memory histogram, the ordered keys held in
// shared memory where they fit.  Then each warp counts its run of positions (those
// above the k-th weight, those equal to it), one scan over the warps gives it its place
// and its share of the equal ones, and it writes its positions in order by ballots.
constexpr int K8_SEL_THREADS = 1024, K8_SEL_KEYS = 49152;   // keys that fit beside the histogram
__global__ void __launch_bounds__(K8_SEL_THREADS) k_kv8_select(K8EvictArgs a, int room) {
    extern __shared__ __align__(16) uint32_t k8_keys[];      // [room]
    __shared__ int hist[2048], s_take[32], s_eq[32], s_sel[2];
    const int H = a.c.n_kv_heads, b = blockIdx.x / H, h = blockIdx.x % H, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    pdl_trigger();
    pdl_wait();
    int n = a.lens[b];
    if (n < 0 || (int64_t) n > (int64_t) a.c.max_pages * K8_PAGE) {
        if (tid == 0 && h == 0) k8_flag(a.c.status, K8_BAD_LEN);
        n = 0;
    }
    const int kept = min(n, a.budget);
    if (h == 0 && tid == 0) a.lens_out[b] = kept;
    // the new pages have to be others than the old ones
    const int np = (n + K8_PAGE - 1) / K8_PAGE, nd = (kept + K8_PAGE - 1) / K8_PAGE;
    for (int t = tid * H + h; t < np; t += H * K8_SEL_THREADS) {
        const int id = a.table[(int64_t) b * a.c.max_pages + t];
        for (int d = 0; d < nd; ++d)
            if (id == a.dst_table[(int64_t) b * a.dst_pages + d]) k8_flag(a.c.status, K8_SHARED_PAGE);
    }
    const float * w = a.weight + ((int64_t) b * H + h) * a.w_stride;
    int32_t * keep = a.keep + ((int64_t) b * H + h) * a.budget;
    float * wo = a.weight_out + ((int64_t) b * H + h) * a.budget;
    for (int i = kept + tid; i < a.budget; i += K8_SEL_THREADS) { keep[i] = -1; wo[i] = 0.0f; }
    if (n <= a.budget) {
        for (int i = tid; i < n; i += K8_SEL_THREADS) { keep[i] = i; wo[i] = w[i]; }
        return;
    }
    const int lo = a.sinks, hi = n - a.recent, total_want = a.budget - a.sinks - a.recent;   // of positions lo .. hi - 1
    const bool held = n <= room;
    if (held)
        for (int i = tid; i < n; i += K8_SEL_THREADS) k8_keys[i] = k8_weight_key(w[i]);
    auto key = [&](int i) { return held ? k8_keys[i] : k8_weight_key(w[i]); };
    uint32_t kth = 0, mask = 0;
    int want = total_want;
    if (want > 0) {
#pragma unroll
        for (int pass = 0; pass < 3; ++pass) {
            const int shift = pass == 0 ? 21 : (pass == 1 ? 10 : 0), bins = pass == 2 ? 1024 : 2048;
            for (int i = tid; i < 2048; i += K8_SEL_THREADS) hist[i] = 0;
            __syncthreads();
            for (int i = lo + tid; i < hi; i += K8_SEL_THREADS) {
                const uint32_t k = key(i);
                if ((k & mask) == kth) atomicAdd(&hist[k >> shift & (bins - 1)], 1);
            }
            __syncthreads();
            // the bin that holds the want-th largest: thread t sums the bins from the top, 2 (or 1) each
            const int per = bins / K8_SEL_THREADS, top_bin = bins - 1 - tid * per;
            int c0 = hist[top_bin], c1 = per == 2 ? hist[top_bin - 1] : 0, x = c0 + c1;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) { const int y = __shfl_up_sync(0xffffffffu, x, o); if (lane >= o) x += y; }
            if (lane == 31) s_take[warp] = x;
            __syncthreads();
            int before = x - c0 - c1;
            for (int i = 0; i < warp; ++i) before += s_take[i];
            if (before < want && before + c0 + c1 >= want) {
                const bool in0 = before + c0 >= want;
                s_sel[0] = in0 ? top_bin : top_bin - 1;
                s_sel[1] = want - before - (in0 ? 0 : c0);
            }
            __syncthreads();
            kth |= (uint32_t) s_sel[0] << shift;
            mask |= (uint32_t)(bins - 1) << shift;
            want = s_sel[1];
        }
    } else if (held) __syncthreads();
    // `want` of those equal to kth stay, the first ones
    const int run = ((n + 31) / 32 + 31) / 32 * 32, i0 = min(n, warp * run), i1 = min(n, i0 + run);
    int take = 0, eq = 0;
    for (int base = i0; base < i1; base += 32) {
        const int i = base + lane;
        const bool mid = i >= lo && i < hi && total_want > 0;
        const uint32_t k = mid && i < i1 ? key(i) : 0;
        take += __popc(__ballot_sync(0xffffffffu, i < i1 && (i < lo || i >= hi || (mid && k > kth))));
        eq += __popc(__ballot_sync(0xffffffffu, i < i1 && mid && k == kth));
    }
    if (lane == 0) { s_take[warp] = take; s_eq[warp] = eq; }
    __syncthreads();
    int out = 0, seen = 0;
    for (int i = 0; i < warp; ++i) {
        out += s_take[i] + max(0, min(s_eq[i], want - seen));
        seen += s_eq[i];
    }
    for (int base = i0; base < i1; base += 32) {
        const int i = base + lane;
        const bool mid = i >= lo && i < hi && total_want > 0;
        const uint32_t k = mid && i < i1 ? key(i) : 0, below = (1u << lane) - 1;
        const uint32_t eqs = __ballot_sync(0xffffffffu, i < i1 && mid && k == kth);
        const bool yes = i < i1 && (i < lo || i >= hi || (mid && (k > kth || (k == kth && seen + __popc(eqs & below) < want))));
        const uint32_t all = __ballot_sync(0xffffffffu, yes);
        if (yes) {
            const int o = out + __popc(all & below);
            keep[o] = i;
            wo[o] = w[i];
        }
        out += __popc(all);
        seen += __popc(eqs);
    }
}

// One warp per (sequence, new block, kv head, K or V): gathers the block's 16 rows
// and requantises them from their codes,
//     scale' = max_r scale_r * (max |code_r| / top),  code' = rn(code_r * (scale_r / scale')),
// so rows whose scale is the block's new one keep their codes, and a block that
// moves whole keeps its values.  Rows past the new length are zero codes.
template <bool E4M3, int D>
__global__ void __launch_bounds__(K8_WARPS * 32) k_kv8_move(K8EvictArgs a) {
    constexpr int LPR = D / 16, RPS = 32 / LPR, STEPS = K8_BLOCK / RPS;
    const int lane = threadIdx.x & 31, H = a.c.n_kv_heads, b = blockIdx.y;
    const int unit = blockIdx.x * K8_WARPS + (threadIdx.x >> 5);
    const int kv = unit & 1, h = (unit >> 1) % H, X = (unit >> 1) / H;
    pdl_trigger();
    pdl_wait();
    const int kept = a.lens_out[b];
    if (X * K8_BLOCK >= kept) return;
    const int dst_page = k8_page(a.dst_table + (int64_t) b * a.dst_pages, X / K8_BPP, a.c.n_pages);
    const int32_t * keep = a.keep + ((int64_t) b * H + h) * a.budget + X * K8_BLOCK;
    const uint8_t * codes = static_cast<const uint8_t *>(kv ? a.c.v : a.c.k);
    const float * scales = kv ? a.c.v_scale : a.c.k_scale;
    const int r0 = lane / LPR, d0 = lane % LPR * 16;
    const float top = Code8<E4M3>::top;
    uint4 x[STEPS];
    float sc[STEPS];
    float best = 0.0f;
    bool nan = false, bad = dst_page < 0;
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
        const int pos = keep[i * RPS + r0];
        x[i] = make_uint4(0, 0, 0, 0);
        sc[i] = 0.0f;
        if (pos >= 0) {
            const int page = k8_page(a.table + (int64_t) b * a.c.max_pages, pos / K8_PAGE, a.c.n_pages);
            if (page >= 0) {
                x[i] = *reinterpret_cast<const uint4 *>(codes + k8_code_off(page, h, pos % K8_PAGE, H, D) + d0);
                sc[i] = scales[k8_scale_off(page, h, pos % K8_PAGE / K8_BLOCK, H)];
            } else bad = true;
        }
    }
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
        const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
        __half2 m = __half2half2(__ushort_as_half(0));
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            uint32_t lo, hi;
            k8_f16x4<E4M3>(w[j], lo, hi);
            m = __hmax2(m, __hmax2(__habs2(*reinterpret_cast<__half2 *>(&lo)), __habs2(*reinterpret_cast<__half2 *>(&hi))));
        }
        float f = fmaxf(__low2float(m), __high2float(m));
#pragma unroll
        for (int o = 1; o < LPR; o <<= 1) f = fmaxf(f, __shfl_xor_sync(0xffffffffu, f, o));
        const float s = __fmul_rn(sc[i], __fdiv_rn(f, top));
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
        const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
        uint32_t o[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            uint32_t lo, hi;
            k8_f16x4<E4M3>(w[j], lo, hi);
            const float2 u = k8_f32x2(lo), v = k8_f32x2(hi);
            o[j] = Code8<E4M3>::pack(k8_clamp(__fmul_rn(u.x, ratio), top), k8_clamp(__fmul_rn(u.y, ratio), top), k8_clamp(__fmul_rn(v.x, ratio), top),
                                     k8_clamp(__fmul_rn(v.y, ratio), top));
        }
        *reinterpret_cast<uint4 *>(dst + (i * RPS + r0) * D + d0) = make_uint4(o[0], o[1], o[2], o[3]);
    }
    if (lane == 0) (kv ? a.c.v_scale : a.c.k_scale)[k8_scale_off(dst_page, h, X % K8_BPP, H)] = nan ? __int_as_float(0x7fffffff) : best;
}

}  // namespace qtts
