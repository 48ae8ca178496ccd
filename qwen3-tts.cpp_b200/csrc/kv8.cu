// kv8.cu — C entry points of the rotary and 8-bit-cache operators: argument
// checks, then launches on the caller's stream.  No entry allocates device memory
// or throws.
#include <atomic>
#include <cmath>
#include <cstdio>
#include <string>

#include "kv8.cuh"
#include "kv8_attend.cuh"
#include "kv8_tile.cuh"
#include "rope.cuh"

namespace qtts {

void set_op_error(const char * msg);   // engine.cu: the text of qtts_create_error()

namespace {

int32_t refuse(const char * who, const char * why) {
    char buf[256];
    snprintf(buf, sizeof(buf), "%s: %s", who, why);
    set_op_error(buf);
    return 0;
}
int32_t result(const char * who, cudaError_t e) { return e == cudaSuccess ? 1 : refuse(who, cudaGetErrorString(e)); }

// The call's device for the launches, the caller's afterwards.
struct OnDevice {
    int was = -1;
    bool ok = false;
    explicit OnDevice(int device) {
        if (cudaGetDevice(&was) != cudaSuccess) { was = -1; cudaGetLastError(); return; }
        ok = was == device || cudaSetDevice(device) == cudaSuccess;
        if (!ok) cudaGetLastError();
        if (was == device) was = -1;
    }
    ~OnDevice() { if (was >= 0) cudaSetDevice(was); }
};

bool aligned(const void * p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

const char * bad_cache(const qtts_kv8 * c) {
    if (!c) return "no cache";
    if (c->device < 0) return "device";
    if (c->code != 0 && c->code != 1) return "code is 0 (int8) or 1 (e4m3)";
    if (c->row_type != 1 && c->row_type != 30) return "row_type is 1 (F16) or 30 (BF16)";
    if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256) return "head_dim is 64, 128 or 256";
    if (c->n_kv_heads < 1 || c->n_kv_heads > 1024) return "n_kv_heads";
    if (c->n_pages < 1 || c->n_seqs < 0 || c->n_seqs > 65535) return "n_pages or n_seqs";
    if (c->max_pages < 1 || c->max_pages > (1 << 24)) return "max_pages";   // positions below 2^30
    if ((int64_t) c->n_pages * c->n_kv_heads * K8_PAGE > 0x7fffffff) return "the pool has 2^31 rows at most";
    if (!c->k || !c->v || !c->k_scale || !c->v_scale || !c->k_open || !c->v_open) return "a buffer of the cache is NULL";
    if (!aligned(c->k, 16) || !aligned(c->v, 16) || !aligned(c->k_scale, 16) || !aligned(c->v_scale, 16) ||
        !aligned(c->k_open, 16) || !aligned(c->v_open, 16))
        return "the cache's buffers are 16-byte aligned";
    return nullptr;
}

// grid of `units` / per, within the launch limit
bool grid_of(int64_t units, int per, unsigned * g) {
    const int64_t n = (units + per - 1) / per;
    if (n > 0x7fffffff) return false;
    *g = (unsigned) n;
    return true;
}

// Programmatic dependent launch: the kernel may be set up while its predecessor runs,
// and waits for it (pdl_wait) before it reads or writes memory.
template <class... P, class... A>
cudaError_t pdl_go(void (*f)(P...), dim3 grid, int block, int smem, cudaStream_t st, A &&... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(block);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, f, std::forward<A>(args)...);
}
template <class T, int MODE> cudaError_t rope_go(const RopeArgs & a, unsigned g, int lanes, cudaStream_t st) {
    if (lanes == 8) return pdl_go(k_rope<T, 8, MODE>, g, ROPE_WARPS * 32, 0, st, a);
    if (lanes == 16) return pdl_go(k_rope<T, 16, MODE>, g, ROPE_WARPS * 32, 0, st, a);
    return pdl_go(k_rope<T, 32, MODE>, g, ROPE_WARPS * 32, 0, st, a);
}
template <class T> int32_t rope_launch(const RopeArgs & a, cudaStream_t st) {
    constexpr int V = 16 / sizeof(T);
    const uintptr_t all = reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.k) | reinterpret_cast<uintptr_t>(a.q_out) |
                          reinterpret_cast<uintptr_t>(a.k_out);
    const int64_t strides = a.qs_row | a.qs_head | a.qo_row | a.qo_head | (a.k ? a.ks_row | a.ks_head | a.ko_row | a.ko_head : 0);
    const int lanes = a.dim / V;
    cudaError_t e;
    if (a.dim % V || (lanes != 8 && lanes != 16 && lanes != 32) || all % 16 || strides % V) {
        const int64_t units = (int64_t) a.rows * (a.q_heads + a.k_heads) * (a.dim - a.rot / 2), g = (units + 255) / 256;
        e = pdl_go(k_rope_any<T>, (unsigned)(g < 148 * 64 ? g : 148 * 64), 256, 0, st, a);
    } else {
        RopeArgs b = a;
        // many rows: a warp takes all heads of a row, so its angles are computed once; few rows: one step's heads each, so
        // that the warps cover the GPU
        const int heads = a.q_heads + a.k_heads, step = 32 / lanes;
        const int64_t warps = 148 * 32, per = ((int64_t) a.rows * heads + warps - 1) / warps;
        b.heads_per_warp = (int)(per >= heads ? heads : (per + step - 1) / step * step);
        b.chunks = (heads + b.heads_per_warp - 1) / b.heads_per_warp;
        unsigned g;
        if (!grid_of((int64_t) a.rows * b.chunks, ROPE_WARPS, &g)) return refuse("qtts_op_rope", "too many rows");
        if (a.interleaved && a.rot % V == 0) e = rope_go<T, ROPE_PAIR>(b, g, lanes, st);
        else if (!a.interleaved && a.rot / 2 % V == 0) e = rope_go<T, ROPE_WORD>(b, g, lanes, st);
        else e = rope_go<T, ROPE_VALUE>(b, g, lanes, st);
    }
    return result("qtts_op_rope", e);
}

// calls f.template operator()<T, E4M3, D>() for the cache's row type, code and head size
template <class F> void by_cache(const qtts_kv8 & c, F f) {
    auto by_dim = [&](auto t, auto e) {
        using T = decltype(t);
        constexpr bool E = decltype(e)::value;
        if (c.head_dim == 64) f(T{}, e, std::integral_constant<int, 64>{});
        else if (c.head_dim == 128) f(T{}, e, std::integral_constant<int, 128>{});
        else f(T{}, e, std::integral_constant<int, 256>{});
        (void) E;
    };
    auto by_code = [&](auto t) {
        if (c.code) by_dim(t, std::true_type{});
        else by_dim(t, std::false_type{});
    };
    if (c.row_type == 1) by_code(__half{});
    else by_code(__nv_bfloat16{});
}

// How an attention call runs.  Few rows of a (sequence, kv head) come in tiles of 8 nt;
// one CTA takes a tile's whole range, or, where that is more than 8 pages, the ranges
// are split evenly over the GPU.  Many rows come in tiles of 256 on tcgen05, one CTA each.
// Where they meet, at 2,000 keys, 8 kv heads, dim 128 (us, split / tile): 32 rows, 1, 8 and
// 32 sequences 31 / 51, 47 / 52, 102 / 103; 64 rows 33 / 51, 66 / 53, 182 / 105.  So from
// 33 rows on the tiles are taken where there are CTAs for half of the SMs, and from 65 on
// always (the split kernel would read the cache once for each 32 rows).
enum : int { PLAN_WHOLE, PLAN_SPLIT, PLAN_TILE };
struct K8Plan { int kind, nt, tiles, ctas, part_rows; int64_t line_bytes, part_bytes; unsigned grid; };   // workspace: line, parts, lse
constexpr int SMS = 148, NW = 4;
bool attend_plan(const qtts_kv8 & c, const qtts_kv8_attend & p, K8Plan * o) {
    const int64_t R = (int64_t) p.max_q * (p.n_heads / c.n_kv_heads);
    if (R > 0x7fffff00) return false;
    const bool tile = c.head_dim <= 128 && (R > 64 || (R > 32 && (int64_t) c.n_seqs * c.n_kv_heads >= 64));
    o->nt = R <= 8 ? 1 : (R <= 16 || c.head_dim == 256 ? 2 : 4);
    const int per = tile ? KT_ROWS : 8 * o->nt;
    const int64_t tiles = (R + per - 1) / per, items = tiles * c.n_kv_heads * c.n_seqs;
    if (items > 0x7fffffff) return false;
    const bool split = !tile && c.max_pages > 8 && R <= 64 && c.n_seqs <= K8_MAX_SPLIT_SEQS && items * c.max_pages < 0x40000000;
    o->kind = tile ? PLAN_TILE : (split ? PLAN_SPLIT : PLAN_WHOLE);
    o->tiles = (int) tiles;
    o->ctas = SMS * k8_ctas_per_sm(c.head_dim, o->nt);
    o->part_rows = (int)(R < 8 * o->nt ? R : 8 * o->nt);
    o->line_bytes = split ? ((int64_t) c.n_seqs + 4) / 4 * 16 : 0;
    o->part_bytes = split ? (int64_t) o->ctas * 2 * o->part_rows * (c.head_dim + 4) * 4 : 0;
    o->grid = (unsigned)(split ? o->ctas : items);
    return true;
}
// The shared memory limit of a kernel, raised once per device.
template <auto F> cudaError_t allow_smem(int bytes, int device) {
    static std::atomic<uint64_t> done{0};   // one for each kernel F
    const uint64_t bit = device < 64 ? 1ull << device : 0;
    if (done.load(std::memory_order_relaxed) & bit) return cudaSuccess;
    const cudaError_t e = cudaFuncSetAttribute(F, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_relaxed);
    return e;
}
// A pool as TMA sees it: rows of D bytes, boxes of `rows` x min(D, 128) bytes, swizzled
// over a row's length.
bool make_map(CUtensorMap * map, void * pool, const qtts_kv8 & c, int rows) {
    static const auto encode = [] {
        void * f = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &found) != cudaSuccess ||
            found != cudaDriverEntryPointSuccess)
            f = nullptr;
        return reinterpret_cast<decltype(&cuTensorMapEncodeTiled)>(f);
    }();
    if (!encode) return false;
    const cuuint64_t dims[2] = {(cuuint64_t) c.head_dim, (cuuint64_t) c.n_pages * c.n_kv_heads * K8_PAGE}, strides[1] = {(cuuint64_t) c.head_dim};
    const cuuint32_t box[2] = {(cuuint32_t)(c.head_dim < 128 ? c.head_dim : 128), (cuuint32_t) rows}, one[2] = {1, 1};
    return encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, pool, dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  c.head_dim == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_NONE,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
template <class T, bool E4M3, int D, int NT>
cudaError_t attend_launch(const K8AttendArgs & a, const K8Plan & p, cudaStream_t st) {
    K8Maps maps;
    constexpr int rows = K8_U<D, NT> * K8_BLOCK;
    if (!make_map(&maps.k, a.c.k, a.c, rows) || !make_map(&maps.v, a.c.v, a.c, rows)) return cudaErrorNotSupported;
    constexpr int base = k8_smem_bytes<D, NT, NW>();
    if (p.kind == PLAN_WHOLE) {
        constexpr auto f = k_kv8_attend_whole<T, E4M3, D, NT, NW>;
        const cudaError_t e = allow_smem<f>(base, a.c.device);
        if (e != cudaSuccess) return e;
        return pdl_go(f, p.grid, NW * 32, base, st, a, maps);
    }
    constexpr auto f = k_kv8_attend_split<T, E4M3, D, NT, NW>;
    const int smem = base + (a.c.n_seqs + 1) * 4;
    cudaError_t e = allow_smem<f>(base + (K8_MAX_SPLIT_SEQS + 1) * 4, a.c.device);
    if (e != cudaSuccess) return e;
    if ((e = pdl_go(f, p.grid, NW * 32, smem, st, a, maps)) != cudaSuccess) return e;
    return pdl_go(k_kv8_join<T, D, NT>, (unsigned)((int64_t) a.c.n_seqs * a.c.n_kv_heads * a.max_q * (a.n_heads / a.c.n_kv_heads)), K8_JOIN_WARPS * 32,
                  0, st, a);
}

template <class T, bool E4M3, int D>
cudaError_t tile_launch(const K8AttendArgs & a, const K8Plan & p, cudaStream_t st) {
    K8Maps maps;
    if (!make_map(&maps.k, a.c.k, a.c, K8_PAGE) || !make_map(&maps.v, a.c.v, a.c, K8_PAGE)) return cudaErrorNotSupported;
    constexpr auto f = k_kv8_attend_tile<T, E4M3, D>;
    const cudaError_t e = allow_smem<f>(KtSmem<D>::total, a.c.device);
    return e != cudaSuccess ? e : pdl_go(f, p.grid, KT_THREADS, KtSmem<D>::total, st, a, maps);
}

}  // namespace
}  // namespace qtts

using namespace qtts;

extern "C" {

int32_t qtts_op_rope(const qtts_rope_args * p, void * stream) {
    const char * who = "qtts_op_rope";
    if (!p) return refuse(who, "no arguments");
    if (p->type != 0 && p->type != 1 && p->type != 30) return refuse(who, "type is 0 (F32), 1 (F16) or 30 (BF16)");
    if (p->rows < 0 || p->q_heads < 1 || p->k_heads < 0 || p->q_heads > 65536 || p->k_heads > 65536) return refuse(who, "rows or heads");
    if (p->dim < 2 || p->dim > 4096) return refuse(who, "dim is 2 to 4096");
    if (p->rot < 2 || p->rot > p->dim || p->rot % 2) return refuse(who, "rot is even, at least 2 and at most dim");
    const bool has_k = p->k_heads > 0;
    if (has_k != (p->k != nullptr)) return refuse(who, "k and k_heads go together");
    if (p->rows == 0) return 1;
    if (!p->pos || !p->freq || !p->q || !p->q_out || (has_k && !p->k_out)) return refuse(who, "a pointer is NULL");
    const size_t el = p->type == 0 ? 4 : 2;
    if (!aligned(p->q, el) || !aligned(p->q_out, el) || !aligned(p->k, el) || !aligned(p->k_out, el) || !aligned(p->pos, 4) || !aligned(p->freq, 8))
        return refuse(who, "a pointer is not aligned to its type");
    if ((p->q == p->q_out && (p->q_row != p->qo_row || p->q_head != p->qo_head)) ||
        (has_k && p->k == p->k_out && (p->k_row != p->ko_row || p->k_head != p->ko_head)))
        return refuse(who, "an output that is its input has its strides");
    OnDevice on(p->device);
    if (!on.ok) return refuse(who, "device");
    RopeArgs a{};
    a.q = p->q; a.k = p->k; a.q_out = p->q_out; a.k_out = p->k_out;
    a.qs_row = p->q_row; a.qs_head = p->q_head; a.ks_row = p->k_row; a.ks_head = p->k_head;
    a.qo_row = p->qo_row; a.qo_head = p->qo_head; a.ko_row = p->ko_row; a.ko_head = p->ko_head;
    a.pos = p->pos; a.freq = p->freq; a.factor = p->factor; a.rows = p->rows; a.q_heads = p->q_heads; a.k_heads = p->k_heads;
    a.dim = p->dim; a.rot = p->rot; a.interleaved = p->interleaved ? 1 : 0;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (p->type == 1) return rope_launch<__half>(a, st);
    if (p->type == 30) return rope_launch<__nv_bfloat16>(a, st);
    return rope_launch<float>(a, st);
}

int32_t qtts_rope_freqs(int32_t scaling, int32_t rot, double theta, double factor, double original_len, double beta_fast,
                        double beta_slow, double * freq, float * value_factor) {
    const char * who = "qtts_rope_freqs";
    if (!freq || rot < 2 || rot % 2 || rot > 4096) return refuse(who, "rot is even, 2 to 4096, and freq a buffer");
    if (!(theta > 1.0) || !std::isfinite(theta)) return refuse(who, "theta is above 1");
    if (scaling < 0 || scaling > 3) return refuse(who, "scaling is 0 to 3");
    if (scaling != 0 && !(factor >= 1.0 && std::isfinite(factor))) return refuse(who, "factor is at least 1");
    if (scaling == 3 && !(original_len >= 1.0 && beta_slow > 0.0 && beta_fast > beta_slow)) return refuse(who, "original_len or the betas");
    double base = theta;
    if (scaling == 2 && rot > 2) base = theta * std::pow(factor, (double) rot / (rot - 2));
    double lo = 0.0, hi = 0.0;
    if (scaling == 3) {
        const double pi2 = 6.283185307179586476925;
        auto dim_of = [&](double turns) { return rot * std::log(original_len / (turns * pi2)) / (2.0 * std::log(theta)); };
        lo = std::fmax(std::floor(dim_of(beta_fast)), 0.0);
        hi = std::fmin(std::ceil(dim_of(beta_slow)), (double) rot - 1.0);
    }
    for (int i = 0; i < rot / 2; ++i) {
        double f = std::pow(base, -2.0 * i / rot);
        if (scaling == 1) f /= factor;
        if (scaling == 3) {
            const double ramp = std::fmin(std::fmax((i - lo) / std::fmax(hi - lo, 0.001), 0.0), 1.0);
            f = f / factor * ramp + f * (1.0 - ramp);
        }
        freq[i] = f;
    }
    if (value_factor) *value_factor = scaling == 3 ? (float)(0.1 * std::log(factor) + 1.0) : 1.0f;
    return 1;
}

int32_t qtts_kv8_check(const qtts_kv8 * c, const int32_t * table, const int32_t * lens, const int32_t * cu, int32_t n_rows,
                       int32_t max_new) {
    const char * why = bad_cache(c);
    if (why || !table || !lens || n_rows < 0) { refuse("qtts_kv8_check", why ? why : "table, lens or n_rows"); return -1; }
    int status = 0;
    for (int b = 0; b < c->n_seqs; ++b) {
        const K8Seq s = k8_seq(b, lens, cu, c->max_pages, n_rows, max_new, true);
        status |= s.status;
        for (int p = 0; p < (s.len + K8_PAGE - 1) / K8_PAGE; ++p)
            if (k8_page(table + (int64_t) b * c->max_pages, p, c->n_pages) < 0) status |= K8_BAD_PAGE;
    }
    return status;
}

int32_t qtts_op_kv8_append(const qtts_kv8 * c, const int32_t * table, const int32_t * lens, const int32_t * cu, const void * k,
                           const void * v, int64_t k_row, int64_t k_head, int64_t v_row, int64_t v_head, int32_t n_rows,
                           int32_t max_new, void * stream) {
    const char * who = "qtts_op_kv8_append";
    if (const char * why = bad_cache(c)) return refuse(who, why);
    if (n_rows < 0 || max_new < 0) return refuse(who, "n_rows or max_new");
    if (!cu && n_rows != c->n_seqs) return refuse(who, "without cu there is one row for each sequence");
    if (n_rows == 0 || c->n_seqs == 0 || max_new == 0) return 1;
    if (!table || !lens || !k || !v) return refuse(who, "a pointer is NULL");
    if (!aligned(k, 2) || !aligned(v, 2)) return refuse(who, "k and v are aligned to their type");
    OnDevice on(c->device);
    if (!on.ok) return refuse(who, "device");
    K8Args a{};
    a.c = *c; a.table = table; a.lens = lens; a.cu = cu;
    a.src[0] = static_cast<const uint16_t *>(k); a.src[1] = static_cast<const uint16_t *>(v);
    a.s_row[0] = k_row; a.s_head[0] = k_head; a.s_row[1] = v_row; a.s_head[1] = v_head;
    a.n_rows = n_rows; a.max_n = max_new;
    a.blocks = (int)(((int64_t) max_new + 2 * K8_BLOCK - 2) / K8_BLOCK);   // a run of max_new rows touches at most this many blocks
    const bool vec = aligned(k, 16) && aligned(v, 16) && (k_row | k_head | v_row | v_head) % 8 == 0;
    unsigned g;
    if (!grid_of((int64_t) a.blocks * c->n_kv_heads * 2, K8_WARPS, &g) || g > 0x7fffffff / K8_WARPS) return refuse(who, "too many rows");
    const dim3 grid(g, (unsigned) c->n_seqs);
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    cudaError_t err = cudaSuccess;
    by_cache(*c, [&](auto t, auto e, auto d) {
        if (vec) err = pdl_go(k_kv8_append<decltype(t), decltype(e)::value, decltype(d)::value, true>, grid, K8_WARPS * 32, 0, st, a);
        else err = pdl_go(k_kv8_append<decltype(t), decltype(e)::value, decltype(d)::value, false>, grid, K8_WARPS * 32, 0, st, a);
    });
    return result(who, err);
}

int32_t qtts_op_kv8_read(const qtts_kv8 * c, const int32_t * table, const int32_t * begin, const int32_t * cu, int32_t out_type,
                         void * k, void * v, int32_t n_rows, int32_t max_rows, void * stream) {
    const char * who = "qtts_op_kv8_read";
    if (const char * why = bad_cache(c)) return refuse(who, why);
    if (n_rows < 0 || max_rows < 0) return refuse(who, "n_rows or max_rows");
    if (!cu && n_rows != c->n_seqs) return refuse(who, "without cu there is one row for each sequence");
    if (out_type != 0 && out_type != 1 && out_type != 30) return refuse(who, "out_type is 0 (F32), 1 (F16) or 30 (BF16)");
    if (n_rows == 0 || c->n_seqs == 0 || max_rows == 0) return 1;
    if (!table || !k || !v) return refuse(who, "a pointer is NULL");
    if (!aligned(k, 16) || !aligned(v, 16)) return refuse(who, "k and v are 16-byte aligned");
    OnDevice on(c->device);
    if (!on.ok) return refuse(who, "device");
    K8ReadArgs a{};
    a.c = *c; a.table = table; a.begin = begin; a.cu = cu; a.n_rows = n_rows; a.max_n = max_rows; a.k = k; a.v = v;
    const int per_row = c->n_kv_heads * (c->head_dim / 16);
    a.rows_per_cta = per_row >= 512 ? 1 : 512 / per_row;
    const dim3 grid((unsigned)((max_rows + (int64_t) a.rows_per_cta - 1) / a.rows_per_cta), (unsigned) c->n_seqs);
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    auto go = [&](auto t) {
        using T = decltype(t);
        return c->code ? pdl_go(k_kv8_read<T, true>, grid, 256, 0, st, a) : pdl_go(k_kv8_read<T, false>, grid, 256, 0, st, a);
    };
    return result(who, out_type == 0 ? go(0.0f) : (out_type == 1 ? go(__half{}) : go(__nv_bfloat16{})));
}

int64_t qtts_kv8_attend_ws(const qtts_kv8 * c, const qtts_kv8_attend * p) {
    if (bad_cache(c) || !p || p->n_rows < 0 || p->n_heads < 1) return -1;
    K8Plan plan;
    if (p->n_heads % c->n_kv_heads || p->max_q < 0 || !attend_plan(*c, *p, &plan)) return -1;
    return plan.line_bytes + plan.part_bytes + (p->weight_out && !p->lse ? ((int64_t) p->n_rows * p->n_heads * 4 + 15) / 16 * 16 : 0);
}

int32_t qtts_op_kv8_attend(const qtts_kv8 * c, const qtts_kv8_attend * p, void * stream) {
    const char * who = "qtts_op_kv8_attend";
    if (const char * why = bad_cache(c)) return refuse(who, why);
    if (!p) return refuse(who, "no arguments");
    if (p->n_heads < 1 || p->n_heads % c->n_kv_heads) return refuse(who, "n_heads is a multiple of n_kv_heads");
    if (p->n_rows < 0 || p->max_q < 0 || p->window < 0) return refuse(who, "n_rows, max_q or window");
    if (!p->cu && p->n_rows != c->n_seqs) return refuse(who, "without cu there is one row for each sequence");
    if (!(p->scale >= 0.0f) || std::isinf(p->scale)) return refuse(who, "scale is finite and not negative");
    if ((p->weight_in == nullptr) != (p->weight_out == nullptr)) return refuse(who, "weight_in and weight_out go together");
    if (p->weight_out && p->weight_stride < (int64_t) c->max_pages * K8_PAGE) return refuse(who, "weight_stride is at least 64 max_pages");
    if (c->n_seqs == 0) return 1;
    // without rows there are no weights to add, but weight_out still gets weight_in
    if ((p->n_rows == 0 || p->max_q == 0) && (!p->weight_out || p->weight_in == p->weight_out)) return 1;
    if (!p->table || !p->lens || (p->n_rows && (!p->q || !p->out))) return refuse(who, "a pointer is NULL");
    if (!aligned(p->q, 2) || !aligned(p->out, 2)) return refuse(who, "q and out are aligned to their type");
    const int64_t ws = qtts_kv8_attend_ws(c, p);
    if (ws > 0 && (!p->ws || p->ws_bytes < ws || !aligned(p->ws, 16))) return refuse(who, "workspace: see qtts_kv8_attend_ws");
    OnDevice on(c->device);
    if (!on.ok) return refuse(who, "device");
    K8AttendArgs a{};
    a.c = *c; a.table = p->table; a.lens = p->lens; a.cu = p->cu; a.q = p->q; a.out = p->out;
    a.q_row = p->q_row; a.q_head = p->q_head; a.o_row = p->o_row; a.o_head = p->o_head;
    a.n_rows = p->n_rows; a.max_q = p->max_q; a.n_heads = p->n_heads; a.window = p->window; a.scale = p->scale; a.lse = p->lse;
    a.w_in = p->weight_in; a.w_out = p->weight_out; a.w_stride = p->weight_stride;
    K8Plan plan;
    if (!attend_plan(*c, *p, &plan)) return refuse(who, "too much work for one call");
    if (p->weight_out && !a.lse) a.lse = reinterpret_cast<float *>(static_cast<uint8_t *>(p->ws) + plan.line_bytes + plan.part_bytes);
    a.line = static_cast<int *>(p->ws);
    a.part = reinterpret_cast<float *>(static_cast<uint8_t *>(p->ws) + plan.line_bytes);
    a.tiles = plan.tiles; a.ctas = plan.ctas; a.part_rows = plan.part_rows;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    cudaError_t err = cudaSuccess;
    by_cache(*c, [&](auto t, auto e, auto d) {
        using T = decltype(t);
        constexpr bool E = decltype(e)::value;
        constexpr int D = decltype(d)::value;
        if (p->n_rows > 0 && p->max_q > 0) {
            if (plan.kind == PLAN_TILE) {
                if constexpr (D < 256) err = tile_launch<T, E, D>(a, plan, st);
            } else if (plan.nt == 1) err = attend_launch<T, E, D, 1>(a, plan, st);
            else if (plan.nt == 2) err = attend_launch<T, E, D, 2>(a, plan, st);
            else if constexpr (D < 256) err = attend_launch<T, E, D, 4>(a, plan, st);
        }
        if (p->weight_out && err == cudaSuccess) {
            constexpr int keys = K8_WEIGH_W<D> * K8_BLOCK * K8_WEIGH_WARPS;
            const dim3 grid((unsigned)(((int64_t) c->max_pages * K8_PAGE + keys - 1) / keys), (unsigned) c->n_kv_heads, (unsigned) c->n_seqs);
            err = pdl_go(k_kv8_weigh<T, E, D>, grid, K8_WEIGH_WARPS * 32, 0, st, a);
        }
    });
    return result(who, err);
}

int32_t qtts_op_kv8_evict(const qtts_kv8 * c, const int32_t * table, const int32_t * lens, const int32_t * dst_table,
                          int32_t dst_pages, const float * weight, int64_t weight_stride, int32_t budget, int32_t sinks,
                          int32_t recent, int32_t * lens_out, int32_t * keep, float * weight_out, void * stream) {
    const char * who = "qtts_op_kv8_evict";
    if (const char * why = bad_cache(c)) return refuse(who, why);
    if (budget < K8_BLOCK || budget % K8_BLOCK) return refuse(who, "budget is a multiple of 16");
    if (sinks < 0 || recent < 0 || sinks > budget || recent > budget - sinks) return refuse(who, "sinks + recent is at most budget");
    if ((int64_t) dst_pages * K8_PAGE < budget) return refuse(who, "dst_pages hold the budget");
    if (weight_stride < (int64_t) c->max_pages * K8_PAGE) return refuse(who, "weight_stride is at least 64 max_pages");
    if (c->n_seqs == 0) return 1;
    if (!table || !lens || !dst_table || !weight || !lens_out || !keep || !weight_out) return refuse(who, "a pointer is NULL");
    if (lens == lens_out || weight == weight_out || table == dst_table) return refuse(who, "the outputs are other buffers than the inputs");
    OnDevice on(c->device);
    if (!on.ok) return refuse(who, "device");
    K8EvictArgs a{};
    a.c = *c; a.table = table; a.lens = lens; a.dst_table = dst_table; a.dst_pages = dst_pages; a.weight = weight; a.w_stride = weight_stride;
    a.budget = budget; a.sinks = sinks; a.recent = recent; a.lens_out = lens_out; a.keep = keep; a.weight_out = weight_out;
    unsigned g;
    if (!grid_of((int64_t)(budget / K8_BLOCK) * c->n_kv_heads * 2, K8_WARPS, &g)) return refuse(who, "too much work for one call");
    const dim3 grid(g, (unsigned) c->n_seqs);
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int64_t cap = (int64_t) c->max_pages * K8_PAGE;
    const int room = cap < K8_SEL_KEYS ? (int) cap : K8_SEL_KEYS;
    cudaError_t err = allow_smem<k_kv8_select>(K8_SEL_KEYS * 4, c->device);
    if (err == cudaSuccess) err = pdl_go(k_kv8_select, (unsigned)(c->n_seqs * c->n_kv_heads), K8_SEL_THREADS, room * 4, st, a, room);
    if (err == cudaSuccess)
        by_cache(*c, [&](auto t, auto e, auto d) {
            (void) t;
            err = pdl_go(k_kv8_move<decltype(e)::value, decltype(d)::value>, grid, K8_WARPS * 32, 0, st, a);
        });
    return result(who, err);
}

}  // extern "C"
