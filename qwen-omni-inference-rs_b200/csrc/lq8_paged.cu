// lq8_paged.cu -- rotary positions with several axes, and the append to a paged K/V cache with
// the q/k RMSNorm and the rotation on the way. Both are bound by HBM (a multiply-add per byte
// or less), so they read each input once, with wide loads of several heads in flight, and write
// each output once.
#include "lq8_async.cuh"
#include "lq8_fused.cuh"
#include "lq8_paged_rows.cuh"

#include <algorithm>

namespace lq {

// =========================================================================================
// Rotary positions with several axes: y_i = x_i cos - x_{i+n} sin, y_{i+n} = x_{i+n} cos +
// x_i sin for the n pairs of a head, the dims past 2n copied. A thread owns V pairs (16 bytes of
// x_i and of x_{i+n}) of H heads of one row: the angles are gathered once for the heads, and 2 H
// 16-byte loads are in flight before the first use. A CTA takes whole rows, so that DRAM sees runs
// of all their heads (a thread that walks over all heads of a row instead, with the CTA spread over
// 32 rows: 180 against 123 us for 32768 rows of 40 heads). Bound: HBM; those rows in 121 to 126 us
// (5.5 TB/s, 85 % of a plain copy), 4805 rows of 32 + 16 heads of 80 dims in f32 in 20 us.
// =========================================================================================
struct MropeArgs {
    const void* x;
    void* y;
    int64_t x_row, x_head, y_row, y_head;
    int64_t rows;
    int heads, head_dim;
    int chunks;      // V-wide chunks of a head: pairs / V rotated ones, then the copied dims
    int units;       // chunks * ceil(heads / H)
    int rows_per_cta;
    float sign;      // -1: the inverse rotation
    int* err;
};

template <typename T, int V, int H>
__global__ void __launch_bounds__(256, 2) mrope_kernel(MropeArgs a, RopeAxes rope) {
    pdl_trigger();
    pdl_wait();
    const T* x = static_cast<const T*>(a.x);
    T* y = static_cast<T*>(a.y);
    const int turned = rope.pairs / V;
    for (int u = threadIdx.x; u < a.units * a.rows_per_cta; u += blockDim.x) {
        const int sub = u / a.units, w = u - sub * a.units;
        const int64_t row = (int64_t)blockIdx.x * a.rows_per_cta + sub;
        if (row >= a.rows) break;
        const int hg = w / a.chunks, c = w - hg * a.chunks;
        const int h0 = hg * H;
        const T* xr = x + row * a.x_row + (int64_t)h0 * a.x_head;
        T* yr = y + row * a.y_row + (int64_t)h0 * a.y_head;
        if (c >= turned) {  // dims past the rotated ones
            if (x == y) continue;
            const int e = 2 * rope.pairs + (c - turned) * V;
#pragma unroll
            for (int j = 0; j < H; j++)
                if (h0 + j < a.heads)
                    *reinterpret_cast<Vec<T, V>*>(yr + j * a.y_head + e) =
                        *reinterpret_cast<const Vec<T, V>*>(xr + j * a.x_head + e);
            continue;
        }
        const int i0 = c * V;
        Vec<T, V> lo[H], hi[H];
#pragma unroll
        for (int j = 0; j < H; j++)
            if (h0 + j < a.heads) {
                lo[j] = *reinterpret_cast<const Vec<T, V>*>(xr + j * a.x_head + i0);
                hi[j] = *reinterpret_cast<const Vec<T, V>*>(xr + j * a.x_head + rope.pairs + i0);
            }
        float cs[V], sn[V];
        const bool ok = angles<V>(rope, row, 0, i0, cs, sn, a.err);
#pragma unroll
        for (int e = 0; e < V; e++) sn[e] *= a.sign;
        if (!ok) continue;
#pragma unroll
        for (int j = 0; j < H; j++)
            if (h0 + j < a.heads) {
                Vec<T, V> o0, o1;
#pragma unroll
                for (int e = 0; e < V; e++) {
                    const float p = to_f32(lo[j].e[e]), q = to_f32(hi[j].e[e]);
                    from_f32(o0.e[e], __fsub_rn(__fmul_rn(p, cs[e]), __fmul_rn(q, sn[e])));
                    from_f32(o1.e[e], __fadd_rn(__fmul_rn(q, cs[e]), __fmul_rn(p, sn[e])));
                }
                *reinterpret_cast<Vec<T, V>*>(yr + j * a.y_head + i0) = o0;
                *reinterpret_cast<Vec<T, V>*>(yr + j * a.y_head + rope.pairs + i0) = o1;
            }
    }
}

template <typename T, int V, int H>
static int launch_mrope_h(lq_ctx* ctx, MropeArgs a, const RopeAxes& rope) {
    a.chunks = rope.pairs / V + (a.head_dim - 2 * rope.pairs) / V;
    a.units = a.chunks * ceil_div(a.heads, H);
    a.rows_per_cta = std::max(1, 256 / a.units);
    const int threads = std::min(256, (a.units * a.rows_per_cta + 31) / 32 * 32);
    return launch_kernel(ctx, mrope_kernel<T, V, H>, dim3((unsigned)ceil_div(a.rows, a.rows_per_cta)), dim3(threads), 0,
                         "mrope", a, rope);
}

template <typename T, int V>
static int launch_mrope(lq_ctx* ctx, const MropeArgs& a, const RopeAxes& rope) {
    // five heads a thread when that leaves no more threads without one than four do (32768 rows of
    // 40 heads, bf16: 123 us with five, 135 with four; six and eight spill, 180 and 218)
    [[maybe_unused]] const bool five = ceil_div(a.heads, 5) * 5 <= ceil_div(a.heads, 4) * 4;
    if constexpr (V > 1)
        if (five) return launch_mrope_h<T, V, 5>(ctx, a, rope);
    return launch_mrope_h<T, V, 4>(ctx, a, rope);
}

// =========================================================================================
// Append to the paged cache: from projection rows [q heads | k heads | v heads], per-head
// RMSNorm of q and k (when weights are given), rotation, q to q_out, k and v to their slots.
// A warp owns some heads of one row; for head dimensions of 64, 128 and 256 that rotate whole a lane
// holds 8 rotary pairs of a head (both members: 16-byte vectors of either half), D / 16 lanes a
// head, so that a warp works on 4 heads of 128 dims at a time and has IT times as many in flight.
// Bound: HBM for large prompts (16 of up to 2000 f32 rows of 32 + 8 heads: 109 us, 6.1 TB/s); for
// smaller ones instructions (2.1 of 4 a cycle) as much as the latency of loads that depend on one
// another (1860 bf16 rows: 23 us).
// =========================================================================================
template <typename S, typename T, int D, int IT>
__global__ void __launch_bounds__(256, 3) paged_append_kernel(AppendArgs a, RopeAxes rope, PagedSeqs seqs, int groups) {
    pdl_trigger();
    pdl_wait();
    append_heads<S, T, D, IT>(a, rope, seqs, groups, (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5));
}

template <typename S, typename T>
__global__ void __launch_bounds__(256) paged_append_any_kernel(AppendArgs a, RopeAxes rope, PagedSeqs seqs) {
    pdl_trigger();
    pdl_wait();
    append_any_head<S, T>(a, rope, seqs, (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5));
}

template <typename S, typename T, int D>
static int launch_append_d(lq_ctx* ctx, const AppendArgs& a, const RopeAxes& rope, const PagedSeqs& s) {
    const int heads = a.n_heads + 2 * a.n_kv, side = 512 / D;  // heads side by side in a warp
    // many rows: two heads a lane in flight, which share the row's slot and angles; a decode step's
    // few rows: one, so that they spread over the SMs
    constexpr int IT = 2;
    const bool few = (int64_t)s.rows * ceil_div(heads, side) < 16ll * ctx->sm_count;
    const int groups = ceil_div(heads, few ? side : side * IT);
    const dim3 grid((unsigned)ceil_div((int64_t)s.rows * groups, 8));
    if (few) return launch_kernel(ctx, paged_append_kernel<S, T, D, 1>, grid, dim3(256), 0, "paged_append", a, rope, s, groups);
    return launch_kernel(ctx, paged_append_kernel<S, T, D, IT>, grid, dim3(256), 0, "paged_append", a, rope, s, groups);
}

template <typename S, typename T>
static int launch_append(lq_ctx* ctx, const AppendArgs& a, const RopeAxes& rope, const PagedSeqs& s) {
    // the lane-local layout needs whole rotation and 16-byte aligned rows, weights and pages
    const int D = a.head_dim;
    auto al = [](const void* p) { return (uintptr_t)p % 16 == 0; };
    const bool whole = rope.pairs * 2 == D && a.row_stride * sizeof(S) % 16 == 0 && a.q_stride * sizeof(T) % 16 == 0 &&
                       a.page_stride * sizeof(T) % 16 == 0 && al(a.qkv) && al(a.q_out) && al(a.k) && al(a.v) &&
                       al(a.q_norm) && al(a.k_norm);
    if (whole && D == 64) return launch_append_d<S, T, 64>(ctx, a, rope, s);
    if (whole && D == 128) return launch_append_d<S, T, 128>(ctx, a, rope, s);
    if (whole && D == 256) return launch_append_d<S, T, 256>(ctx, a, rope, s);
    const int64_t items = (int64_t)s.rows * (a.n_heads + 2 * a.n_kv);
    return launch_kernel(ctx, paged_append_any_kernel<S, T>, dim3((unsigned)ceil_div(items, 8)), dim3(256), 0,
                         "paged_append_any", a, rope, s);
}

int make_rope_axes(lq_ctx* ctx, const char* who, RopeAxes* r, int64_t rot_dim, int64_t head_dim, const float* cos_dev,
                   const float* sin_dev, int64_t table_len, const uint8_t* axis_host, int64_t n_axes,
                   const int32_t* pos_dev, int64_t pos_stride, int64_t rows) {
    LQ_REQUIRE(ctx, rot_dim >= 0 && rot_dim % 2 == 0 && rot_dim <= head_dim,
               "%s: rot_dim %lld must be even and at most head_dim %lld", who, (long long)rot_dim, (long long)head_dim);
    LQ_REQUIRE(ctx, n_axes >= 1 && n_axes <= ROPE_MAX_AXES, "%s: n_axes %lld outside 1..%d", who, (long long)n_axes,
               ROPE_MAX_AXES);
    LQ_REQUIRE(ctx, rot_dim == 0 || (cos_dev && sin_dev && table_len > 0 && table_len < (1ll << 31)),
               "%s: cos/sin tables missing or empty", who);
    LQ_REQUIRE(ctx, aligned_to(cos_dev, 4) && aligned_to(sin_dev, 4) && aligned_to(pos_dev, 4),
               "%s: tables and positions must be aligned to their elements", who);
    LQ_REQUIRE(ctx, !pos_dev || n_axes == 1 || pos_stride >= rows, "%s: pos_stride %lld < rows %lld", who,
               (long long)pos_stride, (long long)rows);
    r->cos = cos_dev;
    r->sin = sin_dev;
    r->pos = pos_dev;
    r->pos_stride = pos_stride;
    r->pos_base = 0;
    r->table_len = (int)table_len;
    r->pairs = (int)(rot_dim / 2);
    for (int i = 0; i < ROPE_MAX_PAIRS; i++) r->axis[i] = 0;
    if (axis_host)
        for (int i = 0; i < r->pairs; i++) {
            LQ_REQUIRE(ctx, axis_host[i] < n_axes, "%s: pair %d on axis %d of %lld", who, i, (int)axis_host[i],
                       (long long)n_axes);
            r->axis[i] = axis_host[i];
        }
    // runs of pairs on one axis whose table entries are 16-byte aligned vectors
    r->same4 = r->same8 = 0;
    if (r->pairs % 4 == 0 && (uintptr_t)cos_dev % 16 == 0 && (uintptr_t)sin_dev % 16 == 0)
        for (int w = 4; w <= 8; w *= 2)
            for (int c = 0; (c + 1) * w <= r->pairs; c++) {
                bool same = true;
                for (int i = 1; i < w; i++) same = same && r->axis[c * w + i] == r->axis[c * w];
                if (same) (w == 4 ? r->same4 : r->same8) |= 1u << c;
            }
    return LQ_OK;
}

int make_paged_seqs(lq_ctx* ctx, const char* who, PagedSeqs* s, int64_t n_seqs, const int32_t* q_start_dev,
                    const int32_t* kv_len_dev, const int32_t* page_table_dev, int64_t table_ld, int64_t rows,
                    int64_t n_pages, int64_t page_size) {
    LQ_REQUIRE(ctx, n_seqs >= 0 && n_seqs < (1 << 24), "%s: n_seqs %lld out of range", who, (long long)n_seqs);
    LQ_REQUIRE(ctx, rows >= 0 && rows < (1ll << 31), "%s: rows %lld out of range", who, (long long)rows);
    LQ_REQUIRE(ctx, q_start_dev || rows <= n_seqs, "%s: without q_start each sequence has one row (%lld rows, %lld sequences)",
               who, (long long)rows, (long long)n_seqs);
    LQ_REQUIRE(ctx, page_size >= 8 && page_size <= 256 && (page_size & (page_size - 1)) == 0,
               "%s: page_size %lld must be a power of two from 8 to 256", who, (long long)page_size);
    LQ_REQUIRE(ctx, n_pages >= 1 && n_pages < (1ll << 31) / page_size, "%s: n_pages %lld out of range", who,
               (long long)n_pages);
    LQ_REQUIRE(ctx, table_ld >= 0 && table_ld < (1ll << 31) / page_size, "%s: table_ld %lld out of range", who,
               (long long)table_ld);
    LQ_REQUIRE(ctx, n_seqs == 0 || rows == 0 || (kv_len_dev && (page_table_dev || table_ld == 0)),
               "%s: NULL sequence lengths or page table", who);
    LQ_REQUIRE(ctx, aligned_to(q_start_dev, 4) && aligned_to(kv_len_dev, 4) && aligned_to(page_table_dev, 4),
               "%s: lengths and page tables must be aligned to their elements", who);
    s->q_start = q_start_dev;
    s->kv_len = kv_len_dev;
    s->table = page_table_dev;
    s->table_ld = table_ld;
    s->n_seqs = (int)n_seqs;
    s->rows = (int)rows;
    s->n_pages = (int)n_pages;
    s->page_shift = 0;
    while ((1 << s->page_shift) < page_size) s->page_shift++;
    return LQ_OK;
}

}  // namespace lq

extern "C" {

int lq_device_status(lq_ctx* ctx) {
    LQ_ENTRY(ctx, "lq_device_status");
    return lq::consume_device_error(ctx, "lq_device_status");
}

int lq_mrope(lq_ctx* ctx, const void* x, lq_dtype dtype, int64_t rows, int64_t heads, int64_t head_dim,
             int64_t row_stride, int64_t head_stride, void* out, int64_t out_row_stride, int64_t out_head_stride,
             int64_t rot_dim, const float* cos_dev, const float* sin_dev, int64_t table_len,
             const uint8_t* pair_axis_host, int64_t n_axes, const int32_t* pos_dev, int64_t pos_stride, int inverse) {
    LQ_ENTRY(ctx, "lq_mrope");
    LQ_REQUIRE(ctx, dtype == LQ_DTYPE_F32 || dtype == LQ_DTYPE_BF16, "lq_mrope: dtype must be F32 or BF16");
    LQ_REQUIRE(ctx, rows >= 0 && rows < (1ll << 31), "lq_mrope: rows %lld out of range", (long long)rows);
    LQ_REQUIRE(ctx, heads >= 1 && heads <= (1 << 16), "lq_mrope: heads %lld out of range", (long long)heads);
    LQ_REQUIRE(ctx, head_dim >= 2 && head_dim <= 256 && head_dim % 2 == 0,
               "lq_mrope: head_dim %lld must be even and at most 256", (long long)head_dim);
    LQ_REQUIRE(ctx, row_stride >= 0 && out_row_stride >= 0 && head_stride >= 0 && out_head_stride >= 0,
               "lq_mrope: negative stride");
    // the output's rows and heads: the ones that lie closer follow each other without overlap, and
    // all of them fit between two of the others
    const bool by_row = rows > 1 && (heads == 1 || out_row_stride < out_head_stride);
    const int64_t near = by_row ? out_row_stride : out_head_stride, n_near = by_row ? rows : heads;
    const int64_t apart = by_row ? out_head_stride : out_row_stride, n_apart = by_row ? heads : rows;
    LQ_REQUIRE(ctx, (n_near <= 1 || near >= head_dim) && (n_apart <= 1 || (apart - head_dim) / std::max<int64_t>(1, near) >= n_near - 1),
               "lq_mrope: output heads overlap");
    LQ_REQUIRE(ctx, x != out || (row_stride == out_row_stride && head_stride == out_head_stride),
               "lq_mrope: in place needs equal strides");
    lq::RopeAxes rope;
    int rc = lq::make_rope_axes(ctx, "lq_mrope", &rope, rot_dim, head_dim, cos_dev, sin_dev, table_len, pair_axis_host,
                                n_axes, pos_dev, pos_stride, rows);
    if (rc) return rc;
    if (rows == 0) return LQ_OK;
    LQ_REQUIRE(ctx, x && out && (pos_dev || rot_dim == 0), "lq_mrope: NULL pointer");
    const size_t size = dtype == LQ_DTYPE_F32 ? 4 : 2;
    LQ_REQUIRE(ctx, lq::aligned_to(x, size) && lq::aligned_to(out, size), "lq_mrope: x and out must be aligned to their elements");
    lq::MropeArgs a;
    a.x = x;
    a.y = out;
    a.x_row = row_stride;
    a.x_head = head_stride;
    a.y_row = out_row_stride;
    a.y_head = out_head_stride;
    a.rows = rows;
    a.heads = (int)heads;
    a.head_dim = (int)head_dim;
    a.sign = inverse ? -1.0f : 1.0f;
    a.err = ctx->err_flag;
    // the widest vector (16 bytes, else one element) that divides the pairs, the copied dims,
    // the strides and the addresses
    const bool f32 = dtype == LQ_DTYPE_F32;
    const int64_t v = f32 ? 4 : 8;
    const bool wide = rope.pairs % v == 0 && head_dim % v == 0 && row_stride % v == 0 && head_stride % v == 0 &&
                      out_row_stride % v == 0 && out_head_stride % v == 0 && (uintptr_t)x % 16 == 0 &&
                      (uintptr_t)out % 16 == 0;
    if (f32) return wide ? lq::launch_mrope<float, 4>(ctx, a, rope) : lq::launch_mrope<float, 1>(ctx, a, rope);
    return wide ? lq::launch_mrope<__nv_bfloat16, 8>(ctx, a, rope) : lq::launch_mrope<__nv_bfloat16, 1>(ctx, a, rope);
}

int lq_paged_append(lq_ctx* ctx, const void* qkv, lq_dtype qkv_dtype, int64_t row_stride, int64_t rows, int64_t n_heads,
                    int64_t n_kv_heads, int64_t head_dim, const uint16_t* q_norm, const uint16_t* k_norm, float eps,
                    int norm_bf16, int64_t rot_dim, const float* cos_dev, const float* sin_dev, int64_t table_len,
                    const uint8_t* pair_axis_host, int64_t n_axes, const int32_t* pos_dev, int64_t pos_stride,
                    int64_t pos_base, int64_t n_seqs, const int32_t* q_start, const int32_t* kv_len,
                    const int32_t* page_table, int64_t table_ld, void* k_pages, void* v_pages, lq_dtype kv_dtype,
                    int64_t n_pages, int64_t page_size, int64_t page_stride, void* q_out, int64_t q_stride) {
    LQ_ENTRY(ctx, "lq_paged_append");
    LQ_REQUIRE(ctx, qkv_dtype == LQ_DTYPE_F32 || qkv_dtype == LQ_DTYPE_BF16, "lq_paged_append: rows must be F32 or BF16");
    LQ_REQUIRE(ctx, kv_dtype == LQ_DTYPE_F32 || kv_dtype == LQ_DTYPE_BF16, "lq_paged_append: cache must be F32 or BF16");
    LQ_REQUIRE(ctx, n_heads >= 0 && n_kv_heads >= 1 && n_heads + 2 * n_kv_heads <= (1 << 16),
               "lq_paged_append: bad head counts");
    LQ_REQUIRE(ctx, head_dim >= 2 && head_dim <= 256 && head_dim % 2 == 0,
               "lq_paged_append: head_dim %lld must be even and at most 256", (long long)head_dim);
    if (row_stride == 0) row_stride = (n_heads + 2 * n_kv_heads) * head_dim;
    if (page_stride == 0) page_stride = n_kv_heads * page_size * head_dim;
    if (q_stride == 0) q_stride = n_heads * head_dim;
    LQ_REQUIRE(ctx, row_stride >= (n_heads + 2 * n_kv_heads) * head_dim, "lq_paged_append: row_stride too small");
    LQ_REQUIRE(ctx, q_stride >= n_heads * head_dim, "lq_paged_append: q_stride too small");
    lq::RopeAxes rope;
    lq::PagedSeqs s;
    int rc = lq::make_rope_axes(ctx, "lq_paged_append", &rope, rot_dim, head_dim, cos_dev, sin_dev, table_len,
                                pair_axis_host, n_axes, pos_dev, pos_stride, rows);
    if (rc) return rc;
    rope.pos_base = pos_base;
    rc = lq::make_paged_seqs(ctx, "lq_paged_append", &s, n_seqs, q_start, kv_len, page_table, table_ld, rows, n_pages,
                             page_size);
    if (rc) return rc;
    LQ_REQUIRE(ctx, page_stride >= n_kv_heads * page_size * head_dim, "lq_paged_append: page_stride too small");
    LQ_REQUIRE(ctx, rows * (n_heads + 2 * n_kv_heads) < (1ll << 33), "lq_paged_append: too many rows");
    if (rows == 0 || n_seqs == 0) return LQ_OK;
    LQ_REQUIRE(ctx, qkv && k_pages && v_pages && (q_out || n_heads == 0), "lq_paged_append: NULL pointer");
    const size_t src_size = qkv_dtype == LQ_DTYPE_F32 ? 4 : 2, size = kv_dtype == LQ_DTYPE_F32 ? 4 : 2;
    LQ_REQUIRE(ctx, lq::aligned_to(qkv, src_size) && lq::aligned_to(k_pages, size) && lq::aligned_to(v_pages, size) &&
                        lq::aligned_to(q_out, size) && lq::aligned_to(q_norm, 2) && lq::aligned_to(k_norm, 2),
               "lq_paged_append: pointers must be aligned to their elements");
    lq::AppendArgs a;
    a.qkv = qkv;
    a.row_stride = row_stride;
    a.n_heads = (int)n_heads;
    a.n_kv = (int)n_kv_heads;
    a.head_dim = (int)head_dim;
    a.q_norm = q_norm;
    a.k_norm = k_norm;
    a.eps = eps;
    a.norm_bf16 = norm_bf16;
    a.k = k_pages;
    a.v = v_pages;
    a.page_stride = page_stride;
    a.q_out = q_out;
    a.q_stride = q_stride;
    a.err = ctx->err_flag;
    const bool sf = qkv_dtype == LQ_DTYPE_F32, tf = kv_dtype == LQ_DTYPE_F32;
    if (sf && tf) return lq::launch_append<float, float>(ctx, a, rope, s);
    if (sf) return lq::launch_append<float, __nv_bfloat16>(ctx, a, rope, s);
    if (tf) return lq::launch_append<__nv_bfloat16, float>(ctx, a, rope, s);
    return lq::launch_append<__nv_bfloat16, __nv_bfloat16>(ctx, a, rope, s);
}

}  // extern "C"
