// lq8_prefix_attn.cu -- attention over a paged K/V cache for a batch whose sequences share a
// prefix: o_r = sum_j exp(scale q_r.k_j - m) v_j / sum_j exp(scale q_r.k_j - m) over the prefix
// positions and over the row's own positions up to itself.
#include "lq8_async.cuh"
#include "lq8_fused.cuh"
#include "lq8_paged.cuh"

#include <algorithm>

namespace lq {

struct PrefixAttnArgs {
    const void* q;
    int64_t q_stride;
    int n_heads, n_kv;
    float scale;
    const void* k;
    const void* v;
    int64_t page_stride;
    const int32_t* prefix_table;
    int prefix_len, max_q, max_kv;
    void* out;
    int64_t out_stride;
    int8_t* xq;
    uint16_t* xd;
    int* err;
};

// own positions that row r sees, in its sequence b; flags lengths the call's bounds do not hold
__device__ __forceinline__ int visible_own(const PrefixAttnArgs& a, const PagedSeqs& s, int b, int r) {
    const int q0 = s.q_start ? s.q_start[b] : b, q1 = s.q_start ? s.q_start[b + 1] : b + 1;
    int kv = s.kv_len[b];
    const int64_t most = min((int64_t)a.max_kv, s.table_ld << s.page_shift);
    if (kv < 0 || kv > most) {
        flag_error(a.err, ERR_KV_LEN, kv);
        kv = kv < 0 ? 0 : (int)most;
    }
    if (q1 - q0 > a.max_q || q1 > s.rows) flag_error(a.err, ERR_ROW_COUNT, q1 - q0);
    return min(kv, max(0, kv - (q1 - r) + 1));
}

template <typename T>
__device__ __forceinline__ float elem(const void* p, int64_t i);
template <>
__device__ __forceinline__ float elem<float>(const void* p, int64_t i) { return static_cast<const float*>(p)[i]; }
template <>
__device__ __forceinline__ float elem<__nv_bfloat16>(const void* p, int64_t i) {
    return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}

// One CTA of 128 threads per (row, query head): 128 positions at a time, a thread a score, then a
// thread a dim, with the running maximum and sum.
template <typename T, int D>
__global__ void __launch_bounds__(128) prefix_attn_row_kernel(PrefixAttnArgs a, PagedSeqs s) {
    __shared__ float q[D], p[128], red[4];
    __shared__ int64_t base[128];
    pdl_trigger();
    pdl_wait();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int row = blockIdx.x, h = blockIdx.y, kh = h / (a.n_heads / a.n_kv);
    int b = row;
    if (s.q_start) b = seq_of_row(s.q_start, s.n_seqs, row, lane);
    if (b >= s.n_seqs) return;
    const int own = visible_own(a, s, b, row), total = a.prefix_len + own;
    if (tid < D) q[tid] = elem<T>(a.q, (int64_t)row * a.q_stride + (int64_t)h * D + tid) * a.scale;
    float m = -INFINITY, l = 0.0f, o = 0.0f;
    const int mask = (1 << s.page_shift) - 1;
    for (int t0 = 0; t0 < total; t0 += 128) {
        __syncthreads();
        const int t = t0 + tid;
        float sc = -INFINITY;
        int64_t at = -1;
        if (t < total) {
            const int u = t < a.prefix_len ? t : t - a.prefix_len;
            const int pg = t < a.prefix_len ? a.prefix_table[u >> s.page_shift]
                                            : s.table[(int64_t)b * s.table_ld + (u >> s.page_shift)];
            if (pg < 0 || pg >= s.n_pages) {
                flag_error(a.err, ERR_PAGE_ID, pg);
            } else {
                at = pg * a.page_stride + (((int64_t)kh << s.page_shift) + (u & mask)) * D;
                sc = 0.0f;
                for (int d = 0; d < D; d++) sc = fmaf(q[d], elem<T>(a.k, at + d), sc);
            }
        }
        base[tid] = at;
        float mx = warp_max(sc);
        if (lane == 0) red[warp] = mx;
        __syncthreads();
        const float m_new = fmaxf(fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])), m);
        const float ref = m_new == -INFINITY ? 0.0f : m_new;
        const float e = expf(sc - ref), f = expf(m - ref);
        p[tid] = e;
        const float sum = warp_sum(e);
        __syncthreads();
        if (lane == 0) red[warp] = sum;
        __syncthreads();
        l = l * f + (red[0] + red[1] + red[2] + red[3]);
        m = m_new;
        if (tid < D) {
            o *= f;
            for (int i = 0; i < 128; i++)
                if (base[i] >= 0) o = fmaf(p[i], elem<T>(a.v, base[i] + tid), o);
        }
    }
    const float y = l > 0.0f ? o / l : 0.0f;
    if (tid < D && a.out) {
        const int64_t at = (int64_t)row * a.out_stride + (int64_t)h * D + tid;
        if constexpr (sizeof(T) == 4) static_cast<float*>(a.out)[at] = y;
        else static_cast<__nv_bfloat16*>(a.out)[at] = __float2bfloat16_rn(y);
    }
    if (a.xq) {
        float amax = warp_max(fabsf(y)), d, id;
        q8_scale(amax, d, id);
        const int64_t blk = ((int64_t)row * a.n_heads + h) * (D / 32) + warp;
        if (warp < D / 32) {
            if (lane == 0) a.xd[blk] = f2h(d);
            a.xq[blk * 32 + lane] = (int8_t)q8_quant(y, id);
        }
    }
}

}  // namespace lq

extern "C" int lq_prefix_attention(lq_ctx* ctx, const void* q, lq_dtype dtype, int64_t q_stride, int64_t rows,
                                   int64_t n_heads, int64_t n_kv_heads, int64_t head_dim, float scale,
                                   const void* k_pages, const void* v_pages, int64_t n_pages, int64_t page_size,
                                   int64_t page_stride, const int32_t* prefix_table, int64_t prefix_len, int64_t n_seqs,
                                   const int32_t* q_start, const int32_t* kv_len, const int32_t* page_table,
                                   int64_t table_ld, int64_t max_q, int64_t max_kv, void* out, int64_t out_stride,
                                   int8_t* xq, uint16_t* xd) {
    LQ_ENTRY(ctx, "lq_prefix_attention");
    LQ_REQUIRE(ctx, dtype == LQ_DTYPE_F32 || dtype == LQ_DTYPE_BF16, "lq_prefix_attention: dtype must be F32 or BF16");
    LQ_REQUIRE(ctx, n_heads >= 1 && n_kv_heads >= 1 && n_heads % n_kv_heads == 0 && n_heads <= 4096,
               "lq_prefix_attention: bad head counts");
    LQ_REQUIRE(ctx, n_heads / n_kv_heads <= 128, "lq_prefix_attention: more than 128 query heads a kv head");
    LQ_REQUIRE(ctx, head_dim == 64 || head_dim == 128, "lq_prefix_attention: head_dim %lld must be 64 or 128",
               (long long)head_dim);
    lq::PagedSeqs s;
    int rc = lq::make_paged_seqs(ctx, "lq_prefix_attention", &s, n_seqs, q_start, kv_len, page_table, table_ld, rows,
                                 n_pages, page_size);
    if (rc) return rc;
    if (page_stride == 0) page_stride = n_kv_heads * page_size * head_dim;
    if (q_stride == 0) q_stride = n_heads * head_dim;
    if (out_stride == 0) out_stride = n_heads * head_dim;
    LQ_REQUIRE(ctx, page_stride >= n_kv_heads * page_size * head_dim, "lq_prefix_attention: page_stride too small");
    LQ_REQUIRE(ctx, q_stride >= n_heads * head_dim && out_stride >= n_heads * head_dim,
               "lq_prefix_attention: row stride too small");
    LQ_REQUIRE(ctx, prefix_len >= 0 && prefix_len < (1ll << 30) && (prefix_len == 0 || prefix_table),
               "lq_prefix_attention: bad prefix");
    LQ_REQUIRE(ctx, max_q >= 1 && max_q < (1ll << 24) && max_kv >= 0 && max_kv < (1ll << 30),
               "lq_prefix_attention: bad bounds max_q %lld, max_kv %lld", (long long)max_q, (long long)max_kv);
    LQ_REQUIRE(ctx, (xq == nullptr) == (xd == nullptr), "lq_prefix_attention: xq and xd go together");
    LQ_REQUIRE(ctx, rows * n_heads < (1ll << 31) / 4, "lq_prefix_attention: too many rows");
    if (rows == 0 || n_seqs == 0) return LQ_OK;
    LQ_REQUIRE(ctx, q && k_pages && v_pages && (out || xq), "lq_prefix_attention: NULL pointer");
    const size_t esize = dtype == LQ_DTYPE_F32 ? 4 : 2;
    auto al = [](const void* p) { return (uintptr_t)p % 16 == 0; };
    LQ_REQUIRE(ctx, al(q) && al(k_pages) && al(v_pages) && al(out) && q_stride * esize % 16 == 0 &&
                        out_stride * esize % 16 == 0 && page_stride * esize % 16 == 0,
               "lq_prefix_attention: pointers and strides must be multiples of 16 bytes");
    lq::PrefixAttnArgs a;
    a.q = q;
    a.q_stride = q_stride;
    a.n_heads = (int)n_heads;
    a.n_kv = (int)n_kv_heads;
    a.scale = scale;
    a.k = k_pages;
    a.v = v_pages;
    a.page_stride = page_stride;
    a.prefix_table = prefix_table;
    a.prefix_len = (int)prefix_len;
    a.max_q = (int)max_q;
    a.max_kv = (int)max_kv;
    a.out = out;
    a.out_stride = out_stride;
    a.xq = xq;
    a.xd = xd;
    a.err = ctx->err_flag;
    const dim3 grid((unsigned)rows, (unsigned)n_heads);
    auto run = [&](auto kern) { return lq::launch_kernel(ctx, kern, grid, dim3(128), 0, "prefix_attn_row", a, s); };
    if (dtype == LQ_DTYPE_F32)
        return head_dim == 64 ? run(lq::prefix_attn_row_kernel<float, 64>) : run(lq::prefix_attn_row_kernel<float, 128>);
    return head_dim == 64 ? run(lq::prefix_attn_row_kernel<__nv_bfloat16, 64>)
                          : run(lq::prefix_attn_row_kernel<__nv_bfloat16, 128>);
}
