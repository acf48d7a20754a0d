// lq8_prefix_attn.cu -- attention over a paged K/V cache for a batch whose sequences share a
// prefix: o_r = sum_j exp(scale q_r.k_j - m) v_j / sum_j exp(scale q_r.k_j - m) over the prefix
// positions and over the row's own positions up to itself.
#include "lq8_async.cuh"
#include "lq8_fused.cuh"
#include "lq8_prefix_attn.cuh"
#include "lq8_prefix_plan.cuh"

#include <algorithm>

namespace lq {

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

// =========================================================================================
// Merge: a warp per (row, head) joins the partials of the workers that had a piece of the row's
// prefix item or own item, in the order of the line: with M the largest of their maxima,
// o = sum 2^(m_i - M) o_i / sum 2^(m_i - M) l_i. A lane looks after one partial's m and l, then
// the warp adds up the vectors, four dims a lane. Rows that a worker had whole are written there.
// =========================================================================================
template <typename T, int D>
__global__ void __launch_bounds__(256) prefix_attn_merge_kernel(PrefixAttnArgs a, PagedSeqs s, PrefixPlan p) {
    pdl_trigger();
    pdl_wait();
    const int lane = threadIdx.x & 31;
    const int idx = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
    const int t = idx / a.n_heads, h = idx - t * a.n_heads;
    if (t >= s.rows) return;
    const int b = s.q_start ? seq_of_row(s.q_start, s.n_seqs, t, lane) : t;
    if (b >= s.n_seqs) return;
    const SeqInfo si = seq_info(a, s, b, false);
    const int kh = h / a.group, gq = h - kh * a.group;
    const OwnSteps os{a, p};
    const Line line(p, p.cum[s.n_seqs]);
    // this row's prefix item and own item: steps [s0, s1), first virtual worker, count, slot, row
    int v0[2] = {0, 0}, cnt[2] = {0, 0}, s0[2], s1[2], item[2], in[2];
    if (p.np > 0) {
        const int r = t * a.group + gq, rb = r / p.pb;
        item[0] = kh * p.n_rb + rb;
        in[0] = r - rb * p.pb;
        s0[0] = item[0] * p.np;
        s1[0] = s0[0] + p.np;
    } else {
        s0[0] = s1[0] = 0;
    }
    s0[1] = s1[1] = 0;
    if (t < si.q0 + si.q) {
        const int r = (t - si.q0) * a.group + gq, rb = r / p.ob, nb = os.blocks(si);
        int before = 0, per = 0;
        for (int i = lane; i < nb; i += 32) {
            const int n = os.tiles(si, i);
            per += n;
            if (i < rb) before += n;
        }
        before = __reduce_add_sync(0xffffffffu, before);
        per = __reduce_add_sync(0xffffffffu, per);
        item[1] = a.n_kv * os.base(si, b) + kh * nb + rb;
        in[1] = r - rb * p.ob;
        s0[1] = p.cum[b] + kh * per + before;
        s1[1] = s0[1] + os.tiles(si, rb);
    }
#pragma unroll
    for (int part = 0; part < 2; part++) {
        if (s0[part] == s1[part]) continue;
        const bool paired = part ? p.pair_o : p.pair_p;
        int w[2];
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const int step = e ? s1[part] - 1 : s0[part];
            w[e] = line.owner(step, part);
            if (!paired) {
                int lo, hi;
                flow_range(line, p, w[e], 0, part, lo, hi);
                w[e] = 2 * w[e] + (step >= hi);
            }
        }
        v0[part] = w[0];
        cnt[part] = w[1] - w[0] + 1;
    }
    if (p.np == 0 && cnt[1] == 1) return;  // written by its only worker
    const int n = cnt[0] + cnt[1];
    float m_i = -INFINITY, l_i = 0.0f;
    int64_t at_i = -1;
    auto look = [&](int i) {  // partial i: its slot row (-1: the worker had no step of the item), m, l
        m_i = -INFINITY;
        l_i = 0.0f;
        at_i = -1;
        if (i >= n) return;
        const int part = i >= cnt[0], v = v0[part] + i - (part ? cnt[0] : 0);
        const bool paired = part ? p.pair_o : p.pair_p;
        int lo, hi;
        flow_range(line, p, paired ? v : v >> 1, paired ? 0 : v & 1, part, lo, hi);
        if (max(lo, s0[part]) >= min(hi, s1[part])) return;
        at_i = (int64_t)(item[part] + v) * (part ? p.cap_o : p.cap_p) + in[part];
        const float2 ml = (part ? p.ml_o : p.ml_p)[at_i];
        m_i = ml.x;
        l_i = ml.y;
    };
    look(lane);
    float M = warp_max(m_i);
    for (int i0 = 32; i0 < n; i0 += 32) {
        look(i0 + lane);
        M = fmaxf(M, warp_max(m_i));
    }
    float L = 0.0f, o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    const bool on = 4 * lane < D;
    for (int i0 = 0; i0 < n; i0 += 32) {
        if (n > 32) look(i0 + lane);
        const float w_i = m_i == -INFINITY ? 0.0f : exp2f(m_i - M);
        L += warp_sum(w_i * l_i);
        const int k = min(32, n - i0);
#pragma unroll 4
        for (int j = 0; j < k; j++) {
            const int64_t at = __shfl_sync(0xffffffffu, at_i, j);
            const float w = __shfl_sync(0xffffffffu, w_i, j);
            if (at >= 0 && on) {
                const float4 x = *reinterpret_cast<const float4*>((i0 + j >= cnt[0] ? p.o_o : p.o_p) + at * D + 4 * lane);
                o[0] = fmaf(w, x.x, o[0]);
                o[1] = fmaf(w, x.y, o[1]);
                o[2] = fmaf(w, x.z, o[2]);
                o[3] = fmaf(w, x.w, o[3]);
            }
        }
    }
    const float inv = L > 0.0f ? 1.0f / L : L;  // a row that saw nothing: zeros; NaN stays
#pragma unroll
    for (int j = 0; j < 4; j++) o[j] *= inv;
    const int64_t col = (int64_t)h * D + 4 * lane;
    if (a.out && on) {
        T* const y = static_cast<T*>(a.out) + (int64_t)t * a.out_stride + col;
        if constexpr (sizeof(T) == 4) *reinterpret_cast<float4*>(y) = make_float4(o[0], o[1], o[2], o[3]);
        else *reinterpret_cast<uint2*>(y) = make_uint2(pack_bf16x2(o[0], o[1]), pack_bf16x2(o[2], o[3]));
    }
    if (a.xq) {
        const int64_t e = (int64_t)t * a.n_heads * D + col;
        const uint32_t q = quant_group8(o, lane & 7, on ? a.xd + (e >> 5) : nullptr);
        if (on) *reinterpret_cast<uint32_t*>(a.xq + e) = q;
    }
}

// The plan of a call for workers of `halves` x `half` stacked rows and `tile` positions, and its
// workspace. Sizes come from the call's bounds; what the lengths really are, the kernels read.
static int make_plan(lq_ctx* ctx, const PrefixAttnArgs& a, const PagedSeqs& s, int half, int tile, int D, PrefixPlan* p) {
    const int64_t R = (int64_t)s.rows * a.group, most_q = std::min<int64_t>((int64_t)a.max_q, s.rows) * a.group;
    p->tile = tile;
    p->pair_p = R > half;
    p->pb = p->pair_p ? 2 * half : half;
    p->pair_o = most_q > half;
    p->ob = p->pair_o ? 2 * half : half;
    p->cap_p = (int)std::min<int64_t>(p->pb, R);
    p->cap_o = (int)std::min<int64_t>(p->ob, most_q);
    p->n_rb = ceil_div(R, p->pb);
    p->np = ceil_div(a.prefix_len, tile);
    const int64_t items_p = (int64_t)a.n_kv * p->n_rb, items_o = a.n_kv * (R / p->ob + s.n_seqs + 1);
    const int64_t steps = items_p * p->np + items_o * ceil_div(a.max_kv, tile);
    LQ_REQUIRE(ctx, steps < (1ll << 26), "lq_prefix_attention: %lld steps, more than a launch can number", (long long)steps);
    p->sp = (int)(items_p * p->np);
    p->workers = (int)std::max<int64_t>(1, std::min<int64_t>(ctx->sm_count, steps));
    p->workers_mul = ((1ull << 40) + p->workers - 1) / p->workers;
    const int64_t slots_p = p->np ? items_p + 2 * p->workers : 0, slots_o = items_o + 2 * p->workers;
    auto al = [](size_t b) { return (b + 255) & ~(size_t)255; };
    const size_t cum = al((size_t)(s.n_seqs + 1) * 4), ml_p = al((size_t)slots_p * p->cap_p * 8),
                 ml_o = al((size_t)slots_o * p->cap_o * 8), o_p = al((size_t)slots_p * p->cap_p * D * 4),
                 o_o = al((size_t)slots_o * p->cap_o * D * 4);
    const int rc = ensure_paged(ctx, cum + ml_p + ml_o + o_p + o_o);
    if (rc) return rc;
    uint8_t* w = static_cast<uint8_t*>(ctx->paged);
    p->cum = reinterpret_cast<int32_t*>(w);
    p->ml_p = reinterpret_cast<float2*>(w += cum);
    p->ml_o = reinterpret_cast<float2*>(w += ml_p);
    p->o_p = reinterpret_cast<float*>(w += ml_o);
    p->o_o = reinterpret_cast<float*>(w += o_p);
    return LQ_OK;
}

template <typename T, int D>
static int launch_merge(lq_ctx* ctx, const PrefixAttnArgs& a, const PagedSeqs& s, const PrefixPlan& p) {
    return launch_kernel(ctx, prefix_attn_merge_kernel<T, D>, dim3((unsigned)ceil_div((int64_t)s.rows * a.n_heads, 8)),
                         dim3(256), 0, "prefix_attn_merge", a, s, p);
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
    LQ_REQUIRE(ctx, scale > 0.0f && scale < INFINITY, "lq_prefix_attention: scale must be positive and finite");
    LQ_REQUIRE(ctx, (xq == nullptr) == (xd == nullptr), "lq_prefix_attention: xq and xd go together");
    LQ_REQUIRE(ctx, rows * n_heads < (1ll << 28), "lq_prefix_attention: too many rows");
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
    a.group = (int)(n_heads / n_kv_heads);
    a.group_mul = ((1ull << 36) + a.group - 1) / a.group;
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
    if (dtype == LQ_DTYPE_BF16) {
        lq::PrefixPlan p;
        if ((rc = lq::make_plan(ctx, a, s, 128, 128, (int)head_dim, &p))) return rc;
        if ((rc = lq::launch_prefix_attn_tc(ctx, a, s, p, (int)head_dim))) return rc;
        return head_dim == 64 ? lq::launch_merge<__nv_bfloat16, 64>(ctx, a, s, p)
                              : lq::launch_merge<__nv_bfloat16, 128>(ctx, a, s, p);
    }
    const dim3 grid((unsigned)rows, (unsigned)n_heads);
    auto run = [&](auto kern) { return lq::launch_kernel(ctx, kern, grid, dim3(128), 0, "prefix_attn_row", a, s); };
    return head_dim == 64 ? run(lq::prefix_attn_row_kernel<float, 64>) : run(lq::prefix_attn_row_kernel<float, 128>);
}
