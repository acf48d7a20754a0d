// lq8_prefix_attn.cu -- attention over a paged K/V cache for a batch whose sequences share a
// prefix: o_r = sum_j exp(scale q_r.k_j - m) v_j / sum_j exp(scale q_r.k_j - m) over the prefix
// positions and over the row's own positions up to itself.
#include "lq8_async.cuh"
#include "lq8_fused.cuh"
#include "lq8_prefix_attn.cuh"
#include "lq8_prefix_plan.cuh"

#include <algorithm>

namespace lq {

// =========================================================================================
// Merge: joins the partials of the workers that had a piece of a row's prefix item or own item, in
// the order of the line: with M the largest of their maxima, o = sum 2^(m_i - M) o_i /
// sum 2^(m_i - M) l_i. A CTA takes up to MR rows of an own item (a sequence's row block and kv
// head), which share the own item's partials and, but for a block's end, those of a prefix item.
// Without prefix items only the items that are cut between workers are left: a worker leaves a note of
// the one that it begins. A thread adds up CH MR / 256 vectors of four dims of one row; rows lie
// next to each other in memory. Bound: latency (launch, lengths, maxima, vectors): 10 us for 64
// sequences, 16 us for 128 behind 32768 positions (9 MB of partials).
// =========================================================================================
constexpr int MERGE_CHUNK = 32;   // partials looked at together

// whose partials: of kernels whose CTAs have flows, of the streaming kernel, or the prefix's of the former and the own
// items' of the latter
enum { MERGE_FLOWS, MERGE_STREAM, MERGE_APART };

template <typename T, int D, int MR, int KIND>
__global__ void __launch_bounds__(256, MR == 32 ? 5 : 4)
prefix_attn_merge_kernel(const __grid_constant__ PrefixAttnArgs a, const __grid_constant__ PagedSeqs s,
                         const __grid_constant__ PrefixPlan p, const __grid_constant__ PrefixPlan prefix_plan) {
    const PrefixPlan& pp = KIND == MERGE_APART ? prefix_plan : p;
    constexpr int CH = D / 4, SUBS = 256 / MR;  // vectors of a row; threads that share a row
    constexpr int VEC = (CH + SUBS - 1) / SUBS, BATCH = VEC == 1 ? 8 : 1;  // partials whose loads go out together
    __shared__ int slot[MERGE_CHUNK];
    __shared__ float weight[MERGE_CHUNK][MR];
    __shared__ float2 red[8][MR];
    __shared__ __align__(16) float stage[MR][D + 4];
    const int tid = threadIdx.x, lane = tid & 31, r = tid % MR, sub = tid / MR;
    const OwnSteps os{a, p};
    const bool with_prefix = p.np > 0;
    // the item, its rows st0 .. st0 + todo - 1 of this CTA, the first one's place in the item
    int st0 = 0, todo = 0, kh = 0, own_item = 0, own_in = blockIdx.y * MR;
    bool own = true;
    if (with_prefix) {  // (the call's inputs: complete before the kernel that this one waits for began)
        const int x = blockIdx.x / a.n_kv;
        kh = blockIdx.x - x * a.n_kv;
        // the last sequence with base(b) <= x
        int lo = 0, n = s.n_seqs - 1;
        while (n > 0) {
            const int step = (n + 31) >> 5, i = lo + min(n, (lane + 1) * step);
            const int q0 = s.q_start ? s.q_start[i] : i;
            const int c = __popc(__ballot_sync(0xffffffffu, q0 * a.group / p.ob + i <= x));
            if (c == 32) {
                lo += n;
                break;
            }
            const int skip = min(n, c * step);
            n = min(step - 1, n - skip);
            lo += skip;
        }
        const SeqInfo si = seq_info(a, s, lo, false);
        const int rb = x - os.base(si, lo), nb = os.blocks(si);
        if (rb < 0 || rb >= nb) {
            // (one CTA at least waits, so that this kernel does not end, and the next one does not begin on the
            // workspace, before the attention is through: with padding rows alone all of them leave here)
            if (blockIdx.x == 0 && blockIdx.y == 0) pdl_wait();
            return;
        }
        st0 = si.q0 * a.group + rb * p.ob + own_in;
        todo = min(MR, min(p.ob, si.q * a.group - rb * p.ob) - own_in);
        own_item = a.n_kv * x + kh * nb + rb - a.n_kv * rb;  // n_kv base + kh nb + rb
        own = os.visible(si, rb) > 0;
    }
    pdl_wait();
    pdl_trigger();
    const int own_steps = *p.own_steps;
    // whether a worker between an item's first and last one has a step of it
    auto works = [&](int part, int v) {
        int lo, hi;
        if (part ? KIND != MERGE_FLOWS : KIND == MERGE_STREAM) {
            Shares(p, own_steps).range(v, part, lo, hi);
        } else {
            const Line line(pp, KIND == MERGE_FLOWS ? own_steps : 0, pp.pair_p, pp.pair_o);
            const bool paired = part ? pp.pair_o : pp.pair_p;
            flow_range(line, paired, paired ? v : v >> 1, paired ? 0 : v & 1, part, lo, hi);
        }
        return lo < hi;
    };
    if (!with_prefix) {
        const SplitItem w = p.split[blockIdx.x];
        st0 = w.row0 + own_in;
        todo = min(MR, w.rows - own_in);
        kh = w.kh;
        own_item = w.item;
    }
#pragma unroll 1
    while (todo > 0) {
        int run = todo, item[2] = {0, own_item}, in[2] = {0, own_in}, v0[2] = {0, 0}, cnt[2] = {0, 0};
        auto workers_of = [&](int k) {  // (within bounds, even where a kernel that gave up left them unwritten)
            const int most = (k ? p : pp).ranges - 1;
            v0[k] = min(max(p.first[k][item[k]], 0), most);
            cnt[k] = min(max(p.last[k][item[k]], 0), most) - v0[k] + 1;
        };
        if (with_prefix) {  // rows that share the prefix item
            const int rb = st0 / pp.pb;
            item[0] = kh * pp.n_rb + rb;
            in[0] = st0 - rb * pp.pb;
            run = min(run, pp.pb - in[0]);
            workers_of(0);
        }
        if (own) workers_of(1);
        const int n = cnt[0] + cnt[1];
        const bool mine = r < run;
        // pass 0: the rows' maxima and sums; pass 1: the vectors
        float M = -INFINITY, L = 0.0f;
        float4 o[VEC];
#pragma unroll
        for (int k = 0; k < VEC; k++) o[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 1
        for (int pass = 0; pass < 2; pass++) {
#pragma unroll 1
            for (int c0 = 0; c0 < n; c0 += MERGE_CHUNK) {
                const int m = min(MERGE_CHUNK, n - c0);
                if (pass == 0 || n > MERGE_CHUNK) {
                    __syncthreads();  // (the last chunk's slots and weights are read no more)
                    if (tid < m) {
                        const int i = c0 + tid, part = i >= cnt[0], k = i - (part ? cnt[0] : 0), v = v0[part] + k;
                        bool has = k == 0 || k == cnt[part] - 1;
                        if (!has) has = works(part, v);  // a worker in between may have no step at all
                        slot[tid] = !has ? -1 : part ? p.own_slot(item[1], v, k == 0) : item[0] + v;
                    } else if (tid < MERGE_CHUNK) {
                        slot[tid] = -1;
                    }
                    __syncthreads();
                }
                // a thread's share of the row's partials: (m, l) in pass 0, weights in pass 1
                for (int i = sub; i < m; i += SUBS) {
                    const int part = c0 + i >= cnt[0];
                    float2 ml = make_float2(-INFINITY, 0.0f);
                    if (mine && slot[i] >= 0) ml = p.ml[part][(int64_t)slot[i] * p.cap[part] + in[part] + r];
                    // (a maximum skips NaN, so that a piece of nothing else has -inf here: its sum tells)
                    if (ml.y != ml.y) ml.x = ml.y;
                    if (pass == 0) {
                        const float up = fmaxf(M, ml.x);
                        if (up != -INFINITY) L = L * exp2f(M - up) + ml.y * exp2f(ml.x - up);
                        M = up;
                    } else {
                        weight[i][r] = ml.x == -INFINITY ? 0.0f : exp2f(ml.x - M);
                    }
                }
                if (pass == 1) {
                    __syncthreads();
                    if (mine) {
#pragma unroll 1
                        for (int i0 = 0; i0 < m; i0 += BATCH) {
                            float4 x[BATCH][VEC];
                            float w[BATCH];
#pragma unroll
                            for (int j = 0; j < BATCH; j++) {
                                const int part = c0 + i0 + j >= cnt[0], at = slot[i0 + j];
                                w[j] = at >= 0 ? weight[i0 + j][r] : 0.0f;
#pragma unroll
                                for (int k = 0; k < VEC; k++) {
                                    x[j][k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                                    if (at >= 0 && !(CH % SUBS && sub + k * SUBS >= CH))
                                        x[j][k] = reinterpret_cast<const float4*>(p.o[part])[((int64_t)at * CH + sub + k * SUBS) * p.cap[part] + in[part] + r];
                                }
                            }
#pragma unroll
                            for (int j = 0; j < BATCH; j++)
#pragma unroll
                                for (int k = 0; k < VEC; k++) {
                                    o[k].x = fmaf(w[j], x[j][k].x, o[k].x);
                                    o[k].y = fmaf(w[j], x[j][k].y, o[k].y);
                                    o[k].z = fmaf(w[j], x[j][k].z, o[k].z);
                                    o[k].w = fmaf(w[j], x[j][k].w, o[k].w);
                                }
                        }
                    }
                }
            }
            if (pass == 0) {  // over the threads of a row: of a warp, then the warps in order
                auto join = [&](float m2, float l2) {
                    const float up = fmaxf(M, m2);
                    if (up != -INFINITY) L = L * exp2f(M - up) + l2 * exp2f(m2 - up);
                    M = up;
                };
#pragma unroll
                for (int d = MR; d < 32; d <<= 1) {
                    const float m2 = __shfl_xor_sync(0xffffffffu, M, d), l2 = __shfl_xor_sync(0xffffffffu, L, d);
                    // (both sides form the same sum: the lower lane's part first)
                    const float up = fmaxf(M, m2), a0 = M == -INFINITY ? 0.0f : L * exp2f(M - up), a1 = m2 == -INFINITY ? 0.0f : l2 * exp2f(m2 - up);
                    L = lane & d ? a1 + a0 : a0 + a1;
                    M = up;
                }
                if (lane < MR) red[tid >> 5][r] = make_float2(M, L);
                __syncthreads();
                M = -INFINITY;
                L = 0.0f;
#pragma unroll
                for (int k = 0; k < 8; k++) join(red[k][r].x, red[k][r].y);
            }
        }
        const float inv = L > 0.0f ? 1.0f / L : L;  // a row that saw nothing: zeros; NaN stays
        if (mine) {
#pragma unroll
            for (int k = 0; k < VEC; k++) {
                if (CH % SUBS && sub + k * SUBS >= CH) break;
                *reinterpret_cast<float4*>(&stage[r][4 * (sub + k * SUBS)]) =
                    make_float4(o[k].x * inv, o[k].y * inv, o[k].z * inv, o[k].w * inv);
            }
        }
        __syncthreads();
        // out, a row's dims side by side
#pragma unroll 1
        for (int base = 0; base < run * CH; base += 256) {
            const int rr = (base + tid) / CH, e = (base + tid) % CH * 4, st = st0 + rr, tok = a.group_div(st);
            const bool on = rr < run;
            float y[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            if (on) {
                const float4 v = *reinterpret_cast<const float4*>(&stage[rr][e]);
                y[0] = v.x, y[1] = v.y, y[2] = v.z, y[3] = v.w;
            }
            const int64_t col = (int64_t)(kh * a.group + st - tok * a.group) * D + e;
            if (a.out && on) {
                T* const dst = static_cast<T*>(a.out) + (int64_t)tok * a.out_stride + col;
                if constexpr (sizeof(T) == 4) *reinterpret_cast<float4*>(dst) = make_float4(y[0], y[1], y[2], y[3]);
                else *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3]));
            }
            if (a.xq) {
                const int64_t at = (int64_t)tok * a.n_heads * D + col;
                const uint32_t q = quant_group8(y, lane & 7, on ? a.xd + (at >> 5) : nullptr);
                if (on) *reinterpret_cast<uint32_t*>(a.xq + at) = q;
            }
        }
        __syncthreads();
        st0 += run;
        own_in += run;
        todo -= run;
    }
}

// LQ_FAULT=prefix_attn_wait: waits inside the kernel run out (tests of what follows then)
static void set_polls(PrefixPlan* p, bool f32) {
    p->hold = fault_injected("prefix_attn_wait");
    p->polls = !p->hold ? 1 << 22 : f32 ? 0 : 1 << 12;
}

// The workspace of a call whose prefix items are cut by pp and whose own items by p (the same plan, but
// where two kernels share the work)
static int make_workspace(lq_ctx* ctx, const char* who, const PrefixAttnArgs& a, const PagedSeqs& s, int D, PrefixPlan* p, PrefixPlan* pp) {
    const int64_t items_p = (int64_t)a.n_kv * pp->n_rb;
    const int64_t items_o = a.n_kv * ((int64_t)s.rows * a.group / p->ob + s.n_seqs + 1);
    const int64_t items[2] = {pp->np ? items_p : 0, items_o};
    // workers, ranges, or flows of a CTA that may have a piece
    for (PrefixPlan* x : {p, pp}) x->ranges = (x->chunks ? 5 : x->streams ? 1 : 2) * x->workers;
    const int64_t most[2] = {pp->ranges, p->ranges};
    size_t at = 0;
    auto place = [&at](int64_t n, size_t size) {
        const size_t here = at;
        at += ((size_t)n * size + 255) & ~(size_t)255;
        return here;
    };
    p->notes = p->streams ? p->ranges : (p->pair_o ? 1 : 2) * p->workers;
    const size_t steps_at = place(1, 4), split_at = place(most[1], sizeof(SplitItem));
    size_t first_at[2], last_at[2], ml_at[2], o_at[2];
    for (int k = 0; k < 2; k++) {
        const int64_t slots = k == 1 && p->np == 0 ? 2 * most[1] : items[k] ? items[k] + most[k] : 0;
        LQ_REQUIRE(ctx, slots < (1ll << 31), "%s: too many partials", who);
        first_at[k] = place(items[k], 4);
        last_at[k] = place(items[k], 4);
        ml_at[k] = place(slots * p->cap[k], 8);
        o_at[k] = place(slots * p->cap[k], (size_t)D * 4);
    }
    void* buffer = nullptr;
    const int rc = ensure_paged(ctx, at, &buffer);
    if (rc) return rc;
    uint8_t* w = static_cast<uint8_t*>(buffer);
    p->own_steps = reinterpret_cast<int32_t*>(w + steps_at);
    p->claimed = reinterpret_cast<unsigned*>(w + steps_at + 128);
    p->split = reinterpret_cast<SplitItem*>(w + split_at);
    for (int k = 0; k < 2; k++) {
        p->first[k] = reinterpret_cast<int32_t*>(w + first_at[k]);
        p->last[k] = reinterpret_cast<int32_t*>(w + last_at[k]);
        p->ml[k] = reinterpret_cast<float2*>(w + ml_at[k]);
        p->o[k] = reinterpret_cast<float*>(w + o_at[k]);
    }
    if (pp != p) {
        pp->own_steps = p->own_steps;
        pp->claimed = p->claimed;
        pp->split = p->split;
        pp->notes = p->notes;
        pp->cap[1] = p->cap[1];
        for (int k = 0; k < 2; k++) pp->first[k] = p->first[k], pp->last[k] = p->last[k], pp->ml[k] = p->ml[k], pp->o[k] = p->o[k];
    }
    return LQ_OK;
}

// the plan of a call and its workspace
static int make_plan(lq_ctx* ctx, const PrefixAttnArgs& a, const PagedSeqs& s, bool f32, int D, PrefixPlan* p) {
    const int64_t steps = plan_cut(a, s, f32, ctx->sm_count, p);
    LQ_REQUIRE(ctx, steps < PREFIX_MAX_STEPS, "lq_prefix_attention: %lld steps, more than a launch can number", (long long)steps);
    set_polls(p, f32);
    return make_workspace(ctx, "lq_prefix_attention", a, s, D, p, p);
}

template <typename T, int D, int KIND = MERGE_FLOWS>
static int launch_merge(lq_ctx* ctx, const PrefixAttnArgs& a, const PagedSeqs& s, const PrefixPlan& p, const PrefixPlan& pp) {
    // a row of few heads leaves most of a 32-row CTA idle
    const int mr = p.cap[1] <= 8 ? 8 : 32;
    const int64_t R = (int64_t)s.rows * a.group;
    const dim3 grid((unsigned)(p.np > 0 ? a.n_kv * (R / p.ob + s.n_seqs) : p.notes),
                    (unsigned)ceil_div(p.cap[1], mr));
    return mr == 8 ? launch_kernel(ctx, prefix_attn_merge_kernel<T, D, 8, KIND>, grid, dim3(256), 0, "prefix_attn_merge", a, s, p, pp)
                   : launch_kernel(ctx, prefix_attn_merge_kernel<T, D, 32, KIND>, grid, dim3(256), 0, "prefix_attn_merge", a, s, p, pp);
}

// An 8-bit cache: which kernel takes which items.
template <int D>
static int attend_q8(lq_ctx* ctx, const PrefixAttnArgs& a, const PagedSeqs& s, const PagedQ8& c) {
    const char* const who = "lq_prefix_attention_q8";
    const int64_t own_rows = std::min<int64_t>(a.max_q, s.rows) * a.group, all_rows = (int64_t)s.rows * a.group;
    const bool stream_own = own_rows <= PREFIX_ATTN_Q8_ROWS;
    const bool stream_prefix = a.prefix_len == 0 ? stream_own : all_rows <= PREFIX_ATTN_Q8_ROWS;
    PrefixPlan tc, st;
    int64_t steps_tc = 0, steps_st = 0;
    const int st_rows = (int)std::min<int64_t>(stream_prefix && a.prefix_len > 0 ? all_rows : own_rows, 16);  // of a block
    if (!stream_own || !stream_prefix) {
        steps_tc = plan_cut(a, s, false, ctx->sm_count, &tc);
        set_polls(&tc, false);
    }
    if (stream_own) {
        steps_st = plan_cut(a, s, true, ctx->sm_count, &st, st_rows > 8 ? 16 : 8, PREFIX_ATTN_Q8_CTAS, 128);
        set_polls(&st, true);
        st.streams = stream_prefix ? 3 : 2;
        st.chunks = 1;
        // an item's beginning and end take as long as three of its tiles (with 0, 1, 2 and 3 of them 48
        // sequences of up to 4000 positions, head dimension 64, took 38, 36.5, 30.5 and 29.4 us: short items
        // in a row held up their CTA)
        st.extra = 3;
        steps_st += 3 * (int64_t)a.n_kv * ((int64_t)s.rows * a.group / st.ob + s.n_seqs + 1);
    }
    LQ_REQUIRE(ctx, steps_tc < PREFIX_MAX_STEPS && steps_st < PREFIX_MAX_STEPS, "%s: %lld steps, more than a launch can number", who,
               (long long)std::max(steps_tc, steps_st));
    PrefixPlan* const own = stream_own ? &st : &tc;
    PrefixPlan* const pre = stream_prefix ? &st : &tc;
    if (own != pre) {  // the prefix for itself, and the own items for themselves
        // (All SMs for the prefix, then for the own items. With the SMs divided between them, by how long
        // either takes, 128 sequences behind 32768 positions took 295 us instead of 216, 64 behind 8191 64
        // instead of 60: an SM with few neighbours at work reads no faster.)
        tc.workers = std::max(1, std::min(ctx->sm_count, tc.sp));
        // Short prefixes: as many CTAs for each item, so that none has the end of one and the beginning of the next
        // (two sets of partials, about two steps more): 64 sequences of 4 rows behind 8191 positions 62.5 -> 57.6
        // us, 64 of 8 behind 9000 51.6 -> 48.5, 128 of 4 behind 8192 80.9 -> 77.6. Not so from about ten steps
        // a CTA on: 100 sequences of 8 rows behind 14900 positions 70.8 -> 77.7, behind 30000 108 -> 130.
        const int items = a.n_kv * tc.n_rb, per = std::min(ctx->sm_count / items, tc.np);
        if (per >= 1 && ceil_div(tc.np, per) <= std::min(8, (int)ceil_div(tc.sp, ctx->sm_count) + 1)) tc.workers = per * items;
        tc.workers_mul = ((1ull << 40) + tc.workers - 1) / tc.workers;
        tc.apart = 1;
        st.sp = 0;
        st.cap[0] = tc.cap[0];
    }
    int rc = make_workspace(ctx, who, a, s, D, own, pre);
    if (rc) return rc;
    if (pre == &tc && (rc = launch_prefix_attn_tc(ctx, a, s, tc, D, &c))) return rc;
    if (own == &st && (rc = launch_prefix_attn_q8_decode(ctx, a, s, c, st, D, st_rows))) return rc;
    if (own != pre) return launch_merge<__nv_bfloat16, D, MERGE_APART>(ctx, a, s, *own, *pre);
    if (own == &tc) return launch_merge<__nv_bfloat16, D>(ctx, a, s, tc, tc);
    return st.np > 0 ? launch_merge<__nv_bfloat16, D, MERGE_STREAM>(ctx, a, s, st, st) : launch_prefix_attn_q8_join(ctx, a, s, st, D);
}

// checks and arguments shared by the entry points; esize: bytes of an element of q and out. page_stride:
// in elements of the cache, which is checked by the caller
static int make_attn_args(lq_ctx* ctx, const char* who, PrefixAttnArgs* a, PagedSeqs* s, const void* q, size_t esize, int64_t q_stride,
                          int64_t rows, int64_t n_heads, int64_t n_kv_heads, int64_t head_dim, float scale, int64_t n_pages,
                          int64_t page_size, const int32_t* prefix_table, int64_t prefix_len, int64_t n_seqs,
                          const int32_t* q_start, const int32_t* kv_len, const int32_t* page_table, int64_t table_ld,
                          int64_t max_q, int64_t max_kv, void* out, int64_t out_stride, int8_t* xq, uint16_t* xd) {
    LQ_REQUIRE(ctx, n_heads >= 1 && n_kv_heads >= 1 && n_heads % n_kv_heads == 0 && n_heads <= 4096, "%s: bad head counts", who);
    LQ_REQUIRE(ctx, n_heads / n_kv_heads <= 128, "%s: more than 128 query heads a kv head", who);
    LQ_REQUIRE(ctx, head_dim == 64 || head_dim == 128, "%s: head_dim %lld must be 64 or 128", who, (long long)head_dim);
    const int rc = make_paged_seqs(ctx, who, s, n_seqs, q_start, kv_len, page_table, table_ld, rows, n_pages, page_size);
    if (rc) return rc;
    if (q_stride == 0) q_stride = n_heads * head_dim;
    if (out_stride == 0) out_stride = n_heads * head_dim;
    LQ_REQUIRE(ctx, q_stride >= n_heads * head_dim && out_stride >= n_heads * head_dim, "%s: row stride too small", who);
    LQ_REQUIRE(ctx, prefix_len >= 0 && prefix_len < (1ll << 30) && (prefix_len == 0 || prefix_table), "%s: bad prefix", who);
    LQ_REQUIRE(ctx, aligned_to(prefix_table, 4), "%s: the prefix's page table must be aligned to its elements", who);
    LQ_REQUIRE(ctx, max_q >= 1 && max_q < (1ll << 24) && max_kv >= 0 && max_kv < (1ll << 30),
               "%s: bad bounds max_q %lld, max_kv %lld", who, (long long)max_q, (long long)max_kv);
    LQ_REQUIRE(ctx, scale > 0.0f && scale < INFINITY, "%s: scale must be positive and finite", who);
    LQ_REQUIRE(ctx, (xq == nullptr) == (xd == nullptr), "%s: xq and xd go together", who);
    LQ_REQUIRE(ctx, rows * n_heads < (1ll << 28), "%s: too many rows", who);
    if (rows == 0 || n_seqs == 0) return LQ_OK;
    LQ_REQUIRE(ctx, q && (out || xq), "%s: NULL pointer", who);
    LQ_REQUIRE(ctx, aligned_to(q, 16) && aligned_to(out, 16) && aligned_to(xq, 16) && aligned_to(xd, 2) &&
                        q_stride * esize % 16 == 0 && out_stride * esize % 16 == 0,
               "%s: pointers and strides must be multiples of 16 bytes (xd: of 2)", who);
    a->q = q;
    a->q_stride = q_stride;
    a->n_heads = (int)n_heads;
    a->n_kv = (int)n_kv_heads;
    a->group = (int)(n_heads / n_kv_heads);
    a->group_mul = ((1ull << 36) + a->group - 1) / a->group;
    a->scale = scale;
    a->k = a->v = nullptr;
    a->page_stride = 0;
    a->prefix_table = prefix_table;
    a->prefix_len = (int)prefix_len;
    a->max_q = (int)max_q;
    a->max_kv = (int)max_kv;
    a->out = out;
    a->out_stride = out_stride;
    a->xq = xq;
    a->xd = xd;
    a->err = ctx->err_flag;
    return LQ_OK;
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
    const bool f32 = dtype == LQ_DTYPE_F32;
    const size_t esize = f32 ? 4 : 2;
    lq::PrefixAttnArgs a;
    lq::PagedSeqs s;
    int rc = lq::make_attn_args(ctx, "lq_prefix_attention", &a, &s, q, esize, q_stride, rows, n_heads, n_kv_heads, head_dim, scale,
                                n_pages, page_size, prefix_table, prefix_len, n_seqs, q_start, kv_len, page_table, table_ld,
                                max_q, max_kv, out, out_stride, xq, xd);
    if (rc) return rc;
    if (page_stride == 0) page_stride = n_kv_heads * page_size * head_dim;
    LQ_REQUIRE(ctx, page_stride >= n_kv_heads * page_size * head_dim, "lq_prefix_attention: page_stride too small");
    if (rows == 0 || n_seqs == 0) return LQ_OK;
    LQ_REQUIRE(ctx, k_pages && v_pages, "lq_prefix_attention: NULL pointer");
    LQ_REQUIRE(ctx, lq::aligned_to(k_pages, 16) && lq::aligned_to(v_pages, 16) && page_stride * esize % 16 == 0,
               "lq_prefix_attention: pointers and strides must be multiples of 16 bytes (xd: of 2)");
    a.k = k_pages;
    a.v = v_pages;
    a.page_stride = page_stride;
    lq::PrefixPlan p;
    const int D = (int)head_dim;
    if ((rc = lq::make_plan(ctx, a, s, f32, D, &p))) return rc;
    rc = f32 ? lq::launch_prefix_attn_f32(ctx, a, s, p, D) : lq::launch_prefix_attn_tc(ctx, a, s, p, D);
    if (rc) return rc;
    if (f32) return D == 64 ? lq::launch_merge<float, 64>(ctx, a, s, p, p) : lq::launch_merge<float, 128>(ctx, a, s, p, p);
    return D == 64 ? lq::launch_merge<__nv_bfloat16, 64>(ctx, a, s, p, p) : lq::launch_merge<__nv_bfloat16, 128>(ctx, a, s, p, p);
}

extern "C" int lq_prefix_attention_q8(lq_ctx* ctx, const uint16_t* q, int64_t q_stride, int64_t rows, int64_t n_heads,
                                      int64_t n_kv_heads, int64_t head_dim, float scale, const int8_t* k_codes,
                                      const int8_t* v_codes, const float* k_scale, const float* v_scale, int64_t n_pages,
                                      int64_t page_size, int64_t page_stride, int64_t block, int64_t scale_stride,
                                      const int32_t* prefix_table, int64_t prefix_len, int64_t n_seqs, const int32_t* q_start,
                                      const int32_t* kv_len, const int32_t* page_table, int64_t table_ld, int64_t max_q,
                                      int64_t max_kv, uint16_t* out, int64_t out_stride, int8_t* xq, uint16_t* xd) {
    LQ_ENTRY(ctx, "lq_prefix_attention_q8");
    lq::PrefixAttnArgs a;
    lq::PagedSeqs s;
    lq::PagedQ8 c;
    int rc = lq::make_attn_args(ctx, "lq_prefix_attention_q8", &a, &s, q, 2, q_stride, rows, n_heads, n_kv_heads, head_dim, scale,
                                n_pages, page_size, prefix_table, prefix_len, n_seqs, q_start, kv_len, page_table, table_ld,
                                max_q, max_kv, out, out_stride, xq, xd);
    if (rc) return rc;
    rc = lq::make_paged_q8(ctx, "lq_prefix_attention_q8", &c, const_cast<int8_t*>(k_codes), const_cast<int8_t*>(v_codes),
                           const_cast<float*>(k_scale), const_cast<float*>(v_scale), n_kv_heads, head_dim, page_size, page_stride,
                           block, scale_stride, rows > 0 && n_seqs > 0);
    if (rc) return rc;
    if (rows == 0 || n_seqs == 0) return LQ_OK;
    return head_dim == 64 ? lq::attend_q8<64>(ctx, a, s, c) : lq::attend_q8<128>(ctx, a, s, c);
}
