// lq8_prefix_attn_f32.cu -- the shared-prefix attention for f32 caches.
//
// The output is held to f32, so the products run as 3xTF32: each operand is split into
// big (the low 13 mantissa bits cleared) and small = x - big, and a product is small.big + big.small
// + big.big with f32 sums (about 22 bits). A worker of the line (lq8_prefix_plan.cuh) is a warp: it
// takes 8 stacked query rows through its steps of 32 positions, 16 at a time,
//   S^T = K Q^T     mma.sync m16n8k8: 16 positions x 8 rows
//   O^T += V^T P^T  16 dims x 8 rows, 8 positions deep
// with K and V straight from global memory into the operand registers: the order of the dims in
// the products is free, so that a lane's elements of K (4 dims of 2 positions) and of V (4 dims of
// 4 positions) are 16-byte vectors and every fetched sector is used whole. No warp waits for
// another; the running maximum and sum of a row lie in the lanes that hold its scores.
// Bound: HBM where few rows share a position (8 rows: 96 MMAs and about 500 other instructions per
// 16 KB), the MMA and split instructions where many do.
#include "lq8_async.cuh"
#include "lq8_fused.cuh"
#include "lq8_prefix_attn.cuh"
#include "lq8_prefix_plan.cuh"

#include <algorithm>

namespace lq {

constexpr int PF_WARPS = PREFIX_ATTN_F32_WARPS;
constexpr int PF_SCAN = 1024;

__device__ __forceinline__ float pf_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t tf_big(float x) { return __float_as_uint(x) & 0xffffe000u; }
__device__ __forceinline__ uint32_t tf_small(float x, uint32_t big) { return __float_as_uint(x - __uint_as_float(big)); }
__device__ __forceinline__ void mma_tf32(float c[4], const uint32_t a[4], uint32_t b0, uint32_t b1) {
    asm(
        "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// c += a b as 3xTF32: the small cross terms into x, big.big into c. The tensor cores cut a sum off
// where an f32 addition rounds it, so c takes few of them in a row: two at a time, then f32 sums
// (chains of eight had the results 1.6 times as far off as plain f32).
__device__ __forceinline__ void mma_3tf32(float c[4], float x[4], float a0, float a1, float a2, float a3, float b0, float b1) {
    const uint32_t ab[4] = {tf_big(a0), tf_big(a1), tf_big(a2), tf_big(a3)};
    const uint32_t as[4] = {tf_small(a0, ab[0]), tf_small(a1, ab[1]), tf_small(a2, ab[2]), tf_small(a3, ab[3])};
    const uint32_t bb0 = tf_big(b0), bb1 = tf_big(b1);
    mma_tf32(x, as, bb0, bb1);
    mma_tf32(x, ab, tf_small(b0, bb0), tf_small(b1, bb1));
    mma_tf32(c, ab, bb0, bb1);
}

template <int D>
__global__ void __launch_bounds__(PF_WARPS * 32, 1)
prefix_attn_f32_kernel(const __grid_constant__ PrefixAttnArgs a, const __grid_constant__ PagedSeqs s,
                       const __grid_constant__ PrefixPlan p) {
    constexpr int KB = D / 16, VB = D / 32;  // 16-byte vectors of a K row, of a V row, per lane
    __shared__ int scan[PF_SCAN + 1];
    __shared__ int4 info[PF_SCAN];  // up to PF_SCAN sequences: q0, q, kv, steps of a head
    __shared__ __align__(16) float prob[PF_WARPS][16][8];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3;
    pdl_wait();
    pdl_trigger();  // (after the wait: the merge reads the call's lengths before its own)
    const int per_entry = (s.n_seqs + PF_SCAN - 1) / PF_SCAN;
    const int n_entries = (s.n_seqs + per_entry - 1) / per_entry;
    const OwnSteps os{a, p};
    auto per_head = [&](const SeqInfo& si) {  // by a warp
        const int n_rb = os.blocks(si);
        int n = 0;
#pragma unroll 1
        for (int rb = lane; rb < n_rb; rb += 32) n += os.tiles(si, rb);
        return __reduce_add_sync(0xffffffffu, n);
    };
    const bool by_warp = a.max_q * a.group > 8 * p.ob;
#pragma unroll 1
    for (int e = by_warp ? warp : tid; e < n_entries; e += by_warp ? PF_WARPS : PF_WARPS * 32) {
        int n = 0;
#pragma unroll 1
        for (int b = e * per_entry; b < min(s.n_seqs, (e + 1) * per_entry); b++) {
            const SeqInfo si = seq_info(a, s, b, blockIdx.x == 0);
            const int per = by_warp ? per_head(si) : os.per_head(si);
            n += per * a.n_kv;
            if (per_entry == 1) info[b] = make_int4(si.q0, si.q, si.kv, per);
        }
        scan[e + 1] = n;
    }
    __syncthreads();
    if (warp == 0) {
        int run = 0;
#pragma unroll 1
        for (int e0 = 0; e0 < n_entries; e0 += 32) {
            int v = e0 + lane < n_entries ? scan[e0 + lane + 1] : 0;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int u = __shfl_up_sync(0xffffffffu, v, o);
                if (lane >= o) v += u;
            }
            if (e0 + lane < n_entries) scan[e0 + lane + 1] = run + v;
            run += __shfl_sync(0xffffffffu, v, 31);
        }
        if (lane == 0) scan[0] = 0;
    }
    __syncthreads();
    const int so = scan[n_entries];
    if (blockIdx.x == 0 && tid == 0) *p.own_steps = so;
    if (a.prefix_len == 0) {  // rows before their sequence's first position see nothing
#pragma unroll 1
        for (int b = blockIdx.x * PF_WARPS + warp; b < s.n_seqs; b += gridDim.x * PF_WARPS) {
            const SeqInfo si = seq_info(a, s, b, false);
            if (si.kv < si.q) zero_rows<float, D>(a, si.q0, si.q - si.kv, lane, 32);
        }
    }
    const int worker = warp * gridDim.x + blockIdx.x;
    if (worker >= p.workers) return;
    const Line line(p, so, true, true);
    if (a.prefix_len == 0 && lane == 0) p.split[worker].rows = 0;
    __syncwarp();
    const float qs = a.scale * 1.44269504088896340736f;  // scores in units of log2
    const int mask = (1 << s.page_shift) - 1;
    float(*const pr)[8] = prob[warp];

#pragma unroll 1
    for (int part = 0; part < 2; part++) {
        const bool own = part;
        int step, hi;
        flow_range(line, true, worker, 0, own, step, hi);
        if (step >= hi) continue;
        // the item of the first step: sequence, kv head, row block, tile
        int b = 0, kh, rb, tile, n_rb = p.n_rb, nt = p.np;
        SeqInfo si{0, s.rows, 0};
        if (!own) {
            const int item = step / p.np;
            tile = step - item * p.np;
            kh = item / n_rb;
            rb = item - kh * n_rb;
        } else {
            int e0 = 0, e1 = n_entries;  // the last entry with scan <= step
#pragma unroll 1
            while (e1 - e0 > 1) {
                const int m = (e0 + e1) >> 1;
                if (scan[m] <= step) e0 = m;
                else e1 = m;
            }
            int rest = step - scan[e0], per = 1;
#pragma unroll 1
            for (b = e0 * per_entry; b < s.n_seqs; b++) {
                si = seq_info(a, s, b, false);
                per = per_entry == 1 ? info[b].w : per_head(si);
                if (rest < per * a.n_kv) break;
                rest -= per * a.n_kv;
            }
            if (b >= s.n_seqs) break;  // lengths that changed under the kernel
            kh = rest / per;
            rest -= kh * per;
            n_rb = os.blocks(si);
            rb = 0;
#pragma unroll 1
            for (; rb < n_rb; rb += 32) {
                int n = rb + lane < n_rb ? os.tiles(si, rb + lane) : 0, upto = n;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int u = __shfl_up_sync(0xffffffffu, upto, o);
                    if (lane >= o) upto += u;
                }
                const int all = __shfl_sync(0xffffffffu, upto, 31);
                if (rest < all) {
                    const int l = __ffs(__ballot_sync(0xffffffffu, upto > rest)) - 1;
                    rest -= __shfl_sync(0xffffffffu, upto - n, l);
                    rb += l;
                    break;
                }
                rest -= all;
            }
            tile = rest;
        }
#pragma unroll 1
        while (step < hi) {
            // ---- a segment: tiles [tile, end) of one item ----
            int kv_end = a.prefix_len;
            if (own) {
                kv_end = os.visible(si, rb);
                nt = (kv_end + p.tile - 1) / p.tile;
            }
            const int end = min(nt, tile + hi - step);
            const int row0 = (own ? si.q0 * a.group : 0) + rb * p.pb;
            const int n = min(p.pb, (own ? si.q : s.rows) * a.group - rb * p.pb);
            const int item = (own ? a.n_kv * os.base(si, b) : 0) + kh * n_rb + rb;
            const bool whole = a.prefix_len == 0 && tile == 0 && end == nt;
            if (lane == 0) {
                if (tile == 0) p.first[part][item] = worker;
                if (end == nt) p.last[part][item] = worker;
                if (a.prefix_len == 0 && tile == 0 && end < nt) p.split[worker] = SplitItem{n, row0, kh, item};
            }
            const int32_t* const table = own ? s.table + (int64_t)b * s.table_ld : a.prefix_table;
            auto row_of = [&](int r, int& tok, int& head) {  // stacked row r of the block
                tok = a.group_div(row0 + r);
                head = kh * a.group + row0 + r - tok * a.group;
            };
            float4 q[KB];
            {
                int tok, head;
                row_of(min(g, n - 1), tok, head);
                const float4* src = reinterpret_cast<const float4*>(static_cast<const float*>(a.q) + (int64_t)tok * a.q_stride +
                                                                    (int64_t)head * D + 4 * t4);
#pragma unroll
                for (int i = 0; i < KB; i++) {
                    const float4 x = g < n ? src[4 * i] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    q[i] = make_float4(x.x * qs, x.y * qs, x.z * qs, x.w * qs);
                }
            }
            // positions that rows 2 t4 and 2 t4 + 1 see
            int vis[2];
#pragma unroll
            for (int k = 0; k < 2; k++) {
                int tok, head;
                row_of(min(2 * t4 + k, n - 1), tok, head);
                vis[k] = own ? min(kv_end, own_visible(si, tok - si.q0)) : kv_end;
            }
            float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f}, o[2 * VB][4];
#pragma unroll
            for (int i = 0; i < 2 * VB; i++) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;

            const int pos0 = tile * p.tile, pos1 = min(end * p.tile, kv_end);
            float4 kr[2][KB], vr[4][VB];
            // 8 positions lie in one page: where the 8 from x on begin, for this kv head, and how
            // many of them count; past the end the last 8 again, their rows from the last one on
            // (finite where a visible row is, and masked)
            struct Eight {
                int64_t at;
                int most;
            };
            const int last8 = (pos1 - 1) & ~7;
            auto eight = [&](int x) {
                x = min(x, last8);
                int pg = table[x >> s.page_shift];
                if ((unsigned)pg >= (unsigned)s.n_pages) {
                    flag_error(a.err, ERR_PAGE_ID, pg);
                    pg = 0;
                }
                return Eight{pg * a.page_stride + (((int64_t)kh << s.page_shift) + (x & mask)) * D, pos1 - 1 - x};
            };
            Eight now[2], then[2];
            auto load_k = [&](const Eight e[2]) {
#pragma unroll
                for (int r = 0; r < 2; r++) {
                    const float4* src = reinterpret_cast<const float4*>(static_cast<const float*>(a.k) + e[r].at) +
                                        min(g, e[r].most) * (D / 4) + t4;
#pragma unroll
                    for (int i = 0; i < KB; i++) kr[r][i] = src[4 * i];
                }
            };
            auto load_v = [&](const Eight e[2]) {
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const float4* src = reinterpret_cast<const float4*>(static_cast<const float*>(a.v) + e[r >> 1].at) +
                                        min(4 * (r & 1) + t4, e[r >> 1].most) * (D / 4) + g;
#pragma unroll
                    for (int i = 0; i < VB; i++) vr[r][i] = src[8 * i];
                }
            };
            now[0] = eight(pos0), now[1] = eight(pos0 + 8);
            load_k(now);
            load_v(now);
#pragma unroll 1
            for (int x = pos0; x < pos1; x += 16) {
                then[0] = eight(x + 16), then[1] = eight(x + 24);
                float sc[4] = {0.0f, 0.0f, 0.0f, 0.0f}, y[2][4];
#pragma unroll
                for (int i = 0; i < 4; i++) y[0][i] = y[1][i] = 0.0f;
#pragma unroll
                for (int i = 0; i < KB; i++) {
                    float c[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                    mma_3tf32(c, y[0], kr[0][i].x, kr[1][i].x, kr[0][i].y, kr[1][i].y, q[i].x, q[i].y);
                    mma_3tf32(c, y[1], kr[0][i].z, kr[1][i].z, kr[0][i].w, kr[1][i].w, q[i].z, q[i].w);
#pragma unroll
                    for (int j = 0; j < 4; j++) sc[j] += c[j];
                }
                load_k(then);
#pragma unroll
                for (int i = 0; i < 4; i++) {  // position x + g + 8 (i / 2), row 2 t4 + i % 2
                    sc[i] += y[0][i] + y[1][i];
                    if (x + g + 8 * (i >> 1) >= vis[i & 1]) sc[i] = -INFINITY;
                }
                float up[2];
#pragma unroll
                for (int k = 0; k < 2; k++) {
                    up[k] = fmaxf(sc[k], sc[2 + k]);
#pragma unroll
                    for (int d = 4; d < 32; d <<= 1) up[k] = fmaxf(up[k], __shfl_xor_sync(0xffffffffu, up[k], d));
                }
                // a maximum that grew by less than 2^8 stays: p <= 256 costs an f32 sum nothing
                if (__any_sync(0xffffffffu, up[0] > m[0] + 8.0f || up[1] > m[1] + 8.0f || x == pos0)) {
#pragma unroll
                    for (int k = 0; k < 2; k++) {
                        const float mn = fmaxf(m[k], up[k]);
                        const float f = mn == -INFINITY ? 1.0f : pf_ex2(m[k] - mn);
                        m[k] = mn;
                        l[k] *= f;
#pragma unroll
                        for (int i = 0; i < 2 * VB; i++) o[i][k] *= f, o[i][2 + k] *= f;
                    }
                }
                float e[4];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    e[i] = pf_ex2(sc[i] - (m[i & 1] == -INFINITY ? 0.0f : m[i & 1]));
                    l[i & 1] += e[i];
                }
                *reinterpret_cast<float2*>(&pr[g][2 * t4]) = make_float2(e[0], e[1]);
                *reinterpret_cast<float2*>(&pr[g + 8][2 * t4]) = make_float2(e[2], e[3]);
                __syncwarp();
                float pb[4];  // positions x + t4 + 4 i, row g
#pragma unroll
                for (int i = 0; i < 4; i++) pb[i] = pr[t4 + 4 * i][g];
                __syncwarp();
                // (16 positions at a time go into the f32 sums)
#pragma unroll
                for (int i = 0; i < VB; i++) {
                    float w[2][4], u[2][4];
#pragma unroll
                    for (int j = 0; j < 4; j++) w[0][j] = w[1][j] = u[0][j] = u[1][j] = 0.0f;
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        mma_3tf32(w[0], u[0], vr[2 * h][i].x, vr[2 * h][i].y, vr[2 * h + 1][i].x, vr[2 * h + 1][i].y, pb[2 * h], pb[2 * h + 1]);
                        mma_3tf32(w[1], u[1], vr[2 * h][i].z, vr[2 * h][i].w, vr[2 * h + 1][i].z, vr[2 * h + 1][i].w, pb[2 * h], pb[2 * h + 1]);
                    }
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        o[2 * i][j] += w[0][j] + u[0][j];
                        o[2 * i + 1][j] += w[1][j] + u[1][j];
                    }
                }
                load_v(then);
                now[0] = then[0], now[1] = then[1];
            }
            // ---- its result: rows 2 t4, 2 t4 + 1, dims 32 i + 4 g .. + 3 ----
#pragma unroll
            for (int k = 0; k < 2; k++) {
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) l[k] += __shfl_xor_sync(0xffffffffu, l[k], d);
                const int r = 2 * t4 + k;
                const bool mine = r < n;
                int tok, head;
                row_of(min(r, n - 1), tok, head);
                const int64_t slot = item + worker;
                const int cap = p.cap[part];
                if (mine && !whole && g == 0) p.ml[part][slot * cap + r] = make_float2(m[k], l[k]);
                const float inv = l[k] > 0.0f ? 1.0f / l[k] : l[k];
#pragma unroll
                for (int i = 0; i < VB; i++) {
                    float v[4] = {o[2 * i][k], o[2 * i][2 + k], o[2 * i + 1][k], o[2 * i + 1][2 + k]};
                    if (!whole) {
                        if (mine)
                            reinterpret_cast<float4*>(p.o[part])[(slot * (D / 4) + 8 * i + g) * cap + r] =
                                make_float4(v[0], v[1], v[2], v[3]);
                        continue;
                    }
#pragma unroll
                    for (int j = 0; j < 4; j++) v[j] = l[k] == 0.0f ? 0.0f : v[j] * inv;
                    if (mine && a.out)
                        *reinterpret_cast<float4*>(static_cast<float*>(a.out) + (int64_t)tok * a.out_stride + (int64_t)head * D +
                                                   32 * i + 4 * g) = make_float4(v[0], v[1], v[2], v[3]);
                    if (a.xq) {  // the 8 lanes of a row hold a block of 32 dims
                        float amax = fmaxf(fmaxf(fabsf(v[0]), fabsf(v[1])), fmaxf(fabsf(v[2]), fabsf(v[3]))), d, id;
#pragma unroll
                        for (int w = 4; w < 32; w <<= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, w));
                        q8_scale(amax, d, id);
                        const int64_t at = ((int64_t)tok * a.n_heads + head) * D + 32 * i;
                        uint32_t w = 0;
#pragma unroll
                        for (int j = 0; j < 4; j++) w |= (uint32_t)(q8_quant(v[j], id) & 0xFF) << (8 * j);
                        if (mine) {
                            if (g == 0) a.xd[at / 32] = f2h(d);
                            *reinterpret_cast<uint32_t*>(a.xq + at + 4 * g) = w;
                        }
                    }
                }
            }
            // ---- the next item with a step ----
            step += end - tile;
            tile = 0;
            while (step < hi) {
                if (++rb >= n_rb) {
                    rb = 0;
                    kh++;
                    if (own && kh == a.n_kv) {
                        kh = 0;
                        if (++b >= s.n_seqs) {  // lengths that changed under the kernel
                            hi = step;
                            break;
                        }
                        si = seq_info(a, s, b, false);
                        n_rb = os.blocks(si);
                        if (n_rb == 0 || si.kv == 0) {  // nothing of this sequence
                            kh = a.n_kv - 1;
                            rb = n_rb;
                            continue;
                        }
                    }
                }
                if (!own || os.tiles(si, rb) > 0) break;
            }
        }
    }
}

int launch_prefix_attn_f32(lq_ctx* ctx, const PrefixAttnArgs& a, const PagedSeqs& s, const PrefixPlan& p, int D) {
    const dim3 grid((unsigned)std::min(ctx->sm_count, p.workers));
    return D == 64 ? launch_kernel(ctx, prefix_attn_f32_kernel<64>, grid, dim3(PF_WARPS * 32), 0, "prefix_attn_f32", a, s, p)
                   : launch_kernel(ctx, prefix_attn_f32_kernel<128>, grid, dim3(PF_WARPS * 32), 0, "prefix_attn_f32", a, s, p);
}

}  // namespace lq
