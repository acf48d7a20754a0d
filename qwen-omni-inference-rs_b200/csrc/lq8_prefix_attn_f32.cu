// lq8_prefix_attn_f32.cu -- the shared-prefix attention for f32 caches.
//
// The output is held to f32, so the products run as 3xTF32: each operand is split into
// big (the low 13 mantissa bits cleared) and small = x - big, and a product is small.big + big.small
// + big.big with f32 sums (about 22 bits). A worker of the line (lq8_prefix_plan.cuh) is a warp: it
// takes 8 stacked query rows through its steps of 32 positions, 16 at a time,
//   S^T = K Q^T     mma.sync m16n8k8: 16 positions x 8 rows
//   O^T += V^T P^T  16 dims x 8 rows, 8 positions deep
// K and V rows come by bulk copies into a ring of three slots of the warp's own (K, V, K, V, ..., 16
// rows each): one is worked on while two are in flight, 128 KB an SM. The order of the dims in the
// products is free, so a lane's elements of K (4 dims of 2 positions) and of V (4 dims of 4
// positions) are 16-byte vectors; the rows are padded so that a warp's reads meet no bank twice. No
// warp waits for another; the running maximum and sum of a row lie in the lanes that hold its scores.
// Bound: the latency of a step's chain (copy, split, MMA, shuffles, exponential, MMA), which two
// warps a scheduler (255 registers a thread) do not hide: no unit is busy. A step of 16 positions
// takes 96 MMAs and about 500 other instructions, and every block of 8 rows splits K and V for
// itself. 8 sequences of 64 heads behind 1024 positions: 27 us (1.1 TB/s, 1.4 instructions of 4 a
// cycle, tensor pipe 18 %), 48 with loads into registers; 64 sequences of 32 heads behind 4096: 230 us
// (20 TFLOP/s) with the merge. An infinity has no second part (it minus itself), so that one in
// Q, K or V gives NaN.
#include "lq8_async.cuh"
#include "lq8_fused.cuh"
#include "lq8_prefix_attn.cuh"
#include "lq8_prefix_plan.cuh"

#include <algorithm>

namespace lq {

constexpr int PF_WARPS = PREFIX_ATTN_F32_WARPS;
constexpr int PF_SCAN = 256;
constexpr int PF_SLOTS = 3;
constexpr int ERR_PF_WAIT = 95;  // a copy did not land

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
__device__ __forceinline__ void mma_3tf32(float c[4], float x[4], float a0, float a1, float a2, float a3, uint32_t b0,
                                          uint32_t b1, uint32_t b0_small, uint32_t b1_small) {
    const uint32_t ab[4] = {tf_big(a0), tf_big(a1), tf_big(a2), tf_big(a3)};
    const uint32_t as[4] = {tf_small(a0, ab[0]), tf_small(a1, ab[1]), tf_small(a2, ab[2]), tf_small(a3, ab[3])};
    mma_tf32(x, as, b0, b1);
    mma_tf32(x, ab, b0_small, b1_small);
    mma_tf32(c, ab, b0, b1);
}

template <int D>
__global__ void __launch_bounds__(PF_WARPS * 32, 1)
prefix_attn_f32_kernel(const __grid_constant__ PrefixAttnArgs a, const __grid_constant__ PagedSeqs s,
                       const __grid_constant__ PrefixPlan p) {
    constexpr int KB = D / 16, VB = D / 32;  // 16-byte vectors of a K row, of a V row, per lane
    constexpr int KS = D * 4 + 64, VS = D * 4 + 32, SLOT = 16 * KS;  // bytes from row to row, of a slot
    extern __shared__ __align__(128) uint8_t slots[];
    __shared__ uint64_t full[PF_WARPS][PF_SLOTS];
    __shared__ int scan[PF_SCAN + 1];
    __shared__ int4 info[PF_SCAN];  // up to PF_SCAN sequences: q0, q, kv, steps of a head
    __shared__ __align__(16) float prob[PF_WARPS][16][8];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3;
    uint8_t* const mine = slots + warp * PF_SLOTS * SLOT;
    if (lane == 0)
        for (int i = 0; i < PF_SLOTS; i++) mbar_init(&full[warp][i], 1);
    mbar_fence_init();
    __syncwarp();
    int slot = 0;       // of the next K or V to be worked on
    unsigned ph = 0;    // and its parity
    bool ok = true;
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
    bool fell = false;
#pragma unroll 1
    for (int e = by_warp ? warp : tid; e < n_entries; e += by_warp ? PF_WARPS : PF_WARPS * 32) {
        int n = 0;
#pragma unroll 1
        for (int b = e * per_entry; b < min(s.n_seqs, (e + 1) * per_entry); b++) {
            const SeqInfo si = seq_info(a, s, b, blockIdx.x == 0);
            fell |= falls(s, b);
            const int per = by_warp ? per_head(si) : os.per_head(si);
            n += per * a.n_kv;
            if (per_entry == 1) info[b] = make_int4(si.q0, si.q, si.kv, per);
        }
        scan[e + 1] = n;
    }
    fell = __syncthreads_or(fell);
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
    const int so = fell ? 0 : scan[n_entries];
    if (blockIdx.x == 0 && tid == 0) *p.own_steps = so;
    if (a.prefix_len == 0) {  // rows before their sequence's first position see nothing
#pragma unroll 1
        for (int b = blockIdx.x * PF_WARPS + warp; b < s.n_seqs; b += gridDim.x * PF_WARPS) {
            const SeqInfo si = seq_info(a, s, b, false);
            if (si.kv < si.q) zero_rows<float, D>(a, si.q0, si.q - si.kv, lane, 32);
        }
    }
    const int worker = warp * gridDim.x + blockIdx.x, live = live_rows(s);
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
        while (step < hi && ok) {
            // ---- a segment: tiles [tile, end) of one item ----
            int kv_end = a.prefix_len;
            if (own) {
                kv_end = os.visible(si, rb);
                nt = (kv_end + p.tile - 1) / p.tile;
            }
            const int end = min(nt, tile + hi - step);
            const int row0 = (own ? si.q0 * a.group : 0) + rb * p.pb;
            // (a block of padding: its first row, for nothing)
            const int n = max(1, min(p.pb, (own ? si.q : live) * a.group - rb * p.pb));
            const int item = (own ? a.n_kv * os.base(si, b) : 0) + kh * n_rb + rb;
            const bool begins = tile == 0, whole = a.prefix_len == 0 && begins && end == nt;
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
            uint32_t qb[KB][4], qm[KB][4];  // big and small parts
            {
                int tok, head;
                row_of(min(g, n - 1), tok, head);
                const float4* src = reinterpret_cast<const float4*>(static_cast<const float*>(a.q) + (int64_t)tok * a.q_stride +
                                                                    (int64_t)head * D + 4 * t4);
#pragma unroll
                for (int i = 0; i < KB; i++) {
                    const float4 x = g < n ? src[4 * i] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    const float v[4] = {x.x * qs, x.y * qs, x.z * qs, x.w * qs};
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        qb[i][j] = tf_big(v[j]);
                        qm[i][j] = tf_small(v[j], qb[i][j]);
                    }
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
            // where position min(x + lane, the last one) lies for this kv head, lanes 0 to 15: rows
            // past the end repeat the last one (finite where that is, and masked)
            auto page_of = [&](int x) { return table[min(x + (lane & 15), pos1 - 1) >> s.page_shift]; };
            auto place = [&](int x, int pg) -> int64_t {
                if ((unsigned)pg >= (unsigned)s.n_pages) {
                    flag_error(a.err, ERR_PAGE_ID, pg);
                    pg = 0;
                }
                return pg * a.page_stride + (((int64_t)kh << s.page_shift) + (min(x + (lane & 15), pos1 - 1) & mask)) * D;
            };
            auto fetch = [&](int to, const void* base, int64_t at, int stride) {
                if (lane == 0) mbar_expect_tx(&full[warp][to], 16 * D * 4);
                __syncwarp();
                if (lane < 16) bulk_g2s(mine + to * SLOT + lane * stride, static_cast<const float*>(base) + at, D * 4, &full[warp][to]);
            };
            auto after = [](int i, int by) { return (i + by) % PF_SLOTS; };
            auto landed = [&]() {
                ok = mbar_wait(&full[warp][slot], ph, p.polls);
                ok = __all_sync(0xffffffffu, ok);
                return ok;
            };
            // after a copy that did not land: it and the later ones of `n` in flight may not land in
            // shared memory that is no longer this kernel's
            auto drain = [&](int n) {
#pragma unroll 1
                for (int i = 0; i < n; i++)
                    mbar_wait_ns(&full[warp][after(slot, i)], slot + i < PF_SLOTS ? ph : ph ^ 1u, 2000000000ull);
            };
            auto done = [&]() {
                __syncwarp();  // (read by every lane)
                if (++slot == PF_SLOTS) slot = 0, ph ^= 1;
            };
            // in flight: K and V of the first 16 positions, K of the next
            int64_t at_v = place(pos0, page_of(pos0)), at_k = 0;
            int pg = page_of(pos0 + 16);
            fetch(slot, a.k, at_v, KS);
            fetch(after(slot, 1), a.v, at_v, VS);
            if (pos0 + 16 < pos1) {
                at_k = place(pos0 + 16, pg);
                fetch(after(slot, 2), a.k, at_k, KS);
            }
#pragma unroll 1
            for (int x = pos0; x < pos1; x += 16) {
                if (x + 32 < pos1) pg = page_of(x + 32);
                float sc[4] = {0.0f, 0.0f, 0.0f, 0.0f}, y[2][4];
#pragma unroll
                for (int i = 0; i < 4; i++) y[0][i] = y[1][i] = 0.0f;
                if (!landed()) {
                    drain(x + 16 < pos1 ? 3 : 2);  // K, V, the next K
                    break;
                }
                {
                    const uint8_t* const k0 = mine + slot * SLOT + g * KS + t4 * 16;
#pragma unroll
                    for (int i = 0; i < KB; i++) {
                        const float4 lo = *reinterpret_cast<const float4*>(k0 + 64 * i);
                        const float4 hi8 = *reinterpret_cast<const float4*>(k0 + 8 * KS + 64 * i);
                        float c[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                        mma_3tf32(c, y[0], lo.x, hi8.x, lo.y, hi8.y, qb[i][0], qb[i][1], qm[i][0], qm[i][1]);
                        mma_3tf32(c, y[1], lo.z, hi8.z, lo.w, hi8.w, qb[i][2], qb[i][3], qm[i][2], qm[i][3]);
#pragma unroll
                        for (int j = 0; j < 4; j++) sc[j] += c[j];
                    }
                }
                done();
                // the slot's next: V of the 16 positions after these
                if (x + 16 < pos1) {
                    fetch(after(slot, 2), a.v, at_k, VS);
                    at_v = at_k;
                }
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
                uint32_t pb[4], pm[4];  // positions x + t4 + 4 i, row g: big and small parts
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float v = pr[t4 + 4 * i][g];
                    pb[i] = tf_big(v);
                    pm[i] = tf_small(v, pb[i]);
                }
                if (!landed()) {
                    drain(x + 16 < pos1 ? 3 : 1);  // V, the next K and V
                    break;
                }
                {
                    const uint8_t* const v0 = mine + slot * SLOT + t4 * VS + g * 16;
#pragma unroll
                    for (int i = 0; i < VB; i++) {  // (16 positions at a time go into the f32 sums)
                        float w[2][4], u[2][4];
#pragma unroll
                        for (int j = 0; j < 4; j++) w[0][j] = w[1][j] = u[0][j] = u[1][j] = 0.0f;
#pragma unroll
                        for (int h = 0; h < 2; h++) {
                            const float4 r0 = *reinterpret_cast<const float4*>(v0 + (8 * h) * VS + 128 * i);
                            const float4 r1 = *reinterpret_cast<const float4*>(v0 + (8 * h + 4) * VS + 128 * i);
                            mma_3tf32(w[0], u[0], r0.x, r0.y, r1.x, r1.y, pb[2 * h], pb[2 * h + 1], pm[2 * h], pm[2 * h + 1]);
                            mma_3tf32(w[1], u[1], r0.z, r0.w, r1.z, r1.w, pb[2 * h], pb[2 * h + 1], pm[2 * h], pm[2 * h + 1]);
                        }
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            o[2 * i][j] += w[0][j] + u[0][j];
                            o[2 * i + 1][j] += w[1][j] + u[1][j];
                        }
                    }
                }
                done();
                // the slot's next: K of the 16 positions after those
                if (x + 32 < pos1) {
                    at_k = place(x + 32, pg);
                    fetch(after(slot, 2), a.k, at_k, KS);
                }
            }
            if (!ok) {
                flag_error(a.err, ERR_PF_WAIT, worker);
                break;
            }
            // ---- its result: rows 2 t4, 2 t4 + 1, dims 32 i + 4 g .. + 3 ----
#pragma unroll
            for (int k = 0; k < 2; k++) {
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) l[k] += __shfl_xor_sync(0xffffffffu, l[k], d);
                const int r = 2 * t4 + k;
                const bool real = r < n;
                int tok, head;
                row_of(min(r, n - 1), tok, head);
                const int64_t slot = own ? p.own_slot(item, worker, begins) : item + worker;
                const int cap = p.cap[part];
                if (real && !whole && g == 0) p.ml[part][slot * cap + r] = make_float2(m[k], l[k]);
                const float inv = l[k] > 0.0f ? 1.0f / l[k] : l[k];
#pragma unroll
                for (int i = 0; i < VB; i++) {
                    float v[4] = {o[2 * i][k], o[2 * i][2 + k], o[2 * i + 1][k], o[2 * i + 1][2 + k]};
                    if (!whole) {
                        if (real)
                            reinterpret_cast<float4*>(p.o[part])[(slot * (D / 4) + 8 * i + g) * cap + r] =
                                make_float4(v[0], v[1], v[2], v[3]);
                        continue;
                    }
#pragma unroll
                    for (int j = 0; j < 4; j++) v[j] = l[k] == 0.0f ? 0.0f : v[j] * inv;
                    if (real && a.out)
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
                        if (real) {
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

template <int D>
static int launch_f32(lq_ctx* ctx, const PrefixAttnArgs& a, const PagedSeqs& s, const PrefixPlan& p) {
    const size_t smem = (size_t)PF_WARPS * PF_SLOTS * 16 * (D * 4 + 64);
    const int rc = ensure_func_smem(ctx, (const void*)prefix_attn_f32_kernel<D>, smem);
    if (rc) return rc;
    return launch_kernel(ctx, prefix_attn_f32_kernel<D>, dim3((unsigned)std::min(ctx->sm_count, p.workers)),
                         dim3(PF_WARPS * 32), smem, "prefix_attn_f32", a, s, p);
}

int launch_prefix_attn_f32(lq_ctx* ctx, const PrefixAttnArgs& a, const PagedSeqs& s, const PrefixPlan& p, int D) {
    return D == 64 ? launch_f32<64>(ctx, a, s, p) : launch_f32<128>(ctx, a, s, p);
}

}  // namespace lq
