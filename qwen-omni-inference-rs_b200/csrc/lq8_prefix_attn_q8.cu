// lq8_prefix_attn_q8.cu -- the shared-prefix attention for 8-bit caches with few query rows a kv head (a
// decode step): K and V stream through warps that turn codes into products without leaving registers.
//
// A worker of the line (lq8_prefix_plan.cuh) is a warp. It takes 8 NR stacked query rows through its
// steps of 32 positions:
//   S = Q K^T   in whole numbers: a row of Q is rounded to 16 bits of its largest value (within
//               amax / 65024) and split into two bytes, the high ones rows 0-7 of the left operand of
//               mma.sync m16n8k32 (s8), the low ones rows 8-15, so that K's codes are the right operand
//               as they lie in memory; 256 hi + lo is exact in 32 bits
//   P = exp2(S f - m), l = sum P, in f32, with f = q's and K's scale
//   O += P' V   mma.sync m16n8k16 (fp16, 16 rows), with V's codes exact in fp16 and P' = exp2(S f + log2
//               V's scale - m' + 7): m' is a running maximum of its own, so that the weights that count
//               lie between 2^7 and 2^15 whatever the scales are, and a rounding is 2^-12 (below 2^-21 of the
//               largest, an absolute 2^-32 of it). The accumulators of Q K^T lie just as the left
//               operand of this product wants them.
// The scales of 16 positions (a block's or a part of one) are one number each, so that they cost
// nothing a code and no more than an addend a score.
// K and V come by TMA, 32 positions a stage, into a ring of the warp's own; swizzled so that a warp's
// 16-byte reads meet every bank once. A lane reads 16 bytes of K of one position and of V of one
// position at a time; which dims they are is the same for all positions, and free. No warp waits
// for another. Page ids and scales of 512 positions at a time lie in the warp's lanes, loaded a
// batch ahead.
// TMA loads here read only this GPU's memory and use no multicast.
#include "lq8_async.cuh"
#include "lq8_fused.cuh"
#include "lq8_paged_q8.cuh"
#include "lq8_prefix_attn.cuh"
#include "lq8_prefix_plan.cuh"
#include "lq8_tma.cuh"

#include <cuda_fp16.h>

#include <algorithm>

namespace lq {

constexpr int PQ_WARPS = PREFIX_ATTN_Q8_WARPS;
constexpr int PQ_SCAN = 256;
constexpr int PQ_STAGE = 32;               // positions of a stage
constexpr int PQ_BATCH = 512;              // positions whose pages and scales lie in the lanes
constexpr int ERR_PQ_WAIT = 96;            // a copy did not land
constexpr int pq_slots(int D) { return D == 64 ? 6 : 3; }

__device__ __forceinline__ float pq_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// a b with s32 sums (FIRST: from zero), c += a b with f32 sums
template <bool FIRST>
__device__ __forceinline__ void pq_mma_s8(int c[4], const uint32_t a[4], uint32_t b0, uint32_t b1) {
    if constexpr (FIRST)
        asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
            : "=r"(c[0]), "=r"(c[1]), "=r"(c[2]), "=r"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "r"(0));
    else
        asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void pq_mma_f16(float c[4], const uint32_t a[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// two bytes of w (sel 0x4140: the lower ones), which are codes + 128, as a pair of fp16: 0x6400 + b has the
// value 1024 + b; less 1152 that is the code, exactly
__device__ __forceinline__ uint32_t pq_f16(uint32_t w, uint32_t sel) {
    const uint32_t x = __byte_perm(w, 0x64646464u, sel), bias = 0x64806480u;
    const __half2 d = __hsub2(*reinterpret_cast<const __half2*>(&x), *reinterpret_cast<const __half2*>(&bias));
    return *reinterpret_cast<const uint32_t*>(&d);
}
__device__ __forceinline__ uint32_t pq_pack(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float pq_max_nan(float a, float b) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}

// D / 4 dims (from dim t4 D / 4) of a row; every lane calls it, those of real rows write
template <int D>
__device__ __forceinline__ void pq_store(const PrefixAttnArgs& a, int tok, int h, int t4, const float* v, bool real) {
    if constexpr (D == 128) {
        if (real) pa_store32<__nv_bfloat16, D>(a, tok, h, 32 * t4, v);
    } else {
        if (a.out && real) {
            uint4* const o = reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(a.out) + (int64_t)tok * a.out_stride + (int64_t)h * D + 16 * t4);
#pragma unroll
            for (int j = 0; j < 2; j++)
                o[j] = make_uint4(pack_bf16x2(v[8 * j], v[8 * j + 1]), pack_bf16x2(v[8 * j + 2], v[8 * j + 3]),
                                  pack_bf16x2(v[8 * j + 4], v[8 * j + 5]), pack_bf16x2(v[8 * j + 6], v[8 * j + 7]));
        }
        if (a.xq) {  // two lanes hold a block of 32 dims
            float amax = 0.0f, d, id;
#pragma unroll
            for (int j = 0; j < 16; j++) amax = fmaxf(amax, fabsf(v[j]));
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
            q8_scale(amax, d, id);
            const int64_t at = ((int64_t)tok * a.n_heads + h) * D + 16 * t4;
            uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
            for (int j = 0; j < 16; j++) w[j / 4] |= (uint32_t)(q8_quant(v[j], id) & 0xFF) << (8 * (j % 4));
            if (real) {
                if (t4 % 2 == 0) a.xd[at / 32] = f2h(d);
                *reinterpret_cast<uint4*>(a.xq + at) = make_uint4(w[0], w[1], w[2], w[3]);
            }
        }
    }
}

struct PqArgs {
    PrefixAttnArgs a;
    PagedSeqs s;
    PrefixPlan p;
    PagedQ8 c;
};

template <int D, int NR>
__global__ void __launch_bounds__(PQ_WARPS * 32, 1)
prefix_attn_q8_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                      const __grid_constant__ PqArgs g) {
    constexpr int SLOTS = pq_slots(D), HALF = PQ_STAGE * D, SLOT = 2 * HALF;  // bytes of K in a stage, of a stage
    constexpr int KS = D / 32, NT = D / 8;   // steps of Q K^T; column tiles of O
    const PrefixAttnArgs& a = g.a;
    const PagedSeqs& s = g.s;
    const PrefixPlan& p = g.p;
    const PagedQ8& cc = g.c;
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t full[PQ_WARPS][SLOTS];
    __shared__ int scan[PQ_SCAN + 1];
    __shared__ int4 info[PQ_SCAN];  // up to PQ_SCAN sequences: q0, q, kv, steps of a head
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, gr = lane >> 2, t4 = lane & 3;
    const uint32_t raw = smem_addr(smem_raw);
    uint8_t* const mine = smem_raw + (((raw + 1023) & ~1023u) - raw) + warp * SLOTS * SLOT;
    if (lane == 0)
        for (int i = 0; i < SLOTS; i++) mbar_init(&full[warp][i], 1);
    mbar_fence_init();
    __syncwarp();
    if (tid == 0) {
        tma_prefetch_map(&map_k);
        tma_prefetch_map(&map_v);
    }
    int slot = 0;       // of the next stage to be worked on
    unsigned ph = 0;    // and its parity
    bool ok = true;
    // Behind the kernel that takes the prefix this one need not wait for it: that one began after its
    // own wait for what came before, and let this one begin after that. It is waited for at the end.
    const bool alone = p.streams == 3;
    if (alone) pdl_wait();
    pdl_trigger();  // (after the wait: the merge reads the call's lengths before its own)
    const int per_entry = (s.n_seqs + PQ_SCAN - 1) / PQ_SCAN;
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
    for (int e = by_warp ? warp : tid; e < n_entries; e += by_warp ? PQ_WARPS : PQ_WARPS * 32) {
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
        for (int b = blockIdx.x * PQ_WARPS + warp; b < s.n_seqs; b += gridDim.x * PQ_WARPS) {
            const SeqInfo si = seq_info(a, s, b, false);
            if (si.kv < si.q) zero_rows<__nv_bfloat16, D>(a, si.q0, si.q - si.kv, lane, 32);
        }
    }
    const int worker = warp * gridDim.x + blockIdx.x;
    const int live = live_rows(s);
    const Shares line(p, so);
    if (a.prefix_len == 0)  // ranges that there are not
        for (int i = worker + line.ranges; i < p.notes; i += PQ_WARPS * gridDim.x)
            if (lane == 0) p.split[i].rows = 0;
    const int box = min(1 << s.page_shift, PQ_STAGE), boxes = PQ_STAGE / box, mask = (1 << s.page_shift) - 1;
    // column n of a tile of Q K^T is position perm(n) of its 8: with D = 64, where two positions share the
    // 128 bytes of all banks, in an order that keeps V's reads apart
    auto perm = [](int n) { return D == 128 ? n : (int)(0x65217430u >> (4 * n)) & 7; };
    const int my_k = perm(gr), my_p[2] = {perm(2 * t4), perm(2 * t4 + 1)};
    // where in a stage vector `ch` (16 bytes) of position x lies
    auto vec = [](int x, int ch) { return D == 128 ? x * 128 + ((ch ^ (x & 7)) << 4) : x * 64 + ((ch ^ ((x >> 1) & 3)) << 4); };

    if (worker >= line.ranges) {
        if (!alone) pdl_wait();
        return;
    }
    if (a.prefix_len == 0 && lane == 0) p.split[worker].rows = 0;
    __syncwarp();
#pragma unroll 1
    for (int part = 0; part < 2; part++) {
        const bool own = part;
        int step, hi;
        line.range(worker, own, step, hi);
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
            const int pos0 = tile * p.tile, pos1 = min(end * p.tile, kv_end);
            // page of the lane's 16 positions of a batch (past the end: none), and their scales
            auto page_at = [&](int x) {
                const int at = x + 16 * lane;
                int id = s.n_pages;
                if (at < pos1) {
                    id = table[at >> s.page_shift];
                    if ((unsigned)id >= (unsigned)s.n_pages) {
                        flag_error(a.err, ERR_PAGE_ID, id);
                        id = s.n_pages;  // zeros
                    }
                }
                return id;
            };
            auto scales_at = [&](int x, int id, float& ks, float& lv) {  // V's as its logarithm
                float vs = 0.0f;
                ks = 0.0f;
                if (id < s.n_pages) {
                    const int64_t at = id * cc.scale_stride + ((int64_t)kh << (s.page_shift - cc.block_shift)) +
                                       (((x + 16 * lane) & mask) >> cc.block_shift);
                    ks = cc.k_scale[at];
                    vs = cc.v_scale[at];
                }
                lv = __log2f(vs);
            };
            int pg = page_at(pos0), pg_next = page_at(pos0 + PQ_BATCH), pg_then = 0;
            int sent = 0;                                 // stages on the way or done
            const int stages = (pos1 - pos0 + PQ_STAGE - 1) / PQ_STAGE;
            int to = slot;                                // slot of the next stage to be sent
            auto send = [&](int at_batch) {               // stage `sent`; at_batch: that of pg
                const int x = sent * PQ_STAGE, in = x & (PQ_BATCH - 1);
                const int from = (x / PQ_BATCH == at_batch) ? pg : pg_next;
                // lanes 0 .. boxes - 1 bring K, the next ones V
                const int piece = lane & (boxes - 1), sub = (in >> 4) + piece * (box >> 4);
                const int id = __shfl_sync(0xffffffffu, from, sub & 31);
                if (lane == 0) mbar_expect_tx(&full[warp][to], SLOT);
                __syncwarp();
                if (lane < 2 * boxes) {
                    const bool v = lane >= boxes;
                    tma_load_4d(mine + to * SLOT + (v ? HALF : 0) + piece * box * D, v ? &map_v : &map_k, 0,
                                (pos0 + x + piece * box) & mask, kh, id, &full[warp][to]);
                }
                sent++;
                if (++to == SLOTS) to = 0;
            };
#pragma unroll 1
            for (int i = 0; i < SLOTS && i < stages; i++) send(0);
            float ks, lv, ks_next = 0.0f, lv_next = 0.0f;
            scales_at(pos0, pg, ks, lv);
            // ---- Q, in two bytes ----
            uint32_t q[NR][KS][4];
            float qf[NR];      // what a whole number of Q K^T counts for, in units of log2, without K's scale
            int vis[NR];       // positions that the row sees
#pragma unroll
            for (int r = 0; r < NR; r++) {
                const int row = min(8 * r + gr, n - 1), tok = a.group_div(row0 + row);
                const int head = kh * a.group + row0 + row - tok * a.group;
                vis[r] = own ? min(kv_end, own_visible(si, tok - si.q0)) : kv_end;
                const uint4* src = reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(a.q) + (int64_t)tok * a.q_stride +
                                                                  (int64_t)head * D + t4 * (D / 4));
                uint32_t w[KS * 4];  // D / 4 values
                uint32_t top = 0;
#pragma unroll
                for (int i = 0; i < KS; i++) {
                    const uint4 u = src[i];
                    w[4 * i] = u.x, w[4 * i + 1] = u.y, w[4 * i + 2] = u.z, w[4 * i + 3] = u.w;
                }
#pragma unroll
                for (int i = 0; i < KS * 4; i++) top = max(top, max(w[i] & 0x7fff0000u, (w[i] << 16) & 0x7fff0000u));
                top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
                const float amax = __uint_as_float(top);
                // (a row of values below 2^-100 counts as zero)
                const bool fine = amax >= 7.8886e-31f && amax < INFINITY;
                const float by = fine ? 32512.0f / amax : 0.0f;
                qf[r] = fine ? amax * (1.0f / 32512.0f) * a.scale * 1.44269504088896340736f : amax < INFINITY ? 0.0f : __uint_as_float(0x7fffffffu);
#pragma unroll
                for (int i = 0; i < KS; i++)
#pragma unroll
                    for (int h = 0; h < 2; h++) {  // four dims: two words
                        uint32_t up = 0, dn = 0;
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            const uint32_t u = w[4 * i + 2 * h + (e >> 1)];
                            const int v = __float2int_rn(__uint_as_float(e & 1 ? u & 0xffff0000u : u << 16) * by);
                            up |= (uint32_t)(((v + 128) >> 8) & 0xff) << (8 * e);
                            dn |= (uint32_t)(v & 0xff) << (8 * e);
                        }
                        q[r][i][2 * h] = up;
                        q[r][i][2 * h + 1] = dn;
                    }
            }
            int all_see = vis[0];  // positions that all of the warp's rows see
#pragma unroll
            for (int r = 1; r < NR; r++) all_see = min(all_see, vis[r]);
            all_see = __reduce_min_sync(0xffffffffu, all_see);
            // running maxima of the scores (for l) and of the scores + log2 V's scale (for O, 2^7 times as
            // large as that says), sums
            float m[NR], mv[NR], l[NR], o[NT][4];
#pragma unroll
            for (int r = 0; r < NR; r++) m[r] = mv[r] = -INFINITY, l[r] = 0.0f;
#pragma unroll
            for (int i = 0; i < NT; i++) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
#pragma unroll 1
            for (int i = 0; i < stages; i++) {
                const int x = pos0 + i * PQ_STAGE, in = (i * PQ_STAGE) & (PQ_BATCH - 1);
                if (in == 0) {
                    if (i > 0) {
                        pg = pg_next;
                        pg_next = pg_then;
                        ks = ks_next;
                        lv = lv_next;
                    }
                    pg_then = page_at(x + 2 * PQ_BATCH);
                    scales_at(x + PQ_BATCH, pg_next, ks_next, lv_next);
                }
                ok = __all_sync(0xffffffffu, mbar_wait(&full[warp][slot], ph, p.polls));
                if (!ok) {  // this copy and the later ones may not land in shared memory that is no longer this kernel's
#pragma unroll 1
                    for (int j = 0; j < sent - i; j++)
                        mbar_wait_ns(&full[warp][(slot + j) % SLOTS], slot + j < SLOTS ? ph : ph ^ 1u, 2000000000ull);
                    break;
                }
                const uint8_t* const kt = mine + slot * SLOT;
                const uint8_t* const vt = kt + HALF;
                // scores, without the factor f of the row and of 16 positions: positions 16 h + 8 t + my_p[e]
                float sc[NR][2][2][2], f[NR][2], l1[2];
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const float k1 = __shfl_sync(0xffffffffu, ks, (in >> 4) + h);
                    l1[h] = __shfl_sync(0xffffffffu, lv, (in >> 4) + h);
                    // (never so small that a masked score loses its minus infinity)
#pragma unroll
                    for (int r = 0; r < NR; r++) f[r][h] = pq_max_nan(qf[r] * k1, 1e-37f);
#pragma unroll
                    for (int t = 0; t < 2; t++) {
                        uint32_t w[KS * 2];
#pragma unroll
                        for (int j = 0; j < KS / 2; j++) {
                            const uint4 u = *reinterpret_cast<const uint4*>(kt + vec(16 * h + 8 * t + my_k, t4 * (KS / 2) + j));
                            w[4 * j] = u.x, w[4 * j + 1] = u.y, w[4 * j + 2] = u.z, w[4 * j + 3] = u.w;
                        }
#pragma unroll
                        for (int r = 0; r < NR; r++) {
                            int c[4];
                            pq_mma_s8<true>(c, q[r][0], w[0], w[1]);
#pragma unroll
                            for (int j = 1; j < KS; j++) pq_mma_s8<false>(c, q[r][j], w[2 * j], w[2 * j + 1]);
#pragma unroll
                            for (int e = 0; e < 2; e++) sc[r][h][t][e] = (float)(c[e] * 256 + c[2 + e]);
                        }
                    }
                }
                if (x + PQ_STAGE > all_see) {
#pragma unroll
                    for (int r = 0; r < NR; r++)
#pragma unroll
                        for (int j = 0; j < 8; j++)
                            if (x + 8 * (j >> 1) + my_p[j & 1] >= vis[r]) sc[r][j >> 2][(j >> 1) & 1][j & 1] = -INFINITY;
                }
                float top[NR], tov[NR];
                bool grows = i == 0;
#pragma unroll
                for (int r = 0; r < NR; r++) {
                    float a0 = fmaxf(fmaxf(sc[r][0][0][0], sc[r][0][0][1]), fmaxf(sc[r][0][1][0], sc[r][0][1][1])) * f[r][0];
                    float a1 = fmaxf(fmaxf(sc[r][1][0][0], sc[r][1][0][1]), fmaxf(sc[r][1][1][0], sc[r][1][1][1])) * f[r][1];
                    top[r] = fmaxf(a0, a1);
                    tov[r] = fmaxf(a0 + l1[0], a1 + l1[1]);
                    // (each lane for itself: a row's lanes follow the one that looks up its own)
                    grows |= top[r] > m[r] + 8.0f || tov[r] > mv[r] + 8.0f;
                }
                // a maximum that grew by less than 2^8 stays: p <= 2^8 costs an f32 sum nothing, and
                // 2^15 is still an fp16
                if (__any_sync(0xffffffffu, grows)) {
#pragma unroll
                    for (int r = 0; r < NR; r++) {
#pragma unroll
                        for (int d = 1; d < 4; d <<= 1) {
                            top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], d));
                            tov[r] = fmaxf(tov[r], __shfl_xor_sync(0xffffffffu, tov[r], d));
                        }
                        const float mn = fmaxf(m[r], top[r]), vn = fmaxf(mv[r], tov[r]);
                        l[r] *= mn == -INFINITY ? 1.0f : pq_ex2(m[r] - mn);
                        const float fo = vn == -INFINITY ? 1.0f : pq_ex2(mv[r] - vn);
                        m[r] = mn;
                        mv[r] = vn;
#pragma unroll
                        for (int j = 0; j < NT; j++) o[j][2 * r] *= fo, o[j][2 * r + 1] *= fo;
                    }
                }
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    uint32_t pa[4] = {0, 0, 0, 0};  // rows 0-7 and 8-15 of either eight positions
#pragma unroll
                    for (int r = 0; r < NR; r++) {
                        const float neg = m[r] == -INFINITY ? 0.0f : -m[r];
                        const float add = mv[r] == -INFINITY ? 0.0f : l1[h] - mv[r] + 7.0f;
#pragma unroll
                        for (int t = 0; t < 2; t++) {
                            l[r] += pq_ex2(fmaf(sc[r][h][t][0], f[r][h], neg)) + pq_ex2(fmaf(sc[r][h][t][1], f[r][h], neg));
                            pa[2 * t + r] = pq_pack(pq_ex2(fmaf(sc[r][h][t][0], f[r][h], add)), pq_ex2(fmaf(sc[r][h][t][1], f[r][h], add)));
                        }
                    }
                    // V of the four positions that this lane's part of the right operand holds
                    constexpr int VW = D / 32;  // words of a position
                    uint32_t w[4][VW];
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const int at = 16 * h + 8 * (j >> 1) + my_p[j & 1];
                        if constexpr (D == 128) {
                            const uint4 u = *reinterpret_cast<const uint4*>(vt + vec(at, gr));
                            w[j][0] = u.x, w[j][1] = u.y, w[j][2] = u.z, w[j][3] = u.w;
                        } else {
                            const uint2 u = *reinterpret_cast<const uint2*>(vt + vec(at, gr >> 1) + (gr & 1) * 8);
                            w[j][0] = u.x, w[j][1] = u.y;
                        }
#pragma unroll
                        for (int k = 0; k < VW; k++) w[j][k] ^= 0x80808080u;
                    }
#pragma unroll
                    for (int j = 0; j < VW; j++)
#pragma unroll
                        for (int e = 0; e < 2; e++) {  // dims 4 j + 2 e, 4 j + 2 e + 1
                            const uint32_t x0 = __byte_perm(w[0][j], w[1][j], e ? 0x7362 : 0x5140);
                            const uint32_t x1 = __byte_perm(w[2][j], w[3][j], e ? 0x7362 : 0x5140);
                            pq_mma_f16(o[4 * j + 2 * e], pa, pq_f16(x0, 0x4140), pq_f16(x1, 0x4140));
                            pq_mma_f16(o[4 * j + 2 * e + 1], pa, pq_f16(x0, 0x4342), pq_f16(x1, 0x4342));
                        }
                }
                __syncwarp();  // (read by every lane)
                if (++slot == SLOTS) slot = 0, ph ^= 1;
                if (sent < stages) send(i * PQ_STAGE / PQ_BATCH);
            }
            if (!ok) {
                flag_error(a.err, ERR_PQ_WAIT, worker);
                break;
            }
            // ---- its result: row gr of each eight, D / 4 dims from t4 (D / 4) on ----
#pragma unroll
            for (int r = 0; r < NR; r++) {
                l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
                l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
                const int row = 8 * r + gr;
                const bool real = row < n;
                const int tok = a.group_div(row0 + min(row, n - 1)), head = kh * a.group + row0 + min(row, n - 1) - tok * a.group;
                const int64_t at = own ? p.own_slot(item, worker, begins) : item + worker;
                const int cap = p.cap[part];
                // O in the units of m
                const float back = m[r] == -INFINITY || mv[r] == -INFINITY ? 0.0f : pq_ex2(mv[r] - 7.0f - m[r]);
                float v[D / 4];
#pragma unroll
                for (int j = 0; j < NT; j++) {
                    v[j] = o[j][2 * r] * back;
                    v[NT + j] = o[j][2 * r + 1] * back;
                }
                if (!whole) {
                    if (real) {
                        if (t4 == 0) p.ml[part][at * cap + row] = make_float2(m[r], l[r]);
#pragma unroll
                        for (int j = 0; j < D / 16; j++)
                            reinterpret_cast<float4*>(p.o[part])[(at * (D / 4) + t4 * (D / 16) + j) * cap + row] =
                                make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
                    }
                    continue;
                }
                const float inv = l[r] > 0.0f ? 1.0f / l[r] : l[r];
#pragma unroll
                for (int j = 0; j < D / 4; j++) v[j] = l[r] == 0.0f ? 0.0f : v[j] * inv;
                pq_store<D>(a, tok, head, t4, v, real);
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
    if (!alone) pdl_wait();
}

template <int D, int NR>
static int launch_q8(lq_ctx* ctx, const PqArgs& g) {
    const int page = 1 << g.s.page_shift;
    const uint64_t dims[4] = {(uint64_t)D, (uint64_t)page, (uint64_t)g.c.n_kv, (uint64_t)g.s.n_pages};
    const uint64_t strides[3] = {(uint64_t)D, (uint64_t)D * page, (uint64_t)g.c.page_stride};
    const uint32_t box[4] = {D, (uint32_t)std::min(page, PQ_STAGE), 1, 1};
    const CUtensorMapSwizzle swz = D == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B;
    CUtensorMap mk, mv;
    int rc = make_tensor_map_4d(ctx, &mk, CU_TENSOR_MAP_DATA_TYPE_UINT8, g.c.k, dims, strides, box, swz);
    if (rc) return rc;
    rc = make_tensor_map_4d(ctx, &mv, CU_TENSOR_MAP_DATA_TYPE_UINT8, g.c.v, dims, strides, box, swz);
    if (rc) return rc;
    const size_t smem = 1024 + (size_t)PQ_WARPS * pq_slots(D) * 2 * PQ_STAGE * D;
    rc = ensure_func_smem(ctx, (const void*)prefix_attn_q8_kernel<D, NR>, smem);
    if (rc) return rc;
    return launch_kernel(ctx, prefix_attn_q8_kernel<D, NR>, dim3((unsigned)std::min(ctx->sm_count, g.p.workers)),
                         dim3(PQ_WARPS * 32), smem, "prefix_attn_q8", mk, mv, g);
}

int launch_prefix_attn_q8(lq_ctx* ctx, const PrefixAttnArgs& a, const PagedSeqs& s, const PagedQ8& c, const PrefixPlan& p, int D) {
    const PqArgs g{a, s, p, c};
    if (D == 64) return p.pb == 8 ? launch_q8<64, 1>(ctx, g) : launch_q8<64, 2>(ctx, g);
    return p.pb == 8 ? launch_q8<128, 1>(ctx, g) : launch_q8<128, 2>(ctx, g);
}

}  // namespace lq
