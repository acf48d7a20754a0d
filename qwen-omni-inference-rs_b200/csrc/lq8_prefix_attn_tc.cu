// lq8_prefix_attn_tc.cu -- the shared-prefix attention for bf16 caches on the tcgen05 tensor
// cores.
//
// One CTA per SM walks its share of the line of steps (lq8_prefix_plan.cuh). It runs two flows of
// up to 128 stacked query rows, each with its own Q tile in shared memory and its own S and O
// accumulators in TMEM, so that one flow's softmax runs while the other's products do:
//   S = Q K^T   (M 128 rows, N 128 positions, K = D; Q and K from shared memory)
//   P = exp2(S c - m), running maximum m and sum l in registers, a row per thread
//   O += P V    (M 128, N = D, K = 128 positions; P bf16 in TMEM over S, V from shared memory as
//                the MN-major operand)
// O stays in TMEM for a whole segment (the steps of one item a flow takes in a row) and is
// multiplied by exp2(m_old - m_new) only when a row's maximum grew by more than 2^8: smaller
// growth leaves p <= 256, exact in the f32 sums and as good in bf16 (a relative rounding).
//
// Warps 0-3: softmax of flow 0 (TMEM lane = row = thread); warps 4-7: flow 1; warp 8: TMA
// producer, which reads the page table and brings K and V tiles page by page into a ring of 32 KB
// stages (128-byte swizzle; pages past the end come as zeros from an out-of-range coordinate);
// warp 9: TMEM allocator and MMA issuer. Per round the MMA warp issues, for each flow, P V of the
// round before and then Q K of this one: the tensor pipe works for one flow while the other is in
// its softmax. Every wait is bounded; a timeout sets the error flag and the CTA tears down.
//
// TMA loads here read only this GPU's memory and use no multicast.
#include "lq8_async.cuh"
#include "lq8_fused.cuh"
#include "lq8_prefix_plan.cuh"
#include "lq8_prefix_attn.cuh"
#include "lq8_tma.cuh"

#include <algorithm>

namespace lq {

constexpr int PA_ROWS = 128;      // rows of a flow (MMA M)
constexpr int PA_TILE = 128;      // positions of a step
constexpr int PA_STAGES = 4;
constexpr int PA_THREADS = 320;
constexpr int PA_SCAN = 1024;     // entries of the scan over the sequences
constexpr int ERR_PA_WAIT = 94;   // a wait ran out

struct PaCtl {
    uint64_t full[PA_STAGES], empty[PA_STAGES];
    uint64_t q_full[2], s_full[2], p_full[2], o_full[2], done;
    uint32_t tmem;
    int abort;
    int scan[PA_SCAN + 1];
};

__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void proxy_fence() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void tc_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_addr(bar))
                 : "memory");
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// 128-byte swizzled operand tiles of 128-byte rows, 8-row groups 1024 bytes apart; lead: distance
// of the 64-element chunks of an MN-major operand
__device__ __forceinline__ uint64_t pa_desc(uint32_t saddr, uint32_t lead) {
    return (uint64_t)((saddr >> 4) & 0x3FFF) | (uint64_t)((lead >> 4) & 0x3FFF) << 16 | (uint64_t)(1024 >> 4) << 32 |
           (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
// D f32, A and B bf16, M 128, N n; B MN-major or K-major
__host__ __device__ constexpr uint32_t pa_idesc(int n, int b_mn) {
    return (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)b_mn << 16) | ((uint32_t)(n >> 3) << 17) | (8u << 24);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, {%5, %5, %5, %5}, p;\n}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(acc), "r"(0));
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%5, %5, %5, %5}, p;\n}\n" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(acc), "r"(0));
}

#define PA_R8(r, o) "=r"(r[o]), "=r"(r[o + 1]), "=r"(r[o + 2]), "=r"(r[o + 3]), "=r"(r[o + 4]), "=r"(r[o + 5]), "=r"(r[o + 6]), "=r"(r[o + 7])
#define PA_I8(r, o) "r"(r[o]), "r"(r[o + 1]), "r"(r[o + 2]), "r"(r[o + 3]), "r"(r[o + 4]), "r"(r[o + 5]), "r"(r[o + 6]), "r"(r[o + 7])
// 32 columns of the warp's 32 TMEM lanes, a lane per thread
__device__ __forceinline__ void tmem_ld32(uint32_t* r, uint32_t addr) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
        "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : PA_R8(r, 0), PA_R8(r, 8), PA_R8(r, 16), PA_R8(r, 24)
        : "r"(addr));
}
__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,"
        "%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};" ::PA_I8(r, 0),
        PA_I8(r, 8), PA_I8(r, 16), PA_I8(r, 24), "r"(addr)
        : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// bounded wait: 2 s, or another warp of the CTA gave up
__device__ __forceinline__ bool pa_wait(PaCtl& c, uint64_t* bar, unsigned parity, int* err) {
    if (mbar_try_wait(bar, parity)) return true;
    const uint64_t t0 = global_ns();
    for (;;) {
        if (mbar_try_wait(bar, parity)) return true;
        if (*reinterpret_cast<volatile int*>(&c.abort)) return false;
        if (global_ns() - t0 > 2000000000ull) {
            *reinterpret_cast<volatile int*>(&c.abort) = 1;
            flag_error(err, ERR_PA_WAIT, 0);
            return false;
        }
    }
}

struct PaArgs {
    PrefixAttnArgs a;
    PagedSeqs s;
    PrefixPlan p;
};

// A flow's place in its part of the line. Every role walks the same sequence by itself.
struct PaCursor {
    bool own;
    int step, hi;       // steps of the part: the next one, and the flow's end
    int b, kh, rb, n_rb;
    int t, nt;          // tile of the item
    int kv_end;         // positions the item sees
    int row0, rows;     // stacked rows of the block
    SeqInfo si;

    __device__ __forceinline__ bool live() const { return step < hi; }

    __device__ __forceinline__ void set_prefix(const PaArgs& g) {
        row0 = rb * g.p.pb;
        rows = min(g.p.pb, g.s.rows * g.a.group - row0);
    }
    __device__ __forceinline__ void set_own(const PaArgs& g) {
        const OwnSteps o{g.a, g.p};
        kv_end = o.visible(si, rb);
        nt = (kv_end + PA_TILE - 1) / PA_TILE;
        row0 = si.q0 * g.a.group + rb * g.p.ob;
        rows = min(g.p.ob, si.q * g.a.group - rb * g.p.ob);
    }
    __device__ __forceinline__ void seek(const PaArgs& g, const int* scan, int per_entry, int n_entries, bool own_part,
                                         int lo, int hi_) {
        own = own_part;
        step = lo;
        hi = hi_;
        if (lo >= hi_) return;
        if (!own) {
            const int item = lo / g.p.np;
            t = lo - item * g.p.np;
            nt = g.p.np;
            kv_end = g.a.prefix_len;
            n_rb = g.p.n_rb;
            kh = item / n_rb;
            rb = item - kh * n_rb;
            b = 0;
            set_prefix(g);
            return;
        }
        int e0 = 0, e1 = n_entries;  // the last entry with scan <= lo
        while (e1 - e0 > 1) {
            const int m = (e0 + e1) >> 1;
            if (scan[m] <= lo) e0 = m;
            else e1 = m;
        }
        const OwnSteps o{g.a, g.p};
        int rest = lo - scan[e0], per = 0;
        for (b = e0 * per_entry; b < g.s.n_seqs; b++) {
            si = seq_info(g.a, g.s, b, false);
            per = o.per_head(si);
            if (rest < per * g.a.n_kv) break;
            rest -= per * g.a.n_kv;
        }
        if (b >= g.s.n_seqs) {  // lengths that changed under the kernel
            hi = step;
            return;
        }
        kh = rest / per;
        rest -= kh * per;
        n_rb = o.blocks(si);
        rb = 0;
        while (rest >= o.tiles(si, rb)) rest -= o.tiles(si, rb++);
        set_own(g);
        t = rest;
    }
    __device__ __forceinline__ void next(const PaArgs& g) {
        step++;
        if (++t < nt || step >= hi) return;
        t = 0;
        if (!own) {
            if (++rb == n_rb) rb = 0, kh++;
            set_prefix(g);
            return;
        }
        do {
            if (++rb >= n_rb) {
                rb = 0;
                if (++kh == g.a.n_kv) {
                    kh = 0;
                    do {
                        if (++b >= g.s.n_seqs) {  // lengths that changed under the kernel
                            hi = step;
                            return;
                        }
                        si = seq_info(g.a, g.s, b, false);
                        n_rb = OwnSteps{g.a, g.p}.blocks(si);
                    } while (n_rb == 0 || si.kv == 0);
                }
            }
            set_own(g);
        } while (nt == 0);
    }
    // rows of flow f: a paired block's halves, else all of them
    __device__ __forceinline__ int flow_rows(const PaArgs& g, int f) const {
        return (own ? g.p.pair_o : g.p.pair_p) ? min(PA_ROWS, max(0, rows - f * PA_ROWS)) : rows;
    }
    __device__ __forceinline__ int flow_row0(const PaArgs& g, int f) const {
        return (own ? g.p.pair_o : g.p.pair_p) ? row0 + f * PA_ROWS : row0;
    }
};

template <int D>
__global__ void __launch_bounds__(PA_THREADS, 1)
prefix_attn_tc_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                      const __grid_constant__ PaArgs g) {
    constexpr int HALVES = D / 64;
    constexpr int Q_BYTES = PA_ROWS * D * 2, KV_BYTES = PA_TILE * D * 2, HALF = 128 * 128;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_addr(smem_raw);
    uint8_t* const sm = smem_raw + (((raw + 1023) & ~1023u) - raw);
    uint8_t* const ring = sm + 2 * Q_BYTES;
    PaCtl& c = *reinterpret_cast<PaCtl*>(ring + PA_STAGES * KV_BYTES);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    int* const err = g.a.err;

    if (tid == 0) {
        for (int i = 0; i < PA_STAGES; i++) mbar_init(&c.full[i], 1), mbar_init(&c.empty[i], 1);
        for (int f = 0; f < 2; f++) {
            mbar_init(&c.q_full[f], 4);
            mbar_init(&c.s_full[f], 1);
            mbar_init(&c.p_full[f], 4);
            mbar_init(&c.o_full[f], 1);
        }
        mbar_init(&c.done, 1);
        c.abort = 0;
        mbar_fence_init();
    }
    if (warp == 8 && lane == 0) {
        tma_prefetch_map(&map_k);
        tma_prefetch_map(&map_v);
    }
    if (warp == 9) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_addr(&c.tmem)));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    pdl_trigger();
    pdl_wait();
    // own steps of every entry (a run of per_entry sequences), then their running sum
    const int per_entry = (g.s.n_seqs + PA_SCAN - 1) / PA_SCAN;
    const int n_entries = (g.s.n_seqs + per_entry - 1) / per_entry;
    const OwnSteps os{g.a, g.p};
    for (int e = tid; e < n_entries; e += PA_THREADS) {
        int n = 0;
        for (int b = e * per_entry; b < min(g.s.n_seqs, (e + 1) * per_entry); b++)
            n += os.per_head(seq_info(g.a, g.s, b, blockIdx.x == 0)) * g.a.n_kv;
        c.scan[e + 1] = n;
    }
    __syncthreads();
    if (warp == 0) {
        int run = 0;
        for (int e0 = 0; e0 < n_entries; e0 += 32) {
            int v = e0 + lane < n_entries ? c.scan[e0 + lane + 1] : 0;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int u = __shfl_up_sync(0xffffffffu, v, o);
                if (lane >= o) v += u;
            }
            if (e0 + lane < n_entries) c.scan[e0 + lane + 1] = run + v;
            run += __shfl_sync(0xffffffffu, v, 31);
        }
        if (lane == 0) c.scan[0] = 0;
    }
    tc_before();
    __syncthreads();
    tc_after();
    const uint32_t tmem = c.tmem;
    const int so = c.scan[n_entries];
    if (blockIdx.x == 0) {  // the sequences' places in the line, for the merge
        for (int e = tid; e < n_entries; e += PA_THREADS) {
            int n = c.scan[e];
            for (int b = e * per_entry; b < min(g.s.n_seqs, (e + 1) * per_entry); b++) {
                g.p.cum[b] = n;
                if (per_entry > 1) n += os.per_head(seq_info(g.a, g.s, b, false)) * g.a.n_kv;
            }
        }
        if (tid == 0) g.p.cum[g.s.n_seqs] = so;
    }
    const Line line(g.p, so);
    const int me = blockIdx.x;

    if (warp < 8) {
        // ------------------------------ softmax ------------------------------
        const int f = warp >> 2, row = tid & 127, wq = warp & 3;
        uint8_t* const sq = sm + f * Q_BYTES;
        const uint32_t t_lane = (uint32_t)(wq * 32) << 16;
        const uint32_t t_s = tmem + t_lane + f * 128, t_o = tmem + t_lane + 256 + f * 128;
        const float cs = g.a.scale * 1.44269504088896340736f;  // scores in units of log2
        unsigned s_ph = 0, o_ph = 0;
        bool ok = true;

        auto load_q = [&](const PaCursor& cu) {
            const int n = cu.flow_rows(g, f), r0 = cu.flow_row0(g, f);
            constexpr int CH = D / 8, PASS = PA_ROWS * CH / 128;
            uint4 v[PASS];
#pragma unroll
            for (int i = 0; i < PASS; i++) {
                const int r = (i * 128 + row) / CH, ch = (i * 128 + row) % CH;
                v[i] = make_uint4(0, 0, 0, 0);
                if (r < n) {
                    const int st = r0 + r, t = st / g.a.group, h = cu.kh * g.a.group + st - t * g.a.group;
                    v[i] = *reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(g.a.q) +
                                                           (int64_t)t * g.a.q_stride + (int64_t)h * D + ch * 8);
                }
            }
#pragma unroll
            for (int i = 0; i < PASS; i++) {
                const int r = (i * 128 + row) / CH, ch = (i * 128 + row) % CH;
                *reinterpret_cast<uint4*>(sq + (ch >> 3) * HALF + r * 128 + (((ch & 7) ^ (r & 7)) << 4)) = v[i];
            }
            proxy_fence();
            __syncwarp();
            if (lane == 0) mbar_arrive(&c.q_full[f]);
        };

        PaCursor cu;
        int part = 0;
        // the next step of this flow that has rows; false: none left
        auto settle = [&](bool fresh) {
            if (!fresh) cu.next(g);
            for (;;) {
                while (cu.live() && cu.flow_rows(g, f) == 0) cu.next(g);
                if (cu.live()) return true;
                if (part == 2) return false;
                int lo, hi;
                flow_range(line, g.p, me, f, part == 1, lo, hi);
                cu.seek(g, c.scan, per_entry, n_entries, part == 1, lo, hi);
                part++;
            }
        };
        cu.step = cu.hi = 0;
        bool more = settle(true);
        if (more) load_q(cu);
        while (more && ok) {
            const PaCursor it = cu;  // the segment's item and first tile
            const int n = it.flow_rows(g, f);
            const bool mine = row < n, busy = wq * 32 < n;
            int vis = it.kv_end;
            if (it.own) vis = own_visible(it.si, (it.flow_row0(g, f) + min(row, n - 1)) / g.a.group - it.si.q0);
            float m = -INFINITY, l = 0.0f;
            bool last;
            do {
                ok = pa_wait(c, &c.s_full[f], s_ph, err);
                if (!ok) break;
                s_ph ^= 1;
                tc_after();
                if (busy) {
                    float s[128];
#pragma unroll
                    for (int i = 0; i < 4; i++) tmem_ld32(reinterpret_cast<uint32_t*>(s) + 32 * i, t_s + 32 * i);
                    tmem_wait_ld();
                    const int lim = vis - cu.t * PA_TILE;
                    if (!__all_sync(0xffffffffu, lim >= PA_TILE)) {
#pragma unroll
                        for (int i = 0; i < 128; i++)
                            if (i >= lim) s[i] = -INFINITY;
                    }
                    float mx[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
                    for (int i = 4; i < 128; i++) mx[i & 3] = fmaxf(mx[i & 3], s[i]);
                    const float mt = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * cs;
                    if (cu.t == it.t) {
                        m = mt;
                    } else if (__any_sync(0xffffffffu, mt > m + 8.0f)) {
                        const float mn = fmaxf(m, mt);
                        const float k = mn == -INFINITY ? 1.0f : ex2(m - mn);
                        l *= k;
                        m = mn;
#pragma unroll 1
                        for (int i = 0; i < D; i += 32) {
                            uint32_t r[32];
                            tmem_ld32(r, t_o + i);
                            tmem_wait_ld();
#pragma unroll
                            for (int j = 0; j < 32; j++) r[j] = __float_as_uint(__uint_as_float(r[j]) * k);
                            tmem_st32(t_o + i, r);
                        }
                    }
                    const float neg = m == -INFINITY ? 0.0f : -m;
                    float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        uint32_t pk[32];
#pragma unroll
                        for (int i = 0; i < 32; i++) {
                            const float p0 = ex2(fmaf(s[64 * h + 2 * i], cs, neg));
                            const float p1 = ex2(fmaf(s[64 * h + 2 * i + 1], cs, neg));
                            sum[i & 1] += p0;
                            sum[2 + (i & 1)] += p1;
                            pk[i] = pack_bf16x2(p0, p1);
                        }
                        tmem_st32(t_s + 32 * h, pk);
                    }
                    l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
                    tmem_wait_st();
                }
                tc_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&c.p_full[f]);
                last = cu.t + 1 == cu.nt || cu.step + 1 == cu.hi;
                if (!last) cu.next(g);
            } while (!last);
            if (!ok) break;
            const int t_last = cu.t;
            more = settle(false);
            if (more) load_q(cu);
            ok = pa_wait(c, &c.o_full[f], o_ph, err);
            if (!ok) break;
            o_ph ^= 1;
            tc_after();
            if (!busy) continue;
            // ---- the segment's result: the row itself, or a partial for the merge ----
            const bool paired = it.own ? g.p.pair_o : g.p.pair_p;
            const int worker = paired ? me : 2 * me + f;
            const int item = it.own ? g.a.n_kv * os.base(it.si, it.b) + it.kh * it.n_rb + it.rb : it.kh * it.n_rb + it.rb;
            const int cap = it.own ? g.p.cap_o : g.p.cap_p;
            const int64_t at = (int64_t)(item + worker) * cap + (paired ? f * PA_ROWS : 0) + row;
            const bool whole = g.a.prefix_len == 0 && it.t == 0 && t_last + 1 == it.nt;
            const int st = it.flow_row0(g, f) + row, tok = st / g.a.group, head = it.kh * g.a.group + st - tok * g.a.group;
            const float inv = l > 0.0f ? 1.0f / l : 0.0f;
            if (mine && !whole) (it.own ? g.p.ml_o : g.p.ml_p)[at] = make_float2(m, l);
            float* const po = (it.own ? g.p.o_o : g.p.o_p) + at * D;
#pragma unroll 1
            for (int i = 0; i < D; i += 32) {
                uint32_t r[32];
                tmem_ld32(r, t_o + i);
                tmem_wait_ld();
                if (mine && !whole) {
#pragma unroll
                    for (int j = 0; j < 32; j += 4)
                        *reinterpret_cast<uint4*>(po + i + j) = make_uint4(r[j], r[j + 1], r[j + 2], r[j + 3]);
                } else if (mine) {
                    float v[32];
#pragma unroll
                    for (int j = 0; j < 32; j++) v[j] = l == 0.0f ? 0.0f : __uint_as_float(r[j]) * inv;
                    pa_store32<__nv_bfloat16, D>(g.a, tok, head, i, v);
                }
                __syncwarp();
            }
            tc_before();
        }
    } else if (warp == 8) {
        // ------------------------------ TMA producer ------------------------------
        const int page = 1 << g.s.page_shift, box = min(page, PA_TILE), boxes = PA_TILE / box;
        int slot = 0, issued = 0;
        unsigned ph = 0;
        bool ok = true;
        PaCursor cu[2];
        int pg[2] = {0, 0}, krow[2] = {0, 0}, kkh[2] = {0, 0};  // this lane's page of the flow's tile, kept from K for V
        bool live_before[2] = {false, false};
        bool paired_before = false;
        auto load = [&](const CUtensorMap* map, int pid, int prow, int kh) {
            if (!ok) return;
            ok = pa_wait(c, &c.empty[slot], ph ^ 1u, err);
            if (!ok) return;
            if (lane == 0) mbar_expect_tx(&c.full[slot], KV_BYTES);
            __syncwarp();
            uint8_t* const dst = ring + slot * KV_BYTES;
            if (lane < boxes) {
#pragma unroll
                for (int h = 0; h < HALVES; h++)
                    tma_load_4d(dst + h * HALF + lane * box * 128, map, h * 64, prow, kh, pid, &c.full[slot]);
            }
            issued++;
            if (++slot == PA_STAGES) slot = 0, ph ^= 1;
        };
        for (int part = 0; part < 2 && ok; part++) {
            const bool paired = part ? g.p.pair_o : g.p.pair_p;
            int lo[2], hi[2];
            for (int f = 0; f < 2; f++) {
                flow_range(line, g.p, me, f, part == 1, lo[f], hi[f]);
                cu[f].seek(g, c.scan, per_entry, n_entries, part == 1, lo[f], hi[f]);
            }
            const int rounds = hi[0] - lo[0];
            // round r brings V of the round before and K of this one; the last V of a part with
            // the next part's first round, or at the end
            for (int r = 0; r < rounds && ok; r++) {
                for (int f = 0; f < 2; f++) {
                    if (live_before[f] && (f == 0 || !paired_before)) load(&map_v, pg[f], krow[f], kkh[f]);
                    const bool live = cu[f].live();
                    if (live && (f == 0 || !paired)) {
                        const int pos = cu[f].t * PA_TILE + lane * box;
                        int id = g.s.n_pages;  // out of range: zeros
                        if (lane < boxes && pos < cu[f].kv_end) {
                            id = cu[f].own ? g.s.table[(int64_t)cu[f].b * g.s.table_ld + (pos >> g.s.page_shift)]
                                           : g.a.prefix_table[pos >> g.s.page_shift];
                            if (id < 0 || id >= g.s.n_pages) {
                                flag_error(err, ERR_PAGE_ID, id);
                                id = g.s.n_pages;
                            }
                        }
                        pg[f] = id;
                        krow[f] = pos & (page - 1);
                        kkh[f] = cu[f].kh;
                        load(&map_k, id, krow[f], kkh[f]);
                    }
                    live_before[f] = live;
                    if (live) cu[f].next(g);
                }
                paired_before = paired;
            }
        }
        for (int f = 0; f < 2; f++)
            if (live_before[f] && (f == 0 || !paired_before)) load(&map_v, pg[f], krow[f], kkh[f]);
        // no copy may still be landing when the CTA exits
        if (!ok) {
            for (int i = max(0, issued - PA_STAGES); i < issued; i++)
                mbar_wait_ns(&c.full[i % PA_STAGES], (unsigned)(i / PA_STAGES) & 1u, 2000000000ull);
        }
    } else {
        // ------------------------------ MMA issuer ------------------------------
        constexpr uint32_t id_qk = pa_idesc(PA_TILE, 0), id_pv = pa_idesc(D, 1);
        int slot = 0;
        unsigned ph = 0, q_ph[2] = {0, 0}, p_ph[2] = {0, 0};
        bool ok = true;
        PaCursor cu[2];
        // what the round before left to do, per flow
        bool pv[2] = {false, false}, pv_first[2] = {false, false}, pv_last[2] = {false, false};
        int pv_valid[2] = {0, 0};
        bool paired_before = false;
        int v_slot = 0, k_slot = 0;
        auto take = [&](int& where) {  // the next stage of the ring
            ok = pa_wait(c, &c.full[slot], ph, err);
            where = slot;
            if (++slot == PA_STAGES) slot = 0, ph ^= 1;
        };
        auto do_pv = [&](int f, bool other) {  // other: the second flow still reads this V
            if (f == 0 || !paired_before) {
                take(v_slot);
                if (!ok) return;
                if (pv_valid[f] < PA_TILE) {
                    // positions past the end share a page with valid ones: whatever is there
                    // (NaN times a zero probability) must not reach the product
                    uint8_t* const v = ring + v_slot * KV_BYTES;
                    for (int i = pv_valid[f] * 8 + lane; i < PA_TILE * 8; i += 32)
#pragma unroll
                        for (int h = 0; h < HALVES; h++)
                            *reinterpret_cast<uint4*>(v + h * HALF + i * 16) = make_uint4(0, 0, 0, 0);
                    proxy_fence();
                    __syncwarp();
                }
            }
            ok = pa_wait(c, &c.p_full[f], p_ph[f], err);
            if (!ok) return;
            p_ph[f] ^= 1;
            tc_after();
            if (lane == 0) {
                const uint32_t v = smem_addr(ring + v_slot * KV_BYTES);
#pragma unroll
                for (int j = 0; j < PA_TILE / 16; j++)
                    mma_ts(tmem + 256 + f * 128, tmem + f * 128 + j * 8, pa_desc(v + j * 2048, HALF), id_pv,
                           (pv_first[f] && j == 0) ? 0u : 1u);
                if (!other) tc_commit(&c.empty[v_slot]);
                if (pv_last[f]) tc_commit(&c.o_full[f]);
            }
            __syncwarp();
        };
        for (int part = 0; part < 2 && ok; part++) {
            const bool paired = part ? g.p.pair_o : g.p.pair_p;
            int lo[2], hi[2];
            bool fresh[2] = {true, true};
            for (int f = 0; f < 2; f++) {
                flow_range(line, g.p, me, f, part == 1, lo[f], hi[f]);
                cu[f].seek(g, c.scan, per_entry, n_entries, part == 1, lo[f], hi[f]);
            }
            const int rounds = hi[0] - lo[0];
            for (int r = 0; r < rounds && ok; r++) {
                const bool act0 = cu[0].live(), act1 = cu[1].live() && cu[1].flow_rows(g, 1) > 0;
                for (int f = 0; f < 2 && ok; f++) {
                    if (pv[f]) do_pv(f, paired_before && f == 0 && pv[1]);
                    if (!ok) break;
                    const bool act = f ? act1 : act0;
                    pv[f] = act;
                    if (act) {
                        if (f == 0 || !paired) take(k_slot);
                        if (!ok) break;
                        if (fresh[f] || cu[f].t == 0) {  // a new segment: its Q
                            ok = pa_wait(c, &c.q_full[f], q_ph[f], err);
                            if (!ok) break;
                            q_ph[f] ^= 1;
                        }
                        tc_after();
                        if (lane == 0) {
                            const uint32_t q = smem_addr(sm + f * Q_BYTES), k = smem_addr(ring + k_slot * KV_BYTES);
#pragma unroll
                            for (int j = 0; j < D / 16; j++) {
                                const uint32_t o = (j >> 2) * HALF + (j & 3) * 32;
                                mma_ss(tmem + f * 128, pa_desc(q + o, 16), pa_desc(k + o, 16), id_qk, j > 0 ? 1u : 0u);
                            }
                            if (!(paired && f == 0 && act1)) tc_commit(&c.empty[k_slot]);
                            tc_commit(&c.s_full[f]);
                        }
                        __syncwarp();
                        pv_first[f] = fresh[f] || cu[f].t == 0;
                        pv_last[f] = cu[f].t + 1 == cu[f].nt || cu[f].step + 1 == cu[f].hi;
                        pv_valid[f] = min(PA_TILE, cu[f].kv_end - cu[f].t * PA_TILE);
                        fresh[f] = false;
                    }
                    if (cu[f].live()) cu[f].next(g);
                }
                paired_before = paired;
            }
        }
        for (int f = 0; f < 2 && ok; f++)
            if (pv[f]) do_pv(f, paired_before && f == 0 && pv[1]);
        if (lane == 0) tc_commit(&c.done);
        __syncwarp();
        if (!mbar_wait_ns(&c.done, 0, 2000000000ull) && lane == 0) flag_error(err, ERR_PA_WAIT, 1);
    }
    tc_before();
    __syncthreads();
    tc_after();
    if (warp == 9) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
}

template <int D>
static int launch_tc(lq_ctx* ctx, const PaArgs& g) {
    const int page = 1 << g.s.page_shift;
    const uint64_t dims[4] = {(uint64_t)D, (uint64_t)page, (uint64_t)g.a.n_kv, (uint64_t)g.s.n_pages};
    const uint64_t strides[3] = {(uint64_t)D * 2, (uint64_t)D * 2 * page, (uint64_t)g.a.page_stride * 2};
    const uint32_t box[4] = {64, (uint32_t)std::min(page, PA_TILE), 1, 1};
    CUtensorMap mk, mv;
    int rc = make_tensor_map_4d(ctx, &mk, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, g.a.k, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
    if (rc) return rc;
    rc = make_tensor_map_4d(ctx, &mv, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, g.a.v, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
    if (rc) return rc;
    const size_t smem = 1024 + 2 * PA_ROWS * D * 2 + PA_STAGES * PA_TILE * D * 2 + sizeof(PaCtl);
    rc = ensure_func_smem(ctx, (const void*)prefix_attn_tc_kernel<D>, smem);
    if (rc) return rc;
    return launch_kernel(ctx, prefix_attn_tc_kernel<D>, dim3((unsigned)g.p.workers), dim3(PA_THREADS), smem,
                         "prefix_attn_tc", mk, mv, g);
}

int launch_prefix_attn_tc(lq_ctx* ctx, const PrefixAttnArgs& a, const PagedSeqs& s, const PrefixPlan& p, int D) {
    const PaArgs g{a, s, p};
    return D == 64 ? launch_tc<64>(ctx, g) : launch_tc<128>(ctx, g);
}

}  // namespace lq
