// lq8_prefix_attn_q8_decode.cu -- the shared-prefix attention for 8-bit caches with few stacked rows a kv
// head (PREFIX_ATTN_Q8_ROWS; decode steps): codes go from memory into int8 products on tcgen05 as they
// are, and no thread ever touches one.
//
// CTAs, two to an SM, which hide each other's latency, claim ranges of the line of steps (Shares in
// lq8_prefix_plan.cuh), 128 positions a step. With blocks of R = 8 or 16 rows:
//   S^T = K Q^T   kind::i8, M 128 positions, N 2 R, K 128 dims: a row of Q is rounded to 16 bits of its
//                 largest value (within amax / 65024) and split into two bytes, which are two
//                 columns; 256 high + low is exact in 32 bits. K's tile as TMA brings it.
//   a thread has one position of all rows: s = S q k_scale, t = s + log2 v_scale, u the tile's largest
//   t of each row (a warp reduction, four warps by way of shared memory), e = 2^(t - u),
//   l += e 2^(u - m) / v_scale, and e rounded to 15 bits as two bytes of P^T in shared memory
//   O^T = V^T P^T kind::i8, M 128 dims, N 2 R, K 128 positions: V's tile as TMA brings it, the
//                 MN-major operand
//   a thread has one dim of all rows: o += (256 high + low) 2^(u - m)
// m is a running maximum of u; o and l are multiplied by 2^(m_old - m_new) when it grew by more than
// 2^8. Since a tile's weights are rounded relative to its own largest one, long tails of small
// weights keep their 15 bits. S and O are double-buffered in TMEM: the next tile's S and the last tile's
// O are in the tensor pipe while a tile is in its softmax.
//
// Warps 0-3: softmax (TMEM lane = position = dim = thread); warp 4: walks the line, reads the page table
// and brings tiles page by page (128-byte swizzle; pages past the end come as zeros); warp 5: TMEM
// allocator and MMA issuer. Every wait is bounded by a number of polls; when one runs out all warps of the CTA
// leave, its copies and MMAs in flight are waited for, and the error flag is set.
// Bound: HBM with long sequences, else the latency of a tile (1900 cycles of a softmax warp: 520 for scales and
// the next tile's loads, 140 for S, 280 to read and mask it, 140 to meet, 420 for P, 200 for O, 220 for the
// sums) and of a segment's start (2 us). 64 sequences of up to 8000 positions, 64 / 8 heads of 128 dims: 88
// us of the 105 us of a call (530 MB, 6.0 TB/s, 92 % of a plain copy), the rest joins cut items; 48 of up to 4000,
// 32 / 4 heads of 64 dims: 26 us (the bytes: 7.5); 16 sequences of 4 rows with up to 8000 positions: 43
// us, where tiles of 128 rows take 61. A kernel of warps that multiplied with mma.sync took 113 us for the
// first of these.
//
// TMA loads here read only this GPU's memory and use no multicast.
#include "lq8_async.cuh"
#include "lq8_fused.cuh"
#include "lq8_paged_q8.cuh"
#include "lq8_prefix_attn.cuh"
#include "lq8_prefix_plan.cuh"
#include "lq8_tcgen05.cuh"
#include "lq8_tma.cuh"

#include <algorithm>

namespace lq {

constexpr int PD_TILE = 128;     // positions of a step
constexpr int pd_stages(int D) { return D == 64 ? 8 : 4; }  // tiles of K or V (64 KB)
constexpr int PD_THREADS = 192;
constexpr int PD_SCAN = 128;     // entries of the scan over the sequences
constexpr int ERR_PD_WAIT = 97;  // a wait ran out
constexpr int PD_CTAS = PREFIX_ATTN_Q8_CTAS;

enum { PD_OWN = 1, PD_END = 2, PD_WHOLE = 4 };
// the steps [t0, t1) of one item
struct alignas(16) PdSeg {
    int t0, t1;     // tiles
    int n;          // rows
    int flags;
    int kh, b;      // kv head; sequence (own items)
    int kv_end;     // positions the item sees
    int row0;       // first stacked row
    int voff;       // own items: the stacked row of token t sees t + voff positions
    int slot;       // slot of the partial
    int pad[2];
};

template <int R>
struct PdCtl {
    uint64_t full[pd_stages(64)], empty[pd_stages(64)], seg_full[2], seg_empty[2];
    uint64_t q_full, s_full[2], p_full[2], o_full[2], met[2], done;
    uint32_t tmem;
    int abort;
    int issued;     // copies that the producer started
    int pad;
    PdSeg seg[2];
    alignas(16) float red[2][4][R];  // a warp's maxima, and at a segment's end its sums
    alignas(16) float qf[R];         // what a whole number of S counts for, without K's scale
    int scan[PD_SCAN + 1];           // own steps before each entry
    int seq[PD_SCAN][3];             // up to so many sequences: q0, q, kv
};

struct PdArgs {
    PrefixAttnArgs a;
    PagedSeqs s;
    PrefixPlan p;
    PagedQ8 c;
};

// D s32, A and B s8, M m, N n; A MN-major or K-major
__host__ __device__ constexpr uint32_t pd_idesc(int m, int n, int a_mn) {
    return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)a_mn << 15) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
// operands of rows of `row` bytes (128 or 64), swizzled over as many, 8-row groups next to each other
template <int row>
__device__ __forceinline__ uint64_t pd_desc(uint32_t saddr) {
    return (uint64_t)((saddr >> 4) & 0x3FFF) | (uint64_t)1 << 16 | (uint64_t)(8 * row >> 4) << 32 | (uint64_t)1 << 46 |
           (uint64_t)(row == 128 ? 2 : 4) << 61;
}
// where in such an operand byte x of row r lies
template <int row>
__device__ __forceinline__ uint32_t pd_at(int r, int x) {
    return r * row + (((x >> 4) ^ (row == 128 ? r & 7 : (r >> 1) & 3)) << 4) + (x & 15);
}
__device__ __forceinline__ void mma_i8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, {%5, %5, %5, %5}, p;\n}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(acc), "r"(0));
}

// Bounded wait by a whole warp: `polls` polls (try_wait sleeps between them), or until another warp of the CTA
// gave up; then the CTA tears down and reports. The vote keeps the warp together.
__device__ __forceinline__ bool pd_wait(int* abort, uint64_t* bar, unsigned parity, int polls) {
#pragma unroll 1
    for (int i = 0; i < polls; i++) {
        if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
        if (__any_sync(0xffffffffu, *reinterpret_cast<volatile int*>(abort))) break;
    }
    *reinterpret_cast<volatile int*>(abort) = 1;
    return false;
}

// 2 R columns of the warp's 32 TMEM lanes
template <int R>
__device__ __forceinline__ void pd_ld(uint32_t* r, uint32_t addr) {
    if constexpr (R == 8) tmem_ld16(r, addr);
    else tmem_ld32(r, addr);
    tmem_wait_ld();
}

// the largest of the warp's values
__device__ __forceinline__ float pd_warp_max(float v) {
    float d;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(d) : "f"(v));
    return d;
}

// sums over the warp of R values a lane; lane 32 / R i has the i-th
template <int R>
__device__ __forceinline__ float pd_warp_sums(float* v, int lane) {
    int half = 16;
#pragma unroll
    for (int n = R / 2; n >= 1; n >>= 1, half >>= 1) {
        const bool up = lane & half;
#pragma unroll
        for (int i = 0; i < n; i++) {
            const float give = up ? v[i] : v[i + n], keep = up ? v[i + n] : v[i];
            v[i] = keep + __shfl_xor_sync(0xffffffffu, give, half);
        }
    }
    float t = v[0];
#pragma unroll
    for (int d = 16 / R; d > 0; d >>= 1) t += __shfl_xor_sync(0xffffffffu, t, d);
    return t;
}

// L: rows of a block that the softmax warps look at (operands hold R, whatever is in the others)
template <int D, int R, int L>
__global__ void __launch_bounds__(PD_THREADS, PD_CTAS)
prefix_attn_q8_decode_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                             const __grid_constant__ PdArgs g) {
    constexpr int N = 2 * R;                      // columns of S^T and O^T
    constexpr int PD_STAGES = pd_stages(D), PD_BYTES = PD_TILE * D;
    constexpr uint32_t OPERAND = N * 128;         // bytes of P^T's planes (and of Q^T's at most)
    constexpr uint32_t COLUMNS = R == 8 ? 64 : 128;
    const PrefixAttnArgs& a = g.a;
    const PagedSeqs& s = g.s;
    const PrefixPlan& p = g.p;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_addr(smem_raw);
    uint8_t* const ring = smem_raw + (((raw + 1023) & ~1023u) - raw);
    uint8_t* const q_sm = ring + PD_STAGES * PD_BYTES;
    uint8_t* const p_sm = q_sm + OPERAND;         // two of them
    PdCtl<R>& c = *reinterpret_cast<PdCtl<R>*>(p_sm + 2 * OPERAND);
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;

    if (tid == 0) {
        for (int i = 0; i < PD_STAGES; i++) mbar_init(&c.full[i], 1), mbar_init(&c.empty[i], 1);
        for (int i = 0; i < 2; i++) {
            mbar_init(&c.seg_full[i], 1);
            mbar_init(&c.seg_empty[i], 5);  // four softmax warps, MMA issuer
            mbar_init(&c.s_full[i], 1);
            mbar_init(&c.p_full[i], 4);
            mbar_init(&c.o_full[i], 1);
            mbar_init(&c.met[i], 4);
        }
        mbar_init(&c.q_full, 4);
        mbar_init(&c.done, 1);
        c.abort = c.issued = 0;
        mbar_fence_init();
    }
    if (warp == 4 && lane == 0) {
        tma_prefetch_map(&map_k);
        tma_prefetch_map(&map_v);
    }
    if (warp == 5) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&c.tmem)), "n"(COLUMNS));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    // Behind the kernel that takes the prefix this one need not wait for it: that one began after its
    // own wait for what came before, and let this one begin after that. It is waited for at the end.
    const bool alone = p.streams == 3;
    if (alone) pdl_wait();
    pdl_trigger();  // (after the wait: the merge reads the call's lengths before its own)
    unsigned claim = 0;  // the first range
    if (warp == 4 && lane == 0) claim = atomicAdd(p.claimed, 1u);
    // own steps of every entry (a run of per_entry sequences), then their running sum
    const int per_entry = (s.n_seqs + PD_SCAN - 1) / PD_SCAN;
    const int n_entries = (s.n_seqs + per_entry - 1) / per_entry;
    const OwnSteps os{a, p};
    // (Up to PD_SCAN sequences' lengths are kept. Looked up again, and with the notes for the join worked out before
    // a segment's first copy instead of behind it, 64 sequences of up to 8000 positions took 106.4 us
    // instead of 105.5, 48 of 64 dims 26.3 instead of 25.7, 2 short ones 14.1 instead of 13.8.)
    auto seq_of = [&](int b) { return per_entry == 1 ? SeqInfo{c.seq[b][0], c.seq[b][1], c.seq[b][2]} : seq_info(a, s, b, false); };
    bool fell = false;
#pragma unroll 1
    for (int e = tid; e < n_entries; e += PD_THREADS) {
        int n = 0;
#pragma unroll 1
        for (int b = e * per_entry; b < min(s.n_seqs, (e + 1) * per_entry); b++) {
            const SeqInfo si = seq_info(a, s, b, blockIdx.x == 0);
            fell |= falls(s, b);
            n += os.per_head(si) * a.n_kv;
            if (per_entry == 1) c.seq[e][0] = si.q0, c.seq[e][1] = si.q, c.seq[e][2] = si.kv;
        }
        c.scan[e + 1] = n;
    }
    fell = __syncthreads_or(fell);
    if (warp == 0) {
        int run = 0;
#pragma unroll 1
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
    const uint32_t tmem = __shfl_sync(0xffffffffu, c.tmem, 0);
    const int so = fell ? 0 : c.scan[n_entries];
    if (blockIdx.x == 0 && tid == 0) *p.own_steps = so;
    // a warp's next segment
    unsigned taken = 0;
    auto fetch = [&](PdSeg& o) {
        if (!pd_wait(&c.abort, &c.seg_full[taken & 1], (taken >> 1) & 1u, p.polls)) return false;
        const int v = reinterpret_cast<const int*>(&c.seg[taken & 1])[lane < 12 ? lane : 0];
        auto field = [&](int k) { return __shfl_sync(0xffffffffu, v, k); };  // uniform in the warp
        o.t0 = field(0), o.t1 = field(1), o.n = field(2), o.flags = field(3), o.kh = field(4), o.b = field(5);
        o.kv_end = field(6), o.row0 = field(7), o.voff = field(8), o.slot = field(9);
        __syncwarp();
        if (lane == 0) mbar_arrive(&c.seg_empty[taken & 1]);
        taken++;
        return !(o.flags & PD_END);
    };

    if (warp < 4) {
        // ------------------------------ softmax ------------------------------
        const uint32_t t_lane = tmem + ((uint32_t)(warp * 32) << 16);
        const float cs = a.scale * 1.44269504088896340736f;  // scores in units of log2
        const int mask = (1 << s.page_shift) - 1;
        int n_tile = 0;          // tiles so far (buffer and parity of S, P, O)
        unsigned meetings = 0, q_ph = 0;
        // values of the warps: each warp's to shared memory, then all of them
        auto meet = [&]() {
            __syncwarp();
            if (lane == 0) mbar_arrive(&c.met[meetings & 1]);
            const bool there = pd_wait(&c.abort, &c.met[meetings & 1], (meetings >> 1) & 1u, p.polls);
            meetings++;
            return there;
        };
        PdSeg sg;
        bool ok = true;
        float m[L], l[L], o[L];
        // this thread's dim of O: TMEM lanes are dims, or, with 64 of them, lanes 0-15 of each warp are
        const int dim = D == 128 ? tid : 16 * warp + lane;
        const bool has = D == 128 || lane < 16;
        auto finish = [&]() {    // rows of sg
#pragma unroll
            for (int r = 0; r < L; r++)
                if (r < sg.n) {
                    const float y = l[r] == 0.0f ? 0.0f : o[r] * (l[r] > 0.0f ? 1.0f / l[r] : l[r]);
                    const int st = sg.row0 + r, tok = a.group_div(st);
                    const int64_t col = (int64_t)(sg.kh * a.group + st - tok * a.group) * D + dim;
                    if (a.out && has) static_cast<__nv_bfloat16*>(a.out)[(int64_t)tok * a.out_stride + col] = __float2bfloat16_rn(y);
                    if (a.xq) {  // a warp has a block of 32 dims, or two warps do
                        float amax = warp_max(has ? fabsf(y) : 0.0f), d, id;
                        if constexpr (D == 64) {
                            const float(*const all)[R] = c.red[meetings & 1];
                            if (lane == 0) c.red[meetings & 1][warp][0] = amax;
                            ok = meet();
                            if (!ok) return;
                            amax = fmaxf(all[warp & 2][0], all[warp | 1][0]);
                        }
                        q8_scale(amax, d, id);
                        const int64_t at = (int64_t)tok * a.n_heads * D + col;
                        if (lane == 0 && dim % 32 == 0) a.xd[at / 32] = f2h(d);
                        if (has) a.xq[at] = (int8_t)q8_quant(y, id);
                    }
                }
        };
        // The next segment is begun while the last tile of one is worked on, if the producer has got
        // there: its pages and Q are on their way, then its scales (without that its start took 1.7 us, 3
        // while memory is busy).
        constexpr int TPR = 128 / R, DIMS = D / TPR;  // threads of a row of Q, dims of a thread
        const int q_row = tid / TPR, q_part = tid % TPR;
        PdSeg nx;
        bool have = false, ended = false;
        int nx_id[2] = {-1, -1};
        uint2 nx_q[DIMS / 4];
        float ks = 0.0f, vs = 1.0f;
        // Pages two tiles ahead, scales one. (A page id is looked at when its scales are asked for: looked at
        // where it is loaded, it held a tile up by a trip to memory.)
        auto page_at = [&](const PdSeg& o, int t) {
            const int32_t* const table = o.flags & PD_OWN ? s.table + (int64_t)o.b * s.table_ld : a.prefix_table;
            const int x = t * PD_TILE + tid;
            int id = -1;
            if (t < o.t1 && x < o.kv_end) id = table[x >> s.page_shift];
            return id;
        };
        auto scales_at = [&](const PdSeg& o, int t, int id) {  // of this position
            ks = 0.0f;
            vs = 1.0f;
            if ((unsigned)id < (unsigned)s.n_pages) {  // (reported by the producer)
                const int64_t at = id * g.c.scale_stride + ((int64_t)o.kh << (s.page_shift - g.c.block_shift)) +
                                   (((t * PD_TILE + tid) & mask) >> g.c.block_shift);
                ks = g.c.k_scale[at];
                vs = g.c.v_scale[at];
            }
        };
        auto begin = [&]() {
            nx_id[0] = page_at(nx, nx.t0);
            nx_id[1] = page_at(nx, nx.t0 + 1);
            const int st = nx.row0 + min(q_row, nx.n - 1), tok = a.group_div(st);
            const uint2* src = reinterpret_cast<const uint2*>(static_cast<const __nv_bfloat16*>(a.q) + (int64_t)tok * a.q_stride +
                                                              (int64_t)(nx.kh * a.group + st - tok * a.group) * D + q_part * DIMS);
#pragma unroll
            for (int i = 0; i < DIMS / 4; i++) nx_q[i] = src[i];
        };
#pragma unroll 1
        while (ok && !ended) {
            if (!have) {
                if (!fetch(nx)) break;
                begin();
                scales_at(nx, nx.t0, nx_id[0]);
            }
            have = false;
            sg = nx;
            int id_next = nx_id[1];
            // ---- Q in two bytes ----
            {
                const int r = q_row, part = q_part;
                uint32_t w[DIMS / 2], top = 0;
#pragma unroll
                for (int i = 0; i < DIMS / 4; i++) w[2 * i] = nx_q[i].x, w[2 * i + 1] = nx_q[i].y;
#pragma unroll
                for (int i = 0; i < DIMS / 2; i++) top = max(top, max(w[i] & 0x7fff0000u, (w[i] << 16) & 0x7fff0000u));
#pragma unroll
                for (int d = 1; d < TPR; d <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, d));
                const float amax = __uint_as_float(top);
                // (a row of values below 2^-100 counts as zero)
                const bool fine = amax >= 7.8886e-31f && amax < INFINITY;
                const float by = fine ? 32512.0f / amax : 0.0f;
                uint32_t up[DIMS / 4], dn[DIMS / 4];
#pragma unroll
                for (int i = 0; i < DIMS / 4; i++) {
                    up[i] = dn[i] = 0;
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const uint32_t u = w[2 * i + (e >> 1)];
                        const int v = __float2int_rn(__uint_as_float(e & 1 ? u & 0xffff0000u : u << 16) * by);
                        up[i] |= (uint32_t)(((v + 128) >> 8) & 0xff) << (8 * e);
                        dn[i] |= (uint32_t)(v & 0xff) << (8 * e);
                    }
                }
#pragma unroll
                for (int i = 0; i < DIMS / 4; i++) {
                    *reinterpret_cast<uint32_t*>(q_sm + pd_at<D>(r, part * DIMS + 4 * i)) = up[i];
                    *reinterpret_cast<uint32_t*>(q_sm + pd_at<D>(R + r, part * DIMS + 4 * i)) = dn[i];
                }
                if (part == 0) c.qf[r] = fine ? amax * (1.0f / 32512.0f) * cs : amax < INFINITY ? 0.0f : __uint_as_float(0x7fffffffu);
                proxy_fence();
                __syncwarp();
                if (lane == 0) mbar_arrive(&c.q_full);
            }
            ok = pd_wait(&c.abort, &c.q_full, q_ph, p.polls);
            if (!ok) break;
            q_ph ^= 1;
            auto seen_by = [&](int r) {  // positions that row r sees
                return sg.flags & PD_OWN ? min(sg.kv_end, max(0, a.group_div(sg.row0 + min(r, sg.n - 1)) + sg.voff)) : sg.kv_end;
            };
            const int all_see = seen_by(0);  // (the first row's token comes first)
            float w[L];                      // what the last tile's O counts for
#pragma unroll
            for (int r = 0; r < L; r++) m[r] = -INFINITY, l[r] = o[r] = w[r] = 0.0f;
            // O of the tile before
            auto take_o = [&](int k) {
                if (!pd_wait(&c.abort, &c.o_full[k & 1], (k >> 1) & 1u, p.polls)) return false;
                tc_after();
                uint32_t v[N];
                pd_ld<R>(v, t_lane + 2 * N + (k & 1) * N);
#pragma unroll
                for (int r = 0; r < L; r++) o[r] = fmaf((float)((int)v[r] * 256 + (int)v[R + r]), w[r], o[r]);
                tc_before();
                return true;
            };
#pragma unroll 1
            for (int t = sg.t0; t < sg.t1; t++, n_tile++) {
                // (a scale that is NaN comes by way of the score, to the rows that see its position, and is no factor of
                // what the others have there: fmaxf takes the least one instead)
                const float k1 = ks, lv = __log2f(max_nan(vs, PREFIX_ATTN_Q8_LEAST)), per = __frcp_rn(fmaxf(vs, PREFIX_ATTN_Q8_LEAST));
                if (t + 1 < sg.t1) {
                    scales_at(sg, t + 1, id_next);
                    id_next = page_at(sg, t + 2);
                } else if (__all_sync(0xffffffffu, mbar_test_wait(&c.seg_full[taken & 1], (taken >> 1) & 1u))) {
                    have = fetch(nx);
                    ended = !have;
                    if (have) begin();
                }
                ok = pd_wait(&c.abort, &c.s_full[n_tile & 1], (n_tile >> 1) & 1u, p.polls);
                if (!ok) break;
                tc_after();
                float e[L];
                {
                    uint32_t v[N];
                    pd_ld<R>(v, t_lane + (n_tile & 1) * N);
#pragma unroll
                    for (int r = 0; r < L; r++) e[r] = fmaf((float)((int)v[r] * 256 + (int)v[R + r]), c.qf[r] * k1, lv);
                }
                if ((t + 1) * PD_TILE > all_see) {
#pragma unroll
                    for (int r = 0; r < L; r++)
                        if (t * PD_TILE + tid >= seen_by(r)) e[r] = -INFINITY;
                }
                float* const mine = c.red[meetings & 1][warp];
                {
                    float top[L];
#pragma unroll
                    for (int r = 0; r < L; r++) top[r] = pd_warp_max(e[r]);
                    if (lane == 0) {
#pragma unroll
                        for (int r = 0; r < L; r += 4) *reinterpret_cast<float4*>(mine + r) = make_float4(top[r], top[r + 1], top[r + 2], top[r + 3]);
                    }
                }
                const float(*const all)[R] = c.red[meetings & 1];
                ok = meet();
                if (!ok) break;
                float u[L];
                bool grows = false;
#pragma unroll
                for (int r = 0; r < L; r++) {
                    u[r] = fmaxf(fmaxf(all[0][r], all[1][r]), fmaxf(all[2][r], all[3][r]));
                    grows |= u[r] > m[r] + 8.0f;
                }
                // ---- P^T: column r the high bytes, R + r the low ones ----
                uint8_t* const pt = p_sm + (n_tile & 1) * OPERAND;
#pragma unroll
                for (int r = 0; r < L; r++) {
                    e[r] = ex2(e[r] - (u[r] == -INFINITY ? 0.0f : u[r]));
                    const uint32_t v = __float_as_uint(fmaf(e[r], 32512.0f, 12582912.0f));  // (whole number in the low bits)
                    const uint32_t at = pd_at<128>(r, tid);  // (rows r and R + r swizzle alike)
                    pt[at] = (uint8_t)((v + 128) >> 8);
                    pt[at + R * 128] = (uint8_t)v;
                }
                proxy_fence();
                tc_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&c.p_full[n_tile & 1]);
                // ---- O of the tile before, then the sums ----
                if (t > sg.t0) {
                    ok = take_o(n_tile - 1);
                    if (!ok) break;
                }
                if (grows) {  // (the same in all threads: u and m are)
#pragma unroll
                    for (int r = 0; r < L; r++) {
                        const float mn = fmaxf(m[r], u[r]), f = mn == -INFINITY ? 1.0f : ex2(m[r] - mn);
                        m[r] = mn;
                        o[r] *= f;
                        l[r] *= f;
                    }
                }
#pragma unroll
                for (int r = 0; r < L; r++) {
                    const float f = m[r] == -INFINITY ? 0.0f : ex2(u[r] - m[r]);
                    l[r] = fmaf(e[r], per * f, l[r]);
                    w[r] = f * (1.0f / 32512.0f);
                }
            }
            if (!ok) break;
            if (have) scales_at(nx, nx.t0, nx_id[0]);
            ok = take_o(n_tile - 1);
            if (!ok) break;
            // ---- the segment's result: one dim of each row ----
            {
                const float sum = pd_warp_sums<L>(l, lane);
                if (lane % (32 / L) == 0) c.red[meetings & 1][warp][lane / (32 / L)] = sum;
                const float(*const all)[R] = c.red[meetings & 1];
                ok = meet();
                if (!ok) break;
#pragma unroll
                for (int r = 0; r < L; r++) l[r] = (all[0][r] + all[1][r]) + (all[2][r] + all[3][r]);
            }
            const bool own = sg.flags & PD_OWN;
            const int cap = p.cap[own];
            if (sg.flags & PD_WHOLE) {
                finish();
            } else {
#pragma unroll
                for (int r = 0; r < L; r++)
                    if (r < sg.n) {
                        if (tid == r) p.ml[own][(int64_t)sg.slot * cap + r] = make_float2(m[r], l[r]);
                        if (has) p.o[own][(((int64_t)sg.slot * (D / 4) + (dim >> 2)) * cap + r) * 4 + (dim & 3)] = o[r];
                    }
            }
        }
    } else if (warp == 4) {
        // ------------------------------ the line, and TMA ------------------------------
        const int page = 1 << s.page_shift, box = min(page, PD_TILE), boxes = PD_TILE / box;
        const Shares line(p, so);
        if (a.prefix_len == 0)  // ranges that there are not
            for (int i = blockIdx.x + line.ranges; i < p.notes; i += gridDim.x)
                if (lane == 0) p.split[i].rows = 0;
        int issued = 0, slot = 0;
        unsigned ph = 0, segs = 0;
        bool ok = true;
        auto put = [&](const PdSeg& o) {
            ok = pd_wait(&c.abort, &c.seg_empty[segs & 1], ((segs >> 1) & 1u) ^ 1u, p.polls);
            if (!ok) return;
            if (lane == 0) {
                c.seg[segs & 1] = o;
                mbar_arrive(&c.seg_full[segs & 1]);
            }
            __syncwarp();
            segs++;
        };
        auto load = [&](const CUtensorMap* map, int kh, int x, int id) {  // a tile from position x on; this lane's page
            ok = pd_wait(&c.abort, &c.empty[slot], ph ^ 1u, p.polls);
            if (!ok) return;
            if (lane == 0) mbar_expect_tx(&c.full[slot], PD_BYTES);
            __syncwarp();
            if (lane < boxes)
                tma_load_4d(ring + slot * PD_BYTES + lane * box * D, map, 0, (x + lane * box) & (page - 1), kh, id, &c.full[slot]);
            issued++;
            if (++slot == PD_STAGES) slot = 0, ph ^= 1;
        };
        int worker = (int)min(__shfl_sync(0xffffffffu, claim, 0), (unsigned)line.ranges);
#pragma unroll 1
        while (worker < line.ranges && ok) {
            if (a.prefix_len == 0 && lane == 0) p.split[worker].rows = 0;
            __syncwarp();
#pragma unroll 1
            for (int part = 0; part < 2 && ok; part++) {
                const bool own = part;
                int step, hi;
                line.range(worker, own, step, hi);
                if (step >= hi) continue;
                // the item of the first step: sequence, kv head, tile
                int b = 0, kh, rb = 0, tile, n_rb = p.n_rb, nt = p.np;
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
                        const int mid = (e0 + e1) >> 1;
                        if (c.scan[mid] <= step) e0 = mid;
                        else e1 = mid;
                    }
                    int rest = step - c.scan[e0], per = 1;
                    if (per_entry == 1) {
                        b = e0;
                        si = seq_of(b);
                        per = max(1, os.per_head(si));
                    } else {
                        // a lane looks at a sequence of the entry
#pragma unroll 1
                        for (b = e0 * per_entry; b < s.n_seqs; b += 32) {
                            int n = 0;
                            if (b + lane < s.n_seqs) {
                                si = seq_info(a, s, b + lane, false);
                                n = os.per_head(si);
                            }
                            int upto = n * a.n_kv;
#pragma unroll
                            for (int d = 1; d < 32; d <<= 1) {
                                const int u = __shfl_up_sync(0xffffffffu, upto, d);
                                if (lane >= d) upto += u;
                            }
                            const unsigned past = __ballot_sync(0xffffffffu, upto > rest);
                            if (past) {
                                const int at = __ffs(past) - 1;
                                rest -= __shfl_sync(0xffffffffu, upto - n * a.n_kv, at);
                                per = __shfl_sync(0xffffffffu, n, at);
                                si.q0 = __shfl_sync(0xffffffffu, si.q0, at);
                                si.q = __shfl_sync(0xffffffffu, si.q, at);
                                si.kv = __shfl_sync(0xffffffffu, si.kv, at);
                                b += at;
                                break;
                            }
                            rest -= __shfl_sync(0xffffffffu, upto, 31);
                        }
                    }
                    if (b >= s.n_seqs) break;  // lengths that changed under the kernel
                    kh = rest / per;
                    rest -= kh * per;
                    n_rb = os.blocks(si);
#pragma unroll 1
                    for (; rb < n_rb; rb++) {
                        const int n = os.steps(si, rb);
                        if (rest < n) break;
                        rest -= n;
                    }
                    tile = rest;
                }
#pragma unroll 1
                while (step < hi && ok) {
                    // ---- a segment: tiles [tile, end) of one item ----
                    int kv_end = a.prefix_len;
                    if (own) {
                        kv_end = os.visible(si, rb);
                        nt = (kv_end + PD_TILE - 1) / PD_TILE;
                    }
                    // (an own item counts for more steps than its tiles: a segment's beginning and end)
                    const int ns = nt + (own && nt > 0 ? p.extra : 0), upto = min(ns, tile + hi - step), end = min(nt, upto);
                    if (upto <= tile) break;  // lengths that changed under the kernel
                    if (end > tile) {
                        const int row0 = (own ? si.q0 * a.group : 0) + rb * p.pb;
                        // (a block of padding: its first row, for nothing)
                        const int n = max(1, min(p.pb, (own ? si.q : live_rows(s)) * a.group - rb * p.pb));
                        const int item = (own ? a.n_kv * os.base(si, b) : 0) + kh * n_rb + rb;
                        const bool begins = tile == 0, whole = a.prefix_len == 0 && begins && end == nt;
                        PdSeg sg;
                        sg.t0 = tile, sg.t1 = end, sg.n = n, sg.flags = (own ? PD_OWN : 0) | (whole ? PD_WHOLE : 0);
                        sg.kh = kh, sg.b = b, sg.kv_end = kv_end, sg.row0 = row0, sg.voff = own ? si.kv - si.q + 1 - si.q0 : 0;
                        sg.slot = own ? p.own_slot(item, worker, begins) : item + worker;
                        sg.pad[0] = sg.pad[1] = 0;
                        const int32_t* const table = own ? s.table + (int64_t)b * s.table_ld : a.prefix_table;
                        // Page ids of 32 / boxes tiles come with one load, while those before are in use, and are looked
                        // at when their tile's turn comes.
                        const int per = 32 / boxes;
                        auto ids_from = [&](int t) {  // lane i: the i-th page from tile t on
                            const int x = t * PD_TILE + lane * box;
                            return x < min(kv_end, end * PD_TILE) ? table[x >> s.page_shift] : -1;
                        };
                        int ids = ids_from(tile), ahead = ids_from(tile + per), base = tile;
                        auto page_of = [&](int t) {  // this lane's page of tile t, asked for in turn; none: zeros
                            if (t == base + per) ids = ahead, base = t, ahead = ids_from(t + per);
                            int id = __shfl_sync(0xffffffffu, ids, ((t - base) * boxes + lane) & 31);
                            if (lane >= boxes || t * PD_TILE + lane * box >= kv_end) {
                                id = s.n_pages;
                            } else if ((unsigned)id >= (unsigned)s.n_pages) {
                                flag_error(a.err, ERR_PAGE_ID, id);
                                id = s.n_pages;
                            }
                            return id;
                        };
                        put(sg);
                        // K of the next tile before V of this one, as the MMA warp takes them
                        int id = page_of(tile);
                        if (ok) load(&map_k, kh, tile * PD_TILE, id);
                        if (lane == 0) {  // (after the copies are on their way)
                            if (tile == 0) p.first[part][item] = worker;
                            if (end == nt) p.last[part][item] = worker;
                            if (a.prefix_len == 0 && tile == 0 && end < nt)
                                p.split[worker] = SplitItem{n, row0, kh, line.owner(line.sp + step + nt - 1)};
                        }
                        __syncwarp();
#pragma unroll 1
                        for (int t = tile; t < end && ok; t++) {
                            int id_next = id;
                            if (t + 1 < end) {
                                id_next = page_of(t + 1);
                                load(&map_k, kh, (t + 1) * PD_TILE, id_next);
                            }
                            if (ok) load(&map_v, kh, t * PD_TILE, id);
                            id = id_next;
                        }
                    }
                    // ---- the next item with a step ----
                    step += upto - tile;
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
                                si = seq_of(b);
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
            // (asked for when all of this is on its way, two tiles before it is done with)
            if (lane == 0) claim = atomicAdd(p.claimed, 1u);
            worker = (int)min(__shfl_sync(0xffffffffu, claim, 0), (unsigned)line.ranges);
        }
        PdSeg last;
        last.t0 = last.t1 = last.n = last.kh = last.b = last.kv_end = last.row0 = last.voff = last.slot = 0;
        last.pad[0] = last.pad[1] = 0;
        last.flags = PD_END;
        if (ok) put(last);
        if (lane == 0) c.issued = issued;
    } else {
        // ------------------------------ MMA issuer ------------------------------
        constexpr uint32_t id_qk = pd_idesc(128, N, 0), id_pv = pd_idesc(D, N, 1);
        int n_tile = 0, slot = 0;
        unsigned ph = 0, q_ph = 0;
        bool ok = true;
        PdSeg sg;
        const uint64_t q = pd_desc<D>(smem_addr(q_sm));
        auto take = [&]() {  // the next stage of the ring
            ok = pd_wait(&c.abort, &c.full[slot], ph, p.polls);
            const int at = slot;
            if (++slot == PD_STAGES) slot = 0, ph ^= 1;
            return at;
        };
        auto scores = [&](int k) {  // of tile k
            const int at = take();
            if (!ok) return;
            tc_after();
            const uint64_t kt = pd_desc<D>(smem_addr(ring + at * PD_BYTES));
            if (elect_one()) {
#pragma unroll
                for (int j = 0; j < D / 32; j++) mma_i8(tmem + (k & 1) * N, kt + 2 * j, q + 2 * j, id_qk, j > 0);
                tc_commit(&c.empty[at]);
                tc_commit(&c.s_full[k & 1]);
            }
            __syncwarp();
        };
#pragma unroll 1
        while (ok && fetch(sg)) {
            ok = pd_wait(&c.abort, &c.q_full, q_ph, p.polls);
            if (!ok) break;
            q_ph ^= 1;
            scores(n_tile);
#pragma unroll 1
            for (int t = sg.t0; t < sg.t1 && ok; t++, n_tile++) {
                if (t + 1 < sg.t1) scores(n_tile + 1);
                if (!ok) break;
                const int at = take();
                if (!ok) break;
                ok = pd_wait(&c.abort, &c.p_full[n_tile & 1], (n_tile >> 1) & 1u, p.polls);
                if (!ok) break;
                tc_after();
                const uint64_t v = pd_desc<D>(smem_addr(ring + at * PD_BYTES));
                const uint64_t pt = pd_desc<128>(smem_addr(p_sm + (n_tile & 1) * OPERAND));
                if (elect_one()) {
#pragma unroll
                    for (int j = 0; j < 4; j++) mma_i8(tmem + 2 * N + (n_tile & 1) * N, v + j * (32 * D >> 4), pt + 2 * j, id_pv, j > 0);
                    tc_commit(&c.empty[at]);
                    tc_commit(&c.o_full[n_tile & 1]);
                }
                __syncwarp();
            }
        }
        if (elect_one()) tc_commit(&c.done);  // (by the thread that issued the MMAs)
        __syncwarp();
        if (!mbar_wait_ns(&c.done, 0, 2000000000ull)) c.abort = 1;
    }
    tc_before();
    __syncthreads();
    tc_after();
    if (a.prefix_len == 0) {  // rows before their sequence's first position see nothing
#pragma unroll 1
        for (int b = blockIdx.x * (PD_THREADS / 32) + warp; b < s.n_seqs; b += gridDim.x * (PD_THREADS / 32)) {
            const SeqInfo si = seq_info(a, s, b, false);
            if (si.kv < si.q) zero_rows<__nv_bfloat16, D>(a, si.q0, si.q - si.kv, lane, 32);
        }
    }
    if (c.abort) {
        if (tid == 0) flag_error(a.err, ERR_PD_WAIT, blockIdx.x);
        // no copy may still be landing when the CTA exits
        if (warp == 4) {
#pragma unroll 1
            for (int i = max(0, c.issued - PD_STAGES); i < c.issued; i++)
                mbar_wait_ns(&c.full[i % PD_STAGES], (unsigned)(i / PD_STAGES) & 1u, 2000000000ull);
        }
    }
    if (warp == 5) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(COLUMNS));
    if (tid == 0) {  // the last CTA leaves the counters at zero
        __threadfence();
        if (atomicAdd(p.claimed + 1, 1u) == gridDim.x - 1) p.claimed[0] = p.claimed[1] = 0;
    }
    if (!alone) pdl_wait();
}

// =========================================================================================
// Joins the pieces of the own items that are cut, without a prefix: o = sum 2^(m_i - M) o_i /
// sum 2^(m_i - M) l_i in the order of the line, M the largest m_i. The range that begins a cut item leaves a
// note of it; a CTA takes some notes, the next one on its way meanwhile. A thread has four dims of a row
// and asks for the first eight pieces' vectors together with their maxima and sums.
// =========================================================================================
constexpr int PD_PIECES = 64;  // pieces looked at together

template <int D, int R>
__global__ void __launch_bounds__(D / 4 * R, 1024 / (D / 4 * R)) prefix_attn_q8_join_kernel(const __grid_constant__ PrefixAttnArgs a, const __grid_constant__ PrefixPlan p, int stacked) {
    constexpr int CH = D / 4, THREADS = CH * R, AHEAD = 8;
    __shared__ float2 ml[PD_PIECES][R];
    __shared__ __align__(16) float stage[R][D + 4];
    const int tid = threadIdx.x, r = tid % R, ch = tid / R, cap = p.cap[1];
    pdl_wait();
    pdl_trigger();
    const int ranges = Shares(p, *p.own_steps).ranges;
    SplitItem next{0, 0, 0, 0};
    if (blockIdx.x < p.notes) next = p.split[blockIdx.x];
#pragma unroll 1
    for (int note = blockIdx.x; note < p.notes; note += gridDim.x) {
        const SplitItem w = next;
        if (note + gridDim.x < p.notes) next = p.split[note + gridDim.x];
        // (a kernel that gave up, or lengths that changed under it, may have left notes unwritten)
        if (w.rows <= 0 || w.rows > cap || w.row0 < 0 || w.row0 > stacked - w.rows || (unsigned)w.kh >= (unsigned)a.n_kv) continue;
        const int v1 = min(max(w.item, note), ranges - 1), n = v1 - note + 1;
        auto slot = [&](int i) { return (int64_t)p.own_slot(0, note + i, i == 0); };
        const float4* const po = reinterpret_cast<const float4*>(p.o[1]) + (int64_t)ch * cap + r;
        const bool mine = r < w.rows;
        float M = -INFINITY, L = 0.0f;
        float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 1
        for (int c0 = 0; c0 < n; c0 += PD_PIECES) {
            const int m = min(PD_PIECES, n - c0);
            float4 x[AHEAD];
            auto ask = [&](int i0) {
#pragma unroll
                for (int j = 0; j < AHEAD; j++) {
                    x[j] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    if (i0 + j < m && mine) x[j] = po[slot(c0 + i0 + j) * CH * cap];
                }
            };
            ask(0);
            __syncthreads();  // (the maxima and sums before these are read no more)
            for (int i = tid; i < m * R; i += THREADS)
                ml[i / R][i % R] = i % R < w.rows ? p.ml[1][slot(c0 + i / R) * cap + i % R] : make_float2(-INFINITY, 0.0f);
            __syncthreads();
            float up = M;
            for (int i = 0; i < m; i++) up = fmaxf(up, ml[i][r].x);
            if (up != -INFINITY) {
                const float k = M == -INFINITY ? 0.0f : exp2f(M - up);
                L *= k;
                o.x *= k, o.y *= k, o.z *= k, o.w *= k;
            }
            M = up;
#pragma unroll 1
            for (int i0 = 0; i0 < m; i0 += AHEAD) {
                if (i0 > 0) ask(i0);
#pragma unroll
                for (int j = 0; j < AHEAD; j++) {
                    if (i0 + j >= m) break;
                    const float2 y = ml[i0 + j][r];
                    const float k = y.x == -INFINITY ? 0.0f : exp2f(y.x - M);
                    L = fmaf(k, y.y, L);
                    o.x = fmaf(k, x[j].x, o.x);
                    o.y = fmaf(k, x[j].y, o.y);
                    o.z = fmaf(k, x[j].z, o.z);
                    o.w = fmaf(k, x[j].w, o.w);
                }
            }
        }
        const float inv = L > 0.0f ? 1.0f / L : L;  // a row that saw nothing: zeros; NaN stays
        *reinterpret_cast<float4*>(&stage[r][4 * ch]) = make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
        __syncthreads();
        // out, a row's dims side by side
        {
            const int rr = tid / CH, e = tid % CH * 4, st = w.row0 + min(rr, w.rows - 1), tok = a.group_div(st);
            const bool on = rr < w.rows;
            const float4 v = *reinterpret_cast<const float4*>(&stage[rr][e]);
            const float y[4] = {v.x, v.y, v.z, v.w};
            const int64_t col = (int64_t)(w.kh * a.group + st - tok * a.group) * D + e;
            if (a.out && on)
                *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(a.out) + (int64_t)tok * a.out_stride + col) =
                    make_uint2(pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3]));
            if (a.xq) {
                const int64_t at = (int64_t)tok * a.n_heads * D + col;
                const uint32_t q = quant_group8(y, tid & 7, on ? a.xd + (at >> 5) : nullptr);
                if (on) *reinterpret_cast<uint32_t*>(a.xq + at) = q;
            }
        }
        __syncthreads();
    }
}

template <int D, int R>
static int launch_join(lq_ctx* ctx, const PrefixAttnArgs& a, const PrefixPlan& p, int stacked) {
    constexpr int THREADS = D / 4 * R;
    return launch_kernel(ctx, prefix_attn_q8_join_kernel<D, R>, dim3((unsigned)std::min(p.notes, 1024 / THREADS * ctx->sm_count)), dim3(THREADS), 0,
                         "prefix_attn_q8_join", a, p, stacked);
}

int launch_prefix_attn_q8_join(lq_ctx* ctx, const PrefixAttnArgs& a, const PagedSeqs& s, const PrefixPlan& p, int D) {
    const int stacked = s.rows * a.group;  // (below 2^28)
    if (D == 64) return p.pb == 8 ? launch_join<64, 8>(ctx, a, p, stacked) : launch_join<64, 16>(ctx, a, p, stacked);
    return p.pb == 8 ? launch_join<128, 8>(ctx, a, p, stacked) : launch_join<128, 16>(ctx, a, p, stacked);
}

template <int D, int R, int L>
static int launch_decode(lq_ctx* ctx, const PdArgs& g) {
    const int page = 1 << g.s.page_shift;
    const uint64_t dims[4] = {(uint64_t)D, (uint64_t)page, (uint64_t)g.c.n_kv, (uint64_t)g.s.n_pages};
    const uint64_t strides[3] = {(uint64_t)D, (uint64_t)D * page, (uint64_t)g.c.page_stride};
    const uint32_t box[4] = {D, (uint32_t)std::min(page, PD_TILE), 1, 1};
    const CUtensorMapSwizzle swz = D == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B;
    CUtensorMap mk, mv;
    int rc = make_tensor_map_4d(ctx, &mk, CU_TENSOR_MAP_DATA_TYPE_UINT8, g.c.k, dims, strides, box, swz);
    if (rc) return rc;
    rc = make_tensor_map_4d(ctx, &mv, CU_TENSOR_MAP_DATA_TYPE_UINT8, g.c.v, dims, strides, box, swz);
    if (rc) return rc;
    const size_t smem = 1024 + pd_stages(D) * PD_TILE * D + 3 * 2 * R * 128 + sizeof(PdCtl<R>);
    rc = ensure_func_smem(ctx, (const void*)prefix_attn_q8_decode_kernel<D, R, L>, smem);
    if (rc) return rc;
    return launch_kernel(ctx, prefix_attn_q8_decode_kernel<D, R, L>, dim3((unsigned)g.p.workers), dim3(PD_THREADS), smem,
                         "prefix_attn_q8_decode", mk, mv, g);
}

// rows: the most of a block. (2 short sequences, groups of 2: 14.4 us with L = 4, 15.0 with 8.)
template <int D>
static int launch_decode_rows(lq_ctx* ctx, const PdArgs& g, int rows) {
    return rows <= 4 ? launch_decode<D, 8, 4>(ctx, g) : rows <= 8 ? launch_decode<D, 8, 8>(ctx, g) : launch_decode<D, 16, 16>(ctx, g);
}

int launch_prefix_attn_q8_decode(lq_ctx* ctx, const PrefixAttnArgs& a, const PagedSeqs& s, const PagedQ8& c, const PrefixPlan& p, int D, int rows) {
    const PdArgs g{a, s, p, c};
    return D == 64 ? launch_decode_rows<64>(ctx, g, rows) : launch_decode_rows<128>(ctx, g, rows);
}

}  // namespace lq
