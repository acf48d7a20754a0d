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
// warp 9: TMEM allocator and MMA issuer; warp 11: zeros for rows that see nothing; warp 10:
// scheduler, the only one that walks the line: it hands each flow its segments (PaSeg) through a
// small ring, so the other roles' code stays short (every role walking by itself came to 300 KB of
// code, and the instruction misses took ten times the arithmetic). Per round the MMA warp issues,
// for each flow, P V of the round before and then
// Q K of this one: the tensor pipe works for one flow while the other is in its softmax. Every
// wait is bounded by a number of polls (4 us each where nothing comes, so 16 s in all; the
// tear-down's by 2 s); when one runs out, all warps of the CTA leave, its copies and MMAs in flight
// are waited for, and the error flag is set.
//
// Bound: a round of two 128-row halves at D = 128 needs 2048 cycles of the tensor pipe and as many
// of the exponentials'; it takes 3550, of which the MMA warp issues for 2880 (QK reads both operands
// from shared memory at its full rate: 86 cycles an MMA instead of 64) and waits 670 for copies and
// P. 128 sequences of 64 heads behind 32768 positions: 164 us for the prefix (837 TFLOP/s), 200 us
// with 1000 own positions; 64 sequences of 32 heads behind 8191: 51 us (3.3 TB/s); 4 chunks of 1000
// tokens behind 8192: 474 us (1047 TFLOP/s), all from cold L2, the merge in the first and last.
//
// TMA loads here read only this GPU's memory and use no multicast.
#include "lq8_async.cuh"
#include "lq8_fused.cuh"
#include "lq8_prefix_plan.cuh"
#include "lq8_prefix_attn.cuh"
#include "lq8_tma.cuh"

#include <algorithm>
#include <type_traits>

namespace lq {

constexpr int PA_ROWS = 128;      // rows of a flow (MMA M)
constexpr int PA_TILE = 128;      // positions of a step
// stages of the ring: 128 KB for either head dimension's tiles of 32 and 16 KB, or what is left
constexpr int pa_stages(int D) { return D == 64 ? 10 : 4; }
constexpr int PA_THREADS = 384;   // warps 0-7 softmax, 8 TMA, 9 MMA, 10 scheduler, 11 empty rows
// registers: 384 x 168 at launch = 256 x 216 for the softmax warps + 128 x 72 for the others
constexpr int PA_REGS = 216, PA_REGS_LOW = 72;
constexpr int PA_SCAN = 512;      // entries of the scan over the sequences
constexpr int PA_BATCH = 16;      // segments a flow gets at a time, worked out by a lane each
constexpr int PA_FEW = 8;         // rows up to which the four warps of a flow share a tile's columns
constexpr int ERR_PA_WAIT = 94;   // a wait ran out

enum { SEG_OWN = 1, SEG_PAIRED = 2, SEG_END = 4, SEG_WHOLE = 8, SEG_HALF = 16 };  // HALF: the second of a block
// the steps [t0, t1) of one item, for one flow
struct alignas(16) PaSeg {
    int t0, t1;     // tiles
    int n;          // rows of the flow (0: it sits this segment out, round by round)
    int flags;
    int kh, b;      // kv head; sequence (own items)
    int kv_end;     // positions the item sees (own items: from the chain's first tile on)
    int row0;       // first stacked row
    int voff;       // own items: the stacked row of token t sees t + voff positions
    int slot;       // slot of the partial
    int n1;         // paired: rows of the second half
    int pad;
};

struct PaCtl {
    uint64_t full[pa_stages(64)], empty[pa_stages(64)];
    uint64_t seg_full[2][2], seg_empty[2][2];  // per flow: two batches of segments
    uint64_t q_full[2], s_full[2], p_full[2], o_full[2], done;
    uint32_t tmem;
    int abort;
    int issued;     // copies that the producer started
    int agreed[2];  // per flow: segments of few rows that its warps went on with, or -1
    int seg_n[2][2];
    PaSeg seg[2][2][PA_BATCH];
    float2 few_ml[2][4][PA_FEW];
    alignas(16) float few_o[2][4][PA_FEW][36];  // 32 dims a row, padded against bank conflicts
    int4 info[PA_SCAN];     // up to PA_SCAN sequences: q0, q, kv, steps of a head
    int scan[PA_SCAN + 1];  // own steps before each entry
};

__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void proxy_fence() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void tc_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_addr(bar))
                 : "memory");
}
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(p));
    return p != 0;
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
__device__ __forceinline__ void tmem_ld16(uint32_t* r, uint32_t addr) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : PA_R8(r, 0), PA_R8(r, 8)
        : "r"(addr));
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::PA_I8(r, 0),
        PA_I8(r, 8), "r"(addr)
        : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

constexpr int PA_POLLS = 1 << 22;
// Bounded wait by a whole warp: PA_POLLS polls (try_wait sleeps between them), or until another warp
// of the CTA gave up; then the CTA tears down and reports. Every lane polls for itself, and the
// vote at the end has the warp go one way: a lane that went on alone would be missing in the
// other's collective instructions. A softmax thread looks at the flag first: with the poll first, 128
// sequences behind 32768 positions took 212 us instead of 202.
__device__ __forceinline__ bool pa_wait(PaCtl& c, uint64_t* bar, unsigned parity) {
    bool there = false;
#pragma unroll 1
    for (int i = 0; i < PA_POLLS && !*reinterpret_cast<volatile int*>(&c.abort); i++)
        if (mbar_try_wait(bar, parity)) {
            there = true;
            break;
        }
    if (__all_sync(0xffffffffu, there)) return true;
    *reinterpret_cast<volatile int*>(&c.abort) = 1;
    return false;
}
// The same by a whole warp, whose control flow the vote keeps uniform: tcgen05.mma and TMA take
// their operands from uniform registers, and moving them there lane by lane made the issue of an
// MMA cost twice its execution. These poll first (202 -> 200 us, a chunk of 2048 tokens 222 -> 218).
// Waits for segments have a limit from the call (a limit from there in every wait: 1 us more).
__device__ __forceinline__ bool pa_wait_warp(PaCtl& c, uint64_t* bar, unsigned parity, int polls = PA_POLLS) {
#pragma unroll 1
    for (int i = 0; i < polls; i++) {
        if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
        if (__any_sync(0xffffffffu, *reinterpret_cast<volatile int*>(&c.abort))) break;
    }
    *reinterpret_cast<volatile int*>(&c.abort) = 1;
    return false;
}
template <typename T>
__device__ __forceinline__ void exchange(T& a, T& b) {
    const T t = a;
    a = b;
    b = t;
}

__device__ __forceinline__ float max3(float a, float b, float c) {  // NaN when one of them is
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ float max_nan(float a, float b) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}

struct PaArgs {
    PrefixAttnArgs a;
    PagedSeqs s;
    PrefixPlan p;
};

__device__ __forceinline__ int warp_scan(int v, int lane) {  // inclusive sum
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += u;
    }
    return v;
}

// steps of one head of a sequence, by a warp
__device__ __forceinline__ int per_head_warp(const OwnSteps& o, const SeqInfo& si, int lane) {
    const int n_rb = o.blocks(si);
    int n = 0;
#pragma unroll 1
    for (int rb = lane; rb < n_rb; rb += 32) n += o.steps(si, rb);
    return __reduce_add_sync(0xffffffffu, n);
}

__device__ __forceinline__ SeqInfo pa_seq(const PaArgs& g, const PaCtl& c, int b) {
    if (g.s.n_seqs > PA_SCAN) return seq_info(g.a, g.s, b, false);
    const int4 v = c.info[b];
    return SeqInfo{v.x, v.y, v.z};
}

// PP, PO: blocks of the prefix / of a sequence's own rows are two halves of 128 rows that share
// their K and V tiles
template <int D, bool PP, bool PO>
__global__ void __launch_bounds__(PA_THREADS, 1)
prefix_attn_tc_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                      const __grid_constant__ PaArgs g) {
    constexpr int HALVES = D / 64, STAGES = pa_stages(D);
    constexpr int Q_BYTES = PA_ROWS * D * 2, KV_BYTES = PA_TILE * D * 2, HALF = 128 * 128;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_addr(smem_raw);
    uint8_t* const sm = smem_raw + (((raw + 1023) & ~1023u) - raw);
    uint8_t* const ring = sm + 2 * Q_BYTES;
    PaCtl& c = *reinterpret_cast<PaCtl*>(ring + STAGES * KV_BYTES);
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    int* const err = g.a.err;

    if (tid == 0) {
        for (int i = 0; i < STAGES; i++) mbar_init(&c.full[i], 1), mbar_init(&c.empty[i], 1);
#pragma unroll 1
        for (int f = 0; f < 2; f++) {
            mbar_init(&c.q_full[f], 4);
            mbar_init(&c.s_full[f], 1);
            mbar_init(&c.p_full[f], 4);
            mbar_init(&c.o_full[f], 1);
            c.agreed[f] = 0;
            for (int i = 0; i < 2; i++) {
                mbar_init(&c.seg_full[f][i], 1);
                mbar_init(&c.seg_empty[f][i], 6);  // four softmax warps, producer, MMA issuer
            }
        }
        mbar_init(&c.done, 1);
        c.abort = c.issued = 0;
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
    pdl_wait();
    pdl_trigger();  // (after the wait: the merge reads the call's lengths before its own)
    // own steps of every entry (a run of per_entry sequences), then their running sum; a warp looks
    // at a sequence of many row blocks, else a thread
    const int per_entry = (g.s.n_seqs + PA_SCAN - 1) / PA_SCAN;
    const int n_entries = per_entry == 1 ? g.s.n_seqs : (g.s.n_seqs + per_entry - 1) / per_entry;
    const OwnSteps os{g.a, g.p};
    const bool by_warp = PO && per_entry == 1 && g.a.max_q * g.a.group > 4 * g.p.ob;
    bool fell = false;
#pragma unroll 1
    for (int e = by_warp ? warp : tid; e < n_entries; e += by_warp ? PA_THREADS / 32 : PA_THREADS) {
        int n = 0;
#pragma unroll 1
        for (int b = e * per_entry; b < min(g.s.n_seqs, (e + 1) * per_entry); b++) {
            const SeqInfo si = seq_info(g.a, g.s, b, blockIdx.x == 0);
            fell |= falls(g.s, b);
            const int per = !PO ? (si.q > 0 ? os.steps(si, 0) : 0) : by_warp ? per_head_warp(os, si, lane) : os.per_head(si);
            n += per * g.a.n_kv;
            if (per_entry == 1) c.info[b] = make_int4(si.q0, si.q, si.kv, per);
        }
        c.scan[e + 1] = n;
    }
    fell = __syncthreads_or(fell);
    if (warp == 0) {
        int run = 0;
#pragma unroll 1
        for (int e0 = 0; e0 < n_entries; e0 += 32) {
            const int v = warp_scan(e0 + lane < n_entries ? c.scan[e0 + lane + 1] : 0, lane);
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
    if (blockIdx.x == 0 && tid == 0) *g.p.own_steps = so;  // for the merge
    const int me = blockIdx.x, polls = g.p.polls;
    // own items count positions from the first tile of the prefix they begin with, whose last tile
    // may be partly empty
    const int chain = PO ? g.p.chain : 0;
    // a warp's place in the segments of a flow
    struct Feed {
        int i = 0, n = 0;   // entry of the batch, entries
        unsigned k = 0;     // batches taken
    };
    auto fetch = [&](int f, Feed& d, PaSeg& o) {
        if (d.i == d.n) {
            if (d.k > 0) {
                __syncwarp();
                if (lane == 0) mbar_arrive(&c.seg_empty[f][(d.k - 1) & 1]);
            }
            if (!pa_wait_warp(c, &c.seg_full[f][d.k & 1], (d.k >> 1) & 1u, polls)) return false;
            d.n = __shfl_sync(0xffffffffu, c.seg_n[f][d.k & 1], 0);
            d.i = 0;
            d.k++;
        }
        const int v = reinterpret_cast<const int*>(&c.seg[f][(d.k - 1) & 1][d.i++])[lane < 12 ? lane : 0];
        auto field = [&](int k) { return __shfl_sync(0xffffffffu, v, k); };  // uniform in the warp
        o.t0 = field(0), o.t1 = field(1), o.n = field(2), o.flags = field(3);
        o.kh = field(4), o.b = field(5), o.kv_end = field(6), o.row0 = field(7);
        o.voff = field(8), o.slot = field(9), o.n1 = field(10);
        return true;
    };
    // Q of a flow: up to 64 rows take one half of the buffer and the next segment's the other, up to
    // PA_FEW rows (in every 32) 8 rows side by side, so that they load a segment ahead; the MMA's
    // other rows read whatever lies there
    auto q_offset = [](const PaSeg& o, unsigned turn) {
        return o.n <= PA_FEW ? (turn & 1) * 1024u : o.n <= PA_ROWS / 2 ? (turn & 1) * (HALF / 2) : 0u;
    };
    auto q_ahead = [](const PaSeg& now, const PaSeg& then) {
        return max(now.n, then.n) <= PA_FEW || (min(now.n, then.n) > PA_FEW && max(now.n, then.n) <= PA_ROWS / 2);
    };

    if (warp < 8) {
        // ------------------------------ softmax ------------------------------
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(PA_REGS));
        const int f = warp >> 2, row = tid & 127, wq = warp & 3;
        const uint32_t sq = smem_addr(sm + f * Q_BYTES);
        const uint32_t t_lane = (uint32_t)(wq * 32) << 16;
        const uint32_t t_s = tmem + t_lane + f * 128, t_o = tmem + t_lane + 256 + f * 128;
        const float cs = g.a.scale * 1.44269504088896340736f;  // scores in units of log2
        unsigned s_ph = 0, o_ph = 0, turn = 0;
        int joint = 0;  // segments of few rows
        Feed feed;

        // The next segment with rows: NX_NONE when there is none (or a wait ran out). Looked for
        // ahead of time, it must not wait for the scheduler (NX_LATER), which may itself wait until
        // the other warps are through with this segment.
        enum { NX_NONE, NX_SEG, NX_LATER };
        PaSeg nx;
        auto next = [&](bool ahead) {
            do {
                if (ahead && feed.i == feed.n &&
                    !__all_sync(0xffffffffu, mbar_try_wait(&c.seg_full[f][feed.k & 1], (feed.k >> 1) & 1u)))
                    return NX_LATER;
                if (!fetch(f, feed, nx) || (nx.flags & SEG_END)) return NX_NONE;
            } while (nx.n == 0);
            return NX_SEG;
        };
        auto q_start = [&]() {  // its Q on the way to shared memory
            const uint32_t base = sq + q_offset(nx, turn++);
            constexpr int CH = D / 8;
            const int copies = nx.n <= PA_FEW ? 4 : 1;  // few rows: one copy for each warp's lanes
#pragma unroll 1
            for (int i = row; i < nx.n * CH * copies; i += 128) {
                const int rr = i / CH, ch = i % CH, r = copies == 4 ? rr >> 2 : rr, t = g.a.group_div(nx.row0 + r);
                const int h = nx.kh * g.a.group + nx.row0 + r - t * g.a.group;
                const int at = copies == 4 ? (rr & 3) * 32 + r : r;
                const uint32_t dst = base + (ch >> 3) * HALF + at * 128 + (((ch & 7) ^ (at & 7)) << 4);
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst),
                             "l"(static_cast<const __nv_bfloat16*>(g.a.q) + (int64_t)t * g.a.q_stride + h * D + ch * 8));
            }
        };
        auto q_finish = [&]() {
            asm volatile("cp.async.wait_all;" ::: "memory");
            proxy_fence();
            __syncwarp();
            if (lane == 0) mbar_arrive(&c.q_full[f]);
        };

        int more = next(false);
        if (more == NX_SEG) {
            q_start();
            q_finish();
        }
        while (more == NX_SEG) {
            const PaSeg sg = nx;
            bool early = false;
            const bool few = sg.n <= PA_FEW;
            const int my_row = few ? lane : row;
            const int st = sg.row0 + min(my_row, sg.n - 1), tok = g.a.group_div(st);
            const bool mine = my_row < sg.n, busy = few || wq * 32 < sg.n;
            const int vis = sg.flags & SEG_OWN ? chain * PA_TILE + max(0, tok + sg.voff) : sg.kv_end;
            float m = -INFINITY, l = 0.0f;
            int t = sg.t0;
#pragma unroll 1
            for (; t < sg.t1; t++) {
                if (!pa_wait(c, &c.s_full[f], s_ph)) break;
                s_ph ^= 1;
                tc_after();
                if (busy) {
                    const int lim = (t < chain ? g.a.prefix_len : vis) - t * PA_TILE;  // columns this row sees
                    // a larger maximum: when a row's grew by more than 2^8, l and O follow
                    auto raise = [&](float mt) {
                        mt *= cs;
                        if (t == sg.t0) {
                            m = mt;
                        } else if (__any_sync(0xffffffffu, mine && !(mt <= m + 8.0f))) {  // (others hold anything)
                            const float mn = max_nan(m, mt);
                            const float k = mn == -INFINITY ? 1.0f : ex2(m - mn);
                            l *= k;
                            m = mn;
#pragma unroll 1
                            for (int i = 0; i < D; i += 16) {
                                uint32_t r[16];
                                tmem_ld16(r, t_o + i);
                                tmem_wait_ld();
#pragma unroll
                                for (int j = 0; j < 16; j++) r[j] = __float_as_uint(__uint_as_float(r[j]) * k);
                                tmem_st16(t_o + i, r);
                            }
                        }
                        return m == -INFINITY ? 0.0f : -m;
                    };
                    if (few) {
                        // warp w takes columns 32 w .. 32 w + 31 of its own copy of the rows, with
                        // a maximum and a sum of its own; its P is zero elsewhere
                        float s[32];
                        tmem_ld32(reinterpret_cast<uint32_t*>(s), t_s + 32 * wq);
                        tmem_wait_ld();
                        const int upto = lim - 32 * wq;
                        if (!__all_sync(0xffffffffu, upto >= 32)) {
#pragma unroll
                            for (int i = 0; i < 32; i++)
                                if (i >= upto) s[i] = -INFINITY;
                        }
                        float mx[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
                        for (int i = 4; i < 28; i += 8)
#pragma unroll
                            for (int j = 0; j < 4; j++) mx[j] = max3(mx[j], s[i + 2 * j], s[i + 2 * j + 1]);
                        const float neg = raise(max_nan(max3(mx[0], s[28], s[29]), max3(max3(mx[1], s[30], s[31]), mx[2], mx[3])));
                        uint32_t pk[16];
                        float2 sum = make_float2(0.0f, 0.0f);
#pragma unroll
                        for (int i = 0; i < 16; i++) {
                            const float2 x = __ffma2_rn(make_float2(s[2 * i], s[2 * i + 1]), make_float2(cs, cs), make_float2(neg, neg));
                            const float2 e = make_float2(ex2(x.x), ex2(x.y));
                            sum = __fadd2_rn(sum, e);
                            pk[i] = pack_bf16x2(e.x, e.y);
                        }
                        l += sum.x + sum.y;
#pragma unroll 1
                        for (int w = 0; w < 4; w++) {
                            tmem_st16(t_s + 16 * ((wq + w) & 3), pk);
#pragma unroll
                            for (int i = 0; i < 16; i++) pk[i] = 0;
                        }
                    } else if (sg.n > 64) {
                        float s[128];
#pragma unroll
                        for (int j = 0; j < 4; j++) tmem_ld32(reinterpret_cast<uint32_t*>(s) + 32 * j, t_s + 32 * j);
                        tmem_wait_ld();
                        if (!__all_sync(0xffffffffu, lim >= PA_TILE)) {
#pragma unroll
                            for (int i = 0; i < 128; i++)
                                if (i >= lim) s[i] = -INFINITY;
                        }
                        float mx[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
                        for (int i = 4; i < 124; i += 8)
#pragma unroll
                            for (int j = 0; j < 4; j++) mx[j] = max3(mx[j], s[i + 2 * j], s[i + 2 * j + 1]);
                        const float neg = raise(max_nan(max3(mx[0], mx[1], max3(mx[2], s[124], s[125])), max3(mx[3], s[126], s[127])));
                        const float2 cs2 = make_float2(cs, cs), neg2 = make_float2(neg, neg);
                        float2 sum[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            uint32_t pk[16];
#pragma unroll
                            for (int i = 0; i < 16; i++) {
                                const float2 x = __ffma2_rn(make_float2(s[32 * j + 2 * i], s[32 * j + 2 * i + 1]), cs2, neg2);
                                const float2 e = make_float2(ex2(x.x), ex2(x.y));
                                sum[i & 1] = __fadd2_rn(sum[i & 1], e);
                                pk[i] = pack_bf16x2(e.x, e.y);
                            }
                            tmem_st16(t_s + 16 * j, pk);
                        }
                        l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
                    } else {
                        // few rows: two passes over S, 32 columns at a time, in a tenth of the code
                        // (they come in many short segments, where fetching the instructions costs
                        // more than the arithmetic)
                        float mt = -INFINITY, sum = 0.0f, neg = 0.0f;
#pragma unroll 1
                        for (int pass = 0; pass < 2; pass++) {
#pragma unroll 1
                            for (int j = 0; j < PA_TILE; j += 32) {
                                float s[32];
                                tmem_ld32(reinterpret_cast<uint32_t*>(s), t_s + j);
                                tmem_wait_ld();
                                if (!__all_sync(0xffffffffu, lim >= j + 32)) {
#pragma unroll
                                    for (int i = 0; i < 32; i++)
                                        if (j + i >= lim) s[i] = -INFINITY;
                                }
                                if (pass == 0) {
#pragma unroll
                                    for (int i = 0; i < 32; i += 2) mt = max3(mt, s[i], s[i + 1]);
                                } else {
                                    uint32_t pk[16];
#pragma unroll
                                    for (int i = 0; i < 16; i++) {
                                        const float p0 = ex2(fmaf(s[2 * i], cs, neg)), p1 = ex2(fmaf(s[2 * i + 1], cs, neg));
                                        sum += p0 + p1;
                                        pk[i] = pack_bf16x2(p0, p1);
                                    }
                                    // P of columns j.. lands on S columns j/2.., which have been read
                                    tmem_st16(t_s + j / 2, pk);
                                }
                            }
                            if (pass == 0) neg = raise(mt);
                        }
                        l += sum;
                    }
                    tmem_wait_st();
                }
                tc_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&c.p_full[f]);
                if (t == sg.t0) {
                    more = next(true);
                    early = more == NX_SEG && q_ahead(sg, nx);
                    if (early) q_start();
                }
            }
            if (t < sg.t1) break;  // a wait ran out
            if (more == NX_LATER) more = next(false);
            if (more == NX_SEG) {
                if (!early) q_start();  // this segment's Q has been read: its last S was complete
                q_finish();
            }
            bool there = pa_wait(c, &c.o_full[f], o_ph);
            if (few) {
                // The flow's warps meet below, so that all of them go on or none: the first one to
                // know decides. One that saw O complete knows that the others come here (all have
                // delivered their last P); one that gave up follows it.
                int was = 0;
                if (lane == 0) was = atomicCAS(&c.agreed[f], joint, there ? joint + 1 : -1);
                was = __shfl_sync(0xffffffffu, was, 0);
                if (was != joint) there = was > joint && mbar_wait(&c.o_full[f], o_ph, PA_POLLS);
                joint++;
            }
            if (!there) break;
            o_ph ^= 1;
            tc_after();
            if (!busy) continue;
            // ---- the segment's result: the row itself, or a partial for the merge ----
            const bool own = sg.flags & SEG_OWN, whole = sg.flags & SEG_WHOLE;
            const int head = sg.kh * g.a.group + st - tok * g.a.group;
            const int cap = g.p.cap[own], half = sg.flags & SEG_HALF ? PA_ROWS : 0;
            if (few) {  // first the sum over the flow's warps
                auto meet = [&]() { asm volatile("bar.sync %0, 128;" ::"r"(1 + f) : "memory"); };
                if (mine) c.few_ml[f][wq][lane] = make_float2(m, l);
                meet();
                float M = -INFINITY, L = 0.0f;
#pragma unroll
                for (int w = 0; w < 4; w++) M = fmaxf(M, c.few_ml[f][w][lane & 7].x);
#pragma unroll
                for (int w = 0; w < 4; w++) {
                    const float2 ml = c.few_ml[f][w][lane & 7];
                    if (ml.x != -INFINITY) L += ml.y * ex2(ml.x - M);
                }
                const float k = m == -INFINITY ? 0.0f : ex2(m - M) * (whole ? (L > 0.0f ? 1.0f / L : L) : 1.0f);
                if (mine && wq == 0 && !whole) g.p.ml[own][(int64_t)sg.slot * cap + half + lane] = make_float2(M, L);
                const int r = row >> 4, e = (row & 15) * 2;  // two dims of a row to write
                const int st_r = sg.row0 + min(r, sg.n - 1), tok_r = g.a.group_div(st_r);
#pragma unroll 1
                for (int i = 0; i < D; i += 32) {
                    uint32_t v[32];
                    tmem_ld32(v, t_o + i);
                    tmem_wait_ld();
                    if (mine) {
#pragma unroll
                        for (int j = 0; j < 32; j += 4)
                            *reinterpret_cast<float4*>(&c.few_o[f][wq][lane][j]) =
                                m == -INFINITY ? make_float4(0.0f, 0.0f, 0.0f, 0.0f)
                                               : make_float4(__uint_as_float(v[j]) * k, __uint_as_float(v[j + 1]) * k,
                                                             __uint_as_float(v[j + 2]) * k, __uint_as_float(v[j + 3]) * k);
                    }
                    meet();
                    float2 y = make_float2(0.0f, 0.0f);
                    if (r < sg.n) {
#pragma unroll
                        for (int w = 0; w < 4; w++) {
                            const float2 x = *reinterpret_cast<const float2*>(&c.few_o[f][w][r][e]);
                            y.x += x.x;
                            y.y += x.y;
                        }
                    }
                    if (!whole) {
                        if (r < sg.n)
                            *reinterpret_cast<float2*>(g.p.o[own] + (((int64_t)sg.slot * (D / 4) + (i + e) / 4) * cap + half + r) * 4 + (e & 2)) = y;
                    } else {
                        store2<__nv_bfloat16, D>(g.a, tok_r, sg.kh * g.a.group + st_r - tok_r * g.a.group, i + e, y, r < sg.n);
                    }
                    meet();
                }
                tc_before();
                continue;
            }
            const float inv = l > 0.0f ? 1.0f / l : 0.0f;
            const int at_o = half + row;
            if (mine && !whole) g.p.ml[own][(int64_t)sg.slot * cap + at_o] = make_float2(m, l);
            // four dims of all rows lie together, so that a warp's stores are 512 bytes each
            float4* po = reinterpret_cast<float4*>(g.p.o[own]) + (int64_t)sg.slot * (D / 4) * cap + at_o;
#pragma unroll 1
            for (int i = 0; i < D; i += 32) {
                uint32_t r[32];
                tmem_ld32(r, t_o + i);
                tmem_wait_ld();
                if (mine && !whole) {
#pragma unroll
                    for (int j = 0; j < 32; j += 4, po += cap)
                        *reinterpret_cast<uint4*>(po) = make_uint4(r[j], r[j + 1], r[j + 2], r[j + 3]);
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
        asm volatile("cp.async.wait_all;" ::: "memory");  // (after a wait that ran out: Q of the next segment)
    } else if (warp == 8) {
        // ------------------------------ TMA producer ------------------------------
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(PA_REGS_LOW));
        const int page = 1 << g.s.page_shift, box = min(page, PA_TILE), boxes = PA_TILE / box;
        int issued = 0, slot = 0;
        unsigned ph = 0;
        bool ok = true;
        struct Flow {
            Feed feed;
            PaSeg sg;
            bool ended, v_due;
            int pg, krow, kh;   // this lane's page of the tile, kept from K for V
        } cur, oth;
        cur.ended = oth.ended = cur.v_due = oth.v_due = false;
        cur.sg.t0 = cur.sg.t1 = oth.sg.t0 = oth.sg.t1 = 0;
        cur.pg = cur.krow = cur.kh = oth.pg = oth.krow = oth.kh = 0;
        // a round brings, per flow, V of the round before and K of this one
#pragma unroll 1
        for (int f = 0; f || !(cur.ended && oth.ended && !cur.v_due && !oth.v_due); f ^= 1) {
            bool k_due = false;
#pragma unroll 1
            for (int which = 0; which < 2 && ok; which++) {
                if (which == 0 ? cur.v_due : k_due) {
                    ok = pa_wait_warp(c, &c.empty[slot], ph ^ 1u);
                    if (!ok) break;
                    if (lane == 0) mbar_expect_tx(&c.full[slot], KV_BYTES);
                    __syncwarp();
                    uint8_t* const dst = ring + slot * KV_BYTES;
                    const CUtensorMap* const map = which ? &map_k : &map_v;
                    if (lane < boxes) {
#pragma unroll
                        for (int h = 0; h < HALVES; h++)
                            tma_load_4d(dst + h * HALF + lane * box * 128, map, h * 64, cur.krow, cur.kh, cur.pg, &c.full[slot]);
                    }
                    issued++;
                    if (++slot == STAGES) slot = 0, ph ^= 1;
                }
                if (which) break;
                cur.v_due = false;
                if (cur.ended) break;
                if (cur.sg.t0 == cur.sg.t1) {
                    ok = fetch(f, cur.feed, cur.sg);
                    cur.ended = !ok || (cur.sg.flags & SEG_END);
                    if (cur.ended) break;
                }
                const int t = cur.sg.t0++;
                if (cur.sg.n == 0 || (f == 1 && (cur.sg.flags & SEG_PAIRED))) break;
                const bool own = (cur.sg.flags & SEG_OWN) && t >= chain;
                const int pos = (own ? t - chain : t) * PA_TILE + lane * box;
                int id = g.s.n_pages;  // out of range: zeros
                if (lane < boxes && pos < (own ? cur.sg.kv_end - chain * PA_TILE : g.a.prefix_len)) {
                    const int32_t* const table = own ? g.s.table + (int64_t)cur.sg.b * g.s.table_ld : g.a.prefix_table;
                    id = table[pos >> g.s.page_shift];
                    if ((unsigned)id >= (unsigned)g.s.n_pages) {
                        flag_error(err, ERR_PAGE_ID, id);
                        id = g.s.n_pages;
                    }
                }
                cur.pg = id;
                cur.krow = pos & (page - 1);
                cur.kh = cur.sg.kh;
                cur.v_due = k_due = true;
            }
            if (!ok) break;
            exchange(cur, oth);
        }
        if (lane == 0) c.issued = issued;
    } else if (warp == 9) {
        // ------------------------------ MMA issuer ------------------------------
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(PA_REGS_LOW));
        constexpr uint32_t id_qk = pa_idesc(PA_TILE, 0), id_pv = pa_idesc(D, 1);
        int slot = 0, k_slot = 0, v_slot = 0;
        unsigned ph = 0;
        bool ok = true, both = false;  // both: this round's K is for the second flow too
        struct Flow {
            Feed feed;
            PaSeg sg;
            bool ended;
            unsigned q_ph, p_ph, turn, q_off;
            // P V of the round before: due, V shared by the flows, first and last of a segment
            bool pv, pv_shared, pv_first, pv_last;
            int pv_valid;
        } cur, oth;
        cur.sg.t0 = cur.sg.t1 = 0;
        cur.ended = cur.pv = cur.pv_shared = cur.pv_first = cur.pv_last = false;
        cur.q_ph = cur.p_ph = cur.turn = cur.q_off = 0;
        cur.pv_valid = 0;
        oth = cur;
        auto take = [&](int& where) {  // the next stage of the ring
            ok = pa_wait_warp(c, &c.full[slot], ph);
            where = slot;
            if (++slot == STAGES) slot = 0, ph ^= 1;
        };
#pragma unroll 1
        for (int f = 0; f || !(cur.ended && oth.ended && !cur.pv && !oth.pv); f ^= 1) {
            const uint32_t t_s = tmem + f * 128, t_o = tmem + 256 + f * 128;
            if (cur.pv) {
                if (f == 0 || !cur.pv_shared) {
                    take(v_slot);
                    if (!ok) break;
                    if (cur.pv_valid < PA_TILE) {
                        // positions past the end share a page with valid ones: whatever is there
                        // (NaN times a zero probability) must not reach the product
                        uint8_t* const v = ring + v_slot * KV_BYTES;
#pragma unroll 1
                        for (int i = cur.pv_valid * 8 + lane; i < PA_TILE * 8; i += 32)
#pragma unroll
                            for (int h = 0; h < HALVES; h++)
                                *reinterpret_cast<uint4*>(v + h * HALF + i * 16) = make_uint4(0, 0, 0, 0);
                        proxy_fence();
                        __syncwarp();
                    }
                }
                ok = pa_wait_warp(c, &c.p_full[f], cur.p_ph);
                if (!ok) break;
                cur.p_ph ^= 1;
                tc_after();
                const uint64_t v = pa_desc(smem_addr(ring + v_slot * KV_BYTES), HALF);
                if (elect_one()) {
#pragma unroll
                    for (int j = 0; j < PA_TILE / 16; j++)
                        mma_ts(t_o, t_s + j * 8, v + j * (2048 >> 4), id_pv, j > 0 || !cur.pv_first);
                    if (!(f == 0 && cur.pv_shared && oth.pv)) tc_commit(&c.empty[v_slot]);
                    if (cur.pv_last) tc_commit(&c.o_full[f]);
                }
                __syncwarp();
                cur.pv = false;
            }
            if (!cur.ended && cur.sg.t0 == cur.sg.t1) {
                ok = fetch(f, cur.feed, cur.sg);
                if (!ok) break;
                cur.ended = cur.sg.flags & SEG_END;
                cur.pv_first = true;
            } else {
                cur.pv_first = false;
            }
            if (!cur.ended) {
                const int t = cur.sg.t0++;
                const bool shared = cur.sg.flags & SEG_PAIRED;
                if (f == 0) both = shared && cur.sg.n1 > 0;
                if (cur.sg.n > 0) {
                    if (f == 0 || !shared) take(k_slot);
                    if (!ok) break;
                    if (cur.pv_first) {  // a new segment: its Q
                        ok = pa_wait_warp(c, &c.q_full[f], cur.q_ph);
                        if (!ok) break;
                        cur.q_ph ^= 1;
                        cur.q_off = q_offset(cur.sg, cur.turn++);
                    }
                    tc_after();
                    const uint64_t q = pa_desc(smem_addr(sm + f * Q_BYTES) + cur.q_off, 16);
                    const uint64_t k = pa_desc(smem_addr(ring + k_slot * KV_BYTES), 16);
                    if (elect_one()) {
#pragma unroll
                        for (int j = 0; j < D / 16; j++) {
                            const uint32_t o = ((j >> 2) * HALF + (j & 3) * 32) >> 4;
                            mma_ss(t_s, q + o, k + o, id_qk, j > 0);
                        }
                        if (!(f == 0 && both)) tc_commit(&c.empty[k_slot]);
                        tc_commit(&c.s_full[f]);
                    }
                    __syncwarp();
                    cur.pv = true;
                    cur.pv_shared = shared;
                    cur.pv_last = cur.sg.t0 == cur.sg.t1;
                    cur.pv_valid = min(PA_TILE, (t < chain ? g.a.prefix_len : cur.sg.kv_end) - t * PA_TILE);
                }
            }
            exchange(cur, oth);
        }
        if (elect_one()) tc_commit(&c.done);  // (by the thread that issued the MMAs)
        __syncwarp();
        if (!mbar_wait_ns(&c.done, 0, 2000000000ull)) c.abort = 1;
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(PA_REGS_LOW));
        if (warp == 10) {
            // ------------------------------ scheduler ------------------------------
            // Half a warp looks after a flow. In a part whose blocks are paired the two flows walk
            // the same items, else each has its half of the CTA's steps.
            const Line line(g.p, so, PP, PO);
            const int f = lane >> 4, hl = lane & 15;
            unsigned batch[2] = {0, 0};
            const unsigned hold = g.p.hold ? me % 8 : ~0u;  // (fault injection: batches handed out)
            bool ok = true;
            // the next batch of the flows with `valid` lanes, in the order of the lanes
            auto put = [&](const PaSeg& o, bool valid) {
                const unsigned all = __ballot_sync(0xffffffffu, valid);
#pragma unroll
                for (int q = 0; q < 2; q++) {
                    const unsigned m = (all >> (16 * q)) & 0xffffu, k = batch[q];
                    if (!m || !ok) continue;
                    ok = batch[0] + batch[1] < hold && pa_wait_warp(c, &c.seg_empty[q][k & 1], ((k >> 1) & 1u) ^ 1u, polls);
                    if (!ok) return;
                    if (valid && f == q) c.seg[q][k & 1][__popc(m & ((1u << hl) - 1))] = o;
                    if (lane == 0) c.seg_n[q][k & 1] = __popc(m);
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&c.seg_full[q][k & 1]);
                    batch[q]++;
                }
            };
            PaSeg o{0, 1, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
            if (g.p.np == 0 && lane < (PO ? 1 : 2)) g.p.split[PO ? me : 2 * me + lane].rows = 0;
            __syncwarp();
            auto part = [&](auto own_part) {
                constexpr bool own = decltype(own_part)::value, paired = own ? PO : PP;
                const int block = own ? g.p.ob : g.p.pb, worker = paired ? me : 2 * me + f;
                const int live = own ? 0 : live_rows(g.s);
                int step, hi, b = 0, j = 0, t = 0, rounds = 0;  // the flow's place
                flow_range(line, paired, me, f, own, step, hi);
                if (step < hi && !own) {
                    j = step / g.p.np;
                    t = step - j * g.p.np;
                }
                if (own && (PO ? __any_sync(0xffffffffu, step < hi) : step < hi)) {
                    int e0 = 0, e1 = n_entries;  // the last entry with scan <= step
#pragma unroll 1
                    while (e1 - e0 > 1) {
                        const int m = (e0 + e1) >> 1;
                        if (c.scan[m] <= step) e0 = m;
                        else e1 = m;
                    }
                    int rest = step - c.scan[e0], per = 1;
                    SeqInfo si{0, 0, 0};
#pragma unroll 1
                    for (b = e0 * per_entry; b < g.s.n_seqs; b++) {
                        si = pa_seq(g, c, b);
                        per = per_entry == 1 ? c.info[b].w : PO ? os.per_head(si) : si.q > 0 ? os.steps(si, 0) : 0;
                        if (rest < per * g.a.n_kv) break;
                        rest -= per * g.a.n_kv;
                    }
                    if (b >= g.s.n_seqs) hi = step;  // lengths that changed under the kernel
                    j = rest / max(per, 1);
                    t = rest - j * per;
                    if constexpr (PO) {  // (both flows are at the same place: the whole warp looks)
                        const int n_rb = os.blocks(si);
                        int rb = 0;
#pragma unroll 1
                        for (; rb < n_rb; rb += 32) {
                            const int n = rb + lane < n_rb ? os.steps(si, rb + lane) : 0;
                            const int upto = warp_scan(n, lane), all = __shfl_sync(0xffffffffu, upto, 31);
                            if (t < all) {
                                const int l = __ffs(__ballot_sync(0xffffffffu, upto > t)) - 1;
                                t -= __shfl_sync(0xffffffffu, upto - n, l);
                                rb += l;
                                break;
                            }
                            t -= all;
                        }
                        j = j * n_rb + rb;
                    }
                }
                bool first = true;
                while (ok && __any_sync(0xffffffffu, step < hi)) {
                    bool go = step < hi;
                    if constexpr (!paired) {
                        const int others = __shfl_xor_sync(0xffffffffu, rounds, 16);
                        const bool other_live = __shfl_xor_sync(0xffffffffu, (int)go, 16);
                        const HandOut turn = hand_out(f, first, go, other_live, rounds, others);
                        go = turn.go;
                        if (__any_sync(0xffffffffu, turn.idle > 0)) {
                            o = PaSeg{0, turn.idle, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
                            put(o, hl == 0 && turn.idle > 0);
                            rounds += turn.idle;
                        }
                    }
                    first = false;
                    // a lane looks at the hl-th item from here on
                    int jj = j + hl, bb = b, n_rb = own ? 1 : g.p.n_rb, nt = g.p.np;
                    SeqInfo si{0, live, 0};
                    o.kv_end = g.a.prefix_len;
                    if constexpr (own) {
                        nt = o.kv_end = 0;
#pragma unroll 1
                        for (; bb < g.s.n_seqs; bb++) {
                            si = pa_seq(g, c, bb);
                            n_rb = PO ? os.blocks(si) : si.q > 0;
                            if (jj < g.a.n_kv * n_rb) break;
                            jj -= g.a.n_kv * n_rb;
                        }
                    }
                    int kh = jj, rb = 0;
                    if ((own ? PO : true) && n_rb > 1) {
                        kh = jj / n_rb;
                        rb = jj - kh * n_rb;
                    }
                    if (own && bb < g.s.n_seqs) {
                        o.kv_end = chain * PA_TILE + os.visible(si, rb);
                        nt = (o.kv_end + PA_TILE - 1) / PA_TILE;
                    }
                    const int ns = nt + (own && nt > 0 ? g.p.extra : 0);  // steps of the item
                    const int from = hl == 0 ? t : 0;
                    int upto = ns - from;  // steps up to here in the batch
#pragma unroll
                    for (int k = 1; k < 16; k <<= 1) {
                        const int u = __shfl_up_sync(0xffffffffu, upto, k, 16);
                        if (hl >= k) upto += u;
                    }
                    o.t0 = min(from, nt);
                    o.t1 = min(nt, from + min(ns - from, hi - (step + upto - (ns - from))));
                    const int n = o.t1 - o.t0;
                    const int rows = si.q * g.a.group - rb * block;  // of the whole block
                    const int item = (own ? g.a.n_kv * os.base(si, bb) : 0) + jj;
                    o.n1 = paired ? max(0, min(PA_ROWS, rows - PA_ROWS)) : 0;
                    o.n = paired && f ? o.n1 : max(0, min(PA_ROWS, rows));  // (0: a block of padding)
                    o.flags = (own ? SEG_OWN : 0) | (paired ? SEG_PAIRED : 0) | (paired && f ? SEG_HALF : 0) |
                              (own && g.p.np == 0 && o.t0 == 0 && o.t1 == nt ? SEG_WHOLE : 0);
                    o.kh = kh;
                    o.b = bb;
                    const int first_row = (own ? si.q0 * g.a.group : 0) + rb * block;
                    o.row0 = first_row + (paired && f ? PA_ROWS : 0);
                    o.voff = own ? si.kv - si.q + 1 - si.q0 : 0;
                    o.slot = own ? g.p.own_slot(item, worker, o.t0 == 0) : item + worker;
                    const bool valid = go && n > 0;
                    if (valid && !(paired && f)) {  // for the merge
                        if (o.t0 == 0) g.p.first[own][item] = worker;
                        if (o.t1 == nt) g.p.last[own][item] = worker;
                        if (own && g.p.np == 0 && o.t0 == 0 && o.t1 < nt)
                            g.p.split[worker] = SplitItem{min(rows, block), first_row, kh, item};
                    }
                    put(o, valid);
                    int tiles = valid ? n : 0;  // rounds the batch takes
#pragma unroll
                    for (int k = 8; k > 0; k >>= 1) tiles += __shfl_xor_sync(0xffffffffu, tiles, k);
                    rounds += tiles;
                    const int all = min(__shfl_sync(0xffffffffu, upto, 15, 16), hi - step);
                    jj = __shfl_sync(0xffffffffu, jj, 15, 16) + 1;
                    bb = __shfl_sync(0xffffffffu, bb, 15, 16);
                    if (go) {
                        step += all;
                        j = jj;
                        b = bb;
                        t = 0;
                        if (own && b >= g.s.n_seqs) hi = step;  // (no more sequences)
                    }
                }
                // both flows take the same number of rounds
                if (!paired && ok) {
                    const int more = __shfl_xor_sync(0xffffffffu, rounds, 16) - rounds;
                    o = PaSeg{0, more, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
                    put(o, hl == 0 && more > 0);
                }
            };
            if (line.sp > 0) part(std::false_type{});
            if (ok) part(std::true_type{});
            o.flags = SEG_END;
            if (ok) put(o, hl == 0);
        } else if (g.a.prefix_len == 0) {
            // warp 11: rows before their sequence's first position see nothing when there is no
            // prefix either
#pragma unroll 1
            for (int b = me; b < g.s.n_seqs; b += gridDim.x) {
                const SeqInfo si = pa_seq(g, c, b);
                if (si.kv < si.q) zero_rows<__nv_bfloat16, D>(g.a, si.q0, si.q - si.kv, lane, 32);
            }
        }
    }
    tc_before();
    __syncthreads();
    tc_after();
    if (c.abort) {
        if (tid == 0) flag_error(err, ERR_PA_WAIT, me);
        // no copy may still be landing when the CTA exits
        if (warp == 8) {
#pragma unroll 1
            for (int i = max(0, c.issued - STAGES); i < c.issued; i++)
                mbar_wait_ns(&c.full[i % STAGES], (unsigned)(i / STAGES) & 1u, 2000000000ull);
        }
    }
    if (warp == 9) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
}

template <int D, bool PP, bool PO>
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
    const size_t smem = 1024 + 2 * PA_ROWS * D * 2 + pa_stages(D) * PA_TILE * D * 2 + sizeof(PaCtl);
    rc = ensure_func_smem(ctx, (const void*)prefix_attn_tc_kernel<D, PP, PO>, smem);
    if (rc) return rc;
    return launch_kernel(ctx, prefix_attn_tc_kernel<D, PP, PO>, dim3((unsigned)g.p.workers), dim3(PA_THREADS), smem,
                         "prefix_attn_tc", mk, mv, g);
}

int launch_prefix_attn_tc(lq_ctx* ctx, const PrefixAttnArgs& a, const PagedSeqs& s, const PrefixPlan& p, int D) {
    const PaArgs g{a, s, p};
    // PO implies PP: one sequence's rows are some of all rows. Without a prefix PP says nothing.
    if (D == 64) return p.pair_o ? launch_tc<64, true, true>(ctx, g) : p.pair_p ? launch_tc<64, true, false>(ctx, g) : launch_tc<64, false, false>(ctx, g);
    return p.pair_o ? launch_tc<128, true, true>(ctx, g) : p.pair_p ? launch_tc<128, true, false>(ctx, g) : launch_tc<128, false, false>(ctx, g);
}

}  // namespace lq
