// lq8_prefix_plan.cuh -- how the shared-prefix attention cuts its work, on the device, from the
// lengths the call finds there.
//
// Query rows of one kv head are stacked: token t's heads g < G of the group are rows t G + g, so
// that all sequences' rows form the tiles of the prefix (its K/V are read once for the batch),
// and one sequence's rows the tiles of its own positions. An item is (kv head, row block); a step
// is one 128-position (f32: 32) tile of an item. Steps of all items form one line, prefix items
// first, then the sequences' own, and every worker takes an equal share of it: no split factors,
// no empty workers, whatever the mix of lengths. An item cut between workers leaves one partial
// (o, m, l) per worker, which the merge kernel joins in order.
//
// Where the sequences bring many rows each (prompt chunks), stacking over sequences saves few
// tiles, while two partials of every row would go through memory. There the prefix has no items of
// its own: its tiles come first in each own item (chain of them).
#pragma once

#include <algorithm>

#include "lq8_paged.cuh"

namespace lq {

struct PrefixAttnArgs {
    const void* q;
    int64_t q_stride;
    int n_heads, n_kv, group;   // group: query heads of a kv head
    uint64_t group_mul;         // ceil(2^36 / group)
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
    // x / group by a multiplication: exact for 0 <= x < 2^28 (group_mul * group < 2^36 + 128)
    __host__ __device__ __forceinline__ int group_div(int x) const { return (int)(((uint64_t)x * group_mul) >> 36); }
};

// an own item that is cut between workers
struct SplitItem {
    int rows;      // rows of its block (0: none)
    int row0, kh, item;
};

struct PrefixPlan {
    int tile;                   // positions of a step
    int pb, ob;                 // rows of a block: prefix items, own items
    int pair_p, pair_o;         // the two halves of a block run side by side in one worker (pb / ob = 2 halves)
    int n_rb;                   // row blocks of the prefix, per kv head
    int np;                     // tiles of a prefix item (0: there are none)
    int chain;                  // tiles of the prefix at the front of every own item
    int sp;                     // steps of the prefix
    int extra;                  // steps that an own item counts for beside its tiles
    int workers;                // CTAs that share the line
    uint64_t workers_mul;       // ceil(2^40 / workers)
    int polls;                  // polls of a wait (f32: for a copy; bf16: for segments) before it gives up
    int hold;                   // fault injection: every CTA stops handing out segments after a few batches
    int cap[2];                 // rows a partial slot holds (prefix, own)
    int32_t* own_steps;         // [1] own steps in all, written by the first CTA
    int32_t* first[2];          // per item (prefix, own): the first worker of its steps,
    int32_t* last[2];           // and the last
    SplitItem* split;           // per worker, without a prefix: the cut item it begins
    float* o[2];                // partials, unnormalised: [slot][D/4][cap] of four dims
    float2* ml[2];              // [slot][cap]: running maximum (log2 units) and sum
    // Where a worker's piece of an own item goes. Without prefix items only cut items leave partials:
    // a worker has one piece at most of an item that it begins and one of an item begun before it.
    __device__ __forceinline__ int own_slot(int item, int worker, bool begins) const {
        return np > 0 ? item + worker : 2 * worker + (begins ? 1 : 0);
    }
};

// a sequence's rows and own length, with what the call's bounds do not hold taken out
struct SeqInfo {
    int q0, q, kv;
};

__device__ __forceinline__ SeqInfo seq_info(const PrefixAttnArgs& a, const PagedSeqs& s, int b, bool flag) {
    int q0 = b, q1 = b + 1;
    if (s.q_start) {
        q0 = s.q_start[b];
        q1 = s.q_start[b + 1];
    }
    SeqInfo r{q0, q1 - q0, s.kv_len[b]};
    if (r.q < 0 || r.q > a.max_q || q0 < 0 || q1 > s.rows) {
        // without q_start, sequences past the rows have none
        if (flag && s.q_start) flag_error(a.err, ERR_ROW_COUNT, r.q);
        r.q = 0;
    }
    const int64_t most = min((int64_t)a.max_kv, s.table_ld << s.page_shift);
    if (r.kv < 0 || r.kv > most) {
        if (flag) flag_error(a.err, ERR_KV_LEN, r.kv);
        r.kv = r.kv < 0 ? 0 : (int)most;
    }
    return r;
}

// Whether the next sequence's rows begin before this one's. Such a batch may name a row several times,
// and more steps than the plan has numbers for: it gets none.
__device__ __forceinline__ bool falls(const PagedSeqs& s, int b) { return s.q_start && s.q_start[b + 1] < s.q_start[b]; }

// rows before the padding: those that the prefix's blocks hold
__device__ __forceinline__ int live_rows(const PagedSeqs& s) {
    return s.q_start ? min(max(s.q_start[s.n_seqs], 0), s.rows) : s.rows;
}

// own positions that token j of the sequence's q sees
__host__ __device__ __forceinline__ int own_visible(const SeqInfo& i, int j) { return max(0, i.kv - i.q + j + 1); }

struct OwnSteps {
    const PrefixAttnArgs& a;
    const PrefixPlan& p;
    __host__ __device__ __forceinline__ int blocks(const SeqInfo& i) const { return (i.q * a.group + p.ob - 1) / p.ob; }
    // own positions that row block rb sees (those of its last row), and its tiles (the chain's too)
    __host__ __device__ __forceinline__ int visible(const SeqInfo& i, int rb) const {
        return own_visible(i, a.group_div(min(i.q * a.group, (rb + 1) * p.ob) - 1));
    }
    __host__ __device__ __forceinline__ int tiles(const SeqInfo& i, int rb) const {
        return p.chain + (visible(i, rb) + p.tile - 1) / p.tile;
    }
    // what the block counts for on the line: its tiles, and p.extra for the segment's beginning and
    // end (after the tiles; a worker whose share has nothing else of the block leaves it alone)
    __host__ __device__ __forceinline__ int steps(const SeqInfo& i, int rb) const {
        const int n = tiles(i, rb);
        return n > 0 ? n + p.extra : 0;
    }
    __host__ __device__ __forceinline__ int per_head(const SeqInfo& i) const {
        int n = 0;
#pragma unroll 1
        for (int rb = blocks(i) - 1; rb >= 0; rb--) n += steps(i, rb);
        return n;
    }
    // numbers a sequence's row blocks from here on; blocks(i) <= base(next) - base(i), so that no
    // scan over the sequences is needed
    __host__ __device__ __forceinline__ int base(const SeqInfo& i, int b) const { return i.q0 * a.group / p.ob + b; }
};

// A step of a paired block weighs 3, one that a flow takes alone 2 (measured: a round of two
// 128-row products takes 3300 cycles, one of two flows' separate tiles 4000). Worker c of n takes
// the steps that start in [W c / n, W (c + 1) / n) of the whole weight W < 2^28.
struct Line {
    int w, split;      // total weight; weight of the prefix part
    int sp, so, n;
    bool pair_p, pair_o;
    int quot, rem;     // W / n
    uint64_t mul;      // ceil(2^40 / n): x / n = x mul / 2^40, exact while x n < 2^40 (x < 2^28, n < 2^11)
    __host__ __device__ __forceinline__ Line(const PrefixPlan& p, int own_steps, bool pair_prefix, bool pair_own)
        : sp(p.sp), so(own_steps), n(p.workers), pair_p(pair_prefix), pair_o(pair_own), mul(p.workers_mul) {
        split = sp * (pair_p ? 3 : 2);
        w = split + so * (pair_o ? 3 : 2);
        quot = (int)(((uint64_t)w * mul) >> 40);
        rem = w - quot * n;
    }
    // floor(W c / n)
    __host__ __device__ __forceinline__ int start(int c) const { return quot * c + (int)(((uint64_t)(rem * c) * mul) >> 40); }
    __host__ __device__ __forceinline__ int first(int c, bool own) const {
        const int x = own ? max(start(c) - split, 0) : start(c);
        return min((own ? pair_o : pair_p) ? (x + 2) / 3 : (x + 1) / 2, own ? so : sp);
    }
};

// [lo, hi) of CTA c's flow f: both halves of a paired block run the same steps, otherwise the
// flows take one half of the steps each
__host__ __device__ __forceinline__ void flow_range(const Line& l, bool paired, int c, int f, bool own, int& lo, int& hi) {
    lo = l.first(c, own);
    hi = l.first(c + 1, own);
    if (!paired) {
        const int mid = lo + (hi - lo + 1) / 2;
        if (f == 0) hi = mid;
        else lo = mid;
    }
}

// What a flow of a CTA gets next in a part whose flows are apart: a batch of its items (go), or
// `idle` rounds without work. The warps that serve the flows take a round of each in turn, and a
// flow's batch is only taken back when they have begun its next one. So a batch goes to the flow
// with fewer rounds, and a flow that ran out of steps is given the rounds that it lacks before the
// other one gets more: else those warps would wait for it, and the scheduler for them. `mine` and
// `other`: rounds that the flows were given; live: steps left.
struct HandOut {
    bool go;
    int idle;
};
__host__ __device__ __forceinline__ HandOut hand_out(int f, bool first, bool live, bool other_live, int mine, int other) {
    return HandOut{live && (first || !other_live || mine < other || (mine == other && f == 0)),
                   !live && other_live && mine < other ? other - mine : 0};
}

// host: cuts a call's work for sm_count SMs, from the bounds that the call gives (what the lengths
// really are, the kernels read); the most steps that there can be, to be checked against
// PREFIX_MAX_STEPS before the plan is used
constexpr int64_t PREFIX_MAX_STEPS = 1ll << 26;
constexpr int PREFIX_ATTN_F32_WARPS = 8;  // workers of a CTA of the f32 kernel
inline int64_t plan_cut(const PrefixAttnArgs& a, const PagedSeqs& s, bool f32, int sm_count, PrefixPlan* p) {
    const int64_t R = (int64_t)s.rows * a.group, most_q = std::min<int64_t>((int64_t)a.max_q, s.rows) * a.group;
    // bf16: blocks of 128 rows, or two halves of 128 that share their K and V tiles; a worker is a
    // CTA with paired halves, else one of its two flows. f32: blocks of 8 rows, a worker is a warp.
    const int half = f32 ? 8 : 128, tile = f32 ? 32 : 128;
    p->tile = tile;
    p->pair_p = f32 || R > half;
    p->pair_o = f32 || most_q > half;
    p->pb = f32 ? half : p->pair_p ? 2 * half : half;
    p->ob = f32 ? half : p->pair_o ? 2 * half : half;
    p->cap[0] = (int)std::min<int64_t>(p->pb, R);
    p->cap[1] = (int)std::min<int64_t>(p->ob, most_q);
    p->n_rb = ceil_div(R, p->pb);
    p->np = ceil_div(a.prefix_len, tile);
    // The prefix's tiles at the front of the own items: that costs at most n_seqs - 1 blocks more of
    // np steps each, and saves a block's two partials and their merge, about as long as 9 steps
    // (a chunk of 2048 tokens behind 2048 positions: 273 us apart, 222 in one line; ten ragged ones behind
    // 2049: 146 and 136).
    p->chain = 0;
    if (!f32 && p->pair_o && (s.n_seqs - 1) * (int64_t)p->np <= 9 * (R / p->pb) &&
        (int64_t)a.prefix_len + a.max_kv < (1 << 30)) {
        p->chain = p->np;
        p->np = 0;
    }
    const int64_t items_p = (int64_t)a.n_kv * p->n_rb, items_o = a.n_kv * (R / p->ob + s.n_seqs + 1);
    const int64_t steps = items_p * p->np + items_o * (p->chain + ceil_div(a.max_kv, tile) + 1);
    p->sp = (int)(items_p * p->np);
    // a segment costs about one more step than its tiles (Q, the masked tile, the store): counted
    // so, short causal items next to a long prefix no longer hold up the last CTAs (a batch of 10
    // prompt chunks: 152 -> 114 us)
    p->extra = f32 ? 0 : 1;
    p->workers = (int)std::max<int64_t>(1, std::min<int64_t>(sm_count * (f32 ? PREFIX_ATTN_F32_WARPS : 1), steps));
    p->workers_mul = ((1ull << 40) + p->workers - 1) / p->workers;
    return steps;
}

}  // namespace lq
