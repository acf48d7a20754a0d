// lq8_paged_q8.cu -- the paged K/V cache in 8 bits: the append that quantises (with q/k norm and rotation
// on the way), and reading rows back.
#include "lq8_paged_q8.cuh"
#include "lq8_paged_rows.cuh"

#include <algorithm>

namespace lq {

// =========================================================================================
// Append. q as in the f32 and bf16 caches (append_heads). k and v by blocks of B positions that
// share a scale: with a = max |x| over the call's rows in the block,
//   s' = a / 127             where the call's rows begin the block,
//   s' = max(s, a / 127)     where older positions do; if that is larger than s, their codes
//                            become rint(c s / s'),
//   c  = rint(x r), r = 1 / s' in f32, the product exact: it is off by up to 127 2^-24 from x / s', which only
//        matters that close to halfway between two codes. (A division takes several instructions for each
//        value, in a kernel that prompt chunks bind by its instructions.)
// A team of B / 16 warps owns a block of one sequence, one kv head, K or V: a warp holds 16
// positions in registers (a lane 8 rotary pairs of a position, D / 16 lanes a position), so that
// rows are read once and the largest value is known before the first code is written. It is found as
// the largest bit pattern, which puts NaN above infinity: either makes the scale NaN, and the
// block reads as NaN until its first position is written anew. A scale below the normal numbers
// becomes zero, with codes of zero.
// Blocks are numbered without a scan over the sequences: those of sequence b from
// q_start[b] / B + 2 b on, which leaves room for one cut at either end.
// Bound: HBM for large prompts, the latency of dependent loads (row, sequence, page, older codes) for small ones.
// 16 prompts of up to 2000 rows of 32 + 16 heads, f32: 91 us with cold caches, 433 MB through DRAM (4.8 TB/s, 73 % of
// a plain copy); 12 prompt chunks, bf16, q/k norm: 25 us (instructions 2.1 a cycle, DRAM 16 %); 8 rows:
// one launch.
// =========================================================================================
struct TeamInfo {
    int q0, p0;      // the sequence's first new row and its position
    int lo, hi;      // new positions of the block
    int first;       // the block's first position
    int page, slot;  // its page, its place there
    int ok;
};

// the last sequence whose blocks begin at or before x (by a warp; base is increasing)
__device__ __forceinline__ int seq_of_block(const PagedSeqs& s, int shift, int64_t x, int lane) {
    int lo = 0, n = s.n_seqs - 1;
    while (n > 0) {
        const int step = (n + 31) >> 5, i = lo + min(n, (lane + 1) * step);
        const int c = __popc(__ballot_sync(0xffffffffu, (int64_t)(s.q_start[i] >> shift) + 2ll * i <= x));
        if (c == 32) return lo + n;
        const int skip = min(n, c * step);
        n = min(step - 1, n - skip);
        lo += skip;
    }
    return lo;
}

__device__ __forceinline__ TeamInfo find_block(const PagedSeqs& s, const PagedQ8& c, int64_t x, int lane, int* err) {
    TeamInfo t{0, 0, 0, 0, 0, 0, 0, 0};
    const int shift = c.block_shift;
    int b = (int)x, q1 = (int)x + 1;
    int64_t j = 0;  // the block's place among those that the sequence's rows touch
    t.q0 = b;
    if (s.q_start) {
        b = seq_of_block(s, shift, x, lane);
        t.q0 = s.q_start[b];
        q1 = s.q_start[b + 1];
        j = x - ((int64_t)(t.q0 >> shift) + 2ll * b);
    } else if (x >= min(s.rows, s.n_seqs)) {
        return t;
    }
    if (q1 <= t.q0 || j < 0) return t;
    const int kv = s.kv_len[b], q = q1 - t.q0;
    if (t.q0 < 0 || q1 > s.rows) {
        if (lane == 0 && j == 0) flag_error(err, ERR_ROW_COUNT, q);
        return t;
    }
    // rows before the sequence's first position have no slot
    if (kv < q && lane == 0 && j == 0) flag_error(err, ERR_KV_LEN, kv);
    if (kv <= 0) return t;
    t.p0 = kv - q;
    const int64_t n = (max(t.p0, 0) >> shift) + j;
    if (n > (kv - 1) >> shift) return t;
    t.first = (int)(n << shift);
    t.lo = max(t.first, t.p0);  // (first >= 0)
    t.hi = (int)min((int64_t)t.first + (1 << shift), (int64_t)kv);
    const int pg = t.first >> s.page_shift;
    if (pg >= s.table_ld) {
        if (lane == 0) flag_error(err, ERR_KV_LEN, kv);
        return t;
    }
    t.page = s.table[(int64_t)b * s.table_ld + pg];
    if ((unsigned)t.page >= (unsigned)s.n_pages) {
        if (lane == 0) flag_error(err, ERR_PAGE_ID, t.page);
        return t;
    }
    t.slot = (t.first & ((1 << s.page_shift) - 1)) >> shift;
    t.ok = 1;
    return t;
}

// rint(x) in the low byte, |x| < 2^22: 1.5 2^23 pushes the fraction out, round to nearest even
__device__ __forceinline__ uint32_t code_bits(float x, float by) { return __float_as_uint(fmaf(x, by, 12582912.0f)); }
__device__ __forceinline__ uint32_t pack_codes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}
__device__ __forceinline__ uint2 codes8(const float x[8], float by) {
    uint32_t u[8];
#pragma unroll
    for (int e = 0; e < 8; e++) u[e] = code_bits(x[e], by);
    return make_uint2(pack_codes(u[0], u[1], u[2], u[3]), pack_codes(u[4], u[5], u[6], u[7]));
}
__device__ __forceinline__ uint32_t codes_again(uint32_t w, float by) {
    uint32_t u[4];
#pragma unroll
    for (int e = 0; e < 4; e++) u[e] = code_bits((float)(int8_t)(w >> (8 * e)), by);
    return pack_codes(u[0], u[1], u[2], u[3]);
}

// Query heads of a row: IT times 32 / (D / 16) of them a warp, as append_heads; where positions are given
// nothing is looked up but whether the row is padding
template <typename S, int D, int IT>
__device__ __forceinline__ void append_query(const AppendArgs& a, const RopeAxes& rope, const PagedSeqs& seqs, int groups, int64_t item) {
    constexpr int LPH = D / 16, HPW = 32 / LPH, N = D / 2;
    const int lane = threadIdx.x & 31;
    const int row = (int)(item / groups);
    const int d0 = 8 * (lane % LPH), mine = (int)(item - (int64_t)row * groups) * (HPW * IT) + lane / LPH;
    if (row >= seqs.rows) return;
    const S* src = static_cast<const S*>(a.qkv) + (int64_t)row * a.row_stride + (int64_t)mine * D + d0;
    Vec<S, 16 / sizeof(S)> raw[IT][2][sizeof(S) / 2];
#pragma unroll
    for (int j = 0; j < IT; j++)
        if (mine + j * HPW < a.n_heads) {
#pragma unroll
            for (int k = 0; k < (int)sizeof(S) / 2; k++) {
                raw[j][0][k] = *reinterpret_cast<const Vec<S, 16 / sizeof(S)>*>(src + j * HPW * D + k * (16 / sizeof(S)));
                raw[j][1][k] = *reinterpret_cast<const Vec<S, 16 / sizeof(S)>*>(src + j * HPW * D + N + k * (16 / sizeof(S)));
            }
        }
    float cs[8], sn[8];
    bool turn = true;
    if (rope.pos) {
        turn = angles<8>(rope, row, 0, d0, cs, sn, nullptr);
        if (row >= (seqs.q_start ? seqs.q_start[seqs.n_seqs] : seqs.n_seqs)) return;  // (padding, whatever its position)
        if (!turn) flag_positions(rope, row, d0, 8, a.err);
    } else {
        int b = row, end = row + 1;
        if (seqs.q_start) {
            b = seq_of_row(seqs.q_start, seqs.n_seqs, row, lane);
            if (b < seqs.n_seqs) end = seqs.q_start[b + 1];
        }
        if (b >= seqs.n_seqs) return;
        const int own = seqs.kv_len[b] - (end - row);
        if ((own < 0 || own >> seqs.page_shift >= seqs.table_ld) && lane == 0) flag_error(a.err, ERR_KV_LEN, own);
        turn = angles<8>(rope, row, rope.pos_base + own, d0, cs, sn, a.err);
    }
    if (!__all_sync(0xffffffffu, turn)) return;
#pragma unroll
    for (int j = 0; j < IT; j++) {
        const bool on = mine + j * HPW < a.n_heads;
        float lo[8], hi[8];
#pragma unroll
        for (int e = 0; e < 8; e++) {
            lo[e] = on ? to_f32(raw[j][0][e / (16 / sizeof(S))].e[e % (16 / sizeof(S))]) : 0.0f;
            hi[e] = on ? to_f32(raw[j][1][e / (16 / sizeof(S))].e[e % (16 / sizeof(S))]) : 0.0f;
        }
        if (a.q_norm) norm_head<D>(a, a.q_norm, d0, lo, hi);
        turn_head(cs, sn, lo, hi);
        if (on) {
            __nv_bfloat16* dst = static_cast<__nv_bfloat16*>(a.q_out) + (int64_t)row * a.q_stride + (int64_t)(mine + j * HPW) * D + d0;
            store_v<8>(dst, lo);
            store_v<8>(dst + N, hi);
        }
    }
}

// WIDE: heads that rotate whole, rows and weights aligned to 16 bytes. P: positions of a warp. ITQ: heads a
// lane of the query part has in flight.
template <typename S, int D, bool WIDE, int P, int ITQ>
__global__ void __launch_bounds__(256, P == 8 ? 3 : 2) paged_append_q8_kernel(AppendArgs a, RopeAxes rope, PagedSeqs seqs, PagedQ8 c,
                                                                             int kv_ctas, int groups) {
    constexpr int LPH = D / 16, HPW = 32 / LPH, IT = P / HPW, N = D / 2;  // lanes a position, positions side by side
    __shared__ TeamInfo info[8];
    __shared__ uint32_t most[8];
    __shared__ float part[WIDE ? 1 : 8][WIDE ? 1 : HPW][WIDE ? 1 : D];
    pdl_trigger();
    pdl_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (blockIdx.x >= kv_ctas) {  // query heads
        AppendArgs qa = a;
        qa.n_kv = 0;
        const int64_t item = (int64_t)(blockIdx.x - kv_ctas) * 8 + warp;
        if constexpr (WIDE) append_query<S, D, ITQ>(qa, rope, seqs, groups, item);
        else append_any_head<S, __nv_bfloat16>(qa, rope, seqs, item);
        return;
    }
    const int wshift = c.block_shift - (P == 8 ? 3 : 4);  // log2 of a team's warps
    const int team = warp >> wshift, sub = warp & ((1 << wshift) - 1);
    const int64_t item = ((int64_t)blockIdx.x << (3 - wshift)) + team;
    const int64_t x = item / (2 * c.n_kv);
    const int hk = (int)(item - x * 2 * c.n_kv);  // K heads, then V heads
    const bool is_v = hk >= c.n_kv;
    const int kh = is_v ? hk - c.n_kv : hk;
    float* const scales = is_v ? c.v_scale : c.k_scale;
    if (sub == 0) {
        const TeamInfo t = find_block(seqs, c, x, lane, a.err);
        if (lane == 0) info[team] = t;
    }
    __syncthreads();
    const TeamInfo t = info[team];
    const int64_t scale_at = t.page * c.scale_stride + ((int64_t)kh << (seqs.page_shift - c.block_shift)) + t.slot;
    const int d0 = 8 * (lane % LPH), r = lane / LPH, base = t.first + P * sub;
    const int head = a.n_heads + hk;
    float lo[IT][8], hi[IT][8];
    unsigned bits = 0;
    uint32_t live = 0;  // iterations whose position this lane has a row for
#pragma unroll
    for (int i = 0; i < IT; i++) {
        const int at = base + i * HPW + r;
        const bool on = t.ok && at >= t.lo && at < t.hi;
        if (on) {
            live |= 1u << i;
            const S* src = static_cast<const S*>(a.qkv) + (int64_t)(t.q0 + (at - t.p0)) * a.row_stride + (int64_t)head * D + d0;
            if constexpr (WIDE) {
                load_v<8>(src, lo[i]);
                load_v<8>(src + N, hi[i]);
            } else {
#pragma unroll
                for (int e = 0; e < 8; e++) lo[i][e] = to_f32(src[e]), hi[i][e] = to_f32(src[N + e]);
            }
        } else {
#pragma unroll
            for (int e = 0; e < 8; e++) lo[i][e] = hi[i][e] = 0.0f;
        }
    }
    float old = t.ok ? scales[scale_at] : 0.0f;
    if (old < 1.17549435e-38f) old = 0.0f;  // (one that a caller put there may have no reciprocal)
    if (!is_v) {
#pragma unroll
        for (int i = 0; i < IT; i++) {
            const int at = base + i * HPW + r;
            const int64_t row = t.q0 + (at - t.p0);
            bool turn = true;
            if constexpr (WIDE) {
                float cs[8], sn[8];
                if (live >> i & 1) turn = angles<8>(rope, row, rope.pos_base + at, d0, cs, sn, a.err);
                if (a.k_norm) norm_head<D>(a, a.k_norm, d0, lo[i], hi[i]);  // (by every lane)
                if (turn && (live >> i & 1)) turn_head(cs, sn, lo[i], hi[i]);
            } else {  // any pairs (d, d + n): the other one by way of shared memory
                if (a.k_norm) norm_head<D, false>(a, a.k_norm, d0, lo[i], hi[i]);
                float* const buf = part[warp][r];
                const int n = rope.pairs;
#pragma unroll
                for (int e = 0; e < 8; e++) buf[d0 + e] = lo[i][e], buf[N + d0 + e] = hi[i][e];
                __syncwarp();
                auto turned = [&](int d, float v) {
                    if (d >= 2 * n || !(live >> i & 1)) return v;
                    const int p = d < n ? d : d - n;
                    const int64_t pos = rope.pos ? (int64_t)rope.pos[(int64_t)rope.axis[p] * rope.pos_stride + row] : rope.pos_base + at;
                    if (pos < 0 || pos >= rope.table_len) {
                        flag_error(a.err, ERR_ROPE_POS, (int)pos);
                        turn = false;
                        return v;
                    }
                    const float cs = rope.cos[pos * n + p], sn = rope.sin[pos * n + p];
                    return d < n ? __fsub_rn(__fmul_rn(v, cs), __fmul_rn(buf[d + n], sn)) : __fadd_rn(__fmul_rn(v, cs), __fmul_rn(buf[p], sn));
                };
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    lo[i][e] = turned(d0 + e, lo[i][e]);
                    hi[i][e] = turned(N + d0 + e, hi[i][e]);
                }
                __syncwarp();
            }
            // a position outside the tables: its row is left out
            const unsigned bad = __ballot_sync(0xffffffffu, !turn);
            if (bad >> (r * LPH) & ((1u << LPH) - 1)) live &= ~(1u << i);
        }
    }
#pragma unroll
    for (int i = 0; i < IT; i++)
        if (live >> i & 1) {
#pragma unroll
            for (int e = 0; e < 8; e++)
                bits = max(bits, max(__float_as_uint(lo[i][e]) & 0x7fffffffu, __float_as_uint(hi[i][e]) & 0x7fffffffu));
        }
    bits = __reduce_max_sync(0xffffffffu, bits);
    const bool any = __any_sync(0xffffffffu, live != 0);
    if (lane == 0) most[warp] = any ? bits : ~0u;  // ~0: no row
    __syncthreads();  // (and every warp of the team has read the scale)
    if (!t.ok) return;
    uint32_t top = 0;
    bool rows = false;
    for (int w = 0; w < 1 << wshift; w++) {
        const uint32_t m = most[(team << wshift) + w];
        if (m != ~0u) top = max(top, m), rows = true;
    }
    if (!rows) return;  // (every row's position was outside the tables)
    const float wants = top >= 0x7f800000u ? __uint_as_float(0x7fffffffu) : __fdiv_rn(__uint_as_float(top), 127.0f);
    const bool fresh = t.lo == t.first;
    float s = wants < 1.17549435e-38f ? 0.0f : wants;
    if (!fresh && !(s > old) && s == s) s = old;
    const float by = s > 0.0f ? __frcp_rn(s) : 0.0f;  // (zero for NaN too)
    int8_t* const page = (is_v ? c.v : c.k) + t.page * c.page_stride + ((int64_t)kh << seqs.page_shift) * D;
    const int in_page = base & ((1 << seqs.page_shift) - 1);
    if (!fresh && s > old) {  // (s not NaN, nor the old one)
        const float ratio = __fdiv_rn(old, s);
#pragma unroll 1
        for (int i = 0; i < IT; i++) {
            if (base + i * HPW + r >= t.lo) continue;
            int8_t* const at = page + (int64_t)(in_page + i * HPW + r) * D + d0;
            uint2 u = *reinterpret_cast<const uint2*>(at), w = *reinterpret_cast<const uint2*>(at + N);
            *reinterpret_cast<uint2*>(at) = make_uint2(codes_again(u.x, ratio), codes_again(u.y, ratio));
            *reinterpret_cast<uint2*>(at + N) = make_uint2(codes_again(w.x, ratio), codes_again(w.y, ratio));
        }
    }
#pragma unroll
    for (int i = 0; i < IT; i++)
        if (live >> i & 1) {
            int8_t* const at = page + (int64_t)(in_page + i * HPW + r) * D + d0;
            *reinterpret_cast<uint2*>(at) = codes8(lo[i], by);
            *reinterpret_cast<uint2*>(at + N) = codes8(hi[i], by);
        }
    if (sub == 0 && lane == 0) scales[scale_at] = s;
}

template <typename S, int D, bool WIDE, int P, int ITQ>
static int launch_append_q8(lq_ctx* ctx, const AppendArgs& a, const RopeAxes& rope, const PagedSeqs& s, const PagedQ8& c) {
    const int64_t blocks = s.q_start ? (int64_t)(s.rows >> c.block_shift) + 2ll * s.n_seqs : (int64_t)std::min(s.rows, s.n_seqs);
    const int teams = 8 >> (c.block_shift - (P == 8 ? 3 : 4));
    const int64_t kv_ctas = (blocks * 2 * c.n_kv + teams - 1) / teams;
    const int groups = WIDE ? ceil_div(a.n_heads, 512 / D * ITQ) : a.n_heads;  // warps a row
    const int64_t q_ctas = ((int64_t)s.rows * groups + 7) / 8;
    LQ_REQUIRE(ctx, kv_ctas + q_ctas < (1ll << 31), "lq_paged_append_q8: too many rows");
    return launch_kernel(ctx, paged_append_q8_kernel<S, D, WIDE, P, ITQ>, dim3((unsigned)(kv_ctas + q_ctas)), dim3(256), 0,
                         "paged_append_q8", a, rope, s, c, (int)kv_ctas, groups);
}

template <typename S, int D>
static int append_q8_d(lq_ctx* ctx, const AppendArgs& a, const RopeAxes& rope, const PagedSeqs& s, const PagedQ8& c, bool wide) {
    if (!wide) return launch_append_q8<S, D, false, 16, 1>(ctx, a, rope, s, c);
    // many rows: two query heads a lane, which share the row's angles; a decode step's few: one, so that they
    // spread over the SMs
    const bool few = (int64_t)s.rows * ceil_div(a.n_heads, 512 / D) < 16ll * ctx->sm_count;
    // a block of 128 positions takes all eight warps of a CTA 16 each; of 8 a warp has twice as many
    // neighbours on its SM
    if (c.block_shift == 7) return few ? launch_append_q8<S, D, true, 16, 1>(ctx, a, rope, s, c) : launch_append_q8<S, D, true, 16, 2>(ctx, a, rope, s, c);
    return few ? launch_append_q8<S, D, true, 8, 1>(ctx, a, rope, s, c) : launch_append_q8<S, D, true, 8, 2>(ctx, a, rope, s, c);
}

template <typename S>
static int append_q8(lq_ctx* ctx, const AppendArgs& a, const RopeAxes& rope, const PagedSeqs& s, const PagedQ8& c) {
    auto al = [](const void* p) { return (uintptr_t)p % 16 == 0; };
    const bool wide = rope.pairs * 2 == a.head_dim && a.row_stride * sizeof(S) % 16 == 0 && a.q_stride * 2 % 16 == 0 &&
                      al(a.qkv) && al(a.q_out) && al(a.q_norm) && al(a.k_norm);
    return a.head_dim == 64 ? append_q8_d<S, 64>(ctx, a, rope, s, c, wide) : append_q8_d<S, 128>(ctx, a, rope, s, c, wide);
}

// =========================================================================================
// Reading rows back: code * scale. The last warp of a CTA looks up where the next 32 rows of the batch lie
// while the others read and write 32 rows: a thread takes 16 codes at a time (one vector), eight of them
// in flight, neighbours along a position's dims and along positions, which lie next to each other in
// a page of a kv head. Bound: HBM, which likes few streams here: 24 whole sequences of up to 9000
// positions to bf16 take 98 us with two CTAs an SM (5.3 TB/s, 81 % of a plain copy), 107 with three, 124 with
// four, 102 to 120 with a CTA for every 32 rows. A call that is done in one round gets three (14054 rows of 4
// heads of 64 dims to f32: 11.7 us instead of 14.3).
// =========================================================================================
constexpr int READ_ROWS = 32, READ_THREADS = 256;
static_assert(READ_ROWS == 32, "a warp looks them up");

struct ReadArgs {
    void* k_out;
    void* v_out;
    int64_t out_stride;
    int parts;  // CTAs that share rows, each with some heads
    int* err;
};

// where row r lies, page * page size + position there, or -1: find_slot by a thread, whose neighbours look up
// the neighbouring rows (a warp a row, four in turn: 6 us of a CTA's life)
__device__ __forceinline__ int slot_of_row(const PagedSeqs& s, int r, int* err) {
    int b = r, end = r + 1;
    if (s.q_start) {
        int n = s.n_seqs;  // the number of ends q_start[1..B] that are <= r lies in [b, b + n]
        b = 0;
        while (n > 0) {
            const int half = n >> 1;
            if (s.q_start[b + half + 1] <= r) b += half + 1, n -= half + 1;
            else n = half;
        }
        if (b >= s.n_seqs) return -1;
        end = s.q_start[b + 1];
    } else if (b >= s.n_seqs) {
        return -1;
    }
    const int own = s.kv_len[b] - (end - r), pg = own >> s.page_shift;
    if (own < 0 || pg >= s.table_ld) {
        flag_error(err, ERR_KV_LEN, own);
        return -1;
    }
    const int page = s.table[(int64_t)b * s.table_ld + pg];
    if ((unsigned)page >= (unsigned)s.n_pages) {
        flag_error(err, ERR_PAGE_ID, page);
        return -1;
    }
    return (page << s.page_shift) + (own & ((1 << s.page_shift) - 1));
}

__device__ __forceinline__ void store_cs(float* p, const float* v) {
#pragma unroll
    for (int i = 0; i < 16; i += 4) __stcs(reinterpret_cast<float4*>(p + i), make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]));
}
__device__ __forceinline__ void store_cs(__nv_bfloat16* p, const float* v) {
#pragma unroll
    for (int i = 0; i < 16; i += 8)
        __stcs(reinterpret_cast<uint4*>(p + i), make_uint4(pack_bf16x2(v[i], v[i + 1]), pack_bf16x2(v[i + 2], v[i + 3]),
                                                           pack_bf16x2(v[i + 4], v[i + 5]), pack_bf16x2(v[i + 6], v[i + 7])));
}

// CTAS: on an SM
template <typename T, int D, int CTAS>
__global__ void __launch_bounds__(READ_THREADS + 32, CTAS) paged_read_q8_kernel(ReadArgs a, PagedSeqs s, PagedQ8 c) {
    constexpr int CH = D / 16;  // vectors of a position
    __shared__ int slots[2][READ_ROWS];  // page * page size + position there, or -1
    pdl_trigger();
    pdl_wait();
    const int tid = threadIdx.x, part = blockIdx.x % a.parts;
    const int groups = (s.rows + READ_ROWS - 1) / READ_ROWS, step = gridDim.x / a.parts;
    const int heads = 2 * c.n_kv, h0 = heads * part / a.parts, h1 = heads * (part + 1) / a.parts;
    const int mask = (1 << s.page_shift) - 1, sshift = s.page_shift - c.block_shift;
    constexpr int STEP = READ_THREADS / CH, BATCH = 8;
    const int ch = tid % CH;
    auto look = [&](int g, int buf) {  // by the last warp: the slots of a group
        const int i = tid - READ_THREADS, row = g * READ_ROWS + i;
        if (g < groups) slots[buf][i] = row < s.rows ? slot_of_row(s, row, part == 0 ? a.err : nullptr) : -1;
    };
    int g = blockIdx.x / a.parts, buf = 0;
    if (tid >= READ_THREADS) look(g, 0);
    __syncthreads();
#pragma unroll 1
    for (; g < groups; g += step, buf ^= 1) {
        if (tid >= READ_THREADS) {
            look(g + step, buf ^ 1);
        } else {
            const int* const slot = slots[buf];
            const int64_t row0 = (int64_t)g * READ_ROWS;
            // (rows fastest, then heads)
#pragma unroll 1
            for (int i0 = h0 * READ_ROWS + tid / CH; i0 < h1 * READ_ROWS; i0 += STEP * BATCH) {
                uint4 w[BATCH];
                float sc[BATCH];
#pragma unroll
                for (int j = 0; j < BATCH; j++) {
                    const int i = i0 + j * STEP, hk = i / READ_ROWS;
                    const int at = i < h1 * READ_ROWS ? slot[i % READ_ROWS] : -1;
                    if (at < 0) continue;
                    const bool is_v = hk >= c.n_kv;
                    const int kh = is_v ? hk - c.n_kv : hk, page = at >> s.page_shift, off = at & mask;
                    w[j] = __ldcs(reinterpret_cast<const uint4*>((is_v ? c.v : c.k) + page * c.page_stride +
                                                                 (((int64_t)kh << s.page_shift) + off) * D + 16 * ch));
                    sc[j] = (is_v ? c.v_scale : c.k_scale)[page * c.scale_stride + ((int64_t)kh << sshift) + (off >> c.block_shift)];
                }
#pragma unroll
                for (int j = 0; j < BATCH; j++) {
                    const int i = i0 + j * STEP, hk = i / READ_ROWS;
                    if (i >= h1 * READ_ROWS || slot[i % READ_ROWS] < 0) continue;
                    const bool is_v = hk >= c.n_kv;
                    T* const dst = static_cast<T*>(is_v ? a.v_out : a.k_out) + (row0 + i % READ_ROWS) * a.out_stride +
                                   (int64_t)(is_v ? hk - c.n_kv : hk) * D + 16 * ch;
                    float v[16];
                    const uint32_t u[4] = {w[j].x, w[j].y, w[j].z, w[j].w};
#pragma unroll
                    for (int e = 0; e < 16; e++) v[e] = (float)(int8_t)(u[e / 4] >> (8 * (e % 4))) * sc[j];
                    store_cs(dst, v);
                }
            }
        }
        __syncthreads();
    }
}

template <typename T, int D>
static int launch_read_q8(lq_ctx* ctx, ReadArgs a, const PagedSeqs& s, const PagedQ8& c) {
    const int64_t groups = ceil_div(s.rows, READ_ROWS);
    // few rows: their heads over several CTAs
    a.parts = (int)std::max<int64_t>(1, std::min<int64_t>(2 * c.n_kv, 3 * ctx->sm_count / groups));
    if (groups * a.parts <= 3 * ctx->sm_count)
        return launch_kernel(ctx, paged_read_q8_kernel<T, D, 3>, dim3((unsigned)(groups * a.parts)), dim3(READ_THREADS + 32), 0,
                             "paged_read_q8", a, s, c);
    const int ctas = std::max(1, 2 * ctx->sm_count / a.parts) * a.parts;
    return launch_kernel(ctx, paged_read_q8_kernel<T, D, 2>, dim3((unsigned)ctas), dim3(READ_THREADS + 32), 0, "paged_read_q8", a, s, c);
}

int make_paged_q8(lq_ctx* ctx, const char* who, PagedQ8* c, int8_t* k, int8_t* v, float* k_scale, float* v_scale,
                  int64_t n_kv_heads, int64_t head_dim, int64_t page_size, int64_t page_stride, int64_t block,
                  int64_t scale_stride, bool any_rows) {
    LQ_REQUIRE(ctx, n_kv_heads >= 1 && n_kv_heads <= 4096, "%s: bad head counts", who);
    LQ_REQUIRE(ctx, head_dim == 64 || head_dim == 128, "%s: head_dim %lld must be 64 or 128", who, (long long)head_dim);
    LQ_REQUIRE(ctx, block >= 16 && block <= 128 && (block & (block - 1)) == 0 && block <= page_size,
               "%s: block %lld must be 16, 32, 64 or 128 positions and no longer than a page of %lld", who, (long long)block,
               (long long)page_size);
    const int64_t dense = n_kv_heads * page_size * head_dim, dense_s = n_kv_heads * (page_size / block);
    if (page_stride == 0) page_stride = dense;
    if (scale_stride == 0) scale_stride = dense_s;
    LQ_REQUIRE(ctx, page_stride >= dense && page_stride % 16 == 0 && page_stride < (1ll << 40),
               "%s: page_stride %lld must be a multiple of 16 and at least %lld", who, (long long)page_stride, (long long)dense);
    LQ_REQUIRE(ctx, scale_stride >= dense_s && scale_stride < (1ll << 40), "%s: scale_stride %lld must be at least %lld", who,
               (long long)scale_stride, (long long)dense_s);
    LQ_REQUIRE(ctx, !any_rows || (k && v && k_scale && v_scale), "%s: NULL pointer", who);
    LQ_REQUIRE(ctx, aligned_to(k, 16) && aligned_to(v, 16) && aligned_to(k_scale, 4) && aligned_to(v_scale, 4),
               "%s: codes must be aligned to 16 bytes, scales to their elements", who);
    c->k = k;
    c->v = v;
    c->k_scale = k_scale;
    c->v_scale = v_scale;
    c->page_stride = page_stride;
    c->scale_stride = scale_stride;
    c->n_kv = (int)n_kv_heads;
    c->block_shift = 0;
    while ((1 << c->block_shift) < block) c->block_shift++;
    return LQ_OK;
}

}  // namespace lq

extern "C" {

int lq_paged_append_q8(lq_ctx* ctx, const void* qkv, lq_dtype qkv_dtype, int64_t row_stride, int64_t rows, int64_t n_heads,
                       int64_t n_kv_heads, int64_t head_dim, const uint16_t* q_norm, const uint16_t* k_norm, float eps,
                       int norm_bf16, int64_t rot_dim, const float* cos_dev, const float* sin_dev, int64_t table_len,
                       const uint8_t* pair_axis_host, int64_t n_axes, const int32_t* pos_dev, int64_t pos_stride,
                       int64_t pos_base, int64_t n_seqs, const int32_t* q_start, const int32_t* kv_len,
                       const int32_t* page_table, int64_t table_ld, int8_t* k_codes, int8_t* v_codes, float* k_scale,
                       float* v_scale, int64_t n_pages, int64_t page_size, int64_t page_stride, int64_t block,
                       int64_t scale_stride, uint16_t* q_out, int64_t q_stride) {
    LQ_ENTRY(ctx, "lq_paged_append_q8");
    LQ_REQUIRE(ctx, qkv_dtype == LQ_DTYPE_F32 || qkv_dtype == LQ_DTYPE_BF16, "lq_paged_append_q8: rows must be F32 or BF16");
    LQ_REQUIRE(ctx, n_heads >= 0 && n_heads <= (1 << 16) && n_kv_heads >= 1 && n_kv_heads <= (1 << 16) &&
                        n_heads + 2 * n_kv_heads <= (1 << 16), "lq_paged_append_q8: bad head counts");
    lq::RopeAxes rope;
    lq::PagedSeqs s;
    lq::PagedQ8 c;
    int rc = lq::make_paged_seqs(ctx, "lq_paged_append_q8", &s, n_seqs, q_start, kv_len, page_table, table_ld, rows, n_pages,
                                 page_size);
    if (rc) return rc;
    rc = lq::make_paged_q8(ctx, "lq_paged_append_q8", &c, k_codes, v_codes, k_scale, v_scale, n_kv_heads, head_dim, page_size,
                           page_stride, block, scale_stride, rows > 0 && n_seqs > 0);
    if (rc) return rc;
    rc = lq::make_rope_axes(ctx, "lq_paged_append_q8", &rope, rot_dim, head_dim, cos_dev, sin_dev, table_len, pair_axis_host,
                            n_axes, pos_dev, pos_stride, rows);
    if (rc) return rc;
    rope.pos_base = pos_base;
    if (row_stride == 0) row_stride = (n_heads + 2 * n_kv_heads) * head_dim;
    if (q_stride == 0) q_stride = n_heads * head_dim;
    LQ_REQUIRE(ctx, row_stride >= (n_heads + 2 * n_kv_heads) * head_dim, "lq_paged_append_q8: row_stride too small");
    LQ_REQUIRE(ctx, q_stride >= n_heads * head_dim, "lq_paged_append_q8: q_stride too small");
    if (rows == 0 || n_seqs == 0) return LQ_OK;
    LQ_REQUIRE(ctx, qkv && (q_out || n_heads == 0), "lq_paged_append_q8: NULL pointer");
    LQ_REQUIRE(ctx, lq::aligned_to(qkv, qkv_dtype == LQ_DTYPE_F32 ? 4 : 2) && lq::aligned_to(q_out, 2) &&
                        lq::aligned_to(q_norm, 2) && lq::aligned_to(k_norm, 2),
               "lq_paged_append_q8: pointers must be aligned to their elements");
    lq::AppendArgs a;
    a.qkv = qkv;
    a.row_stride = row_stride;
    a.n_heads = (int)n_heads;
    a.n_kv = (int)n_kv_heads;
    a.head_dim = (int)head_dim;
    a.q_norm = q_norm;
    a.k_norm = k_norm;
    a.eps = eps;
    a.norm_bf16 = norm_bf16;
    a.k = a.v = nullptr;
    a.page_stride = 0;
    a.q_out = q_out;
    a.q_stride = q_stride;
    a.err = ctx->err_flag;
    return qkv_dtype == LQ_DTYPE_F32 ? lq::append_q8<float>(ctx, a, rope, s, c) : lq::append_q8<__nv_bfloat16>(ctx, a, rope, s, c);
}

int lq_paged_read_q8(lq_ctx* ctx, const int8_t* k_codes, const int8_t* v_codes, const float* k_scale, const float* v_scale,
                     int64_t n_kv_heads, int64_t head_dim, int64_t n_pages, int64_t page_size, int64_t page_stride,
                     int64_t block, int64_t scale_stride, int64_t n_seqs, const int32_t* q_start, const int32_t* kv_len,
                     const int32_t* page_table, int64_t table_ld, int64_t rows, void* k_out, void* v_out,
                     lq_dtype out_dtype, int64_t out_stride) {
    LQ_ENTRY(ctx, "lq_paged_read_q8");
    LQ_REQUIRE(ctx, out_dtype == LQ_DTYPE_F32 || out_dtype == LQ_DTYPE_BF16, "lq_paged_read_q8: rows must be F32 or BF16");
    lq::PagedSeqs s;
    lq::PagedQ8 c;
    int rc = lq::make_paged_seqs(ctx, "lq_paged_read_q8", &s, n_seqs, q_start, kv_len, page_table, table_ld, rows, n_pages,
                                 page_size);
    if (rc) return rc;
    rc = lq::make_paged_q8(ctx, "lq_paged_read_q8", &c, const_cast<int8_t*>(k_codes), const_cast<int8_t*>(v_codes),
                           const_cast<float*>(k_scale), const_cast<float*>(v_scale), n_kv_heads, head_dim, page_size,
                           page_stride, block, scale_stride, rows > 0 && n_seqs > 0);
    if (rc) return rc;
    if (out_stride == 0) out_stride = n_kv_heads * head_dim;
    LQ_REQUIRE(ctx, out_stride >= n_kv_heads * head_dim, "lq_paged_read_q8: out_stride too small");
    if (rows == 0 || n_seqs == 0) return LQ_OK;
    LQ_REQUIRE(ctx, k_out && v_out, "lq_paged_read_q8: NULL pointer");
    LQ_REQUIRE(ctx, lq::aligned_to(k_out, 16) && lq::aligned_to(v_out, 16) &&
                        out_stride * (out_dtype == LQ_DTYPE_F32 ? 4 : 2) % 16 == 0,
               "lq_paged_read_q8: outputs and their rows must be aligned to 16 bytes");
    const lq::ReadArgs a{k_out, v_out, out_stride, 1, ctx->err_flag};
    if (out_dtype == LQ_DTYPE_F32)
        return head_dim == 64 ? lq::launch_read_q8<float, 64>(ctx, a, s, c) : lq::launch_read_q8<float, 128>(ctx, a, s, c);
    return head_dim == 64 ? lq::launch_read_q8<__nv_bfloat16, 64>(ctx, a, s, c)
                          : lq::launch_read_q8<__nv_bfloat16, 128>(ctx, a, s, c);
}

}  // extern "C"
