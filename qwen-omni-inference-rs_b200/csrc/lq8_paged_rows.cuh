// lq8_paged_rows.cuh -- device code that the appends to a paged cache share: wide loads, rotary
// angles, a row's slot, norm and rotation of a head, and the heads of a row in a cache of f32 or bf16.
#pragma once

#include "lq8_async.cuh"
#include "lq8_fused.cuh"
#include "lq8_paged.cuh"

namespace lq {

// V consecutive elements of T as f32, and back (bf16 by round to nearest even)
template <typename T, int V>
struct alignas(sizeof(T) * V) Vec {
    T e[V];
};
__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void from_f32(float& d, float v) { d = v; }
__device__ __forceinline__ void from_f32(__nv_bfloat16& d, float v) { d = __float2bfloat16_rn(v); }

// V consecutive values as f32, in vectors of 16 bytes (V elements aligned so)
template <int V>
__device__ __forceinline__ void load_v(const float* p, float v[V]) {
#pragma unroll
    for (int i = 0; i < V; i += 4) {
        const float4 t = *reinterpret_cast<const float4*>(p + i);
        v[i] = t.x, v[i + 1] = t.y, v[i + 2] = t.z, v[i + 3] = t.w;
    }
}
template <int V>
__device__ __forceinline__ void load_v(const __nv_bfloat16* p, float v[V]) {
    const Vec<__nv_bfloat16, V> t = *reinterpret_cast<const Vec<__nv_bfloat16, V>*>(p);
#pragma unroll
    for (int i = 0; i < V; i++) v[i] = to_f32(t.e[i]);
}
template <int V>
__device__ __forceinline__ void store_v(float* p, const float v[V]) {
#pragma unroll
    for (int i = 0; i < V; i += 4) *reinterpret_cast<float4*>(p + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
}
template <int V>
__device__ __forceinline__ void store_v(__nv_bfloat16* p, const float v[V]) {
    Vec<__nv_bfloat16, V> t;
#pragma unroll
    for (int i = 0; i < V; i++) t.e[i] = __float2bfloat16_rn(v[i]);
    *reinterpret_cast<Vec<__nv_bfloat16, V>*>(p) = t;
}

// cos and sin of pairs i0 .. i0 + V - 1 of a row (`at`: its position when the call gives none);
// false, and the error flag, when a position lies outside the tables
template <int V>
__device__ __forceinline__ bool angles(const RopeAxes& rope, int64_t row, int64_t at, int i0, float cs[V], float sn[V], int* err) {
    if (V >= 4 && ((V == 8 ? rope.same8 : rope.same4) >> (i0 / V) & 1)) {
        const int64_t p = rope.pos ? (int64_t)rope.pos[(int64_t)rope.axis[i0] * rope.pos_stride + row] : at;
        if (p < 0 || p >= rope.table_len) {
            flag_error(err, ERR_ROPE_POS, (int)p);
            return false;
        }
        if constexpr (V >= 4) {
            load_v<V>(rope.cos + p * rope.pairs + i0, cs);
            load_v<V>(rope.sin + p * rope.pairs + i0, sn);
        }
        return true;
    }
    bool ok = true;
#pragma unroll
    for (int e = 0; e < V; e++) {
        const int64_t p = rope.pos ? (int64_t)rope.pos[(int64_t)rope.axis[i0 + e] * rope.pos_stride + row] : at;
        const bool in = p >= 0 && p < rope.table_len;
        if (!in) flag_error(err, ERR_ROPE_POS, (int)p);
        ok &= in;
        const int64_t o = (in ? p : 0) * rope.pairs + i0 + e;
        cs[e] = rope.cos[o];
        sn[e] = rope.sin[o];
    }
    return ok;
}

// flags a position of pairs i0 .. i0 + n - 1 of a row that lies outside the tables
__device__ __forceinline__ void flag_positions(const RopeAxes& rope, int64_t row, int i0, int n, int* err) {
#pragma unroll 1
    for (int i = i0; i < i0 + n; i++) {
        const int p = rope.pos[(int64_t)rope.axis[i] * rope.pos_stride + row];
        if (p < 0 || p >= rope.table_len) flag_error(err, ERR_ROPE_POS, p);
    }
}

struct AppendArgs {
    const void* qkv;
    int64_t row_stride;
    int n_heads, n_kv, head_dim;
    const uint16_t* q_norm;
    const uint16_t* k_norm;
    float eps;
    int norm_bf16;   // the rounding points of lq_rmsnorm: input and normalised output to bf16
    void* k;
    void* v;
    int64_t page_stride;
    void* q_out;
    int64_t q_stride;
    int* err;
};

// RMSNorm of a head of D dims by the D / 16 lanes that hold it, dims d0 .. d0 + 7 and those of its upper
// half each; every lane of the warp calls it, nw NULL: nothing to do. WIDE: weights aligned to 16 bytes
template <int D, bool WIDE = true>
__device__ __forceinline__ void norm_head(const AppendArgs& a, const uint16_t* nw, int d0, float lo[8], float hi[8]) {
    constexpr int LPH = D / 16, N = D / 2;
    if (nw && a.norm_bf16) {
#pragma unroll
        for (int e = 0; e < 8; e++) lo[e] = round_bf16(lo[e]), hi[e] = round_bf16(hi[e]);
    }
    // the sum of squares in the order of lq_qk_norm_rope_kv, where a lane has dims 2 v,
    // 2 v + 1 and theirs of the upper half and a butterfly joins the lanes from bit 4 down:
    // here v = 4 (lane % LPH) + k, so bits 4 to 2 are lanes and bits 1 and 0 are k
    float t[4];
#pragma unroll
    for (int k = 0; k < 4; k++)
        t[k] = __fadd_rn(__fadd_rn(__fmul_rn(lo[2 * k], lo[2 * k]), __fmul_rn(lo[2 * k + 1], lo[2 * k + 1])),
                         __fadd_rn(__fmul_rn(hi[2 * k], hi[2 * k]), __fmul_rn(hi[2 * k + 1], hi[2 * k + 1])));
#pragma unroll
    for (int d = LPH / 2; d > 0; d >>= 1)
#pragma unroll
        for (int k = 0; k < 4; k++) t[k] = __fadd_rn(t[k], __shfl_xor_sync(0xffffffffu, t[k], d));
    const float ss = __fadd_rn(__fadd_rn(t[0], t[2]), __fadd_rn(t[1], t[3]));
    if (nw) {
        const float inv = __frcp_rn(__fsqrt_rn(__fadd_rn(__fmul_rn(ss, 1.0f / D), a.eps)));  // (1 / D is exact)
        float w0[8], w1[8];
        if constexpr (WIDE) {
            load_v<8>(reinterpret_cast<const __nv_bfloat16*>(nw) + d0, w0);
            load_v<8>(reinterpret_cast<const __nv_bfloat16*>(nw) + N + d0, w1);
        } else {
#pragma unroll
            for (int e = 0; e < 8; e++) w0[e] = bf16_to_f32(nw[d0 + e]), w1[e] = bf16_to_f32(nw[N + d0 + e]);
        }
#pragma unroll
        for (int e = 0; e < 8; e++) {
            lo[e] = __fmul_rn(__fmul_rn(lo[e], inv), w0[e]);
            hi[e] = __fmul_rn(__fmul_rn(hi[e], inv), w1[e]);
            if (a.norm_bf16) lo[e] = round_bf16(lo[e]), hi[e] = round_bf16(hi[e]);
        }
    }
}

// the rotation of 8 pairs of a lane
__device__ __forceinline__ void turn_head(const float cs[8], const float sn[8], float lo[8], float hi[8]) {
#pragma unroll
    for (int e = 0; e < 8; e++) {
        const float p = lo[e], q = hi[e];
        lo[e] = __fsub_rn(__fmul_rn(p, cs[e]), __fmul_rn(q, sn[e]));
        hi[e] = __fadd_rn(__fmul_rn(q, cs[e]), __fmul_rn(p, sn[e]));
    }
}

// where row r's k and v go: page id and slot in the page; false: nowhere (padding, or an error)
struct RowSlot {
    int own;         // position in the sequence's own pages
    int page, off;
    bool live;       // the row belongs to a sequence
    bool ok;         // ... and has a slot
};

__device__ __forceinline__ RowSlot find_slot(const PagedSeqs& s, int r, int lane, int* err) {
    RowSlot o{0, 0, 0, false, false};
    int b = r, end = r + 1;
    if (s.q_start) {
        b = seq_of_row(s.q_start, s.n_seqs, r, lane);
        if (b >= s.n_seqs) return o;
        end = s.q_start[b + 1];
    } else if (b >= s.n_seqs) {
        return o;
    }
    o.live = true;
    o.own = s.kv_len[b] - (end - r);
    const int pg = o.own >> s.page_shift;
    if (o.own < 0 || pg >= s.table_ld) {
        if (lane == 0) flag_error(err, ERR_KV_LEN, o.own);
        return o;
    }
    o.page = s.table[(int64_t)b * s.table_ld + pg];
    o.off = o.own & ((1 << s.page_shift) - 1);
    if (o.page < 0 || o.page >= s.n_pages) {
        if (lane == 0) flag_error(err, ERR_PAGE_ID, o.page);
        return o;
    }
    o.ok = true;
    return o;
}

// A warp's heads of one row: q, k and v of an append into a cache of T (n_kv 0: q alone). `groups` warps
// share a row; item: row * groups + the warp's place in it.
template <typename S, typename T, int D, int IT>
__device__ __forceinline__ void append_heads(const AppendArgs& a, const RopeAxes& rope, const PagedSeqs& seqs, int groups, int64_t item) {
    constexpr int LPH = D / 16, HPW = 32 / LPH, N = D / 2;  // lanes a head, heads side by side
    const int lane = threadIdx.x & 31;
    const int row = (int)(item / groups);
    const int h0 = (int)(item - (int64_t)row * groups) * (HPW * IT);  // the warp's first head
    if (row >= seqs.rows) return;
    const int heads = a.n_heads + 2 * a.n_kv, d0 = 8 * (lane % LPH), mine = h0 + lane / LPH;
    const S* src = static_cast<const S*>(a.qkv) + (int64_t)row * a.row_stride + (int64_t)mine * D + d0;
    Vec<S, 16 / sizeof(S)> raw[IT][2][sizeof(S) / 2];
#pragma unroll
    for (int j = 0; j < IT; j++)
        if (mine + j * HPW < heads) {
#pragma unroll
            for (int k = 0; k < (int)sizeof(S) / 2; k++) {
                raw[j][0][k] = *reinterpret_cast<const Vec<S, 16 / sizeof(S)>*>(src + j * HPW * D + k * (16 / sizeof(S)));
                raw[j][1][k] = *reinterpret_cast<const Vec<S, 16 / sizeof(S)>*>(src + j * HPW * D + N + k * (16 / sizeof(S)));
            }
        }
    // (given positions do not wait for the row's place, whose loads depend on one another)
    float cs[8], sn[8];
    bool turn = true;
    const bool turned = h0 < a.n_heads + a.n_kv;
    if (turned && rope.pos) turn = angles<8>(rope, row, 0, d0, cs, sn, nullptr);
    const RowSlot slot = find_slot(seqs, row, lane, a.err);
    if (!slot.live) return;  // (padding, whatever its position)
    if (!turn) flag_positions(rope, row, d0, 8, a.err);
    if (turned && !rope.pos) turn = angles<8>(rope, row, rope.pos_base + slot.own, d0, cs, sn, a.err);
    turn = __all_sync(0xffffffffu, turn);
    T* const page_k = static_cast<T*>(a.k) + slot.page * a.page_stride;
    T* const page_v = static_cast<T*>(a.v) + slot.page * a.page_stride;
#pragma unroll
    for (int j = 0; j < IT; j++) {
        if (h0 + j * HPW >= heads) break;
        const int h = mine + j * HPW;
        const bool is_q = h < a.n_heads, is_v = h >= a.n_heads + a.n_kv, on = h < heads && (is_q || slot.ok) && (is_v || turn);
        float lo[8], hi[8];
        if (h < heads) {
#pragma unroll
            for (int e = 0; e < 8; e++) {
                lo[e] = to_f32(raw[j][0][e / (16 / sizeof(S))].e[e % (16 / sizeof(S))]);
                hi[e] = to_f32(raw[j][1][e / (16 / sizeof(S))].e[e % (16 / sizeof(S))]);
            }
        } else {
#pragma unroll
            for (int e = 0; e < 8; e++) lo[e] = hi[e] = 0.0f;
        }
        const uint16_t* const nw = is_q ? a.q_norm : is_v ? nullptr : a.k_norm;
        if (a.q_norm || a.k_norm) norm_head<D>(a, nw, d0, lo, hi);  // (by every lane, weights or none)
        if (!is_v && turn) turn_head(cs, sn, lo, hi);
        if (on) {
            T* dst;
            if (is_q) {
                dst = static_cast<T*>(a.q_out) + (int64_t)row * a.q_stride + (int64_t)h * D;
            } else {
                const int kh = h - a.n_heads - (is_v ? a.n_kv : 0);
                dst = (is_v ? page_v : page_k) + (((int64_t)kh << seqs.page_shift) + slot.off) * D;
            }
            store_v<8>(dst + d0, lo);
            store_v<8>(dst + d0 + N, hi);
        }
    }
}

// any even head dimension up to 256, rotated in part or whole: one warp a head, a lane's
// elements 32 apart, the other member of a pair read again
template <typename S, typename T>
__device__ __forceinline__ void append_any_head(const AppendArgs& a, const RopeAxes& rope, const PagedSeqs& seqs, int64_t item) {
    const int lane = threadIdx.x & 31, D = a.head_dim;
    const int heads = a.n_heads + 2 * a.n_kv;
    const int row = (int)(item / heads), h = (int)(item - (int64_t)row * heads);
    if (row >= seqs.rows) return;
    const RowSlot slot = find_slot(seqs, row, lane, a.err);
    if (!slot.live || (h >= a.n_heads && !slot.ok)) return;
    const S* src = static_cast<const S*>(a.qkv) + (int64_t)row * a.row_stride + (int64_t)h * D;
    T* dst;
    if (h < a.n_heads) {
        dst = static_cast<T*>(a.q_out) + (int64_t)row * a.q_stride + (int64_t)h * D;
    } else {
        const bool is_k = h < a.n_heads + a.n_kv;
        const int kh = h - a.n_heads - (is_k ? 0 : a.n_kv);
        dst = static_cast<T*>(is_k ? a.k : a.v) + slot.page * a.page_stride +
              (((int64_t)kh << seqs.page_shift) + slot.off) * D;
    }
    if (h >= a.n_heads + a.n_kv) {
        for (int e = lane; e < D; e += 32) from_f32(dst[e], to_f32(src[e]));
        return;
    }
    const uint16_t* nw = h < a.n_heads ? a.q_norm : a.k_norm;
    float inv = 1.0f;
    if (nw) {
        float ss = 0.0f;
        for (int e = lane; e < D; e += 32) {
            const float v = a.norm_bf16 ? round_bf16(to_f32(src[e])) : to_f32(src[e]);
            ss = __fadd_rn(ss, __fmul_rn(v, v));
        }
        ss = warp_sum(ss);
        inv = __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn(__fdiv_rn(ss, (float)D), a.eps)));
    }
    auto value = [&](int e) {
        float v = to_f32(src[e]);
        if (nw) {
            if (a.norm_bf16) v = round_bf16(v);
            v = __fmul_rn(__fmul_rn(v, inv), bf16_to_f32(nw[e]));
            if (a.norm_bf16) v = round_bf16(v);
        }
        return v;
    };
    bool ok = true;
    for (int i = lane; i < rope.pairs; i += 32) {
        const int64_t p = rope.pos ? (int64_t)rope.pos[(int64_t)rope.axis[i] * rope.pos_stride + row]
                                   : rope.pos_base + slot.own;
        if (p < 0 || p >= rope.table_len) {
            flag_error(a.err, ERR_ROPE_POS, (int)p);
            ok = false;
        }
    }
    if (!__all_sync(0xffffffffu, ok)) return;
    for (int i = lane; i < rope.pairs; i += 32) {
        const int64_t p = rope.pos ? (int64_t)rope.pos[(int64_t)rope.axis[i] * rope.pos_stride + row]
                                   : rope.pos_base + slot.own;
        const float c = rope.cos[p * rope.pairs + i], s = rope.sin[p * rope.pairs + i];
        const float u = value(i), w = value(i + rope.pairs);
        from_f32(dst[i], __fsub_rn(__fmul_rn(u, c), __fmul_rn(w, s)));
        from_f32(dst[i + rope.pairs], __fadd_rn(__fmul_rn(w, c), __fmul_rn(u, s)));
    }
    for (int e = 2 * rope.pairs + lane; e < D; e += 32) from_f32(dst[e], value(e));
}

}  // namespace lq
