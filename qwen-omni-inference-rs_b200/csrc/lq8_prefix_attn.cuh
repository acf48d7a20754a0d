// lq8_prefix_attn.cuh -- the kernels behind lq_prefix_attention, and how they write a finished row.
#pragma once

#include "lq8_fused.cuh"
#include "lq8_paged_q8.cuh"
#include "lq8_prefix_plan.cuh"

namespace lq {

// 32 consecutive dims (from dim `at`) of row tok, head h, by one thread: cache type and/or Q8_0
template <typename T, int D>
__device__ __forceinline__ void pa_store32(const PrefixAttnArgs& a, int tok, int h, int at, const float v[32]) {
    if (a.out) {
        T* const o = static_cast<T*>(a.out) + (int64_t)tok * a.out_stride + (int64_t)h * D + at;
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int j = 0; j < 32; j += 4)
                *reinterpret_cast<float4*>(o + j) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
        } else {
#pragma unroll
            for (int j = 0; j < 32; j += 8)
                *reinterpret_cast<uint4*>(o + j) = make_uint4(pack_bf16x2(v[j], v[j + 1]), pack_bf16x2(v[j + 2], v[j + 3]),
                                                              pack_bf16x2(v[j + 4], v[j + 5]), pack_bf16x2(v[j + 6], v[j + 7]));
        }
    }
    if (a.xq) {
        float amax = 0.0f, d, id;
#pragma unroll
        for (int j = 0; j < 32; j++) amax = fmaxf(amax, fabsf(v[j]));
        q8_scale(amax, d, id);
        const int64_t blk = ((int64_t)tok * a.n_heads + h) * (D / 32) + at / 32;
        a.xd[blk] = f2h(d);
        uint32_t w[8];
#pragma unroll
        for (int j = 0; j < 8; j++) {
            w[j] = 0;
#pragma unroll
            for (int i = 0; i < 4; i++) w[j] |= (uint32_t)(q8_quant(v[4 * j + i], id) & 0xFF) << (8 * i);
        }
        uint4* const q = reinterpret_cast<uint4*>(a.xq + blk * 32);
        q[0] = make_uint4(w[0], w[1], w[2], w[3]);
        q[1] = make_uint4(w[4], w[5], w[6], w[7]);
    }
}

// two dims (at, at + 1) of row tok, head h, by the 16 lanes that hold the 32 dims of a block; every
// lane of the warp calls it, those with `on` write
template <typename T, int D>
__device__ __forceinline__ void store2(const PrefixAttnArgs& a, int tok, int h, int at, float2 y, bool on) {
    if (a.out && on) {
        T* const o = static_cast<T*>(a.out) + (int64_t)tok * a.out_stride + (int64_t)h * D + at;
        if constexpr (sizeof(T) == 4) *reinterpret_cast<float2*>(o) = y;
        else *reinterpret_cast<uint32_t*>(o) = pack_bf16x2(y.x, y.y);
    }
    if (a.xq) {
        float amax = fmaxf(fabsf(y.x), fabsf(y.y)), d, id;
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
        q8_scale(amax, d, id);
        const int64_t i = ((int64_t)tok * a.n_heads + h) * D + at;
        if (on) {
            if (at % 32 == 0) a.xd[i / 32] = f2h(d);
            *reinterpret_cast<uint16_t*>(a.xq + i) = (uint16_t)((q8_quant(y.x, id) & 0xFF) | (q8_quant(y.y, id) & 0xFF) << 8);
        }
    }
}

// rows tok0 .. tok0 + n - 1, which see no position: zeros, by `threads` threads
template <typename T, int D>
__device__ __forceinline__ void zero_rows(const PrefixAttnArgs& a, int tok0, int n, int thread, int threads) {
    const uint4 z = make_uint4(0, 0, 0, 0);
    const int blocks = a.n_heads * (D / 32);  // of 32 dims
#pragma unroll 1
    for (int tok = tok0; tok < tok0 + n; tok++)
#pragma unroll 1
        for (int i = thread; i < blocks; i += threads) {
            if (a.out) {
                uint4* const o = reinterpret_cast<uint4*>(static_cast<T*>(a.out) + (int64_t)tok * a.out_stride + i * 32);
#pragma unroll
                for (int j = 0; j < (int)sizeof(T) * 2; j++) o[j] = z;
            }
            if (a.xq) {
                const int64_t at = (int64_t)tok * blocks + i;
                uint4* const q = reinterpret_cast<uint4*>(a.xq + at * 32);
                q[0] = q[1] = z;
                a.xd[at] = 0;
            }
        }
}

// 8-bit caches: a score gets log2 of V's scale on top, of no less than 2^-80. A block of zeros so still has its
// weight in the sums, and sums of weight / scale stay finite.
constexpr float PREFIX_ATTN_Q8_LEAST = 8.2718061e-25f;

int launch_prefix_attn_f32(lq_ctx* ctx, const PrefixAttnArgs& a, const PagedSeqs& s, const PrefixPlan& p, int D);
int launch_prefix_attn_q8_decode(lq_ctx* ctx, const PrefixAttnArgs& a, const PagedSeqs& s, const PagedQ8& c, const PrefixPlan& p, int D, int rows);
int launch_prefix_attn_q8_join(lq_ctx* ctx, const PrefixAttnArgs& a, const PagedSeqs& s, const PrefixPlan& p, int D);  // its merge without a prefix
// q8: a cache in 8 bits (else bf16)
int launch_prefix_attn_tc(lq_ctx* ctx, const PrefixAttnArgs& a, const PagedSeqs& s, const PrefixPlan& p, int D, const PagedQ8* q8 = nullptr);

}  // namespace lq
