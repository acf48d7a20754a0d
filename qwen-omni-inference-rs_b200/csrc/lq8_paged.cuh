// lq8_paged.cuh -- what the paged-cache kernels share: the batch of sequences with their new
// rows, the page layout, and rotary angles with several axes.
#pragma once

#include <cuda_bf16.h>

#include "lq8_internal.cuh"

namespace lq {

constexpr int ROPE_MAX_PAIRS = 128;  // head_dim <= 256
constexpr int ROPE_MAX_AXES = 4;

// device error codes of these kernels (lq_device_status)
constexpr int ERR_ROPE_POS = 90;    // a position outside the cos/sin tables
constexpr int ERR_KV_LEN = 91;      // a sequence's length outside its page table or max_kv
constexpr int ERR_PAGE_ID = 92;     // a page id outside the cache
constexpr int ERR_ROW_COUNT = 93;   // q_start names more rows than the call has, or a sequence more than max_q

__device__ __forceinline__ void flag_error(int* flag, int code, int value) {
    if (flag && atomicCAS(flag, 0, code) == 0) flag[1] = value;
}

// Rotary angles: pair i of a head turns by the table row of its axis' position,
// cos[pos[axis[i]][row]][i].
struct RopeAxes {
    const float* cos;
    const float* sin;
    const int32_t* pos;     // [n_axes][pos_stride]; NULL: one axis, the row's own position + pos_base
    int64_t pos_stride;
    int64_t pos_base;
    int table_len, pairs;
    uint32_t same4, same8;  // bit c: pairs 4 c .. 4 c + 3 (8 c .. 8 c + 7) share an axis and load as vectors
    uint8_t axis[ROPE_MAX_PAIRS];
};

// Sequences of a call. Row r belongs to the sequence b with q_start[b] <= r < q_start[b+1]
// (q_start NULL: row b is sequence b's only one) and sits at position
// kv_len[b] - (q_start[b+1] - r) of the sequence's own pages.
struct PagedSeqs {
    const int32_t* q_start;
    const int32_t* kv_len;
    const int32_t* table;
    int64_t table_ld;
    int n_seqs, rows;
    int page_shift;         // log2 of the page size
    int n_pages;
};

// The sequence of row r by a whole warp: the number of ends q_start[1..B] that are <= r, counted
// over 32 samples at a time (two dependent loads up to 1024 sequences). B when r is past the
// last sequence's rows.
__device__ __forceinline__ int seq_of_row(const int32_t* __restrict__ q_start, int B, int r, int lane) {
    int lo = 0, n = B;  // the answer is in [lo, lo + n]
    while (n > 0) {
        const int step = (n + 31) >> 5;
        const int i = lo + min(n, (lane + 1) * step);  // samples at lo + step, lo + 2 step, ..., lo + n
        const bool le = q_start[i] <= r;
        const int c = __popc(__ballot_sync(0xffffffffu, le));
        if (c == 32) return lo + n;
        // the first c samples are <= r: the answer lies in [lo + c step, lo + (c + 1) step - 1]
        const int base = min(n, c * step);
        n = min(step - 1, n - base);
        lo += base;
    }
    return lo;
}

__device__ __forceinline__ uint32_t pack_bf16x2(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// host: whether a device pointer (or NULL) is aligned to elements of n bytes
inline bool aligned_to(const void* p, size_t n) { return (uintptr_t)p % n == 0; }
// host: the rotary tables of a call; axis_host NULL puts every pair on axis 0
int make_rope_axes(lq_ctx* ctx, const char* who, RopeAxes* r, int64_t rot_dim, int64_t head_dim, const float* cos_dev,
                   const float* sin_dev, int64_t table_len, const uint8_t* axis_host, int64_t n_axes,
                   const int32_t* pos_dev, int64_t pos_stride, int64_t rows);
// host: checks shared by the append and the attention
int make_paged_seqs(lq_ctx* ctx, const char* who, PagedSeqs* s, int64_t n_seqs, const int32_t* q_start_dev,
                    const int32_t* kv_len_dev, const int32_t* page_table_dev, int64_t table_ld, int64_t rows,
                    int64_t n_pages, int64_t page_size);

}  // namespace lq
