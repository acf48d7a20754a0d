// lq8_paged_q8.cuh -- the paged K/V cache held in 8 bits: int8 codes [page][kv head][position][dim]
// and f32 scales [page][kv head][position / block] for K and V; a value is code * scale.
#pragma once

#include "lq8_paged.cuh"

namespace lq {

struct PagedQ8 {
    int8_t* k;
    int8_t* v;
    float* k_scale;
    float* v_scale;
    int64_t page_stride;    // codes from page to page
    int64_t scale_stride;   // scales from page to page
    int n_kv;
    int block_shift;        // log2 of the positions that share a scale
};

// host: checks shared by the operators on such a cache (page_size: checked by make_paged_seqs);
// strides 0 become the dense ones
int make_paged_q8(lq_ctx* ctx, const char* who, PagedQ8* c, int8_t* k, int8_t* v, float* k_scale, float* v_scale,
                  int64_t n_kv_heads, int64_t head_dim, int64_t page_size, int64_t page_stride, int64_t block,
                  int64_t scale_stride, bool any_rows);

}  // namespace lq
