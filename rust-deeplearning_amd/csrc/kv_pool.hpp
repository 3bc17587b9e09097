// kv_pool.hpp -- a checked rdl_kv_pool and the argument checks that the
// entry points of include/rdl_attention.h share (kv_plan.hip).
#pragma once

#include <hip/hip_runtime.h>

#include <string>

#include "../../include/rdl_attention.h"

namespace rdl {

struct PoolView {
    void *k, *v;
    int32_t dtype;  // RDL_DTYPE_F16, RDL_DTYPE_F32 or RDL_KV_Q4 (strides in bytes)
    int n_pages, shift;  // shift: log2(page_positions)
    int n_kv_heads, head_dim;
    int64_t page_stride, head_stride, position_stride;
    // element offset (4 bits: that of the codes) of position pos (any multiple of the page size may be added) on page pg
    __device__ __forceinline__ int64_t at(int pg, int kvh, int pos) const {
        return pg * page_stride + kvh * head_stride + (pos & ((1 << shift) - 1)) * position_stride;
    }
};

rdl_status check_pool(const rdl_kv_pool* p, PoolView* v);
rdl_status check_page_positions(size_t n, int* shift);
rdl_status check_head_dim(size_t hd);
// elements between two positions: 16 of them within a 32-bit offset
rdl_status check_position_stride(size_t n);
// m rows of `width` elements, `stride` apart, 16-byte aligned and not NULL
rdl_status check_rows(const char* what, const void* p, size_t stride, size_t width, size_t m, size_t elem);
// whether two sets of m >= 1 rows, pitch bytes apart and width bytes long, share a byte
bool rows_overlap(const void* a, size_t a_pitch, size_t a_width, const void* b, size_t b_pitch, size_t b_width, size_t m);
// RDL_ERR_INVALID_DATA for a stream of another device than the current one
rdl_status check_stream(hipStream_t s);

}  // namespace rdl
