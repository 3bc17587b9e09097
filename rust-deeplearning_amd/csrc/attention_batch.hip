// attention_batch.hip -- causal attention of a step's rows over a paged cache
// or over packed prompts (include/rdl_attention.h).
#include <hip/hip_runtime.h>
#include <limits.h>
#include <math.h>

#include "../../include/rdl_attention.h"
#include "kv_pool.hpp"
#include "rdl_device.hpp"
#include "rdl_internal.hpp"

namespace rdl {
namespace {

// Keys and values of a launch: pages through a table, or (table NULL) the rows
// of the step itself.
struct KvSource {
    const void *k, *v;
    int64_t k_position, v_position, head, page;  // strides in elements
    const int32_t* tables;
    int64_t table_stride;
    int n_pages, shift;
    // element offsets of key j of sequence b (its first row row0) and KV head kvh; false: not in the pool
    __device__ __forceinline__ bool at(int b, int64_t row0, int kvh, int j, int64_t* ko, int64_t* vo) const {
        if (!tables) {
            *ko = (row0 + j) * k_position + kvh * head;
            *vo = (row0 + j) * v_position + kvh * head;
            return true;
        }
        const int32_t pg = tables[b * table_stride + (j >> shift)];
        const int64_t base = pg * page + kvh * head;
        const int o = j & ((1 << shift) - 1);
        *ko = base + o * k_position;
        *vo = base + o * v_position;
        return (uint32_t)pg < (uint32_t)n_pages;
    }
};

struct BatchArgs {
    KvSource kv;
    const float* q;
    int64_t q_stride;
    float* out;
    int64_t out_stride;
    int n_heads, n_kv, hd;
    int64_t m;
    const int32_t *row_start, *kv_len;  // kv_len NULL: the sequence's rows
    int n_seq;
    float scale;
};

// The rows of sequence b: [r0, r0 + n) of the step, cut to [0, m) by the
// caller; t: its keys, cut to what the table can name.
__device__ __forceinline__ void sequence(const BatchArgs& a, int b, int64_t* r0, int64_t* n, int64_t* t) {
    *r0 = a.row_start[b];
    *n = (int64_t)a.row_start[b + 1] - *r0;
    *t = a.kv_len ? a.kv_len[b] : *n;
    if (a.kv.tables) *t = min(*t, a.kv.table_stride << a.kv.shift);
}

// One workgroup a (row, head): scores of 256 keys at a time, a running
// maximum and sum, a thread a value dim.
template <typename KV>
__global__ __launch_bounds__(256) void rows_kernel(BatchArgs a) {
    __shared__ float qs[256], ws[256], red[4];
    __shared__ int64_t vofs[256];
    const int64_t r = blockIdx.x;  // < m
    const int h = blockIdx.y, kvh = h / (a.n_heads / a.n_kv), tid = threadIdx.x;
    int64_t r0 = 0, n = 0, t = 0;
    int lo = 0;
    for (; lo < a.n_seq; lo++) {
        sequence(a, lo, &r0, &n, &t);
        if (r0 >= 0 && r >= r0 && r - r0 < n) break;
    }
    if (lo == a.n_seq) return;
    const int64_t limit = (a.kv_len ? a.kv_len[lo] : n) - n + (r - r0) + 1;
    const int64_t seen = min(t, limit);
    if (tid < a.hd) qs[tid] = a.q[r * a.q_stride + (int64_t)h * a.hd + tid];
    float M = -__builtin_inff(), L = 0.0f, o = 0.0f;
    for (int64_t j0 = 0; j0 < seen; j0 += 256) {
        __syncthreads();
        float s = -__builtin_inff();
        int64_t ko = 0, vo = -1;
        if (j0 + tid < seen && a.kv.at(lo, r0, kvh, (int)(j0 + tid), &ko, &vo)) {
            const KV* k = reinterpret_cast<const KV*>(a.kv.k) + ko;
            float acc = 0.0f;
            for (int d = 0; d < a.hd; d++) acc += qs[d] * (float)k[d];
            s = acc * a.scale;
        } else {
            vo = -1;
        }
        vofs[tid] = vo;
        float mx = s;
        for (int d = 32; d; d >>= 1) mx = fmaxf(mx, __shfl_xor(mx, d));
        if ((tid & 63) == 0) red[tid >> 6] = mx;
        __syncthreads();
        const float Mn = fmaxf(M, fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])));
        if (Mn > -__builtin_inff()) {
            const float corr = expf(M - Mn);
            L *= corr, o *= corr, M = Mn;
        }
        ws[tid] = vo >= 0 ? expf(s - M) : 0.0f;
        __syncthreads();
        if (tid < a.hd)
            for (int j = 0; j < 256; j++)
                if (vofs[j] >= 0) {
                    L += ws[j];
                    o += ws[j] * (float)(reinterpret_cast<const KV*>(a.kv.v) + vofs[j])[tid];
                }
    }
    if (tid < a.hd) a.out[r * a.out_stride + (int64_t)h * a.hd + tid] = L != 0.0f ? o / L : 0.0f;
}

rdl_status run(const BatchArgs& a, bool f16, size_t max_rows, size_t max_kv, hipStream_t s) {
    const dim3 grid((unsigned)a.m, (unsigned)a.n_heads);
    if (f16)
        hipLaunchKernelGGL(rows_kernel<_Float16>, grid, dim3(256), 0, s, a);
    else
        hipLaunchKernelGGL(rows_kernel<float>, grid, dim3(256), 0, s, a);
    HIP_TRY(hipGetLastError());
    return api_ok();
}

// The checks that both entry points share; fills the fields of `a` that they name.
rdl_status check_attention(BatchArgs* a, const float* q, size_t q_stride, size_t n_heads, size_t n_kv, size_t hd,
                           size_t m, const int32_t* row_start, size_t n_seq, float scale, float* out,
                           size_t out_stride, void* stream) {
    if (n_heads == 0 || n_heads > 65535 || n_heads % n_kv)
        return api_fail(RDL_ERR_INVALID_DATA, "%zu query heads over %zu KV heads", n_heads, n_kv);
    if (!(scale > 0.0f) || !isfinite(scale)) return api_fail(RDL_ERR_INVALID_DATA, "scale %g: positive, finite", scale);
    if (n_seq > (size_t)1 << 24) return api_fail(RDL_ERR_UNSUPPORTED, "%zu sequences", n_seq);
    if (m == 0 || n_seq == 0) return RDL_OK;
    rdl_status st = check_rows("q", q, q_stride, n_heads * hd, m, 4);
    if (st != RDL_OK) return st;
    if ((st = check_rows("out", out, out_stride, n_heads * hd, m, 4)) != RDL_OK) return st;
    if (rows_overlap(q, q_stride, n_heads * hd, out, out_stride, n_heads * hd, m))
        return api_fail(RDL_ERR_INVALID_DATA, "out overlaps q");
    if (!row_start) return api_fail(RDL_ERR_NULL_POINTER, "row_start is NULL");
    if ((st = check_stream((hipStream_t)stream)) != RDL_OK) return st;
    a->q = q;
    a->q_stride = (int64_t)q_stride;
    a->out = out;
    a->out_stride = (int64_t)out_stride;
    a->n_heads = (int)n_heads;
    a->n_kv = (int)n_kv;
    a->hd = (int)hd;
    a->m = (int64_t)m;
    a->row_start = row_start;
    a->n_seq = (int)n_seq;
    a->scale = scale;
    return RDL_OK;
}

}  // namespace
}  // namespace rdl

using rdl::api_fail;
using rdl::api_ok;

extern "C" {

rdl_status rdl_attention_paged_dev(const rdl_kv_pool* pool, const float* q_dev, size_t q_stride, size_t n_heads,
                                   size_t m, const int32_t* row_start_dev, const int32_t* kv_len_dev, size_t n_seq,
                                   const int32_t* tables_dev, size_t table_stride, float scale, float* out_dev,
                                   size_t out_stride, size_t max_rows, size_t max_kv, void* stream) {
    rdl::PoolView p;
    rdl_status st = rdl::check_pool(pool, &p);
    if (st != RDL_OK) return st;
    rdl::BatchArgs a{};
    st = rdl::check_attention(&a, q_dev, q_stride, n_heads, (size_t)p.n_kv_heads, (size_t)p.head_dim, m, row_start_dev,
                              n_seq, scale, out_dev, out_stride, stream);
    if (st != RDL_OK) return st;
    if (table_stride > (size_t)1 << 30) return api_fail(RDL_ERR_UNSUPPORTED, "%zu table entries", table_stride);
    if (m == 0 || n_seq == 0) return api_ok();
    if (!kv_len_dev || !tables_dev) return api_fail(RDL_ERR_NULL_POINTER, "NULL device pointer");
    a.kv = {p.k, p.v, p.position_stride, p.position_stride, p.head_stride, p.page_stride, tables_dev,
            (int64_t)table_stride, p.n_pages, p.shift};
    a.kv_len = kv_len_dev;
    return rdl::run(a, p.f16, max_rows, max_kv, (hipStream_t)stream);
}

rdl_status rdl_attention_packed_dev(const float* q_dev, size_t q_stride, size_t n_heads, const void* k_dev,
                                    size_t k_stride, const void* v_dev, size_t v_stride, int32_t kv_dtype,
                                    size_t n_kv_heads, size_t head_dim, size_t m, const int32_t* row_start_dev,
                                    size_t n_seq, float scale, float* out_dev, size_t out_stride, size_t max_rows,
                                    void* stream) {
    if (kv_dtype != RDL_DTYPE_F16 && kv_dtype != RDL_DTYPE_F32)
        return api_fail(RDL_ERR_DTYPE_MISMATCH, "k / v dtype %d: F32 (0) or F16 (1)", kv_dtype);
    rdl_status st = rdl::check_head_dim(head_dim);
    if (st != RDL_OK) return st;
    if (n_kv_heads == 0 || n_kv_heads > 65535) return api_fail(RDL_ERR_INVALID_DATA, "%zu KV heads", n_kv_heads);
    rdl::BatchArgs a{};
    st = rdl::check_attention(&a, q_dev, q_stride, n_heads, n_kv_heads, head_dim, m, row_start_dev, n_seq, scale,
                              out_dev, out_stride, stream);
    if (st != RDL_OK) return st;
    if (m == 0 || n_seq == 0) return api_ok();
    const size_t elem = kv_dtype == RDL_DTYPE_F16 ? 2 : 4, width = n_kv_heads * head_dim;
    if ((st = rdl::check_rows("k", k_dev, k_stride, width, m, elem)) != RDL_OK) return st;
    if ((st = rdl::check_rows("v", v_dev, v_stride, width, m, elem)) != RDL_OK) return st;
    a.kv = {k_dev, v_dev, (int64_t)k_stride, (int64_t)v_stride, (int64_t)head_dim, 0, nullptr, 0, 0, 0};
    return rdl::run(a, kv_dtype == RDL_DTYPE_F16, max_rows, max_rows, (hipStream_t)stream);
}

}  // extern "C"
