// kv_plan.hip -- the cache bookkeeping of a step that serves several sequences
// (include/rdl_attention.h): page tables, positions and slots from request
// lengths, and RoPE with the write of k and v rows through the slots.
#include <hip/hip_runtime.h>
#include <limits.h>
#include <math.h>

#include <algorithm>
#include <utility>

#include "../../include/rdl_attention.h"
#include "kv_pool.hpp"
#include "kv_q4.hpp"
#include "kv_store_norm.hpp"
#include "rdl_device.hpp"
#include "rdl_internal.hpp"

namespace rdl {
namespace {

// ---- plan ---------------------------------------------------------------------------
// Two prefix sums over the sequences: rows (sum of new) and pages (sum of the
// pages each takes beyond those it has).  Every workgroup forms them for
// itself, PLAN_CHUNK sequences at a time, because a sum over a thousand
// lengths (8 KB, in every L2) takes less time than a second launch would; it
// then writes its own PLAN_ROWS rows and its own share of the new table
// entries, a thread a row or an entry, each finding its sequence by bisection
// in LDS.  Nothing passes between workgroups: the slot of a row on a new page
// comes from the free list, not from the table entry that another workgroup
// writes.  Past PLAN_WG workgroups each takes more rows, since every one of them walks
// all the sequences.  Sums stop at 2^31 - 1, which no row or free page number reaches.
// Latency bounds it (one load of the lengths, the scan, a bisection and a
// dependent load): 4.1 us for 16 sequences, 7.4 us for 1500 with 20600 rows, where
// an empty launch takes about as much as the former.
constexpr int PLAN_NT = 512, PLAN_PER = 4, PLAN_CHUNK = PLAN_NT * PLAN_PER;
constexpr int PLAN_ROWS = 1024, PLAN_WG = 2048;  // rows a workgroup, at least; workgroups, at most

struct PlanArgs {
    const int32_t *cached, *new_rows;
    int n_seq;
    const int32_t* free_pages;
    int n_free;
    int shift;  // log2(page_positions)
    int32_t* tables;
    int table_stride;
    int32_t *row_start, *kv_len;
    int m, wg_rows;  // rows; of a workgroup
    int32_t *row_seq, *positions, *slots, *summary;
};

__device__ __forceinline__ int add_cut(int a, int b) {  // of non-negative values
    return (int)min((uint32_t)a + (uint32_t)b, (uint32_t)INT32_MAX);
}
__device__ __forceinline__ int wave_scan(int v) {  // inclusive, over the 64 lanes
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(v, d);
        if (lane >= d) v = add_cut(v, o);
    }
    return v;
}
// the last of n ascending values that is <= x (the first is)
__device__ __forceinline__ int bisect(const int* v, int n, int x) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (v[mid] <= x) lo = mid;
        else hi = mid;
    }
    return lo;
}

__global__ __launch_bounds__(PLAN_NT) void plan_kernel(PlanArgs a) {
    // of the chunk's sequences: first row, first place in the free list, pages had, positions had
    __shared__ int start[PLAN_CHUNK], first[PLAN_CHUNK], have[PLAN_CHUNK], before[PLAN_CHUNK];
    __shared__ int wrows[PLAN_NT / 64], wpages[PLAN_NT / 64], wflag[PLAN_NT / 64], wlong[PLAN_NT / 64];
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    const int r_lo = min((int)blockIdx.x * a.wg_rows, a.m), r_hi = min(r_lo + a.wg_rows, a.m);  // m <= 2^30
    const int mask = (1 << a.shift) - 1;
    int rows = 0, pages = 0;  // of the chunks before this one
    int flags = 0, longest = 0;
    for (int c0 = 0; c0 < a.n_seq; c0 += PLAN_CHUNK) {
        const int live = min(PLAN_CHUNK, a.n_seq - c0);
        int c[PLAN_PER], k[PLAN_PER], h[PLAN_PER], n[PLAN_PER];
#pragma unroll
        for (int i = 0; i < PLAN_PER; i++) {
            const int s = tid * PLAN_PER + i;
            c[i] = s < live ? a.cached[c0 + s] : 0;
            k[i] = s < live ? a.new_rows[c0 + s] : 0;
        }
        int sr = 0, sp = 0;
#pragma unroll
        for (int i = 0; i < PLAN_PER; i++) {
            const int s = tid * PLAN_PER + i;
            if (c[i] < 0 || k[i] < 0) flags |= RDL_PLAN_BAD_LENGTH;
            c[i] = max(c[i], 0), k[i] = max(k[i], 0);
            const int t = add_cut(c[i], k[i]);
            if (t - c[i] != k[i]) flags |= RDL_PLAN_BAD_LENGTH;
            k[i] = t - c[i];
            // ceil(x / page) of x < 2^31
            const int hp = (c[i] >> a.shift) + ((c[i] & mask) != 0), tp = (t >> a.shift) + ((t & mask) != 0);
            if (tp > a.table_stride) flags |= RDL_PLAN_TABLE_FULL;
            h[i] = min(hp, a.table_stride);
            n[i] = min(tp, a.table_stride) - h[i];
            longest = max(longest, t);
            if (blockIdx.x == 0 && s < live) a.kv_len[c0 + s] = t;
            sr = add_cut(sr, k[i]), sp = add_cut(sp, n[i]);
        }
        const int ir = wave_scan(sr), ip = wave_scan(sp);
        __syncthreads();  // the previous chunk's LDS reads are done
        if (lane == 63) wrows[w] = ir, wpages[w] = ip;
        __syncthreads();
        const int rows0 = rows, pages0 = pages;
        // what lies before this thread's first sequence
        int xr = __shfl_up(ir, 1), xp = __shfl_up(ip, 1);
        if (lane == 0) xr = xp = 0;
        xr = add_cut(rows, xr), xp = add_cut(pages, xp);
#pragma unroll
        for (int i = 0; i < PLAN_NT / 64; i++) {
            if (i < w) xr = add_cut(xr, wrows[i]), xp = add_cut(xp, wpages[i]);
            rows = add_cut(rows, wrows[i]), pages = add_cut(pages, wpages[i]);
        }
#pragma unroll
        for (int i = 0; i < PLAN_PER; i++) {
            const int s = tid * PLAN_PER + i;
            start[s] = xr, first[s] = xp, have[s] = h[i], before[s] = c[i];
            if (blockIdx.x == 0 && s < live) a.row_start[c0 + s] = xr;
            xr = add_cut(xr, k[i]), xp = add_cut(xp, n[i]);
        }
        __syncthreads();
        for (int r = max(r_lo, rows0) + tid; r < min(r_hi, rows); r += PLAN_NT) {
            const int s = bisect(start, live, r);
            const int pos = before[s] + (r - start[s]), p = pos >> a.shift;
            int page = -1;
            if (p < a.table_stride) {
                if (p < have[s]) {
                    page = a.tables[(int64_t)(c0 + s) * a.table_stride + p];
                } else {
                    const int f = add_cut(first[s], p - have[s]);
                    if (f < a.n_free) page = a.free_pages[f];
                }
            }
            const int64_t slot = ((int64_t)page << a.shift) + (pos & mask);
            a.row_seq[r] = c0 + s;
            a.positions[r] = pos;
            a.slots[r] = page < 0 || slot > INT32_MAX ? -1 : (int)slot;
        }
        // entries of pages past the free list too: -1
        for (int f = add_cut(pages0, (int)blockIdx.x * PLAN_NT + tid); f < pages; f = add_cut(f, (int)gridDim.x * PLAN_NT)) {
            const int s = bisect(first, live, f);
            a.tables[(int64_t)(c0 + s) * a.table_stride + have[s] + (f - first[s])] = f < a.n_free ? a.free_pages[f] : -1;
        }
    }
    for (int r = max(r_lo, rows) + tid; r < r_hi; r += PLAN_NT) {
        a.row_seq[r] = -1;
        a.positions[r] = 0;
        a.slots[r] = -1;
    }
    if (blockIdx.x != 0) return;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        flags |= __shfl_xor(flags, d);
        longest = max(longest, __shfl_xor(longest, d));
    }
    if (lane == 0) wflag[w] = flags, wlong[w] = longest;
    __syncthreads();
    if (tid == 0) {
        for (int i = 1; i < PLAN_NT / 64; i++) flags |= wflag[i], longest = max(longest, wlong[i]);
        if (pages > a.n_free) flags |= RDL_PLAN_NO_PAGES;
        if (rows > a.m) flags |= RDL_PLAN_NO_ROWS;
        a.row_start[a.n_seq] = rows;
        a.summary[0] = rows;
        a.summary[1] = min(pages, a.n_free);
        a.summary[2] = flags;
        a.summary[3] = longest;
    }
}

// ---- store ----------------------------------------------------------------------------
// A thread takes four pairs (i .. i + 3, i + half ..) of one head of one row:
// 16-byte loads and stores throughout (8-byte ones of an f16 cache).  Reads and
// writes each value once, so HBM bounds it: 4096 rows of 32 + 2 * 8 heads of 128
// take 34.5 us, 5.4 TB/s.
struct StoreArgs {
    PoolView pool;
    int64_t m;
    const float* q;
    int64_t q_stride;
    float* q_out;
    int64_t q_out_stride;
    int n_heads;
    const float *k, *v;
    int64_t k_stride, v_stride;
    const int32_t *positions, *slots;
    const float *cos_t, *sin_t;
    int64_t n_positions;
};
typedef float f4 __attribute__((ext_vector_type(4)));

template <typename KV>
__device__ __forceinline__ void store4(KV* p, f4 v) {
    typedef KV kv4 __attribute__((ext_vector_type(4)));
    kv4 o;
#pragma unroll
    for (int i = 0; i < 4; i++) o[i] = (KV)v[i];
    *reinterpret_cast<kv4*>(p) = o;
}

constexpr int STORE_NT = 256;
template <typename KV>
__global__ __launch_bounds__(STORE_NT) void store_kernel(StoreArgs a) {
    const int hd = a.pool.head_dim, half = hd >> 1, quads = half >> 2;
    const int n_kv = a.pool.n_kv_heads;
    const int u = (int)(blockIdx.x * STORE_NT + threadIdx.x);
    const int head = u / quads, i = (u % quads) * 4;
    if (head >= a.n_heads + 2 * n_kv) return;
    const int64_t capacity = (int64_t)a.pool.n_pages << a.pool.shift;
    for (int64_t r = blockIdx.y; r < a.m; r += gridDim.y) {
        const int32_t slot = a.slots[r];
        if (slot < 0 || slot >= capacity) continue;
        f4 c = {1.0f, 1.0f, 1.0f, 1.0f}, s = {0.0f, 0.0f, 0.0f, 0.0f};
        if (a.cos_t) {
            const int32_t pos = a.positions[r];
            if (pos < 0 || pos >= a.n_positions) continue;
            c = *reinterpret_cast<const f4*>(a.cos_t + (int64_t)pos * half + i);
            s = *reinterpret_cast<const f4*>(a.sin_t + (int64_t)pos * half + i);
        }
        const bool is_q = head < a.n_heads, is_v = head >= a.n_heads + n_kv;
        const float* src = is_q ? a.q + r * a.q_stride + (int64_t)head * hd
                         : is_v ? a.v + r * a.v_stride + (int64_t)(head - a.n_heads - n_kv) * hd
                                : a.k + r * a.k_stride + (int64_t)(head - a.n_heads) * hd;
        const f4 x1 = *reinterpret_cast<const f4*>(src + i), x2 = *reinterpret_cast<const f4*>(src + half + i);
        f4 y1 = x1, y2 = x2;
        if (!is_v && a.cos_t) {
            y1 = x1 * c - x2 * s;
            y2 = x1 * s + x2 * c;
        }
        if (is_q) {
            float* o = a.q_out + r * a.q_out_stride + (int64_t)head * hd;
            *reinterpret_cast<f4*>(o + i) = y1;
            *reinterpret_cast<f4*>(o + half + i) = y2;
        } else {
            const int kvh = is_v ? head - a.n_heads - n_kv : head - a.n_heads;
            KV* o = reinterpret_cast<KV*>(is_v ? a.pool.v : a.pool.k) + a.pool.at(slot >> a.pool.shift, kvh, slot);
            store4<KV>(o + i, y1);
            store4<KV>(o + half + i, y2);
        }
    }
}

}  // namespace

rdl_status check_pool(const rdl_kv_pool* p, PoolView* v) {
    if (!p) return api_fail(RDL_ERR_NULL_POINTER, "pool is NULL");
    const bool q4 = p->dtype == RDL_KV_Q4;
    if (p->dtype != RDL_DTYPE_F16 && p->dtype != RDL_DTYPE_F32 && !q4)
        return api_fail(RDL_ERR_DTYPE_MISMATCH, "cache dtype %d: F32 (0), F16 (1) or Q4 (%d)", p->dtype, RDL_KV_Q4);
    int shift = 0;
    rdl_status st = check_page_positions(p->page_positions > 0 ? (size_t)p->page_positions : 0, &shift);
    if (st != RDL_OK) return st;
    if ((st = check_head_dim(p->head_dim > 0 ? (size_t)p->head_dim : 0)) != RDL_OK) return st;
    if (q4 && p->head_dim % Q4_BLOCK)
        return api_fail(RDL_ERR_UNSUPPORTED, "head_dim %d in 4 bits: a multiple of 32", p->head_dim);
    if (p->n_kv_heads <= 0 || p->n_kv_heads > 65535 || p->n_pages < 0)
        return api_fail(RDL_ERR_INVALID_DATA, "pool of %d pages, %d KV heads", p->n_pages, p->n_kv_heads);
    if (q4 && p->position_stride != p->head_dim / 2)
        return api_fail(RDL_ERR_SHAPE_MISMATCH, "position stride %lld: %d bytes of codes", (long long)p->position_stride,
                        p->head_dim / 2);
    const int64_t unit = q4 ? 16 : p->dtype == RDL_DTYPE_F16 ? 8 : 4;
    if (p->page_stride % unit || p->head_stride % unit || (!q4 && p->position_stride % unit) || ((uintptr_t)p->k_dev & 15) ||
        ((uintptr_t)p->v_dev & 15))
        return api_fail(RDL_ERR_INVALID_DATA, "pool strides and bases must be multiples of 16 bytes");
    if (p->position_stride > 0 && (st = check_position_stride((size_t)p->position_stride)) != RDL_OK) return st;
    // the axes from the innermost out: each must step over all that the ones inside it span
    struct Axis {
        int64_t stride, count;
    } ax[3] = {{p->page_stride, p->n_pages}, {p->head_stride, p->n_kv_heads}, {p->position_stride, q4 ? 1 : p->page_positions}};
    for (int i = 0; i < 3; i++)
        for (int j = i + 1; j < 3; j++)
            if (ax[j].stride < ax[i].stride) {
                const Axis t = ax[i];
                ax[i] = ax[j];
                ax[j] = t;
            }
    // elements the axes inside take (4 bits: bytes of a head's page, which is one run)
    int64_t span = q4 ? q4_run_bytes(p->page_positions, p->head_dim) : p->head_dim;
    for (const Axis& x : ax) {
        if (x.count <= 1) continue;
        int64_t reach = 0;
        if (x.stride < span || __builtin_mul_overflow(x.stride, x.count - 1, &reach) ||
            __builtin_add_overflow(reach, span, &span) || span > ((int64_t)1 << 60))
            return api_fail(RDL_ERR_SHAPE_MISMATCH, "pool strides (page %lld, head %lld, position %lld) overlap",
                            (long long)p->page_stride, (long long)p->head_stride, (long long)p->position_stride);
    }
    if (p->n_pages > 0 && (!p->k_dev || !p->v_dev)) return api_fail(RDL_ERR_NULL_POINTER, "NULL pool memory");
    *v = PoolView{p->k_dev, p->v_dev, p->dtype, p->n_pages, shift, p->n_kv_heads, p->head_dim,
                  p->page_stride, p->head_stride, p->position_stride};
    return RDL_OK;
}

rdl_status check_page_positions(size_t n, int* shift) {
    for (int s = 4; s <= 10; s++)
        if (n == (size_t)1 << s) {
            *shift = s;
            return RDL_OK;
        }
    return api_fail(RDL_ERR_UNSUPPORTED, "%zu positions a page: a power of two, 16 .. 1024", n);
}

rdl_status check_position_stride(size_t n) {
    if (n >= (size_t)1 << 24) return api_fail(RDL_ERR_UNSUPPORTED, "%zu elements between positions: below 2^24", n);
    return RDL_OK;
}

rdl_status check_head_dim(size_t hd) {
    if (hd < 8 || hd > 256 || hd % 8)
        return api_fail(RDL_ERR_UNSUPPORTED, "head_dim %zu: a multiple of 8, 8 .. 256", hd);
    return RDL_OK;
}

rdl_status check_rows(const char* what, const void* p, size_t stride, size_t width, size_t m, size_t elem) {
    if (stride < width) return api_shape_fail((std::string(what) + " row stride").c_str(), {width}, {stride});
    if ((stride * elem) & 15 || (uintptr_t)p & 15)
        return api_fail(RDL_ERR_INVALID_DATA, "%s rows must be 16-byte aligned (stride %zu)", what, stride);
    if (stride > ((size_t)1 << 56) || m > (size_t)INT32_MAX || (m && stride > ((size_t)1 << 58) / m))
        return api_fail(RDL_ERR_UNSUPPORTED, "%s: %zu rows of stride %zu", what, m, stride);
    if (!p) return api_fail(RDL_ERR_NULL_POINTER, "%s is NULL", what);
    return RDL_OK;
}

bool rows_overlap(const void* a, size_t a_pitch, size_t a_width, const void* b, size_t b_pitch, size_t b_width, size_t m) {
    const uintptr_t a0 = (uintptr_t)a, a1 = a0 + (m - 1) * a_pitch + a_width;
    const uintptr_t b0 = (uintptr_t)b, b1 = b0 + (m - 1) * b_pitch + b_width;
    if (a1 <= b0 || b1 <= a0) return false;
    if (a_pitch != b_pitch || m == 1) return true;
    // rows of one pitch: columns apart (q and out as two parts of the same rows)
    const size_t off = (b0 + a_pitch - a0 % a_pitch) % a_pitch;  // b's column in a's rows
    return off < a_width || off + b_width > a_pitch;
}

rdl_status check_stream(hipStream_t s) {
    if (!s) return RDL_OK;
    int cur = 0, dev = 0;
    HIP_TRY(hipGetDevice(&cur));
    HIP_TRY(hipStreamGetDevice(s, &dev));
    if (cur != dev)
        return api_fail(RDL_ERR_INVALID_DATA, "the stream is device %d's, the current device is %d", dev, cur);
    return RDL_OK;
}

// The checks of the two cache writes; fills all of `a` but the norms. (m 0: the pool alone is checked.)
static rdl_status check_store(const rdl_kv_pool* pool, size_t m, const float* q_dev, size_t q_stride, float* q_out_dev,
                              size_t q_out_stride, size_t n_heads, const float* k_dev, size_t k_stride,
                              const float* v_dev, size_t v_stride, const int32_t* positions_dev,
                              const int32_t* slots_dev, const float* cos_dev, const float* sin_dev, size_t n_positions,
                              void* stream, StoreNormArgs* out) {
    StoreNormArgs& a = *out;
    rdl_status st = check_pool(pool, &a.pool);
    if (st != RDL_OK || m == 0) return st;
    const size_t hd = (size_t)pool->head_dim, kvw = (size_t)pool->n_kv_heads * hd;
    if (n_heads > 65535) return api_fail(RDL_ERR_UNSUPPORTED, "%zu heads", n_heads);
    if (n_heads) {
        if ((st = check_rows("q", q_dev, q_stride, n_heads * hd, m, 4)) != RDL_OK) return st;
        if ((st = check_rows("q_out", q_out_dev, q_out_stride, n_heads * hd, m, 4)) != RDL_OK) return st;
        if (!(q_dev == q_out_dev && q_stride == q_out_stride) &&
            rows_overlap(q_dev, q_stride * 4, n_heads * hd * 4, q_out_dev, q_out_stride * 4, n_heads * hd * 4, m))
            return api_fail(RDL_ERR_INVALID_DATA, "q_out overlaps q (the same rows, or none of them)");
    }
    if ((st = check_rows("k", k_dev, k_stride, kvw, m, 4)) != RDL_OK) return st;
    if ((st = check_rows("v", v_dev, v_stride, kvw, m, 4)) != RDL_OK) return st;
    if (n_heads)
        for (const auto& x : {std::make_pair(k_dev, k_stride), std::make_pair(v_dev, v_stride)})
            if (rows_overlap(x.first, x.second * 4, kvw * 4, q_out_dev, q_out_stride * 4, n_heads * hd * 4, m))
                return api_fail(RDL_ERR_INVALID_DATA, "q_out overlaps k or v");
    if (!slots_dev || !cos_dev != !sin_dev || (cos_dev && !positions_dev))
        return api_fail(RDL_ERR_NULL_POINTER, "NULL device pointer");
    if (((uintptr_t)cos_dev | (uintptr_t)sin_dev) & 15)
        return api_fail(RDL_ERR_INVALID_DATA, "cos and sin must be 16-byte aligned");
    if ((st = check_stream((hipStream_t)stream)) != RDL_OK) return st;
    a.m = (int64_t)m;
    a.q = q_dev;
    a.q_stride = (int64_t)q_stride;
    a.q_out = q_out_dev;
    a.q_out_stride = (int64_t)q_out_stride;
    a.n_heads = (int)n_heads;
    a.k = k_dev;
    a.v = v_dev;
    a.k_stride = (int64_t)k_stride;
    a.v_stride = (int64_t)v_stride;
    a.positions = positions_dev;
    a.slots = slots_dev;
    a.cos_t = cos_dev;
    a.sin_t = sin_dev;
    a.n_positions = (int64_t)n_positions;
    return RDL_OK;
}

}  // namespace rdl

using rdl::api_fail;
using rdl::api_ok;

extern "C" {

rdl_status rdl_kv_plan_dev(const int32_t* cached_dev, const int32_t* new_rows_dev, size_t n_seq,
                           const int32_t* free_pages_dev, size_t n_free, size_t page_positions, int32_t* tables_dev,
                           size_t table_stride, int32_t* row_start_dev, int32_t* kv_len_dev, size_t m,
                           int32_t* row_seq_dev, int32_t* positions_dev, int32_t* slots_dev, int32_t* summary_dev,
                           void* stream) {
    rdl::PlanArgs a{};
    rdl_status st = rdl::check_page_positions(page_positions, &a.shift);
    if (st != RDL_OK) return st;
    if (n_seq > (size_t)1 << 24 || m > (size_t)1 << 30 || table_stride > (size_t)1 << 30 || n_free > (size_t)INT32_MAX)
        return api_fail(RDL_ERR_UNSUPPORTED, "%zu sequences, %zu rows, %zu table entries, %zu free pages", n_seq, m,
                        table_stride, n_free);
    if (!row_start_dev || !summary_dev || (n_seq && (!cached_dev || !new_rows_dev || !kv_len_dev)) ||
        (n_free && !free_pages_dev) || (n_seq && table_stride && !tables_dev) ||
        (m && (!row_seq_dev || !positions_dev || !slots_dev)))
        return api_fail(RDL_ERR_NULL_POINTER, "NULL device pointer");
    if ((st = rdl::check_stream((hipStream_t)stream)) != RDL_OK) return st;
    a.cached = cached_dev;
    a.new_rows = new_rows_dev;
    a.n_seq = (int)n_seq;
    a.free_pages = free_pages_dev;
    a.n_free = (int)n_free;
    a.tables = tables_dev;
    a.table_stride = (int)table_stride;
    a.row_start = row_start_dev;
    a.kv_len = kv_len_dev;
    a.m = (int)m;
    a.row_seq = row_seq_dev;
    a.positions = positions_dev;
    a.slots = slots_dev;
    a.summary = summary_dev;
    const size_t rows = std::max((size_t)rdl::PLAN_ROWS, (m + rdl::PLAN_WG - 1) / rdl::PLAN_WG);
    const size_t wg = (m + rows - 1) / rows;
    a.wg_rows = (int)rows;
    hipLaunchKernelGGL(rdl::plan_kernel, dim3((unsigned)(wg ? wg : 1)), dim3(rdl::PLAN_NT), 0, (hipStream_t)stream, a);
    HIP_TRY(hipGetLastError());
    return api_ok();
}

rdl_status rdl_kv_store_dev(const rdl_kv_pool* pool, size_t m, const float* q_dev, size_t q_stride, float* q_out_dev,
                            size_t q_out_stride, size_t n_heads, const float* k_dev, size_t k_stride,
                            const float* v_dev, size_t v_stride, const int32_t* positions_dev,
                            const int32_t* slots_dev, const float* cos_dev, const float* sin_dev, size_t n_positions,
                            void* stream) {
    rdl::StoreNormArgs n{};
    const rdl_status st = rdl::check_store(pool, m, q_dev, q_stride, q_out_dev, q_out_stride, n_heads, k_dev, k_stride,
                                           v_dev, v_stride, positions_dev, slots_dev, cos_dev, sin_dev, n_positions,
                                           stream, &n);
    if (st != RDL_OK) return st;
    if (m == 0) return api_ok();
    if (n.pool.dtype == RDL_KV_Q4) {
        HIP_TRY(rdl::launch_store_norm(n, (hipStream_t)stream));
        return api_ok();
    }
    const rdl::StoreArgs a{n.pool, n.m, n.q, n.q_stride, n.q_out, n.q_out_stride, n.n_heads, n.k, n.v, n.k_stride, n.v_stride,
                           n.positions, n.slots, n.cos_t, n.sin_t, n.n_positions};
    const size_t units = (n_heads + 2 * (size_t)pool->n_kv_heads) * ((size_t)pool->head_dim / 8);
    const dim3 grid((unsigned)((units + rdl::STORE_NT - 1) / rdl::STORE_NT), (unsigned)(m < 65535 ? m : 65535));
    if (a.pool.dtype == RDL_DTYPE_F16)
        hipLaunchKernelGGL(rdl::store_kernel<_Float16>, grid, dim3(rdl::STORE_NT), 0, (hipStream_t)stream, a);
    else
        hipLaunchKernelGGL(rdl::store_kernel<float>, grid, dim3(rdl::STORE_NT), 0, (hipStream_t)stream, a);
    HIP_TRY(hipGetLastError());
    return api_ok();
}

rdl_status rdl_kv_store_norm_dev(const rdl_kv_pool* pool, size_t m, const float* q_dev, size_t q_stride,
                                 float* q_out_dev, size_t q_out_stride, size_t n_heads, const float* k_dev,
                                 size_t k_stride, const float* v_dev, size_t v_stride, const float* q_gamma_dev,
                                 const float* k_gamma_dev, float eps, const int32_t* positions_dev,
                                 const int32_t* slots_dev, const float* cos_dev, const float* sin_dev,
                                 size_t n_positions, void* stream) {
    rdl::StoreNormArgs n{};
    if (!(eps >= 0.0f) || !isfinite(eps)) return api_fail(RDL_ERR_INVALID_DATA, "eps %g: finite, not negative", eps);
    if (((uintptr_t)q_gamma_dev | (uintptr_t)k_gamma_dev) & 15)
        return api_fail(RDL_ERR_INVALID_DATA, "q_gamma and k_gamma must be 16-byte aligned");
    const rdl_status st = rdl::check_store(pool, m, q_dev, q_stride, q_out_dev, q_out_stride, n_heads, k_dev, k_stride,
                                           v_dev, v_stride, positions_dev, slots_dev, cos_dev, sin_dev, n_positions,
                                           stream, &n);
    if (st != RDL_OK) return st;
    if (m == 0) return api_ok();
    n.q_gamma = q_gamma_dev;
    n.k_gamma = k_gamma_dev;
    n.eps = eps;
    HIP_TRY(rdl::launch_store_norm(n, (hipStream_t)stream));
    return api_ok();
}

}  // extern "C"
