// kv_pages.hip -- sequences forked over shared pages, and pages copied within
// and between pools (rdl_kv_fork_dev, rdl_kv_copy_pages_dev, include/rdl_attention.h).
#include <hip/hip_runtime.h>
#include <limits.h>

#include <algorithm>
#include <utility>

#include "../../include/rdl_attention.h"
#include "kv_pool.hpp"
#include "kv_q4.hpp"
#include "rdl_device.hpp"
#include "rdl_internal.hpp"

namespace rdl {
namespace {

// ---- fork -----------------------------------------------------------------------------
// A pair's place in the free list is the number of pairs before it that need a
// page, counted by the parents' lengths from before the call: the children's are
// written when all counts are done, so that a child which is another pair's parent
// spoils nothing but its own copies.  Latency is what it costs: a call of 1, 32, 64 pairs of rows of 16 entries takes
// 2.4, 2.6, 3.0 us as one workgroup, one of 65 or 300 5.2, 5.4 as a workgroup a pair with a launch behind (with
// rows of 128 entries 2.5, 2.9, 3.6 and 5.2, 5.4).  One workgroup copies long rows alone: of 1024 entries 16, 32 and 64 pairs
// take 4.2, 6.3 and 10.6 so, 5.5 the other way, so it has at most 16 rows' worth of those.
constexpr int FORK_SMALL = 64, FORK_SMALL_WAVES = 16;
constexpr size_t FORK_SMALL_ENTRIES = 16384;
constexpr int FORK_NT = 256, FORK_WG = 2048;

struct ForkArgs {
    int32_t* tables;
    int64_t table_stride;
    int32_t* kv_len;
    int n_seq, shift;
    const int32_t *parents, *children;
    int n;
    const int32_t* free_pages;
    int n_free;
    int32_t *src, *dst, *summary;
};
struct ForkPair {
    int parent, child, pages, flags;  // pages: full ones
    int length;
    bool ok, part;
};
__device__ __forceinline__ ForkPair fork_pair(const ForkArgs& a, int i) {
    ForkPair p{a.parents[i], a.children[i], 0, 0, 0, false, false};
    p.ok = (uint32_t)p.parent < (uint32_t)a.n_seq && (uint32_t)p.child < (uint32_t)a.n_seq && p.parent != p.child;
    if (!p.ok) {
        p.flags = RDL_FORK_BAD_SEQUENCE;
        return p;
    }
    const int64_t len = a.kv_len[p.parent], most = min((int64_t)INT32_MAX, a.table_stride << a.shift);
    p.length = (int)max((int64_t)0, min(len, most));
    if (p.length != len) p.flags = RDL_FORK_BAD_LENGTH;
    p.pages = p.length >> a.shift;
    p.part = (p.length & ((1 << a.shift) - 1)) != 0;
    return p;
}
// Up to 64 pairs: one workgroup, whose waves have a pair a lane and copy the rows of every
// 16th.
__global__ __launch_bounds__(FORK_SMALL_WAVES * 64) void fork_small_kernel(ForkArgs a) {
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    ForkPair p{-1, -1, 0, 0, 0, false, false};
    if (lane < a.n) p = fork_pair(a, lane);
    const uint64_t wanted = __builtin_amdgcn_ballot_w64(p.part), ok = __builtin_amdgcn_ballot_w64(p.ok);
    for (int i = w; i < a.n; i += FORK_SMALL_WAVES) {
        if (!(ok >> i & 1)) continue;
        const int pages = __builtin_amdgcn_readlane(p.pages, i);
        const int32_t* from = a.tables + __builtin_amdgcn_readlane(p.parent, i) * a.table_stride;
        int32_t* to = a.tables + __builtin_amdgcn_readlane(p.child, i) * a.table_stride;
        for (int k = lane; k < pages; k += 64) to[k] = from[k];
    }
    if (w == 0) {
        const int before = (int)__builtin_popcountll(wanted & (((uint64_t)1 << lane) - 1)), needed = (int)__builtin_popcountll(wanted);
        int fresh = -1, last = -1;
        if (p.part) {
            fresh = before < a.n_free ? a.free_pages[before] : -1;
            last = a.tables[p.parent * a.table_stride + p.pages];
            a.tables[p.child * a.table_stride + p.pages] = fresh;
        }
        if (lane < a.n) {
            a.src[lane] = fresh < 0 ? -1 : last;
            a.dst[lane] = fresh;
        }
        const bool bad = __builtin_amdgcn_ballot_w64((p.flags & RDL_FORK_BAD_SEQUENCE) != 0) != 0;
        const bool cut = __builtin_amdgcn_ballot_w64((p.flags & RDL_FORK_BAD_LENGTH) != 0) != 0;
        if (lane == 0) {
            a.summary[0] = min(needed, a.n_free);
            a.summary[1] = (bad ? RDL_FORK_BAD_SEQUENCE : 0) | (cut ? RDL_FORK_BAD_LENGTH : 0) |
                           (needed > a.n_free ? RDL_FORK_NO_PAGES : 0);
        }
    }
    __syncthreads();  // every wave has read the lengths
    if (w == 0 && p.ok) a.kv_len[p.child] = p.length;
}

// More pairs: a workgroup each, which counts the pairs before its own for itself (a length and two
// numbers a pair, in every L2); the lengths come from a launch behind.
// Sum over the workgroup (twice in a row: a barrier between).
__device__ __forceinline__ int block_sum(int v, int* red) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) v += __shfl_xor(v, d);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    int s = 0;
#pragma unroll
    for (int w = 0; w < FORK_NT / 64; w++) s += red[w];
    return s;
}

__global__ __launch_bounds__(FORK_NT) void fork_kernel(ForkArgs a) {
    __shared__ int red[FORK_NT / 64];
    const int tid = threadIdx.x;
    int before = 0, counted = 0;
    for (int i = (int)blockIdx.x; i < a.n; i += (int)gridDim.x) {
        int more = 0;
        for (int j = counted + tid; j < i; j += FORK_NT) more += fork_pair(a, j).part;
        before += block_sum(more, red);
        counted = i;
        const ForkPair p = fork_pair(a, i);
        const int fresh = p.part && before < a.n_free ? a.free_pages[before] : -1;
        int last = -1;
        if (p.ok) {
            const int32_t* from = a.tables + p.parent * a.table_stride;
            int32_t* to = a.tables + p.child * a.table_stride;
            for (int k = tid; k < p.pages; k += FORK_NT) to[k] = from[k];
            if (p.part) last = from[p.pages];
            if (tid == 0 && p.part) to[p.pages] = fresh;
        }
        if (tid == 0) {
            a.src[i] = fresh < 0 ? -1 : last;
            a.dst[i] = fresh;
        }
    }
    if (blockIdx.x != 0) return;
    int needed = 0, flags = 0;
    for (int j = tid; j < a.n; j += FORK_NT) {
        const ForkPair p = fork_pair(a, j);
        needed += p.part;
        flags |= p.flags;
    }
    needed = block_sum(needed, red);
    const int bad = block_sum((flags & RDL_FORK_BAD_SEQUENCE) != 0, red), cut = block_sum((flags & RDL_FORK_BAD_LENGTH) != 0, red);
    if (tid == 0) {
        a.summary[0] = min(needed, a.n_free);
        a.summary[1] = (bad ? RDL_FORK_BAD_SEQUENCE : 0) | (cut ? RDL_FORK_BAD_LENGTH : 0) |
                       (needed > a.n_free ? RDL_FORK_NO_PAGES : 0);
    }
}
__global__ __launch_bounds__(FORK_NT) void fork_lengths_kernel(ForkArgs a) {
    for (int i = (int)(blockIdx.x * FORK_NT + threadIdx.x); i < a.n; i += (int)(gridDim.x * FORK_NT)) {
        const ForkPair p = fork_pair(a, i);
        if (p.ok) a.kv_len[p.child] = p.length;
    }
}

// ---- copy -------------------------------------------------------------------------------
// A workgroup takes a piece of one head's page of K or V of one pool, threads
// COPY_DEEP units of 8 values each (4-bit runs of the same type: 16 bytes), whose
// loads are all on their way before the first store.  HBM bounds it: 32 copies of 4 pages in 32 layers (268 MB
// written, 34 read and then 235 again from the caches) 77 us, 480 pages of 64 positions and 8 heads of 128, f16 to 4 bits 35 us,
// back 25 (161 MB each).  A workgroup has 1024 units, the values of such a page's head; smaller ones leave threads without
// any: as many bytes in pages of 32 positions take 51 and 28 us, in pages of 16 and heads of 64 151 and 83.
constexpr int COPY_NT = 256, COPY_DEEP = 4, COPY_POOLS = 32;

struct CopySide {
    void *k[COPY_POOLS], *v[COPY_POOLS];
    int64_t page_stride, head_stride, position_stride;
    int n_pages;
};
struct CopyArgs {
    CopySide src, dst;
    const int32_t *src_pages, *dst_pages;
    int64_t n;
    int page_positions, head_dim;
    int head_blocks, head_units;  // workgroups and units a head's page
    int row_units;                // units a position
};
struct Q4 {};
typedef float f4 __attribute__((ext_vector_type(4)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));

// 8 values (or 16 bytes) on their way.
template <typename S, bool RAW>
struct Unit;
template <bool RAW>
struct Unit<float, RAW> {
    f4 x[2];
    __device__ __forceinline__ void load(const void* head, const CopyArgs& a, int pos, int col, int) {
        const float* p = reinterpret_cast<const float*>(head) + pos * a.src.position_stride + col * 8;
        x[0] = *reinterpret_cast<const f4*>(p);
        x[1] = *reinterpret_cast<const f4*>(p + 4);
    }
    __device__ __forceinline__ void get(float (&v)[8]) const {
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = x[i >> 2][i & 3];
    }
};
template <bool RAW>
struct Unit<_Float16, RAW> {
    h8 x;
    __device__ __forceinline__ void load(const void* head, const CopyArgs& a, int pos, int col, int) {
        x = *reinterpret_cast<const h8*>(reinterpret_cast<const _Float16*>(head) + pos * a.src.position_stride + col * 8);
    }
    __device__ __forceinline__ void get(float (&v)[8]) const {
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = (float)x[i];
    }
};
template <>
struct Unit<Q4, true> {
    u32x4 x;
    __device__ __forceinline__ void load(const void* head, const CopyArgs&, int, int, int u) {
        x = reinterpret_cast<const u32x4*>(head)[u];
    }
};
template <>
struct Unit<Q4, false> {
    uint32_t w, d;
    __device__ __forceinline__ void load(const void* head, const CopyArgs& a, int pos, int col, int u) {
        const uint8_t* run = reinterpret_cast<const uint8_t*>(head);
        w = reinterpret_cast<const uint32_t*>(run)[u];
        d = *reinterpret_cast<const uint16_t*>(run + q4_scale_at(a.page_positions, a.head_dim, pos, col * 8)) * 0x10001u;
    }
    __device__ __forceinline__ u32x4 halves() const { return Q4Decoder().word(w, __builtin_bit_cast(q4h2, d)); }
    __device__ __forceinline__ void get(float (&v)[8]) const {
        const h8 x = __builtin_bit_cast(h8, halves());
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = (float)x[i];
    }
};

// Every lane comes here, those without a unit (on false) too: 4 lanes are a 4-bit block.
template <typename S, typename D>
__device__ __forceinline__ void store_unit(const Unit<S, __is_same(S, D)>& u, void* head, const CopyArgs& a, int pos, int col,
                                           int at, bool on) {
    if constexpr (__is_same(S, Q4) && __is_same(D, Q4)) {
        if (on) reinterpret_cast<u32x4*>(head)[at] = u.x;
    } else if constexpr (__is_same(S, D)) {
        if (!on) return;
        D* p = reinterpret_cast<D*>(head) + pos * a.dst.position_stride + col * 8;
        if constexpr (__is_same(D, float)) {
            *reinterpret_cast<f4*>(p) = u.x[0];
            *reinterpret_cast<f4*>(p + 4) = u.x[1];
        } else {
            *reinterpret_cast<h8*>(p) = u.x;
        }
    } else if constexpr (__is_same(S, Q4) && __is_same(D, _Float16)) {
        if (on)
            *reinterpret_cast<u32x4*>(reinterpret_cast<D*>(head) + pos * a.dst.position_stride + col * 8) = u.halves();
    } else {
        float v[8];
        u.get(v);
        if constexpr (__is_same(D, Q4)) {
            uint32_t mag = 0;
            float top = -__builtin_inff();
#pragma unroll
            for (int i = 0; i < 8; i++) mag = max(mag, abs_bits(v[i])), top = fmaxf(top, v[i]);
            mag = max4_u32(mag);
            top = max4_f32(top);
            const uint32_t scale = q4_scale(mag, top == as_f32((int32_t)mag));
            const float by = q4_divisor(scale), inv = __builtin_amdgcn_rcpf(by);
            uint32_t w = 0;
#pragma unroll
            for (int i = 0; i < 8; i++) w |= q4_code<__is_same(S, _Float16)>(v[i], by, inv) << ((i >> 1) * 4 + (i & 1) * 16);
            if (!on) return;
            uint8_t* run = reinterpret_cast<uint8_t*>(head);
            reinterpret_cast<uint32_t*>(run)[at] = w;
            if ((col & 3) == 0)
                *reinterpret_cast<uint16_t*>(run + q4_scale_at(a.page_positions, a.head_dim, pos, col * 8)) = (uint16_t)scale;
        } else if (on) {
            D* p = reinterpret_cast<D*>(head) + pos * a.dst.position_stride + col * 8;
            if constexpr (__is_same(D, float)) {
                *reinterpret_cast<f4*>(p) = f4{v[0], v[1], v[2], v[3]};
                *reinterpret_cast<f4*>(p + 4) = f4{v[4], v[5], v[6], v[7]};
            } else {
                h8 h;
#pragma unroll
                for (int i = 0; i < 8; i++) h[i] = (_Float16)v[i];
                *reinterpret_cast<h8*>(p) = h;
            }
        }
    }
}

template <typename T>
__device__ __forceinline__ void* head_of(const CopySide& s, int pool, bool v, int64_t page, int kvh) {
    constexpr int E = __is_same(T, Q4) ? 1 : (int)sizeof(T);
    uint8_t* base = reinterpret_cast<uint8_t*>(v ? s.v[pool] : s.k[pool]);
    return base + (page * s.page_stride + kvh * s.head_stride) * E;
}

template <typename S, typename D>
__global__ __launch_bounds__(COPY_NT) void copy_kernel(CopyArgs a) {
    constexpr bool SAME = __is_same(S, D), RUNS = SAME && __is_same(S, Q4);
    const int kvh = (int)blockIdx.x / a.head_blocks, u0 = ((int)blockIdx.x % a.head_blocks) * COPY_NT * COPY_DEEP + (int)threadIdx.x;
    const int pool = (int)blockIdx.z >> 1;
    const bool v = blockIdx.z & 1;
    for (int64_t i = blockIdx.y; i < a.n; i += gridDim.y) {
        const int from = a.src_pages[i], to = a.dst_pages[i];
        if ((uint32_t)from >= (uint32_t)a.src.n_pages || (uint32_t)to >= (uint32_t)a.dst.n_pages) continue;
        const void* sh = head_of<S>(a.src, pool, v, from, kvh);
        void* dh = head_of<D>(a.dst, pool, v, to, kvh);
        Unit<S, SAME> u[COPY_DEEP];
        int pos[COPY_DEEP], col[COPY_DEEP];
#pragma unroll
        for (int j = 0; j < COPY_DEEP; j++) {
            const int at = u0 + j * COPY_NT, in = at < a.head_units ? at : 0;
            pos[j] = RUNS ? 0 : in / a.row_units;
            col[j] = RUNS ? 0 : in - pos[j] * a.row_units;
            u[j].load(sh, a, pos[j], col[j], in);
        }
#pragma unroll
        for (int j = 0; j < COPY_DEEP; j++) {
            const int at = u0 + j * COPY_NT;
            store_unit<S, D>(u[j], dh, a, pos[j], col[j], at, at < a.head_units);
        }
    }
}

template <typename S, typename D>
void copy_go(const CopyArgs& a, int n_kv, int pools, hipStream_t s) {
    const dim3 grid((unsigned)(n_kv * a.head_blocks), (unsigned)std::min<int64_t>(a.n, 65535), (unsigned)(2 * pools));
    hipLaunchKernelGGL((copy_kernel<S, D>), grid, dim3(COPY_NT), 0, s, a);
}
template <typename S>
void copy_to(const CopyArgs& a, int32_t dtype, int n_kv, int pools, hipStream_t s) {
    if (dtype == RDL_KV_Q4) copy_go<S, Q4>(a, n_kv, pools, s);
    else if (dtype == RDL_DTYPE_F16) copy_go<S, _Float16>(a, n_kv, pools, s);
    else copy_go<S, float>(a, n_kv, pools, s);
}

// One list of pools: checked, alike in everything but their addresses.
rdl_status check_pools(const rdl_kv_pool* p, size_t n, PoolView* first) {
    for (size_t l = 0; l < n; l++) {
        PoolView v;
        const rdl_status st = check_pool(p + l, &v);
        if (st != RDL_OK) return st;
        if (l == 0) *first = v;
        const PoolView& f = *first;
        if (v.dtype != f.dtype || v.n_pages != f.n_pages || v.shift != f.shift || v.n_kv_heads != f.n_kv_heads ||
            v.head_dim != f.head_dim || v.page_stride != f.page_stride || v.head_stride != f.head_stride ||
            v.position_stride != f.position_stride)
            return api_fail(RDL_ERR_INVALID_DATA, "pool %zu differs from pool 0 in more than its addresses", l);
    }
    return RDL_OK;
}

}  // namespace
}  // namespace rdl

using rdl::api_fail;
using rdl::api_ok;

extern "C" {

rdl_status rdl_kv_fork_dev(int32_t* tables_dev, size_t table_stride, int32_t* kv_len_dev, size_t n_seq,
                           size_t page_positions, const int32_t* parents_dev, const int32_t* children_dev, size_t n,
                           const int32_t* free_pages_dev, size_t n_free, int32_t* src_pages_dev,
                           int32_t* dst_pages_dev, int32_t* summary_dev, void* stream) {
    rdl::ForkArgs a{};
    rdl_status st = rdl::check_page_positions(page_positions, &a.shift);
    if (st != RDL_OK) return st;
    if (n_seq > (size_t)1 << 24 || n > (size_t)1 << 24 || table_stride > (size_t)1 << 30 || n_free > (size_t)INT32_MAX)
        return api_fail(RDL_ERR_UNSUPPORTED, "%zu sequences, %zu pairs, %zu table entries, %zu free pages", n_seq, n,
                        table_stride, n_free);
    if (!summary_dev || (n && (!parents_dev || !children_dev || !src_pages_dev || !dst_pages_dev)) ||
        (n_seq && (!kv_len_dev || (table_stride && !tables_dev))) || (n_free && !free_pages_dev))
        return api_fail(RDL_ERR_NULL_POINTER, "NULL device pointer");
    if ((st = rdl::check_stream((hipStream_t)stream)) != RDL_OK) return st;
    a.tables = tables_dev;
    a.table_stride = (int64_t)table_stride;
    a.kv_len = kv_len_dev;
    a.n_seq = (int)n_seq;
    a.parents = parents_dev;
    a.children = children_dev;
    a.n = (int)n;
    a.free_pages = free_pages_dev;
    a.n_free = (int)n_free;
    a.src = src_pages_dev;
    a.dst = dst_pages_dev;
    a.summary = summary_dev;
    if (n <= (size_t)rdl::FORK_SMALL && n * table_stride <= rdl::FORK_SMALL_ENTRIES) {
        hipLaunchKernelGGL(rdl::fork_small_kernel, dim3(1), dim3(rdl::FORK_SMALL_WAVES * 64), 0, (hipStream_t)stream, a);
    } else {
        const size_t lengths = (n + rdl::FORK_NT - 1) / rdl::FORK_NT;
        hipLaunchKernelGGL(rdl::fork_kernel, dim3((unsigned)std::min<size_t>(n, rdl::FORK_WG)), dim3(rdl::FORK_NT), 0,
                           (hipStream_t)stream, a);
        hipLaunchKernelGGL(rdl::fork_lengths_kernel, dim3((unsigned)std::min<size_t>(lengths, rdl::FORK_WG)), dim3(rdl::FORK_NT), 0,
                           (hipStream_t)stream, a);
    }
    HIP_TRY(hipGetLastError());
    return api_ok();
}

rdl_status rdl_kv_copy_pages_dev(const rdl_kv_pool* src, const rdl_kv_pool* dst, size_t n_pools,
                                 const int32_t* src_pages_dev, const int32_t* dst_pages_dev, size_t n, void* stream) {
    if (n_pools > 65535) return api_fail(RDL_ERR_UNSUPPORTED, "%zu pools", n_pools);
    if (n_pools && (!src || !dst)) return api_fail(RDL_ERR_NULL_POINTER, "pools are NULL");
    if (n > (size_t)INT32_MAX) return api_fail(RDL_ERR_UNSUPPORTED, "%zu pages", n);
    rdl::PoolView s, d;
    rdl_status st = rdl::check_pools(src, n_pools, &s);
    if (st != RDL_OK || (st = rdl::check_pools(dst, n_pools, &d)) != RDL_OK) return st;
    if (n == 0 || n_pools == 0) return api_ok();
    if (s.shift != d.shift || s.n_kv_heads != d.n_kv_heads || s.head_dim != d.head_dim)
        return rdl::api_shape_fail("pages (positions, KV heads, head_dim)",
                                   {(size_t)1 << s.shift, (size_t)s.n_kv_heads, (size_t)s.head_dim},
                                   {(size_t)1 << d.shift, (size_t)d.n_kv_heads, (size_t)d.head_dim});
    if (!src_pages_dev || !dst_pages_dev) return api_fail(RDL_ERR_NULL_POINTER, "NULL device pointer");
    if ((st = rdl::check_stream((hipStream_t)stream)) != RDL_OK) return st;
    rdl::CopyArgs a{};
    a.src_pages = src_pages_dev;
    a.dst_pages = dst_pages_dev;
    a.n = (int64_t)n;
    a.page_positions = 1 << s.shift;
    a.head_dim = s.head_dim;
    a.row_units = s.head_dim / 8;
    const bool runs = s.dtype == RDL_KV_Q4 && d.dtype == RDL_KV_Q4;
    a.head_units = runs ? (int)(rdl::q4_run_bytes(a.page_positions, s.head_dim) / 16) : a.page_positions * a.row_units;
    const int per = rdl::COPY_NT * rdl::COPY_DEEP;
    a.head_blocks = (a.head_units + per - 1) / per;
    for (auto [side, view] : {std::make_pair(&a.src, &s), std::make_pair(&a.dst, &d)}) {
        side->page_stride = view->page_stride;
        side->head_stride = view->head_stride;
        side->position_stride = view->position_stride;
        side->n_pages = view->n_pages;
    }
    for (size_t l0 = 0; l0 < n_pools; l0 += rdl::COPY_POOLS) {
        const int pools = (int)std::min<size_t>(n_pools - l0, rdl::COPY_POOLS);
        for (int l = 0; l < pools; l++) {
            a.src.k[l] = src[l0 + l].k_dev, a.src.v[l] = src[l0 + l].v_dev;
            a.dst.k[l] = dst[l0 + l].k_dev, a.dst.v[l] = dst[l0 + l].v_dev;
        }
        auto to = s.dtype == RDL_KV_Q4 ? rdl::copy_to<rdl::Q4> : s.dtype == RDL_DTYPE_F16 ? rdl::copy_to<_Float16> : rdl::copy_to<float>;
        to(a, d.dtype, s.n_kv_heads, pools, (hipStream_t)stream);
        HIP_TRY(hipGetLastError());
    }
    return api_ok();
}

}  // extern "C"
