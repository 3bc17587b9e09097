// kv_store_norm.hip -- RMS norms of the q and k heads of a step's rows, RoPE
// and the cache write in one pass (rdl_kv_store_norm_dev, include/rdl_attention.h),
// and rdl_kv_store_dev's rows of a 4-bit cache.
#include "kv_store_norm.hpp"

#include <hip/hip_runtime.h>

#include "kv_q4.hpp"
#include "rdl_device.hpp"
#include "rdl_internal.hpp"

namespace rdl {
namespace {

typedef float f4 __attribute__((ext_vector_type(4)));

// G lanes hold one head of one row, four neighbouring dims each: the norm is a sum
// over the lanes, a rotation's other half comes from the lane half / 4 further
// on, and 8 lanes are a 4-bit block.
constexpr int STORE_NT = 256;

struct Q4 {};

template <int CTRL>
__device__ __forceinline__ double dpp_f64(double v) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t)dpp_i32<CTRL>((int)(uint32_t)u), hi = (uint32_t)dpp_i32<CTRL>((int)(uint32_t)(u >> 32));
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
template <int G>
__device__ __forceinline__ double group_sum(double v) {
    if constexpr (G >= 2) v += dpp_f64<DPP_QUAD_XOR1>(v);
    if constexpr (G >= 4) v += dpp_f64<DPP_QUAD_XOR2>(v);
    if constexpr (G >= 8) v += dpp_f64<DPP_ROW_HALF_MIRROR>(v);
    if constexpr (G >= 16) v += dpp_f64<DPP_ROW_MIRROR>(v);
    if constexpr (G >= 32) v += __shfl_xor(v, 16);
    if constexpr (G >= 64) v += __shfl_xor(v, 32);
    return v;
}
// f32(1 / sqrt(a)): two steps of Newton's method from the 24 bits of the instruction.
__device__ __forceinline__ float inverse_root(double a) {
    double y = __builtin_amdgcn_rsq(a);
    if (!(a > 0.0 && a < __builtin_inf())) return (float)y;  // 0, infinity, NaN as they are
    y = y * (1.5 - 0.5 * a * (y * y));
    y = y * (1.5 - 0.5 * a * (y * y));
    return (float)y;
}

// A thread's four dims of a cached row.
template <typename KV>
__device__ __forceinline__ void put(const PoolView& p, void* base, int64_t page, int kvh, int pos, int dim, bool live, f4 y) {
    if constexpr (__is_same(KV, Q4)) {
        // (lanes of 8 that are a block agree on live: head_dim is a multiple of 32)
        uint32_t mag = 0;
        float top = -__builtin_inff();
#pragma unroll
        for (int i = 0; i < 4; i++) mag = max(mag, abs_bits(y[i])), top = fmaxf(top, y[i]);
        mag = max8_u32(mag);
        top = max8_f32(top);
        const uint32_t scale = q4_scale(mag, __builtin_bit_cast(uint32_t, top) == mag);
        const float d = h2f(scale), by = d == 0.0f ? __builtin_inff() : d, inv = __builtin_amdgcn_rcpf(by);
        uint32_t w = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) w |= q4_code(y[i], by, inv) << ((i >> 1) * 4 + (i & 1) * 16);
        const bool odd = (dim & 4) != 0;  // the upper four codes of a word
        w <<= odd ? 8 : 0;
        w |= (uint32_t)dpp_i32<DPP_QUAD_XOR1>((int)w);
        if (!live) return;
        uint8_t* run = reinterpret_cast<uint8_t*>(base) + page * p.page_stride + kvh * p.head_stride;
        if (!odd) *reinterpret_cast<uint32_t*>(run + (pos * p.head_dim + dim) / 2) = w;
        if ((dim & 31) == 0)
            *reinterpret_cast<uint16_t*>(run + q4_scale_at(1 << p.shift, p.head_dim, pos, dim)) = (uint16_t)scale;
    } else {
        typedef KV kv4 __attribute__((ext_vector_type(4)));
        kv4 o;
#pragma unroll
        for (int i = 0; i < 4; i++) o[i] = (KV)y[i];
        if (live) *reinterpret_cast<kv4*>(reinterpret_cast<KV*>(base) + p.at((int)page, kvh, pos) + dim) = o;
    }
}

template <typename KV, int G>
__global__ __launch_bounds__(STORE_NT) void store_norm_kernel(StoreNormArgs a) {
#pragma clang fp contract(off)
    const int hd = a.pool.head_dim, quarter = hd >> 3, n_kv = a.pool.n_kv_heads;  // quarter: lanes of half a head
    const int l = (int)threadIdx.x % G, head = (int)(blockIdx.x * (STORE_NT / G) + threadIdx.x / G);
    if (head >= a.n_heads + 2 * n_kv) return;  // whole groups
    const int dim = 4 * l;
    const bool live = dim < hd, is_q = head < a.n_heads, is_v = head >= a.n_heads + n_kv;
    const int kvh = is_v ? head - a.n_heads - n_kv : head - a.n_heads;
    const float* gamma = is_q ? a.q_gamma : is_v ? nullptr : a.k_gamma;
    const f4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
    const f4 g = gamma && live ? *reinterpret_cast<const f4*>(gamma + dim) : zero;
    const int64_t capacity = (int64_t)a.pool.n_pages << a.pool.shift;
    for (int64_t r = blockIdx.y; r < a.m; r += gridDim.y) {
        const float* src = is_q ? a.q + r * a.q_stride + (int64_t)head * hd
                         : is_v ? a.v + r * a.v_stride + (int64_t)kvh * hd
                                : a.k + r * a.k_stride + (int64_t)kvh * hd;
        f4 x = live ? *reinterpret_cast<const f4*>(src + dim) : zero;
        const int32_t slot = a.slots[r];
        if (slot < 0 || slot >= capacity) continue;
        if (a.cos_t) {
            const int32_t pos = a.positions[r];
            if (pos < 0 || pos >= a.n_positions) continue;
        }
        if (gamma) {
            double ss = 0.0;
#pragma unroll
            for (int i = 0; i < 4; i++) ss = __builtin_fma((double)x[i], (double)x[i], ss);
            const float inv = inverse_root(group_sum<G>(ss) / (double)hd + (double)a.eps);
            x = x * inv;
            x = x * g;
        }
        if (a.cos_t && !is_v) {
            const int64_t at = (int64_t)a.positions[r] * (hd >> 1) + (l < quarter ? dim : dim - (hd >> 1));
            const f4 c = live ? *reinterpret_cast<const f4*>(a.cos_t + at) : zero;
            const f4 s = live ? *reinterpret_cast<const f4*>(a.sin_t + at) : zero;
            f4 other;
#pragma unroll
            for (int i = 0; i < 4; i++) other[i] = __shfl(x[i], l < quarter ? l + quarter : l - quarter, G);
            x = l < quarter ? x * c - other * s : other * s + x * c;
        }
        if (is_q) {
            if (live) *reinterpret_cast<f4*>(a.q_out + r * a.q_out_stride + (int64_t)head * hd + dim) = x;
        } else {
            put<KV>(a.pool, is_v ? a.pool.v : a.pool.k, slot >> a.pool.shift, kvh, slot & ((1 << a.pool.shift) - 1), dim, live, x);
        }
    }
}

template <typename KV, int G>
void go(const StoreNormArgs& a, hipStream_t s) {
    const unsigned heads = (unsigned)(a.n_heads + 2 * a.pool.n_kv_heads), per = STORE_NT / G;
    const dim3 grid((heads + per - 1) / per, (unsigned)(a.m < 65535 ? a.m : 65535));
    hipLaunchKernelGGL((store_norm_kernel<KV, G>), grid, dim3(STORE_NT), 0, s, a);
}
template <typename KV>
void go_hd(const StoreNormArgs& a, hipStream_t s) {
    const int hd = a.pool.head_dim;
    if (hd <= 32) go<KV, 8>(a, s);
    else if (hd <= 64) go<KV, 16>(a, s);
    else if (hd <= 128) go<KV, 32>(a, s);
    else go<KV, 64>(a, s);
}

}  // namespace

hipError_t launch_store_norm(const StoreNormArgs& a, hipStream_t s) {
    if (a.pool.dtype == RDL_KV_Q4) go_hd<Q4>(a, s);
    else if (a.pool.dtype == RDL_DTYPE_F16) go_hd<_Float16>(a, s);
    else go_hd<float>(a, s);
    return hipGetLastError();
}

}  // namespace rdl
