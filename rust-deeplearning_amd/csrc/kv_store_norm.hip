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

template <typename F>
__device__ __forceinline__ double two_words(double v, F&& f) {  // another lane's value, a word at a time
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_bit_cast(uint32_t, f(as_f32((int32_t)(uint32_t)u)));
    const uint32_t hi = __builtin_bit_cast(uint32_t, f(as_f32((int32_t)(uint32_t)(u >> 32))));
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
template <int CTRL>
__device__ __forceinline__ double dpp_f64(double v) {
    return two_words(v, [](float w) { return dpp_f32<CTRL>(w); });
}
template <int G>
__device__ __forceinline__ double group_sum(double v) {
    if constexpr (G >= 2) v += dpp_f64<DPP_QUAD_XOR1>(v);
    if constexpr (G >= 4) v += dpp_f64<DPP_QUAD_XOR2>(v);
    if constexpr (G >= 8) v += dpp_f64<DPP_ROW_HALF_MIRROR>(v);
    if constexpr (G >= 16) v += dpp_f64<DPP_ROW_MIRROR>(v);
    if constexpr (G >= 32) v += two_words(v, [](float w) { return other16(w); });
    if constexpr (G >= 64) v += two_words(v, [](float w) { return other32(w); });
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

// The value of the lane that holds the other half of the rotation's pairs.  Where the head fills its G
// lanes that is lane ^ G / 2, without a way through LDS.
template <int G>
__device__ __forceinline__ float half_away(float v, int l, int quarter) {
    if (2 * quarter == G) {
        if constexpr (G == 16) return dpp_f32<0x128>(v);  // row_ror:8
        if constexpr (G == 32) return other16(v);
        if constexpr (G == 64) return other32(v);
    }
    return __shfl(v, l < quarter ? l + quarter : l - quarter, G);
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
        const uint32_t scale = q4_scale(mag, top == as_f32((int32_t)mag));
        const float by = q4_divisor(scale), inv = __builtin_amdgcn_rcpf(by);
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

// ROWS rows at a time, whose loads are on their way together: slot and position,
// then cos and sin, are two trips to memory one behind the other, and what is in
// flight meanwhile bounds the rate, with the norm's 64-bit sums behind it.  4096 rows of 32 + 2 * 8
// heads of 128 took 45 us one at a time, 40 by two, 42 by four and 48 by eight, whose registers
// leave fewer waves.  Now 33 where the 256 MB cache still holds the rows, three quarters of the cycles VALU issue; 42 with
// other rows in turn, 4.4 TB/s of the 5.1 to 5.3 that a copy of 1 GiB reaches.
// Few rows take one each, so that they spread over the CUs.  The first rows' loads stand before the loop and the next
// ones' behind those of cos and sin: with all of a turn's in the turn the same took 49 us from cold caches, so 44, and
// with 1536 .. 4096 workgroups that take several turns 46 to 56.
template <typename KV, int G, int ROWS>
__global__ __launch_bounds__(STORE_NT) void store_norm_kernel(StoreNormArgs a) {
#pragma clang fp contract(off)
    const int hd = a.pool.head_dim, quarter = hd >> 3, n_kv = a.pool.n_kv_heads;  // quarter: lanes of half a head
    const int l = (int)threadIdx.x % G, head = (int)(blockIdx.x * (STORE_NT / G) + threadIdx.x / G);
    if (head >= a.n_heads + 2 * n_kv) return;  // whole groups
    const int dim = 4 * l;
    const bool live = dim < hd, is_q = head < a.n_heads, is_v = head >= a.n_heads + n_kv;
    const int kvh = is_v ? head - a.n_heads - n_kv : head - a.n_heads;
    const float* gamma = is_q ? a.q_gamma : is_v ? nullptr : a.k_gamma;
    const float* src = is_q ? a.q + (int64_t)head * hd : is_v ? a.v + (int64_t)kvh * hd : a.k + (int64_t)kvh * hd;
    const int64_t stride = is_q ? a.q_stride : is_v ? a.v_stride : a.k_stride;
    const f4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
    const f4 g = gamma && live ? *reinterpret_cast<const f4*>(gamma + dim) : zero;
    const int64_t capacity = (int64_t)a.pool.n_pages << a.pool.shift;
    const bool turns = a.cos_t && !is_v;
    f4 x[ROWS], c[ROWS], s[ROWS], x_next[ROWS];
    int32_t slot[ROWS], pos[ROWS], slot_next[ROWS], pos_next[ROWS];
    auto fetch = [&](int64_t r0) {
#pragma unroll
        for (int i = 0; i < ROWS; i++) {
            const int64_t r = min(r0 + i, a.m - 1);
            slot_next[i] = a.slots[r];
            pos_next[i] = a.cos_t ? a.positions[r] : 0;
            x_next[i] = live ? *reinterpret_cast<const f4*>(src + r * stride + dim) : zero;
        }
    };
    const int64_t step = (int64_t)gridDim.y * ROWS;
    fetch((int64_t)blockIdx.y * ROWS);
    for (int64_t r0 = (int64_t)blockIdx.y * ROWS; r0 < a.m; r0 += step) {
#pragma unroll
        for (int i = 0; i < ROWS; i++) x[i] = x_next[i], slot[i] = slot_next[i], pos[i] = pos_next[i];
#pragma unroll
        for (int i = 0; i < ROWS; i++) {
            // (no short circuits: from branches around the assignment the compiler lost that of an even row)
            const bool in = (r0 + i < a.m) & (slot[i] >= 0) & (slot[i] < capacity) &
                            (!a.cos_t | ((pos[i] >= 0) & (pos[i] < a.n_positions)));
            slot[i] = in ? slot[i] : -1;
            const int64_t at = (int64_t)(slot[i] < 0 ? 0 : pos[i]) * (hd >> 1) + (l < quarter ? dim : dim - (hd >> 1));
            const bool load = turns && live && slot[i] >= 0;
            c[i] = load ? *reinterpret_cast<const f4*>(a.cos_t + at) : zero;
            s[i] = load ? *reinterpret_cast<const f4*>(a.sin_t + at) : zero;
        }
        if (r0 + step < a.m) fetch(r0 + step);
#pragma unroll
        for (int i = 0; i < ROWS; i++) {
            if (slot[i] < 0) continue;  // (the same in all lanes)
            if (gamma) {
                double ss = 0.0;
#pragma unroll
                for (int e = 0; e < 4; e++) ss = __builtin_fma((double)x[i][e], (double)x[i][e], ss);
                const float inv = inverse_root(__builtin_fma(group_sum<G>(ss), a.share, (double)a.eps));
                x[i] = x[i] * inv;
                x[i] = x[i] * g;
            }
            if (turns) {
                f4 other;
#pragma unroll
                for (int e = 0; e < 4; e++) other[e] = half_away<G>(x[i][e], l, quarter);
                x[i] = l < quarter ? x[i] * c[i] - other * s[i] : other * s[i] + x[i] * c[i];
            }
            if (is_q) {
                if (live) *reinterpret_cast<f4*>(a.q_out + (r0 + i) * a.q_out_stride + (int64_t)head * hd + dim) = x[i];
            } else {
                put<KV>(a.pool, is_v ? a.pool.v : a.pool.k, slot[i] >> a.pool.shift, kvh, slot[i] & ((1 << a.pool.shift) - 1), dim, live, x[i]);
            }
        }
    }
}

constexpr int STORE_ROWS = 2;
constexpr int64_t STORE_MANY = 512;  // rows from which on a workgroup takes STORE_ROWS at a time
template <typename KV, int G>
void go(const StoreNormArgs& a, hipStream_t s) {
    const unsigned heads = (unsigned)(a.n_heads + 2 * a.pool.n_kv_heads), per = STORE_NT / G;
    const bool many = a.m >= STORE_MANY;
    const int64_t rows = many ? (a.m + STORE_ROWS - 1) / STORE_ROWS : a.m;
    const dim3 grid((heads + per - 1) / per, (unsigned)(rows < 65535 ? rows : 65535));
    if (many) hipLaunchKernelGGL((store_norm_kernel<KV, G, STORE_ROWS>), grid, dim3(STORE_NT), 0, s, a);
    else hipLaunchKernelGGL((store_norm_kernel<KV, G, 1>), grid, dim3(STORE_NT), 0, s, a);
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

hipError_t launch_store_norm(StoreNormArgs a, hipStream_t s) {
    a.share = 1.0 / a.pool.head_dim;
    if (a.pool.dtype == RDL_KV_Q4) go_hd<Q4>(a, s);
    else if (a.pool.dtype == RDL_DTYPE_F16) go_hd<_Float16>(a, s);
    else go_hd<float>(a, s);
    return hipGetLastError();
}

}  // namespace rdl
