// logprobs.hip -- log probabilities of given tokens, entropies and the most
// likely tokens of logit rows (rdl_logprobs_dev, include/rdl_llama.h).
#include <hip/hip_runtime.h>
#include <limits.h>
#include <math.h>

#include <algorithm>

#include "../../include/rdl_llama.h"
#include "kv_pool.hpp"
#include "rdl_device.hpp"
#include "rdl_internal.hpp"

namespace rdl {
namespace {

// One pass over the logits.  A wave takes a range of a row, PER values a lane at
// a time, and holds, a lane each: the running maximum M, S = sum e^(x - M) and
// T = sum e^(x - M) (x - M), so that
//   lse = M + log S,  entropy = lse - sum p x = log S - T / S;
// and the range's largest values so far, the i-th in lane i as a 64-bit key of
// value and place.  A step without a value that passes the last of those costs a comparison; one
// that does costs two passes over the step's registers, and each wave's range has some n log(range / n) of
// them behind its first list: five alternatives take a sixth longer than one (a third, from the cache), more take a multiple.  The waves of a
// workgroup join through LDS, the workgroups of a row (rows that are few are split, down to a
// step a wave) through partial results that the last of them to arrive joins.
// Few rows: latency.  16 rows of 32000, five alternatives: 10.5 us (8.7 with one alternative); one workgroup of 16 waves a
// row took 16.3, the waves' lists then share one CU.  Many rows with one alternative: HBM bounds it: 2000 rows of
// 32003 take 52 us, 4.9 TB/s, from memory, 44 where the 256 MB cache holds a part of them; with 5, 20 and 64
// alternatives 61, 117 and 405, which those candidates and the lists' begin bound.
constexpr int NT = 256, W = NT / 64, PER = 16, STEP = 64 * PER, TOP = 64;
constexpr int WG_TARGET = 1024, MOST_PARTS = 64;
// A list begins by counting (first_list), where that is faster than one by one: 16 rows of 32000 with 5,
// 20 and 64 alternatives take 10.4, 12.8 and 71.7 us so, 10.5, 23.7 and 50.5 one by one; 2000 rows of 32003 with 5 and 20
// 57 and 116 instead of 61 and 152.
__host__ __device__ constexpr bool counted(int n) { return n > 4 && n <= 32; }
constexpr float LOG2E = 1.44269504088896340736f;
typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f4a4 __attribute__((ext_vector_type(4), aligned(4)));

struct Args {
    const float* logits;
    int64_t stride;
    int64_t m;
    int vocab, n_top;
    const int32_t* tokens;
    float *logprobs, *entropies;
    int32_t* ids;
    float* tops;
    int parts;       // workgroups a row
    float* stats;    // [m][parts][4]: M, S, T, whether a value was not finite
    uint64_t* keys;  // [m][parts][n_top]
    int* counters;   // [m], zero between launches
};

// Orders by value, then by place, the lower one larger; 0 is below them all.
__device__ __forceinline__ uint64_t key_of(float x, int at) {
    const uint32_t u = __builtin_bit_cast(uint32_t, x + 0.0f);  // one zero
    const uint32_t s = u & 0x80000000u ? ~u : u | 0x80000000u;
    return (uint64_t)s << 32 | (uint32_t)~at;
}
__device__ __forceinline__ float value_of(uint64_t key) {
    const uint32_t s = (uint32_t)(key >> 32);
    return __builtin_bit_cast(float, s & 0x80000000u ? s & 0x7FFFFFFFu : ~s);
}
__device__ __forceinline__ int place_of(uint64_t key) { return (int)~(uint32_t)key; }

__device__ __forceinline__ float wave_max(float v) {
    v = max8_f32(v);
    v = fmaxf(v, dpp_f32<DPP_ROW_MIRROR>(v));
    v = fmaxf(v, other16(v));
    return fmaxf(v, other32(v));
}
__device__ __forceinline__ float wave_sum(float v) {
    v = sum8_f32(v);
    v += dpp_f32<DPP_ROW_MIRROR>(v);
    v += other16(v);
    return v + other32(v);
}
__device__ __forceinline__ uint64_t lane_key(uint64_t v, int lane) {  // lane's, uniform
    return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(v >> 32), lane) << 32 |
           (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, lane);
}
// The value of the lane before (0 in lane 0).
__device__ __forceinline__ uint64_t lane_before(uint64_t v) {
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)v, 0x138, 0xF, 0xF, false);  // wave_shr:1
    const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(v >> 32), 0x138, 0xF, 0xF, false);
    return (uint64_t)hi << 32 | lo;
}

// Orders a wave's LDS accesses between its lanes.
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}
// How many of n keys in LDS (8-byte, from a 16-byte boundary, a 0 behind an odd number) are larger than k.
__device__ __forceinline__ int larger(const uint64_t* keys, int n, uint64_t k) {
    int c = 0;
#pragma unroll 4
    for (int i = 0; i < n; i += 2) {  // (reads of LDS in flight together)
        const u32x4 two = *reinterpret_cast<const u32x4*>(keys + i);
        c += ((uint64_t)two[1] << 32 | two[0]) > k;
        c += ((uint64_t)two[3] << 32 | two[2]) > k;
    }
    return c;
}

struct Stats {
    float M, S, T;
};
__device__ __forceinline__ float exp_of(float d) { return __builtin_amdgcn_exp2f(d * LOG2E); }
// The statistics of the wave's lanes together, in every lane.
__device__ __forceinline__ Stats join(Stats a) {
    const float M = wave_max(a.M);
    // (a lane that has seen nothing: S and T are 0)
    const float d = a.M == -__builtin_inff() ? 0.0f : fmaxf(a.M - M, -200.0f), c = exp_of(d);
    return {M, wave_sum(a.S * c), wave_sum((a.T + d * a.S) * c)};
}

// The lane's part of a running list of the wave's largest keys, sorted over the lanes.
__device__ __forceinline__ uint64_t insert(uint64_t list, uint64_t key) {
    const int lane = threadIdx.x & 63;
    const int at = (int)__builtin_popcountll(__builtin_amdgcn_ballot_w64(list > key));
    const uint64_t up = lane_before(list);
    return lane < at ? list : lane == at ? key : up;
}

// 4 values of a row from place i; past `hi` NaN, which no maximum or sum takes.
__device__ __forceinline__ f4 load4(const float* row, int i, int hi) {
    if (i + 4 <= hi) return *reinterpret_cast<const f4a4*>(row + i);
    f4 x;
#pragma unroll
    for (int t = 0; t < 4; t++) x[t] = i + t < hi ? row[i + t] : __builtin_nanf("");
    return x;
}

// The n largest keys of the wave's step x, the i-th in lane i, by counting: the n-th
// largest of the lanes' own largest keys is a bound that n lanes' values at most reach, whose places in
// the order are then counted.  room: room_of(n) keys of LDS.
__device__ __forceinline__ uint64_t first_list(const f4 (&x)[PER / 4], float top, int i0, int n, uint64_t* room) {
    const int lane = threadIdx.x & 63;
    int at = INT_MAX;
#pragma unroll
    for (int j = PER / 4 - 1; j >= 0; j--)
#pragma unroll
        for (int t = 3; t >= 0; t--)
            if (x[j][t] == top) at = i0 + (j * 64 + lane) * 4 + t;
    const uint64_t own = at == INT_MAX ? 0 : key_of(top, at);
    room[lane] = own;
    wave_sync();
    const int before = larger(room, 64, own);
    const uint64_t nth = __builtin_amdgcn_ballot_w64(own != 0 && before == n - 1);
    uint64_t bound = 1;
    if (nth) {
        bound = lane_key(own, (int)__builtin_ctzll(nth));
    }
    wave_sync();
    int count = 0;
#pragma unroll
    for (int j = 0; j < PER / 4; j++)
#pragma unroll
        for (int t = 0; t < 4; t++) {
            const uint64_t k = x[j][t] == x[j][t] ? key_of(x[j][t], i0 + (j * 64 + lane) * 4 + t) : 0;
            const uint64_t m = __builtin_amdgcn_ballot_w64(k >= bound);
            if (k >= bound) room[count + (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0))] = k;
            count += (int)__builtin_popcountll(m);
        }
    if (lane == 0) room[count] = 0;
    wave_sync();
    // into order: the lanes' keys, 64 at a time, to their places (room for n behind the others)
    uint64_t* sorted = room + n * PER + 2;
    if (lane < n) sorted[lane] = 0;
    wave_sync();
    for (int i = lane; i < count; i += 64) {
        const uint64_t k = room[i];
        const int place = larger(room, count, k);
        if (place < n) sorted[place] = k;
    }
    wave_sync();
    return lane < n ? sorted[lane] : 0;
}
__host__ __device__ constexpr int room_of(int n) { return counted(n) ? n * PER + 2 + ((n + 1) & ~1) : 0; }
// `count` lists of n keys each in LDS, largest first, to one, by counting, four at a
// time, between src and dst; both have a key's room behind their lists.
__device__ __forceinline__ const uint64_t* merge_lists(uint64_t* src, uint64_t* dst, int count, int n) {
    const int tid = threadIdx.x;
    while (count > 1) {
        const int groups = (count + 3) / 4;
        for (int i = tid; i <= groups * n; i += NT) dst[i] = 0;
        if (tid == 0) src[count * n] = 0;
        __syncthreads();
        for (int i = tid; i < count * n; i += NT) {
            const uint64_t k = src[i];
            const int g = i / (4 * n), lists = min(4, count - 4 * g);
            const int place = k ? larger(src + g * 4 * n, lists * n, k) : n;
            if (place < n) dst[g * n + place] = k;
        }
        __syncthreads();
        uint64_t* t = src;
        src = dst, dst = t;
        count = groups;
    }
    return src;
}

template <bool TOPS>
__global__ __launch_bounds__(NT, 4) void logprobs_kernel(Args a) {
    __shared__ float wave_stats[W][4];
    // the waves' rooms for their first lists, the lists of the waves or parts, and those merged
    extern __shared__ __attribute__((aligned(16))) uint64_t smem[];
    uint64_t *lists = smem + W * room_of(a.n_top), *merged = lists + ((max(W, a.parts) * a.n_top + 2) & ~1);
    __shared__ int flag;
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int64_t r = blockIdx.x / a.parts;
    const int part = (int)(blockIdx.x % a.parts);
    const float* row = a.logits + r * a.stride;
    // the given token's logit, on its way with the others
    const int32_t token = a.logprobs ? a.tokens[r] : -1;
    const float given = (uint32_t)token < (uint32_t)a.vocab ? row[token] : __builtin_nanf("");
    // this wave's range: whole steps, the last waves' fewer
    const int steps = (a.vocab + STEP - 1) / STEP, waves = a.parts * W, share = (steps + waves - 1) / waves;
    const int lo = (int)min((int64_t)a.vocab, (int64_t)(part * W + w) * share * STEP);
    const int hi = (int)min((int64_t)a.vocab, (int64_t)lo + (int64_t)share * STEP);
    Stats s{-__builtin_inff(), 0.0f, 0.0f};
    bool bad = false;
    uint64_t list = 0, least = 0;  // least: the n_top-th
    f4 next[PER / 4];
#pragma unroll
    for (int j = 0; j < PER / 4; j++) next[j] = load4(row, lo + (j * 64 + lane) * 4, hi);
    for (int i0 = lo; i0 < hi; i0 += STEP) {
        f4 x[PER / 4];
#pragma unroll
        for (int j = 0; j < PER / 4; j++) x[j] = next[j];
        if (i0 + STEP < hi)
#pragma unroll
            for (int j = 0; j < PER / 4; j++) next[j] = load4(row, i0 + STEP + (j * 64 + lane) * 4, hi);
        float top = -__builtin_inff();
        bool odd = false;
#pragma unroll
        for (int j = 0; j < PER / 4; j++)
#pragma unroll
            for (int t = 0; t < 4; t++) {
                top = fmaxf(top, x[j][t]);
                odd |= !(x[j][t] < __builtin_inff());
            }
        if (i0 + STEP <= hi) bad |= odd;
        else
#pragma unroll
            for (int j = 0; j < PER / 4; j++)
#pragma unroll
                for (int t = 0; t < 4; t++) bad |= i0 + (j * 64 + lane) * 4 + t < hi && !(x[j][t] < __builtin_inff());
        const float M = fmaxf(s.M, top);
        const float d0 = s.M == -__builtin_inff() ? 0.0f : fmaxf(s.M - M, -200.0f), c = exp_of(d0);
        s.T = (s.T + d0 * s.S) * c;
        s.S *= c;
        s.M = M;
#pragma unroll
        for (int j = 0; j < PER / 4; j++)
#pragma unroll
            for (int t = 0; t < 4; t++) {
                const float d = fmaxf(x[j][t] - M, -200.0f);  // of nothing (NaN) too
                const float e = exp_of(d);
                s.S += e;
                s.T = fmaf(e, d, s.T);
            }
        if constexpr (TOPS) {
            if (i0 == lo && counted(a.n_top)) {
                list = first_list(x, top, i0, a.n_top, smem + w * room_of(a.n_top));
                least = lane_key(list, a.n_top - 1);
                continue;
            }
            // the step's values that belong into the list, largest first; one that is as large as the list's last
            // lies behind it in the row
            while (__builtin_amdgcn_ballot_w64(least == 0 || top > value_of(least))) {
                const float V = wave_max(top);
                // the first place with it
                int at = INT_MAX;
#pragma unroll
                for (int j = PER / 4 - 1; j >= 0; j--)
#pragma unroll
                    for (int t = 3; t >= 0; t--)
                        if (x[j][t] == V) at = i0 + (j * 64 + lane) * 4 + t;
                at = (int)~wave_max_u32(~(uint32_t)at);
                if (at == INT_MAX) break;  // nothing left of the step
                list = insert(list, key_of(V, at));
                least = lane_key(list, a.n_top - 1);
                top = -__builtin_inff();
#pragma unroll
                for (int j = 0; j < PER / 4; j++)
#pragma unroll
                    for (int t = 0; t < 4; t++) {
                        if (i0 + (j * 64 + lane) * 4 + t == at) x[j][t] = __builtin_nanf("");
                        top = fmaxf(top, x[j][t]);
                    }
            }
        }
    }
    s = join(s);
    bad = __builtin_amdgcn_ballot_w64(bad) != 0;
    if (lane == 0) {
        wave_stats[w][0] = s.M;
        wave_stats[w][1] = s.S;
        wave_stats[w][2] = s.T;
        wave_stats[w][3] = bad ? 1.0f : 0.0f;
    }
    if constexpr (TOPS)
        if (lane < a.n_top) lists[w * a.n_top + lane] = list;
    __syncthreads();
    uint64_t best = 0;  // wave 0: the largest keys, the i-th in lane i
    auto merge = [&](int n) {
        if constexpr (TOPS) {
            const uint64_t* r = merge_lists(lists, merged, n, a.n_top);
            best = lane < a.n_top ? r[lane] : 0;
        }
    };
    merge(W);
    if (w == 0) {
        s = lane < W ? Stats{wave_stats[lane][0], wave_stats[lane][1], wave_stats[lane][2]} : Stats{-__builtin_inff(), 0.0f, 0.0f};
        bad = __builtin_amdgcn_ballot_w64(lane < W && wave_stats[lane & (W - 1)][3] != 0.0f) != 0;
        s = join(s);
    }
    if (a.parts > 1) {
        // the workgroup's result, agent-coherent, then its arrival
        if (w == 0) {
            uint64_t* to = reinterpret_cast<uint64_t*>(a.stats + (r * a.parts + part) * 4);
            typedef float f2 __attribute__((ext_vector_type(2)));
            if (lane < 2)
                __hip_atomic_store(to + lane, __builtin_bit_cast(uint64_t, lane ? f2{s.T, bad ? 1.0f : 0.0f} : f2{s.M, s.S}),
                                   __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            if (TOPS && lane < a.n_top)
                __hip_atomic_store(a.keys + (r * a.parts + part) * a.n_top + lane, best, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (threadIdx.x == 0) {
            const int old = __hip_atomic_fetch_add(a.counters + r, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            flag = old == a.parts - 1;
            if (old == a.parts - 1) __hip_atomic_store(a.counters + r, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        __syncthreads();
        if (!flag) return;
        if constexpr (TOPS)
            for (int i = threadIdx.x; i < a.parts * a.n_top; i += NT)
                lists[i] = __hip_atomic_load(a.keys + r * a.parts * a.n_top + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __syncthreads();
        if (w == 0) {
            s = Stats{-__builtin_inff(), 0.0f, 0.0f};
            bool b = false;
            if (lane < a.parts) {
                typedef float f2 __attribute__((ext_vector_type(2)));
                const uint64_t* from = reinterpret_cast<const uint64_t*>(a.stats + (r * a.parts + lane) * 4);
                const f2 x = __builtin_bit_cast(f2, __hip_atomic_load(from, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
                const f2 y = __builtin_bit_cast(f2, __hip_atomic_load(from + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
                s = Stats{x[0], x[1], y[0]};
                b = y[1] != 0.0f;
            }
            bad = __builtin_amdgcn_ballot_w64(b) != 0;
            s = join(s);
        }
        merge(a.parts);
    }
    if (w != 0) return;
    const bool none = bad || s.M == -__builtin_inff();
    const float log_s = logf(s.S), nan = __builtin_nanf("");
    if (lane == 0) {
        if (a.logprobs) a.logprobs[r] = none ? nan : given - s.M - log_s;
        if (a.entropies) a.entropies[r] = none ? nan : log_s - s.T / s.S;
    }
    if (TOPS && lane < a.n_top) {
        a.ids[r * a.n_top + lane] = none ? -1 : place_of(best);
        a.tops[r * a.n_top + lane] = none ? nan : value_of(best) - s.M - log_s;
    }
}

}  // namespace
}  // namespace rdl

using rdl::api_fail;
using rdl::api_ok;

extern "C" rdl_status rdl_logprobs_dev(const float* logits_dev, size_t stride, size_t m, size_t vocab,
                                       const int32_t* tokens_dev, float* logprobs_dev, float* entropies_dev,
                                       size_t n_top, int32_t* top_ids_dev, float* top_logprobs_dev, void* stream) {
    if (vocab == 0 || vocab > (size_t)1 << 28) return api_fail(RDL_ERR_UNSUPPORTED, "vocabulary of %zu: 1 .. 2^28", vocab);
    if (stride < vocab) return rdl::api_shape_fail("logits row stride", {vocab}, {stride});
    if (n_top > (size_t)rdl::TOP || n_top > vocab)
        return api_fail(RDL_ERR_UNSUPPORTED, "%zu alternatives of %zu tokens: at most %d", n_top, vocab, rdl::TOP);
    if (m > (size_t)1 << 23 || stride > (size_t)1 << 32) return api_fail(RDL_ERR_UNSUPPORTED, "%zu rows of stride %zu", m, stride);
    if (!tokens_dev != !logprobs_dev || (n_top && (!top_ids_dev || !top_logprobs_dev)))
        return api_fail(RDL_ERR_NULL_POINTER, "NULL device pointer");
    if (m == 0) return api_ok();
    if (!logits_dev) return api_fail(RDL_ERR_NULL_POINTER, "logits is NULL");
    if ((uintptr_t)logits_dev & 3) return api_fail(RDL_ERR_INVALID_DATA, "logits must be 4-byte aligned");
    rdl_status st = rdl::check_stream((hipStream_t)stream);
    if (st != RDL_OK) return st;
    rdl::Args a{logits_dev, (int64_t)stride, (int64_t)m, (int)vocab, (int)n_top, tokens_dev, logprobs_dev, entropies_dev,
                top_ids_dev, top_logprobs_dev, 1, nullptr, nullptr, nullptr};
    const size_t whole = (vocab + rdl::STEP * rdl::W - 1) / (rdl::STEP * rdl::W);  // workgroups that a step a wave makes
    a.parts = (int)std::min<size_t>({std::max<size_t>(1, rdl::WG_TARGET / m), whole, (size_t)rdl::MOST_PARTS});
    rdl::CallScratch work;
    if (a.parts > 1) {
        const size_t n = m * (size_t)a.parts;
        st = rdl::call_scratch((hipStream_t)stream, n * 16 + n * n_top * 8, m, &work);
        if (st != RDL_OK) return st;
        a.stats = reinterpret_cast<float*>(work.p);
        a.keys = reinterpret_cast<uint64_t*>(a.stats + 4 * n);
        a.counters = work.counters;
    }
    const dim3 grid((unsigned)(m * (size_t)a.parts));
    const int lists = std::max(rdl::W, a.parts);
    const size_t lds = n_top ? 8 * (size_t)(rdl::W * rdl::room_of(a.n_top) + ((lists * a.n_top + 2) & ~1) + (lists + 3) / 4 * a.n_top + 2) : 0;
    static_assert(8 * (rdl::W * rdl::room_of(32) + rdl::MOST_PARTS * 32 * 5 / 4 + 4) <= 64 * 1024 &&
                  8 * (rdl::W * rdl::room_of(rdl::TOP) + rdl::MOST_PARTS * rdl::TOP * 5 / 4 + 4) <= 64 * 1024, "LDS of a launch");
    hipLaunchKernelGGL(n_top ? rdl::logprobs_kernel<true> : rdl::logprobs_kernel<false>, grid, dim3(rdl::NT), lds, (hipStream_t)stream, a);
    const hipError_t e = hipGetLastError();
    const rdl_status done = a.parts > 1 ? rdl::call_scratch_done((hipStream_t)stream, &work) : RDL_OK;
    HIP_TRY(e);
    return done == RDL_OK ? api_ok() : done;
}
