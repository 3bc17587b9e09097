// attention_batch.hip -- causal attention of a step's rows over a paged cache
// or over packed prompts (include/rdl_attention.h).
#include <hip/hip_runtime.h>
#include <limits.h>
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "../../include/rdl_attention.h"
#include "attention.hpp"
#include "kv_pool.hpp"
#include "rdl_device.hpp"
#include "rdl_internal.hpp"

namespace rdl {
namespace {

// Keys and values of a launch: pages through a table, or (table NULL) the rows
// of the step itself.  Strides in elements.
struct KvSource {
    const void *k, *v;
    int64_t k_position, v_position, head, page;
    const int32_t* tables;
    int64_t table_stride;
    int n_pages, shift;
};

struct BatchArgs {
    KvSource kv;
    const float* q;
    int64_t q_stride;
    float* out;
    int64_t out_stride;
    int n_heads, n_kv, hd, group;  // group: n_heads / n_kv
    int64_t m;
    const int32_t *row_start, *kv_len;  // kv_len NULL: the sequence's rows
    int n_seq;
    float scale;
    uint32_t group_mul, group_shift;  // p / group = (mulhi(p, group_mul) + p) >> group_shift, p < 2^31
    // The launch: tile workgroups first, then few-row ones, KV heads fastest
    // (of 8 KV heads each has an XCD and its L2 to itself).
    int tiles, tile_splits, few_splits;
    int tile_span, few_span;  // keys a split
    int tile_slots;           // not 0: the splits of all tiles that the launch has room for (tile_plan)
    int few_rows;             // sequences of at most this many (row, head of a group) pairs are few-row ones
    float* part;              // [m][n_heads][part_splits][hd]
    float* part_ml;           // [m][n_heads][part_splits][2]
    int part_splits;
    int* counters;            // [n_seq][n_kv] of few rows, zero between launches
    // Split sources: tiles of TK keys as LDS holds them, numbered as row tiles
    // are (tile of TK rows * n_kv + KV head), and their exponents and flags
    const _Float16* images;
    const int4* notes;
    const int2* exps;  // [image][TK]
};

struct Pair {  // (row, head of the group) pair p of a sequence
    int row, head;
};
__device__ __forceinline__ Pair pair_of(const BatchArgs& a, int p) {
    const int row = (int)((__umulhi((uint32_t)p, a.group_mul) + (uint32_t)p) >> a.group_shift);
    return {row, p - row * a.group};
}

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef short s4 __attribute__((ext_vector_type(4)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f16v __attribute__((ext_vector_type(16)));

constexpr float LOG2E = 1.44269504088896340736f;
// Weights are held as 2^(x - M + SHIFT), M a running maximum that moves only
// when a score passes it by SLACK: at most 2^15, so hi and lo fit f16, and
// f16's smallest step, 2^-24, lies 2^-35 below the largest weight.  (8 and 7
// instead take the same time: M seldom moves after a sequence's first tiles.)
constexpr float SHIFT = 11.0f, SLACK = 4.0f;

// a as two f16 parts of 11 bits each.  NEAREST (with f32 keys and values): both are rounded
// to nearest, hi is off by at most 2^-11 of a, and lo, by its own half step, leaves
// 2^-23.  Else both are cut toward zero and leave less than 2^-21, which with f16
// keys and values, exact as they are, is below what the f32 sums are off by; the instruction
// that rounds takes longer (1 % of a long chunk, 1 to 2 % of f32 prompts and chunks).
template <bool NEAREST>
__device__ __forceinline__ void split2(float a, float b, uint32_t* hi, uint32_t* lo) {
    auto two = [](float x, float y) {
        if constexpr (NEAREST) return h2{(_Float16)x, (_Float16)y};  // v_cvt_pk_f16_f32
        else return __builtin_bit_cast(h2, __builtin_amdgcn_cvt_pkrtz(x, y));
    };
    const h2 h = two(a, b);
    *hi = __builtin_bit_cast(uint32_t, h);
    *lo = __builtin_bit_cast(uint32_t, two(fmaf((float)h[0], -1.0f, a), fmaf((float)h[1], -1.0f, b)));
}
// scale 2^e, the factor from a product of scaled parts (below 2^39) to a power of 2, e
// the exponents of both factors together.  Not below 2^-126, where it stands for scores
// of nothing in any case: masked scores are -infinity before it.
__device__ __forceinline__ float score_factor(float scale, int e) {
    return fmaxf(__builtin_amdgcn_ldexpf(scale, e) * LOG2E, 0x1p-126f);
}
// And not above 2^FACTOR_MAX or so: past f32's range it would make NaN of a score
// of 0, which queries and keys have however large they are.  f16 keys: a
// row's products are whole steps of 2^-48, so from there on any two that differ are 2^40
// apart, before a cap as behind it.  f32 keys: what is cut off the exponent, `lift`, comes on the
// products first, as their rows' own exponents do.
constexpr int FACTOR_MAX = 88;
__device__ __forceinline__ float f16_factor(float scale, int e) {
    return fminf(score_factor(scale, e), __builtin_bit_cast(float, (uint32_t)(FACTOR_MAX + 127) << 23));
}
__device__ __forceinline__ int lift_of(float scale, int e) {
    return max(0, e + (int)(__builtin_bit_cast(uint32_t, scale) >> 23) - 127 - FACTOR_MAX);
}
__device__ __forceinline__ float weight(float s, float f, float off) { return __builtin_amdgcn_exp2f(fmaf(s, f, off)); }
__device__ __forceinline__ float other32(float v) {  // the value of lane ^ 32
    const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, v),
                                                    false, false);
    const uint32_t a = r[0], b = r[1];
    return __builtin_bit_cast(float, threadIdx.x & 32 ? a : b);
}
__device__ __forceinline__ float max32(float v) { return fmaxf(v, other32(v)); }
__device__ __forceinline__ float other16(float v) {  // the value of lane ^ 16
    const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, v),
                                                    false, false);
    const uint32_t a = r[0], b = r[1];
    return __builtin_bit_cast(float, threadIdx.x & 16 ? a : b);
}
__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v) {
    v = max8_u32(v);
    v = max(v, (uint32_t)dpp_i32<DPP_ROW_MIRROR>((int)v));
    v = max(v, __builtin_bit_cast(uint32_t, other16(__builtin_bit_cast(float, v))));
    v = max(v, __builtin_bit_cast(uint32_t, other32(__builtin_bit_cast(float, v))));
    return (uint32_t)__builtin_amdgcn_readfirstlane((int)v);
}
// Maximum over the first N lanes of each N (4 or 8), uniform.
template <int N>
__device__ __forceinline__ int lanes_max(int v) {
    v = max(v, dpp_i32<DPP_QUAD_XOR1>(v));
    v = max(v, dpp_i32<DPP_QUAD_XOR2>(v));
    if constexpr (N == 8) v = max(v, dpp_i32<DPP_ROW_HALF_MIRROR>(v));
    return __builtin_amdgcn_readfirstlane(v);
}
__device__ __forceinline__ int lanes_sum(int v) {  // over the wave, uniform
    v += dpp_i32<DPP_QUAD_XOR1>(v);
    v += dpp_i32<DPP_QUAD_XOR2>(v);
    v += dpp_i32<DPP_ROW_HALF_MIRROR>(v);
    v += dpp_i32<DPP_ROW_MIRROR>(v);
    v += __builtin_bit_cast(int, other16(__builtin_bit_cast(float, v)));
    v += __builtin_bit_cast(int, other32(__builtin_bit_cast(float, v)));
    return __builtin_amdgcn_readfirstlane(v);
}
__device__ __forceinline__ int lanes_before(int v) {  // the sum over the lanes before this one
    int t = v;
    t += __builtin_amdgcn_update_dpp(0, t, 0x111, 0xF, 0xF, false);  // row_shr:1, 2, 4, 8
    t += __builtin_amdgcn_update_dpp(0, t, 0x112, 0xF, 0xF, false);
    t += __builtin_amdgcn_update_dpp(0, t, 0x114, 0xF, 0xF, false);
    t += __builtin_amdgcn_update_dpp(0, t, 0x118, 0xF, 0xF, false);
    t += __builtin_amdgcn_update_dpp(0, t, 0x142, 0xA, 0xF, false);  // row_bcast:15 to rows 1 and 3
    t += __builtin_amdgcn_update_dpp(0, t, 0x143, 0xC, 0xF, false);  // row_bcast:31 to rows 2 and 3
    return t - v;
}
// floor(log2(v)) of a positive finite f32 given by its bits (-127 below 2^-126)
__device__ __forceinline__ int exponent(uint32_t bits) { return (int)(bits >> 23) - 127; }

// Splits 8 f32 values times 2^-e.
__device__ __forceinline__ void split8(const u32x4 (&x)[2], int e, u32x4* hi, u32x4* lo) {
#pragma unroll
    for (int p = 0; p < 2; p++)
#pragma unroll
        for (int c = 0; c < 2; c++) {
            const float a = __builtin_amdgcn_ldexpf(as_f32((int32_t)(c ? x[p].z : x[p].x)), -e);
            const float b = __builtin_amdgcn_ldexpf(as_f32((int32_t)(c ? x[p].w : x[p].y)), -e);
            uint32_t h, l;
            split2<true>(a, b, &h, &l);
            (*hi)[2 * p + c] = h;
            (*lo)[2 * p + c] = l;
        }
}
// Where a launch's keys and values come from: _Float16 and float as they
// are, Split as f32 rows that split_kernel has made f16 parts of before.
struct Split {};

// LDS rows of one key, HDP f16 values without a pad (direct loads fill them
// 16 bytes a lane in order).  The 16-byte pieces of a row stand in the order
// piece ^ k_swap (K) or ^ v_swap (V) of the row, so that 16 rows' reads of one
// piece (K) and the transposed reads of 4 rows' 64 bytes (V) fall on all 64 banks.
template <typename KV, int HD>
struct Geo {
    static constexpr bool TWO = !std::is_same<KV, _Float16>::value;  // hi, lo parts
    static constexpr int PARTS = TWO ? 2 : 1;
    static constexpr int HDP = HD == 96 ? 128 : HD;
    static constexpr int KEY = 2 * HDP * PARTS;              // f16 elements a key
    static constexpr int W = 4;                              // waves of a workgroup, 32 pairs each of a tile
    static constexpr int TK = HD == 64 ? 64 : TWO || HD == 256 ? 32 : 64;  // keys of a tile
    static constexpr int FK = TWO ? 16 : 32;                 // keys a wave takes at a time for few rows
    static constexpr size_t TILE_LDS = (size_t)2 * TK * KEY * 2, FEW_LDS = (size_t)W * FK * KEY * 2;
    static constexpr size_t LDS = TILE_LDS > FEW_LDS ? TILE_LDS : FEW_LDS;
    static_assert(LDS <= 160 * 1024 - 6144, "LDS of a CU");
    static __device__ __forceinline__ int k_swap(int row) { return HDP == 64 ? (row >> 1) & 7 : row & 15; }
    static __device__ __forceinline__ int v_swap(int row) {
        return (HDP == 64 ? (row & 2) << 1 : (row & 3) << 2) | (row & 4) >> 1;
    }
};

// What a wave's slab of keys needs beside its LDS rows.  f32 keys and values
// are held times 2^-ke and 2^-ve, except the rows of a flagged slab that are
// too small for that: each row's own exponents (x: key, y: value) stand beside
// the LDS rows.
struct Meta {
    int valid;   // the keys' page is in the pool
    int flags;
    int ke, ve;
};
constexpr int SLAB_WIDE = 1;     // values that are not finite were zeroed: wide4 brings them
constexpr int SLAB_OTHER_K = 2;  // some keys have an exponent of their own
constexpr int SLAB_OTHER_V = 4;  // some values have one

// The exponent to hold a row of largest magnitude `bits` with: the one in use,
// `ref`, where the row begins at most 2^HOLD below it or is all zero, so that
// rows seldom differ; else its own.  Held below 2^15 a row's f16 parts end at
// 2^-24, 2^-33 of its largest.  For values the 2^HOLD also come off the weights,
// which are held for the largest exponent (weigh_two).
constexpr int HOLD = 5, NO_EXPONENT = -1000;
__device__ __forceinline__ int hold(uint32_t bits, int ref) {
    const int e = exponent(bits) - 14;
    return (e <= ref && e >= ref - HOLD) || bits == 0 ? ref : e;
}
// The same for a slab or tile as a whole, whose own exponent is rounded up to
// an even one: those of one size then mostly agree from the first on.
__device__ __forceinline__ int hold_all(uint32_t bits, int ref) {
    const int e = hold(bits, ref);
    return e == ref ? ref : (e + 1) & ~1;
}
// Largest magnitude of 8 values as f32 bits (finite: of the finite ones).  As
// integers, the largest signed value is the largest positive f32 (NaN above
// infinity) and the largest unsigned one, where its sign is set, the
// negative f32 of the largest magnitude.
__device__ __forceinline__ uint32_t largest8(const u32x4 (&x)[2], bool finite) {
    int32_t pos = 0;
    uint32_t neg = 0;
#pragma unroll
    for (int p = 0; p < 2; p++)
#pragma unroll
        for (int c = 0; c < 4; c++) {
            uint32_t b = x[p][c];
            if (finite && (b & 0x7F800000u) == 0x7F800000u) b = 0;
            pos = max(pos, (int32_t)b);
            neg = max(neg, b);
        }
    return max((uint32_t)pos, neg & 0x80000000u ? neg & 0x7FFFFFFFu : 0u);
}
// Maximum over each aligned group of C = 8, 16 or 32 lanes: a row's pieces.
template <int C>
__device__ __forceinline__ uint32_t row_max(uint32_t v) {
    v = max8_u32(v);
    if constexpr (C >= 16) v = max(v, (uint32_t)dpp_i32<DPP_ROW_MIRROR>((int)v));
    if constexpr (C == 32) v = max(v, __builtin_bit_cast(uint32_t, other16(__builtin_bit_cast(float, v))));
    return v;
}
// Of N pieces a lane, C lanes a row: their largest magnitudes (as largest8).
// Those that are not finite count as zero; zero: and become zero.  Returns
// whether there were any in the wave.
template <int N>
__device__ __forceinline__ bool piece_sizes(u32x4 (&x)[N][2], uint32_t (&m)[N], bool zero) {
    uint32_t t = 0;
#pragma unroll
    for (int i = 0; i < N; i++) t = max(t, m[i] = largest8(x[i], false));
    if (!__builtin_amdgcn_ballot_w64(t >= 0x7F800000u)) return false;
#pragma unroll
    for (int i = 0; i < N; i++) {
        m[i] = largest8(x[i], true);
        if (zero)
#pragma unroll
            for (int p = 0; p < 2; p++)
#pragma unroll
                for (int c = 0; c < 4; c++)
                    if ((x[i][p][c] & 0x7F800000u) == 0x7F800000u) x[i][p][c] = 0;
    }
    return true;
}
// The rows' exponents where the wave's or tile's is E, at least the largest
// row's: e; whether any differs from E.  Two ballots a piece find that none
// does, without the rows' maxima.
template <int C, int N>
__device__ __forceinline__ bool row_exponents(const uint32_t (&m)[N], int E, int (&e)[N]) {
    const uint32_t low = (uint32_t)max(E + 14 - HOLD + 127, 0) << 23;  // what begins at most 2^HOLD below
    constexpr uint64_t STARTS = C == 8 ? 0x0101010101010101u : C == 16 ? 0x0001000100010001u : 0x0000000100000001u;
    uint64_t other = 0;
#pragma unroll
    for (int i = 0; i < N; i++) {
        uint64_t some = __builtin_amdgcn_ballot_w64(m[i] != 0), enough = __builtin_amdgcn_ballot_w64(m[i] >= low);
#pragma unroll
        for (int k = 1; k < C; k *= 2) some |= some >> k, enough |= enough >> k;  // at a row's first lane: any of it
        other |= some & ~enough & STARTS;
        e[i] = E;
    }
    if (!other) return false;
#pragma unroll
    for (int i = 0; i < N; i++) e[i] = hold(row_max<C>(m[i]), E);
    return true;
}

// One wave's slab of SK keys on its way from memory to LDS: loads into
// registers (issued a step ahead), then the f16 parts into LDS.  A slab of 16
// keys or fewer lies on one page, so each load is a buffer load from a uniform
// base; keys past the sequence and pages outside the pool read as zeros.
template <typename KV, int HD, int SK>
struct Slab {
    using G = Geo<KV, HD>;
    static constexpr bool F32 = G::TWO;
    static constexpr int E = (int)sizeof(KV);
    static constexpr int CPR = G::HDP / 8;          // 8-element pieces a key
    static constexpr int NL = SK * CPR / 64;        // pieces a lane
    static constexpr int GK = SK < 16 ? SK : 16, NG = SK / GK, LPG = NL / NG;
    static_assert(NL * 64 == SK * CPR && LPG * NG == NL, "whole pieces");
    u32x4 k[NL][G::PARTS], v[NL][G::PARTS];
    uint32_t koff[LPG], voff[LPG];
    int pg[NG];  // table entries of the next slab to load

    __device__ __forceinline__ void init(const KvSource& s, int hd) {
#pragma unroll
        for (int i = 0; i < LPG; i++) {
            const int pc = (threadIdx.x & 63) + 64 * i, key = pc / CPR, col = pc % CPR;
            const bool in = col * 8 < hd;
            koff[i] = in ? (uint32_t)(key * (int)s.k_position + col * 8) * E : RSRC_OOB;
            voff[i] = in ? (uint32_t)(key * (int)s.v_position + col * 8) * E : RSRC_OOB;
        }
    }
    // the table entries of the slab at key j (of t)
    __device__ __forceinline__ void pages(const KvSource& s, const int32_t* table, int j, int t) {
#pragma unroll
        for (int g = 0; g < NG; g++) pg[g] = s.tables && j + g * GK < t ? table[(j + g * GK) >> s.shift] : 0;
    }
    // issues the loads of the slab at key j; valid: bit g for group g's page in the pool
    __device__ __forceinline__ int load(const KvSource& s, int64_t row0, int kvh, int j, int t) {
        int valid = 0;
#pragma unroll
        for (int g = 0; g < NG; g++) {
            const int jg = j + g * GK, nv = max(0, min(GK, t - jg));
            int64_t kb, vb;
            bool ok = true;
            if (s.tables) {
                const int p = __builtin_amdgcn_readfirstlane(pg[g]);
                ok = (uint32_t)p < (uint32_t)s.n_pages;
                const int64_t at = (ok ? p : 0) * s.page + kvh * s.head;
                const int o = jg & ((1 << s.shift) - 1);
                kb = at + o * s.k_position;
                vb = at + o * s.v_position;
            } else {
                kb = (row0 + jg) * s.k_position + kvh * s.head;
                vb = (row0 + jg) * s.v_position + kvh * s.head;
            }
            valid |= (int)ok << g;
            const int rows = ok ? nv : 0;
            if (rows == 0) kb = vb = 0;
            const auto kr = make_rsrc(reinterpret_cast<const KV*>(s.k) + kb, (uint32_t)(rows * (int)s.k_position * E));
            const auto vr = make_rsrc(reinterpret_cast<const KV*>(s.v) + vb, (uint32_t)(rows * (int)s.v_position * E));
#pragma unroll
            for (int i = 0; i < LPG; i++)
#pragma unroll
                for (int p = 0; p < G::PARTS; p++) {
                    k[g * LPG + i][p] = buf_load_b128(kr, koff[i] + 16 * p);
                    v[g * LPG + i][p] = buf_load_b128(vr, voff[i] + 16 * p);
                }
        }
        return valid;
    }
    // Registers to LDS rows row0 .. of ks and vs (the lo parts `part` elements
    // further on) and, f32, the rows' exponents to exps.  check: whether values that are not finite
    // have to be found (f16; f32 finds them on the way to the exponent).
    __device__ __forceinline__ Meta store(_Float16* ks, _Float16* vs, int2* exps, int row0, int part, int valid, bool check,
                                          int kref, int vref) {
        const int lane = threadIdx.x & 63;
        Meta mt{valid, 0, 0, 0};
        [[maybe_unused]] int ek[NL], ev[NL];
        if constexpr (F32) {
            uint32_t km[NL], vm[NL], kt = 0, vt = 0;
            piece_sizes(k, km, false);
            if (piece_sizes(v, vm, true)) mt.flags |= SLAB_WIDE;
#pragma unroll
            for (int i = 0; i < NL; i++) kt = max(kt, km[i]), vt = max(vt, vm[i]);
            mt.ke = hold_all(wave_max_u32(kt), kref);
            mt.ve = hold_all(wave_max_u32(vt), vref);
            if (row_exponents<CPR>(km, mt.ke, ek)) mt.flags |= SLAB_OTHER_K;
            if (row_exponents<CPR>(vm, mt.ve, ev)) mt.flags |= SLAB_OTHER_V;
            if (mt.flags & (SLAB_OTHER_K | SLAB_OTHER_V)) {
#pragma unroll
                for (int i = 0; i < NL; i++)
                    if (lane % CPR == 0) exps[row0 + (lane + 64 * i) / CPR] = int2{ek[i], ev[i]};
            } else if (lane < SK) {
                exps[row0 + lane] = int2{mt.ke, mt.ve};
            }
        } else if (check) {
            bool found = false;
#pragma unroll
            for (int i = 0; i < NL; i++)
#pragma unroll
                for (int c = 0; c < 4; c++)
                    found |= ((((v[i][0][c] & 0x7C007C00u) + 0x04000400u) & 0x80008000u) != 0);
            if (__builtin_amdgcn_ballot_w64(found)) {
                mt.flags = SLAB_WIDE;
#pragma unroll
                for (int i = 0; i < NL; i++)
#pragma unroll
                    for (int c = 0; c < 4; c++) {
                        if ((v[i][0][c] & 0x7C00u) == 0x7C00u) v[i][0][c] &= 0xFFFF0000u;
                        if ((v[i][0][c] & 0x7C000000u) == 0x7C000000u) v[i][0][c] &= 0xFFFFu;
                    }
            }
        }
#pragma unroll
        for (int i = 0; i < NL; i++) {
            const int pc = lane + 64 * i, key = pc / CPR, col = pc % CPR;
            const int row = row0 + key;
            u32x4* kd = reinterpret_cast<u32x4*>(ks + row * G::HDP + (col ^ G::k_swap(row)) * 8);
            u32x4* vd = reinterpret_cast<u32x4*>(vs + row * G::HDP + (col ^ G::v_swap(row)) * 8);
            if constexpr (F32) {
                u32x4 kh, kl, vh, vl;
                split8(k[i], ek[i], &kh, &kl);
                split8(v[i], ev[i], &vh, &vl);
                *kd = kh;
                kd[part / 8] = kl;
                *vd = vh;
                vd[part / 8] = vl;
            } else {
                *kd = k[i][0];
                *vd = v[i][0];
            }
        }
        return mt;
    }
};

// One load of 16 bytes a lane from a buffer straight to LDS (lane l's at lds + 16
// l; an offset past the buffer writes zeros).  In asm, because the compiler
// makes every LDS read wait for all such loads that it knows of, the next
// tile's among them; they have no output register, and loads_done() stands
// before the barrier that precedes the reads.  The compiler does not look into asm for the
// 5 wait states between a v_readfirstlane, which forms the buffer's words, and a
// load that reads them either: the block brings them (check_lds_loads.py looks).
// M0 is named as written, so that the compiler sets it anew where it needs it (it warns that it
// would not keep a value there over the block; it has none).
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void load_to_lds(i32x4 rsrc, uint32_t off, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(lds), "v"(off), "s"(rsrc)
                 : "memory", "m0");
}
#pragma clang diagnostic pop
__device__ __forceinline__ void loads_done() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
__device__ __forceinline__ i32x4 uniform_rsrc(const void* base, int bytes) {
    const uint64_t b = (uint64_t)base;
    return {__builtin_amdgcn_readfirstlane((int)(uint32_t)b), __builtin_amdgcn_readfirstlane((int)(uint32_t)(b >> 32) & 0xFFFF),
            __builtin_amdgcn_readfirstlane(bytes), 0x00020000};
}
__device__ __forceinline__ uint32_t lds_address(const void* p) {
    return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)p;
}

// A wave's slab of SK f16 keys straight to its LDS rows.
template <int HD, int SK>
struct DirectSlab {
    using G = Geo<_Float16, HD>;
    static constexpr int C = G::HDP / 8, KI = 64 / C, NL = SK / KI;  // pieces a row, rows a load, loads
    static_assert(SK <= 16 && NL * KI == SK, "whole loads of one page");
    uint32_t koff[NL], voff[NL];
    int pg;
    __device__ __forceinline__ void init(const KvSource& s, int hd, int row0) {
#pragma unroll
        for (int i = 0; i < NL; i++) {
            const int key = KI * i + (threadIdx.x & 63) / C, piece = (threadIdx.x & 63) % C;
            const int kc = piece ^ G::k_swap(row0 + key), vc = piece ^ G::v_swap(row0 + key);
            koff[i] = kc * 8 < hd ? (uint32_t)(key * (int)s.k_position + kc * 8) * 2 : RSRC_OOB;
            voff[i] = vc * 8 < hd ? (uint32_t)(key * (int)s.v_position + vc * 8) * 2 : RSRC_OOB;
        }
    }
    __device__ __forceinline__ void pages(const KvSource& s, const int32_t* table, int j, int t) {
        pg = s.tables && j < t ? table[j >> s.shift] : 0;
    }
    // issues the loads of the slab at key j to LDS rows at byte addresses ks, vs; whether its page is in the pool
    __device__ __forceinline__ int load(const KvSource& s, int64_t row0, int kvh, int j, int t, uint32_t ks, uint32_t vs) {
        int64_t kb, vb;
        bool ok = true;
        if (s.tables) {
            const int p = __builtin_amdgcn_readfirstlane(pg);
            ok = (uint32_t)p < (uint32_t)s.n_pages;
            const int64_t at = (ok ? p : 0) * s.page + kvh * s.head;
            const int o = j & ((1 << s.shift) - 1);
            kb = at + o * s.k_position;
            vb = at + o * s.v_position;
        } else {
            kb = (row0 + j) * s.k_position + kvh * s.head;
            vb = (row0 + j) * s.v_position + kvh * s.head;
        }
        const int rows = ok ? max(0, min(SK, t - j)) : 0;
        if (rows == 0) kb = vb = 0;
        const i32x4 kr = uniform_rsrc(reinterpret_cast<const _Float16*>(s.k) + kb, rows * (int)s.k_position * 2);
        const i32x4 vr = uniform_rsrc(reinterpret_cast<const _Float16*>(s.v) + vb, rows * (int)s.v_position * 2);
#pragma unroll
        for (int i = 0; i < NL; i++) {
            load_to_lds(kr, koff[i], ks + 1024 * i);
            load_to_lds(vr, voff[i], vs + 1024 * i);
        }
        return ok;
    }
    // Zeroes the values of the slab's LDS rows that are not finite; whether there were any.
    static __device__ __forceinline__ int clean(_Float16* vs) {
        u32x4* v = reinterpret_cast<u32x4*>(vs) + (threadIdx.x & 63);
        bool found = false;
#pragma unroll
        for (int i = 0; i < NL; i++) {
            const u32x4 x = v[64 * i];
#pragma unroll
            for (int c = 0; c < 4; c++) found |= ((((x[c] & 0x7C007C00u) + 0x04000400u) & 0x80008000u) != 0);
        }
        if (!__builtin_amdgcn_ballot_w64(found)) return 0;
#pragma unroll
        for (int i = 0; i < NL; i++) {
            u32x4 x = v[64 * i];
#pragma unroll
            for (int c = 0; c < 4; c++) {
                if ((x[c] & 0x7C00u) == 0x7C00u) x[c] &= 0xFFFF0000u;
                if ((x[c] & 0x7C000000u) == 0x7C000000u) x[c] &= 0xFFFFu;
            }
            v[64 * i] = x;
        }
        return 1;
    }
};

// 4 keys (consecutive LDS rows from `row`) of 16 dims, transposed: lane i of
// each 16 gets dim i's 4 values.
__device__ __forceinline__ h4 read_t(const void* p) {
    typedef __attribute__((address_space(3))) s4 lds_s4;
    return __builtin_bit_cast(h4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(p)));
}

// Orders a wave's LDS accesses between its lanes.
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// Row of V of key j (NULL: its page is not in the pool).
template <typename KV>
__device__ __forceinline__ const KV* value_row(const KvSource& s, int64_t row0, const int32_t* table, int kvh, int j) {
    int64_t at;
    if (s.tables) {
        const int32_t p = table[j >> s.shift];
        if ((uint32_t)p >= (uint32_t)s.n_pages) return nullptr;
        at = p * s.page + kvh * s.head + (j & ((1 << s.shift) - 1)) * s.v_position;
    } else {
        at = (row0 + j) * s.v_position + kvh * s.head;
    }
    return reinterpret_cast<const KV*>(s.v) + at;
}

// Of 4 values those that are not finite, the others (and all without `on`) as 0.
template <typename KV>
__device__ __forceinline__ f4 wide4(const KV* v, bool on) {
    typedef KV kv4 __attribute__((ext_vector_type(4)));
    const kv4 x = *reinterpret_cast<const kv4*>(v);
    f4 y;
#pragma unroll
    for (int i = 0; i < 4; i++) y[i] = on && abs_bits((float)x[i]) >= 0x7F800000u ? (float)x[i] : 0.0f;
    return y;
}

// What is not finite is summed apart from the products, where an infinity times a weight
// of 0 (its small part, or underflown) would be NaN in one tile and not in the next:
// values of masked tiles are zeroed before the products; of the others' outputs, of which
// `all` is 0 times their sum, those that are not finite begin again from 0, but not where the
// sum of weights L is NaN itself; wide4 then brings the values.
__device__ __forceinline__ bool not_finite_of_values(float all, float L) {
    return __builtin_amdgcn_ballot_w64(all != 0.0f && L == L) != 0;
}
__device__ __forceinline__ float finite_or(float x, bool zero) {
    return zero && abs_bits(x) >= 0x7F800000u ? 0.0f : x;
}
// Partial outputs likewise, joined by y = sum(w x): an infinite x keeps its place
// whatever its weight.  y tells whether there was any; if so its element is the
// sum of those, which `partial` gives one by one.
__device__ __forceinline__ bool some_not_finite(f4 y) {
    return !(fmaf(y[0], 0.0f, fmaf(y[1], 0.0f, fmaf(y[2], 0.0f, y[3] * 0.0f))) == 0.0f);
}
template <typename Partial>
__device__ __forceinline__ f4 sum_not_finite(f4 y, int n, Partial&& partial) {
    f4 x = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int z = 0; z < n; z++) {
        const f4 u = partial(z);
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (abs_bits(u[i]) >= 0x7F800000u) x[i] += u[i];
    }
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (abs_bits(y[i]) >= 0x7F800000u) y[i] = x[i];
    return y;
}

// The rows of a sequence that a launch works on.
struct Seq {
    int64_t row0;   // its first row
    int pairs;      // (row, head of the group) pairs, rows cut to m
    int64_t first;  // last key that row 0 sees
    int t;          // keys
};
__device__ __forceinline__ Seq sequence(const BatchArgs& a, int b) {
    Seq s;
    const int64_t r0 = a.row_start[b], n = (int64_t)a.row_start[b + 1] - r0;
    int64_t t = a.kv_len ? (int64_t)a.kv_len[b] : n;
    s.row0 = r0;
    s.pairs = r0 < 0 ? 0 : (int)(max((int64_t)0, min(n, a.m - r0)) * a.group);  // m * group < 2^31
    s.first = t - n;
    // keys that the table can name, or that are rows of the step
    t = min(t, a.kv.tables ? a.kv.table_stride << a.kv.shift : a.m - r0);
    s.t = (int)max((int64_t)0, min(t, (int64_t)INT32_MAX - 4096));
    return s;
}
// Key ranges are split until the launch has about this many workgroups, as far
// as a span has keys enough.  Measured (us): 48 single rows over up to 8192
// keys with FEW_TARGET 512, 1024, 2048, 4096: 157.8, 163, 154.6, 163; 2048 rows over
// 16048 keys with TILE_TARGET 512 (two workgroups a CU) and 768: 910 and 951, as each
// split of a tile writes 65 KB that join_kernel reads; chunks and single rows in
// one step (841 rows of 16 sequences) with MIXED_TARGET 512, 384, 320: 104, 95,
// 126: the single rows run on what the tiles leave; 63 rows of 9 sequences over up
// to 1900 f32 keys with TILE_MIN_SPAN 128, 256, 512: 22.8, 25.0, 36.7.
constexpr int64_t FEW_TARGET = 2048, TILE_TARGET = 512, MIXED_TARGET = 384;
constexpr int FEW_MIN_SPAN = 128, TILE_MIN_SPAN = 128;

// Tiles are numbered so that a sequence is found from row_start alone:
// sequence b's are TILE_PAIRS pairs each and numbered from row_start[b] group
// / TILE_PAIRS + b on, which leaves at least as many numbers as it has tiles before
// those of b + 1.
constexpr int TILE_PAIRS = 128, FEW_PAIRS = 16;
template <int TILE>
__device__ __forceinline__ int tiles_of(int n) { return (int)(((uint32_t)n + TILE - 1) / TILE); }
template <int TILE>
__device__ __forceinline__ int first_tile(int64_t row0, int unit, int b) {
    return (int)((uint64_t)max((int64_t)0, row0 * unit) / TILE) + b;  // row0 * unit < 2^31: rows lie below m
}
// The sequence of number t among tiles of TILE units, `unit` units a row, or -1
// (the same in every lane): 64 samples of row_start a step narrow it down, the last
// step looks at 64 sequences.
template <int TILE>
__device__ __forceinline__ int sequence_of(const BatchArgs& a, int t, int unit) {
    const int lane = threadIdx.x & 63;
    int lo = 0, n = a.n_seq;
    while (n > 64) {
        const int step = (n + 63) / 64, b = lo + lane * step;
        const bool in = lane * step < n && first_tile<TILE>(min((int64_t)a.row_start[min(b, a.n_seq)], a.m), unit, b) <= t;
        const uint64_t mask = __builtin_amdgcn_ballot_w64(in);
        if (mask == 0) return -1;
        const int k = (63 - __builtin_clzll(mask)) * step;
        lo += k;
        n = min(step, n - k);
    }
    const int b = lo + lane;
    bool hit = false;
    if (lane < n) {
        const Seq s = sequence(a, b);
        const int rows = unit == 1 ? pair_of(a, s.pairs).row : s.pairs;  // units: rows, or pairs
        const int f = rows ? first_tile<TILE>(s.row0, unit, b) : 0;
        hit = rows && t >= f && t - f < tiles_of<TILE>(rows);
    }
    const uint64_t mask = __builtin_amdgcn_ballot_w64(hit);
    return mask ? __builtin_amdgcn_readfirstlane(lo + __builtin_ctzll(mask)) : -1;
}
// The last key that pair p sees (-1: none).
__device__ __forceinline__ int last_key(const BatchArgs& a, const Seq& s, int p) {
    const int64_t l = s.first + pair_of(a, p).row;
    return (int)max((int64_t)-1, min(l, (int64_t)s.t - 1));
}

// ---- joining split key ranges ---------------------------------------------------------
// A split's partial result: each pair's normalised outputs (part) with their
// maximum and sum (part_ml).  Tiles' are joined by join_kernel.  Few rows' are published
// as attention.hpp describes it: agent-coherent stores, each wave waits for its own, a
// barrier, then the counter; the last split to arrive joins all of them in order (so results
// do not depend on which it is) and leaves the counter at zero.  A counter belongs
// to the workgroups of one slot of the launch, not to rows: whatever
// row_start holds, they agree on how many they are.
__device__ __forceinline__ int64_t place(const BatchArgs& a, const Seq& s, int kvh, int p) {
    const Pair x = pair_of(a, p);
    return (s.row0 + x.row) * a.n_heads + kvh * a.group + x.head;
}
__device__ __forceinline__ float* out_at(const BatchArgs& a, const Seq& s, int kvh, int p) {
    const Pair x = pair_of(a, p);
    return a.out + (s.row0 + x.row) * a.out_stride + (kvh * a.group + x.head) * a.hd;
}
__device__ __forceinline__ const float* q_at(const BatchArgs& a, const Seq& s, int kvh, int p) {
    const Pair x = pair_of(a, p);
    return a.q + (s.row0 + x.row) * a.q_stride + (kvh * a.group + x.head) * a.hd;
}
typedef float f2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ void put2(float* p, float x, float y) {
    __hip_atomic_store(reinterpret_cast<uint64_t*>(p), __builtin_bit_cast(uint64_t, f2{x, y}), __ATOMIC_RELAXED,
                       __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ f2 get2(const float* p) {
    return __builtin_bit_cast(f2, __hip_atomic_load(reinterpret_cast<const uint64_t*>(p), __ATOMIC_RELAXED,
                                                    __HIP_MEMORY_SCOPE_AGENT));
}
// Pair p's partial of split z: outputs, maximum and sum.
__device__ __forceinline__ void put_ml(const BatchArgs& a, int64_t at, int z, float M, float L) {
    put2(a.part_ml + (at * a.part_splits + z) * 2, M, L);
}
// Joins up to FEW_PAIRS pairs: JOIN_LANES lanes a pair form the splits' weights
// while the first outputs are on their way, then a thread takes four dims of a
// pair at a time, by weights of at most 1 (large values stay in f32's range).  Its
// latency is what it costs.  COHERENT: the partials come from the same launch.
constexpr int JOIN_DEEP = 16, JOIN_AHEAD = 4;  // splits a lane, at most; splits whose outputs are read ahead
constexpr int JOIN_THREADS = 256, JOIN_LANES = JOIN_THREADS / FEW_PAIRS, JOIN_SPLITS = JOIN_LANES * JOIN_DEEP;
constexpr int JOIN_FLOATS = FEW_PAIRS * (JOIN_SPLITS + 1);  // of LDS
template <bool COHERENT>
__device__ __forceinline__ void join(const BatchArgs& a, const Seq& s, int kvh, int p0, int pairs, int splits, float* wt) {
    constexpr int NT = JOIN_THREADS, PAIRS = FEW_PAIRS;
    const int tid = threadIdx.x;
    auto get2 = [](const float* p) {
        if constexpr (COHERENT) return rdl::get2(p);
        else return *reinterpret_cast<const f2*>(p);
    };
    constexpr int LP = NT / PAIRS;
    const int quads = a.hd >> 2;
    auto outputs = [&](int i) {  // item i's first split
        const int pi = i / quads;
        return a.part + place(a, s, kvh, p0 + pi) * a.part_splits * a.hd + (i - pi * quads) * 4;
    };
    const int pi = tid / LP, l = tid % LP;
    const float* ml_at = a.part_ml + place(a, s, kvh, p0 + min(pi, pairs - 1)) * a.part_splits * 2;
    auto ml = [&](int z) { return get2(ml_at + z * 2); };
    const f2 own = ml(min(l, splits - 1));  // the lane's first split; more of them are read twice
    const float* o0 = outputs(min(tid, pairs * quads - 1));
    f2 ahead[JOIN_AHEAD][2];
#pragma unroll
    for (int z = 0; z < JOIN_AHEAD; z++) {
        ahead[z][0] = get2(o0 + min(z, splits - 1) * a.hd);
        ahead[z][1] = get2(o0 + min(z, splits - 1) * a.hd + 2);
    }
    auto top = [](f2 x, float M) { return x[1] != 0.0f ? fmaxf(M, x[0]) : M; };
    auto weigh = [](f2 x, float M) { return x[1] != 0.0f ? x[1] * __builtin_amdgcn_exp2f(x[0] - M) : 0.0f; };
    float M = l < splits ? top(own, -__builtin_inff()) : -__builtin_inff();
#pragma unroll 4
    for (int z = l + LP; z < splits; z += LP) M = top(ml(z), M);
#pragma unroll
    for (int d = 1; d < LP; d <<= 1) M = fmaxf(M, __shfl_xor(M, d));
    float L = l < splits ? weigh(own, M) : 0.0f;
    if (l < splits && pi < pairs) wt[pi * splits + l] = L;
#pragma unroll 4
    for (int z = l + LP; z < splits; z += LP) {
        const float x = weigh(ml(z), M);
        if (pi < pairs) wt[pi * splits + z] = x;
        L += x;
    }
#pragma unroll
    for (int d = 1; d < LP; d <<= 1) L += __shfl_xor(L, d);
    float* inv = wt + PAIRS * JOIN_SPLITS;
    if (l == 0 && pi < pairs) inv[pi] = L != 0.0f ? 1.0f / L : 0.0f;
    __syncthreads();
    for (int i = tid; i < pairs * quads; i += NT) {
        const int pr = i / quads;
        const float *o = outputs(i), *w = wt + pr * splits, unit = inv[pr];
        f4 y = {0.0f, 0.0f, 0.0f, 0.0f};
        int z0 = 0;
        if (i == tid) {
#pragma unroll
            for (int z = 0; z < JOIN_AHEAD; z++)
                if (z < splits) y += w[z] * unit * f4{ahead[z][0][0], ahead[z][0][1], ahead[z][1][0], ahead[z][1][1]};
            z0 = min(JOIN_AHEAD, splits);
        }
        auto partial = [&](int z) {
            const f2 u = get2(o + z * a.hd), v = get2(o + z * a.hd + 2);
            return f4{u[0], u[1], v[0], v[1]};
        };
#pragma unroll 4
        for (int z = z0; z < splits; z++) y += w[z] * unit * partial(z);
        if (some_not_finite(y)) y = sum_not_finite(y, splits, partial);
        *reinterpret_cast<f4*>(out_at(a, s, kvh, p0 + pr) + (i - pr * quads) * 4) = y;
    }
}

// q of one pair as f16 parts: NS steps of 8 dims, step i at dim d0 + i * step.
// Scaled by the power of two that brings the row's largest value (over all
// lanes of the pair: `reduce`) into [2^14, 2^15).  Returns the exponent.
template <int NS>
struct QRow {
    f4 x[NS][2];
    __device__ __forceinline__ void load(const float* q, bool live, int d0, int step, int hd) {
#pragma unroll
        for (int i = 0; i < NS; i++) {
            const int d = d0 + i * step;
#pragma unroll
            for (int c = 0; c < 2; c++)
                x[i][c] = live && d < hd ? *reinterpret_cast<const f4*>(q + d + 4 * c) : f4{0.0f, 0.0f, 0.0f, 0.0f};
        }
    }
};
template <bool NEAREST, int NS, typename R>
__device__ __forceinline__ int split_q(const QRow<NS>& row, h8 (&hi)[NS], h8 (&lo)[NS], R&& reduce) {
    const f4 (&x)[NS][2] = row.x;
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < NS; i++)
#pragma unroll
        for (int c = 0; c < 2; c++)
#pragma unroll
            for (int e = 0; e < 4; e++) m = max(m, abs_bits(x[i][c][e]));
    m = reduce(m);
    const int e = m >= 0x7F800000u ? 0 : exponent(m) - 14;
#pragma unroll
    for (int i = 0; i < NS; i++) {
        u32x4 h, l;
#pragma unroll
        for (int c = 0; c < 4; c++) {
            uint32_t a, b;
            split2<NEAREST>(__builtin_amdgcn_ldexpf(x[i][c >> 1][(c & 1) * 2], -e),
                            __builtin_amdgcn_ldexpf(x[i][c >> 1][(c & 1) * 2 + 1], -e), &a, &b);
            h[c] = a;
            l[c] = b;
        }
        hi[i] = __builtin_bit_cast(h8, h);
        lo[i] = __builtin_bit_cast(h8, l);
    }
    return e;
}

// 2^ref as a factor, where it is below f32's normal numbers too.
struct Power {
    float part;
    int whole;
    __device__ __forceinline__ explicit Power(float ref) {
        const float w = floorf(fmaxf(ref, (float)NO_EXPONENT));
        part = ref < w ? 1.0f : __builtin_amdgcn_exp2f(ref - w);
        whole = (int)w;
    }
    __device__ __forceinline__ float times(float x) const { return __builtin_amdgcn_ldexpf(x * part, whole); }
};

// The softmax step of f32 values.  A value is held times 2^-ve, so the weight
// that enters the product with it is 2^(x - M + SHIFT + ve - ref): ref, a pair's
// own, follows the largest x - M + ve of the keys that it sees, as M follows x.
// (By the largest ve alone, values that a pair does not see or hardly weighs
// would push its own below f16's smallest step.)  A weight's step of 2^-24 times a
// value's 2^15 is so 2^-28 of the largest weighted row's size at most, 2^HOLD
// of it for rows held with a larger one's exponent.  L sums 2^(x - M + SHIFT).
// Where all keys have one exponent E the two differ by a factor only, which goes into the
// exponent's offset, but not beside a maximum past 2^8: it would be rounded away there.
// N scores of a lane: get(i), put(i, weight); value(i): key i's exponent;
// rescale(c): o *= c; reduce: the maximum over a pair's lanes; mx: the pair's largest x.
template <int N, typename Get, typename Put, typename Value, typename Rescale, typename Reduce>
__device__ __forceinline__ void weigh_two(Get&& get, Put&& put, Value&& value, Rescale&& rescale, Reduce&& reduce, float f,
                                          float mx, int E, bool other, float& M, float& L, float& ref) {
    if (__builtin_amdgcn_ballot_w64(mx > M + SLACK)) {
        const float Mn = fmaxf(M, mx);
        if (Mn != M) {
            L *= __builtin_amdgcn_exp2f(M - Mn);
            ref += M - Mn;
            M = Mn;
        }
    }
    const float Mu = M == -__builtin_inff() ? 0.0f : M;
    float top = mx - Mu + (float)E;
    if (other) {
        top = -__builtin_inff();
#pragma unroll
        for (int i = 0; i < N; i++) top = fmaxf(top, fmaf(get(i), f, -Mu) + (float)value(i));
        top = reduce(top);
    }
    if (__builtin_amdgcn_ballot_w64(top > ref + SLACK)) {
        const float rn = fmaxf(ref, ceilf(top));
        rescale(rn == ref ? 1.0f : __builtin_amdgcn_exp2f(ref - rn));
        ref = rn;
    }
    const float r = ref == -__builtin_inff() ? (float)E : ref;
    const float base = SHIFT - Mu, up = (float)E - r;
    if (!other && !__builtin_amdgcn_ballot_w64(up < -60.0f || fabsf(Mu) > 256.0f)) {
        const float off = base + up;
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < N; i++) {
            const float w = weight(get(i), f, off);
            sum += w;
            put(i, w);
        }
        L += sum * __builtin_amdgcn_exp2f(-up);
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) {
            const float x = fmaf(get(i), f, base);
            L += __builtin_amdgcn_exp2f(x);
            put(i, __builtin_amdgcn_exp2f(x + (other ? (float)value(i) - r : up)));
        }
    }
}

// Of a few-row workgroup whose split's partial is stored: whether it is the last
// of its splits, which the counter c knows.
__device__ __forceinline__ bool last_to_arrive(int splits, int* c, int* flag) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (threadIdx.x == 0) {
        const int old = __hip_atomic_fetch_add(c, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        *flag = old == splits - 1;
        if (old == splits - 1) __hip_atomic_store(c, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    return *flag;
}

// How a tile's keys are split: into at most `parts` (its sequence's number), `share`
// keys each, the last one's fewer.
struct TileSplit {
    int keys, share, splits;
};
__device__ __forceinline__ TileSplit tile_split(const BatchArgs& a, const Seq& s, int p0, int parts) {
    TileSplit t;
    t.keys = last_key(a, s, min(p0 + TILE_PAIRS - 1, s.pairs - 1)) + 1;
    t.share = max(64, ((t.keys + parts - 1) / parts + 63) & ~63);
    t.splits = max(1, (t.keys + t.share - 1) / t.share);
    return t;
}
// (Nearly a division rounded up; what matters is that all who ask get the same.)
__device__ __forceinline__ int parts_of(const BatchArgs& a, int keys, int span) {
    return min(a.tile_splits, max(1, (int)fmaf((float)keys, __builtin_amdgcn_rcpf((float)span), 0.999f)));
}
// The tile of slot number `slot`: its sequence's last rows, which see the most keys, first.
__device__ __forceinline__ int tile_start(const BatchArgs& a, const Seq& s, int b, int slot) {
    return (tiles_of<TILE_PAIRS>(s.pairs) - 1 - (slot - first_tile<TILE_PAIRS>(s.row0, a.group, b))) * TILE_PAIRS;
}

// ---- many rows: waves of 32 pairs, tiles of TK keys shared through LDS -------------------
// Each wave holds 32 pairs as the columns of both products, S^T = K Q^T and
// O^T = V^T P^T (v_mfma_f32_32x32x16_f16): a lane has 16 scores of one pair, so
// the softmax needs one exchange with lane ^ 32, and its weights are already
// the second product's B operand once the keys of a 16-key step are taken in
// the order 4h .. 4h + 3, 8 + 4h .. (h = lane / 32), in which the transposed LDS reads of V
// fetch them.  q and the weights are f16 pairs, so each product takes two
// instructions (three with f32 keys and values); the matrix cores bound it: 2048 rows
// over 16048 f16 keys (32 / 8 heads of 128) take 870 to 935 us from card to card,
// 1160 to 1080 TFLOP/s of those instructions (a large f16 library product on
// the first card: 1191).  32 pairs a wave and 4 waves a workgroup: 64 pairs a wave left one
// wave a SIMD and took twice the time, 8 waves a workgroup and wave priorities gave nothing.  f16
// keys go straight to LDS (DirectSlab), two tiles deep, one barrier a tile.
template <typename KV, int HD>
__device__ __forceinline__ void tile_rows(const BatchArgs& a, const Seq& s, const int32_t* table, int b, int kvh,
                                         int p0, int z, int parts, _Float16* lds, Meta* meta, int2* exps) {
    using G = Geo<KV, HD>;
    typedef typename std::conditional<std::is_same<KV, Split>::value, float, KV>::type Elem;
    constexpr int TK = G::TK, W = G::W, SK = TK / W, KS = HD / 16, DT = HD / 32, HDP = G::HDP;
    constexpr bool TWO = G::TWO, RAW32 = std::is_same<KV, float>::value, PRE = std::is_same<KV, Split>::value;
    // blocks of 32 keys that take one softmax step together: two where registers hold their scores
    constexpr int NB = TWO || HD == 256 ? 1 : 2;
    constexpr int PART = TK * HDP;  // a part's elements
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int h = lane >> 5, c = lane & 31;
    // this tile's keys and the split's share of them
    static_assert(32 * W == TILE_PAIRS, "a wave 32 pairs");
    const TileSplit ts = tile_split(a, s, p0, parts);
    const int splits = ts.splits;
    if (z >= splits) return;
    const int j_lo = z * ts.share, j_hi = min(ts.keys, j_lo + ts.share);
    const int p = p0 + 32 * w + c;
    const bool live = p < s.pairs, work = p0 + 32 * w < s.pairs;
    const int last = live ? last_key(a, s, p) : -1;
    const int w_first = __builtin_amdgcn_readfirstlane(last_key(a, s, p0 + 32 * w));   // the wave's first pair sees
    const int w_last = __builtin_amdgcn_readfirstlane(last_key(a, s, min(p0 + 32 * w + 31, s.pairs - 1)));
    const int wg_first = last_key(a, s, p0);
    f16v o[DT];
#pragma unroll
    for (int d = 0; d < DT; d++)
#pragma unroll
        for (int e = 0; e < 16; e++) o[d][e] = 0.0f;
    float M = -__builtin_inff(), L = 0.0f;
    [[maybe_unused]] float ref = -__builtin_inff();      // f32 values: o is held times 2^-ref
    [[maybe_unused]] int kref = NO_EXPONENT, vref = NO_EXPONENT;  // f32: the exponents last used
    int wide = 0;     // some values were not finite

    // LDS addresses of this lane's operands; a step further along a row is an
    // exclusive or, because the pieces' order is one
    const uint32_t k_off = (c * HDP + (h ^ G::k_swap(c)) * 8) * 2;
    const int v_row = 4 * h + ((lane & 15) >> 2);
    const uint32_t v_off = (PART * G::PARTS + v_row * HDP +
                            ((2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) ^ G::v_swap(v_row)) * 8 + 4 * (lane & 1)) * 2;
    typedef typename std::conditional<RAW32, Slab<float, HD, SK>, DirectSlab<HD, (SK < 16 ? SK : 16)>>::type Stage;
    Stage slab;
    int valid = 1;
    [[maybe_unused]] int4 note_next = {0, 0, 0, 0};
    const uint32_t lds0 = lds_address(lds);
    [[maybe_unused]] const int64_t image = PRE ? ((int64_t)(s.row0 / TK) + b) * a.n_kv + kvh : 0;  // of the sequence's first tile
    auto fetch = [&](int j, int to) {  // a wave's share of the tile at key j, to buffer `to`
        if constexpr (PRE) {
            const int64_t im = image + (int64_t)(j / TK) * a.n_kv;
            note_next = a.notes[im];
            constexpr int SHARE = TK * G::KEY * 2 / W;  // bytes
            const i32x4 r = uniform_rsrc(a.images + im * (TK * G::KEY) + w * (SHARE / 2), SHARE);
#pragma unroll
            for (int i = 0; i < SHARE / 1024; i++)
                load_to_lds(r, 1024 * i + 16 * lane, lds0 + to * TK * G::KEY * 2 + w * SHARE + 1024 * i);
        } else if constexpr (RAW32) {
            valid = slab.load(a.kv, s.row0, kvh, j + SK * w, j_hi);
            slab.pages(a.kv, table, j + TK + SK * w, s.t);
        } else {
            const uint32_t at = lds0 + (to * TK * G::KEY + SK * w * HDP) * 2;
            valid = slab.load(a.kv, s.row0, kvh, j + SK * w, j_hi, at, at + PART * 2);
            slab.pages(a.kv, table, j + TK + SK * w, s.t);
        }
    };
    if (j_lo < j_hi) {
        if constexpr (RAW32) slab.init(a.kv, a.hd);
        else if constexpr (!PRE) slab.init(a.kv, a.hd, SK * w);
        if constexpr (!PRE) slab.pages(a.kv, table, j_lo + SK * w, s.t);
    }
    // the rows of q on their way while the page numbers are
    QRow<KS> q;
    q.load(q_at(a, s, kvh, p), live, 8 * h, 16, a.hd);
    if (j_lo < j_hi) fetch(j_lo, 0);
    h8 qh[KS], ql[KS];
    const int qe = split_q<TWO, KS>(q, qh, ql, [](uint32_t m) {
        return max(m, __builtin_bit_cast(uint32_t, other32(__builtin_bit_cast(float, m))));
    });
    [[maybe_unused]] const float f16_f = f16_factor(a.scale, qe);  // (f32 keys have exponents too)
    int buf = 0;
    for (int j0 = j_lo; j0 < j_hi; j0 += TK, buf ^= 1) {
        const int at = buf * TK * G::KEY;  // elements
        Meta note;
        [[maybe_unused]] const int2* key_exps = exps + buf * TK;
        if constexpr (RAW32) {
            const Meta mine = slab.store(lds + at, lds + at + PART * 2, exps + buf * TK, SK * w, PART, valid, true, kref, vref);
            if (lane == 0) meta[buf * W + w] = mine;
            if (j0 + TK < j_hi) fetch(j0 + TK, 0);
            __syncthreads();
            note = meta[buf * W + (lane & (W - 1))];
        } else if constexpr (PRE) {
            note = Meta{1, note_next.z, note_next.x, note_next.y};
            key_exps = a.exps + (image + (int64_t)(j0 / TK) * a.n_kv) * TK;
            loads_done();
            __syncthreads();
            if (j0 + TK < j_hi) fetch(j0 + TK, buf ^ 1);
        } else {
            if (lane == 0) meta[buf * W + w] = Meta{valid, 0, 0, 0};
            loads_done();
            __syncthreads();
            if (j0 + TK - 1 > wg_first) {  // some of its values are masked
                if (Stage::clean(lds + at + PART + SK * w * HDP) && lane == 0) meta[buf * W + w].flags = SLAB_WIDE;
                __syncthreads();
            }
            if (j0 + TK < j_hi) fetch(j0 + TK, buf ^ 1);
            note = meta[buf * W + (lane & (W - 1))];
        }
        if (!work || j0 > w_last) continue;
        // the slabs' notes, a lane a slab
        [[maybe_unused]] const Meta* notes = meta + buf * W;
        const bool masked = j0 + TK - 1 > w_first || __builtin_amdgcn_ballot_w64(!note.valid);
        wide |= __builtin_amdgcn_ballot_w64(note.flags & SLAB_WIDE) != 0;
        float f = f16_f;
        [[maybe_unused]] int lift = 0;
        bool other_k = false, other_v = false;  // f32: keys held with other exponents than the rest
        if constexpr (TWO) {
            kref = lanes_max<W>(note.ke);
            vref = lanes_max<W>(note.ve);
            lift = lift_of(a.scale, qe + kref);
            f = score_factor(a.scale, qe + kref - lift);
            other_k = __builtin_amdgcn_ballot_w64((note.ke != kref && note.ke != NO_EXPONENT) || (note.flags & SLAB_OTHER_K) || lift);
            other_v = __builtin_amdgcn_ballot_w64((note.ve != vref && note.ve != NO_EXPONENT) || (note.flags & SLAB_OTHER_V));
        }
#pragma unroll
        for (int b0 = 0; b0 < TK / 32; b0 += NB) {
            f16v sc[NB];
#pragma unroll
            for (int b = 0; b < NB; b++) {
#pragma unroll
                for (int e = 0; e < 16; e++) sc[b][e] = 0.0f;
                const char* kr = reinterpret_cast<const char*>(lds) + (size_t)(at + 32 * (b0 + b) * HDP) * 2;
#pragma unroll
                for (int k = 0; k < KS; k++) {
                    const uint32_t ko = k_off ^ (32 * k);
                    const h8 kf = *reinterpret_cast<const h8*>(kr + ko);
                    sc[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf, qh[k], sc[b], 0, 0, 0);
                    sc[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf, ql[k], sc[b], 0, 0, 0);
                    if constexpr (TWO) {
                        const h8 kl = *reinterpret_cast<const h8*>(kr + ko + PART * 2);
                        sc[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kl, qh[k], sc[b], 0, 0, 0);
                    }
                }
            }
            if (TWO && other_k)
#pragma unroll
                for (int b = 0; b < NB; b++)
#pragma unroll
                    for (int e = 0; e < 16; e++)
                        sc[b][e] = __builtin_amdgcn_ldexpf(
                            sc[b][e], key_exps[32 * (b0 + b) + 8 * (e >> 2) + 4 * h + (e & 3)].x - kref + lift);
            if (masked)
#pragma unroll
                for (int b = 0; b < NB; b++) {
                    const int rel = last - (j0 + 32 * (b0 + b)) - 4 * h;
#pragma unroll
                    for (int e = 0; e < 16; e++) {
                        const bool in = (PRE || notes[(32 * (b0 + b) + 8 * (e >> 2)) / SK].valid) && 8 * (e >> 2) + (e & 3) <= rel;
                        sc[b][e] = in ? sc[b][e] : -__builtin_inff();
                    }
                }
            float mx = sc[0][0];
#pragma unroll
            for (int b = 0; b < NB; b++)
#pragma unroll
                for (int e = b == 0; e < 16; e++) mx = fmaxf(mx, sc[b][e]);
            mx = max32(mx) * f;
            auto rescale = [&](float corr) {
#pragma unroll
                for (int d = 0; d < DT; d++)
#pragma unroll
                    for (int e = 0; e < 16; e++) o[d][e] *= corr;
            };
            [[maybe_unused]] float off = 0.0f;
            if constexpr (TWO) {
                weigh_two<16>([&](int e) { return sc[0][e]; }, [&](int e, float v) { sc[0][e] = v; },
                              [&](int e) { return key_exps[32 * b0 + 8 * (e >> 2) + 4 * h + (e & 3)].y; }, rescale,
                              [](float v) { return max32(v); }, f, mx, vref, other_v, M, L, ref);
            } else {
                if (__builtin_amdgcn_ballot_w64(mx > M + SLACK)) {
                    const float Mn = fmaxf(M, mx);
                    const float corr = Mn == M ? 1.0f : __builtin_amdgcn_exp2f(M - Mn);
                    L *= corr;
                    rescale(corr);
                    M = Mn;
                }
                off = SHIFT - (M == -__builtin_inff() ? 0.0f : M);
            }
#pragma unroll
            for (int b = 0; b < NB; b++) {
                if constexpr (!TWO)
#pragma unroll
                    for (int e = 0; e < 16; e++) {
                        sc[b][e] = weight(sc[b][e], f, off);
                        L += sc[b][e];
                    }
#pragma unroll
                for (int k = 0; k < 2; k++) {  // 16 keys a step
                    u32x4 ph, pl;
#pragma unroll
                    for (int u = 0; u < 4; u++) {
                        uint32_t hi, lo;
                        split2<TWO>(sc[b][8 * k + 2 * u], sc[b][8 * k + 2 * u + 1], &hi, &lo);
                        ph[u] = hi;
                        pl[u] = lo;
                    }
                    const h8 p8 = __builtin_bit_cast(h8, ph), q8 = __builtin_bit_cast(h8, pl);
                    const char* vr = reinterpret_cast<const char*>(lds) + (size_t)(at + (32 * (b0 + b) + 16 * k) * HDP) * 2;
#pragma unroll
                    for (int d = 0; d < DT; d++) {
                        const char* vd = vr + (v_off ^ (64 * d));
                        const h4 v0 = read_t(vd), v1 = read_t(vd + 16 * HDP);
                        const h8 vf = __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7);
                        o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf, p8, o[d], 0, 0, 0);
                        o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf, q8, o[d], 0, 0, 0);
                        if constexpr (TWO) {
                            const h4 w0 = read_t(vd + PART * 2), w1 = read_t(vd + PART * 2 + 16 * HDP);
                            const h8 vl = __builtin_shufflevector(w0, w1, 0, 1, 2, 3, 4, 5, 6, 7);
                            o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vl, p8, o[d], 0, 0, 0);
                        }
                    }
                }
            }
        }
    }
    L += other32(L);
    const float inv = L != 0.0f ? 1.0f / L : 0.0f;
    [[maybe_unused]] const Power unit(ref);
#pragma unroll
    for (int d = 0; d < DT; d++)
#pragma unroll
        for (int e = 0; e < 16; e++) {
            const float x = o[d][e] * inv;
            o[d][e] = TWO ? unit.times(x) : x;
        }
    if constexpr (!TWO) {
        float all = 0.0f;
#pragma unroll
        for (int d = 0; d < DT; d++)
#pragma unroll
            for (int e = 0; e < 16; e++) all = fmaf(o[d][e], 0.0f, all);
        if (not_finite_of_values(all, L)) {
            wide = 1;
#pragma unroll
            for (int d = 0; d < DT; d++)
#pragma unroll
                for (int e = 0; e < 16; e++) o[d][e] = finite_or(o[d][e], L == L);
        }
    }
    if (wide)  // rows that see a value that is not finite
        for (int j = j_lo; j < min(j_hi, w_last + 1); j++) {
            const Elem* v = value_row<Elem>(a.kv, s.row0, table, kvh, j);
            if (!v) continue;
#pragma unroll
            for (int d = 0; d < DT; d++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int dim = 32 * d + 8 * i + 4 * h;
                    const f4 x = wide4(v + (dim < a.hd ? dim : 0), j <= last && dim < a.hd);
#pragma unroll
                    for (int t = 0; t < 4; t++) o[d][4 * i + t] += x[t];
                }
        }
    // the wave's rows through LDS of its own, OD dims at a time, so that each
    // store covers whole rows: a lane's own values lie 16 bytes apart in 32 rows,
    // and as write-through stores those took longer than the keys of a split
    __syncthreads();
    constexpr int OD = HD < 128 ? HD : 128, OROW = HDP < 128 ? HDP : 128;
    static_assert((size_t)W * 32 * OROW * 4 <= G::TILE_LDS, "outputs fit the tiles' LDS");
    float* os = reinterpret_cast<float*>(lds) + w * 32 * OROW;
    const int rows = min(32, s.pairs - p0 - 32 * w);
#pragma unroll
    for (int d0 = 0; d0 < HD; d0 += OD) {
#pragma unroll
        for (int d = 0; d < OD / 32; d++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const f16v& x = o[d0 / 32 + d];
                *reinterpret_cast<f4*>(os + c * OROW + ((8 * d + 2 * i + h) ^ (c & 15)) * 4) =
                    f4{x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]};
            }
        wave_sync();
        constexpr int QR = OD / 4;  // float4 a row
        for (int i = lane; i < rows * QR; i += 64) {
            const int r = i / QR, d = d0 + i % QR * 4;
            if (d >= a.hd) continue;
            const f4 y = *reinterpret_cast<const f4*>(os + r * OROW + ((i % QR) ^ (r & 15)) * 4);
            const int pr = p0 + 32 * w + r;
            if (splits == 1) {
                *reinterpret_cast<f4*>(out_at(a, s, kvh, pr) + d) = y;
            } else {
                *reinterpret_cast<f4*>(a.part + (place(a, s, kvh, pr) * a.part_splits + z) * a.hd + d) = y;
            }
        }
        wave_sync();
    }
    if (splits > 1 && live && h == 0)
        *reinterpret_cast<f2*>(a.part_ml + (place(a, s, kvh, p) * a.part_splits + z) * 2) = f2{M, L};
}

// ---- few rows: up to 16 pairs, each wave its own keys ------------------------------------------
// A decode step reads the cache once and computes little: the waves of a
// workgroup take the split's keys 32 at a time in turn, each through LDS rows
// of its own without a barrier, with the next keys' loads in flight; at
// the end they join through LDS.  The products as above, 16 columns wide
// (v_mfma_f32_16x16x32_f16): a lane has the scores of keys 4g .. 4g + 3 and 16 +
// 4g .. (g = lane / 16) of one pair.  HBM bounds it: 48 rows over 187420 keys of
// 8 KV heads of 128 in f16, 769 MB, take 158 us, 4.9 TB/s (a large copy reaches
// 4.7); a single row over 778 keys takes 11.4 us, which is latency: lengths,
// page numbers, keys, then the splits' partials one behind the other.
// Returns the splits to join (1: the output is written, 0: no such split).
template <typename KV, int HD>
__device__ __forceinline__ int few_rows(const BatchArgs& a, const Seq& s, const int32_t* table, int kvh, int p0, int z,
                                        _Float16* lds, float* wml, int2* exps) {
    using G = Geo<KV, HD>;
    constexpr int KS = HD / 32, DT = HD / 16, FK = G::FK, NB = FK / 16, W = G::W, HDP = G::HDP;
    constexpr bool F32 = G::TWO;
    constexpr int PART = FK * HDP;
    constexpr int OROW = HD + 4;  // f32 elements of a pair's joined output
    static_assert(16 * OROW * 4 <= FK * G::KEY * 2, "the output fits the wave's key rows");
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int g = lane >> 4, c = lane & 15;
    const int pairs = min(FEW_PAIRS, s.pairs - p0);
    const int keys = last_key(a, s, p0 + pairs - 1) + 1;
    const int splits = p0 ? 1 : min(a.few_splits, max(1, (keys + a.few_span - 1) / a.few_span));
    if (z >= splits) return 0;
    const int j_lo = z * a.few_span, j_hi = z == splits - 1 ? keys : min(keys, j_lo + a.few_span);
    const int p = p0 + c;
    const bool live = c < pairs;
    const int last = live ? last_key(a, s, p) : -1;
    const int first = last_key(a, s, p0);
    _Float16* ks = lds + w * FK * G::KEY;
    _Float16* vs = ks + PART * G::PARTS;
    const int v_row = 4 * g + ((lane & 15) >> 2);
    const uint32_t k_off = (c * HDP + (g ^ G::k_swap(c)) * 8) * 2;
    const uint32_t v_off = (v_row * HDP + (((lane & 3) >> 1) ^ G::v_swap(v_row)) * 8 + 4 * (lane & 1)) * 2;
    float M = -__builtin_inff(), L = 0.0f;
    f4 o[DT];
#pragma unroll
    for (int d = 0; d < DT; d++) o[d] = f4{0.0f, 0.0f, 0.0f, 0.0f};
    int wide = 0;
    [[maybe_unused]] float ref = -__builtin_inff();  // f32 values: o is held times 2^-ref
    {
        Slab<KV, HD, FK> slab;
        slab.init(a.kv, a.hd);
        const int step = W * FK, j_w = j_lo + FK * w;
        // the row of q on its way while the page numbers are
        int valid = 0;
        if (j_w < j_hi) slab.pages(a.kv, table, j_w, s.t);
        QRow<KS> q;
        q.load(q_at(a, s, kvh, p), live, 8 * g, 32, a.hd);
        if (j_w < j_hi) {
            valid = slab.load(a.kv, s.row0, kvh, j_w, j_hi);
            slab.pages(a.kv, table, j_w + step, s.t);
        }
        h8 qh[KS], ql[KS];
        const int qe = split_q<F32, KS>(q, qh, ql, [](uint32_t m) {
            m = max(m, __builtin_bit_cast(uint32_t, other16(__builtin_bit_cast(float, m))));
            return max(m, __builtin_bit_cast(uint32_t, other32(__builtin_bit_cast(float, m))));
        });
        [[maybe_unused]] const float f16_f = f16_factor(a.scale, qe);  // (f32 keys have exponents too)
        for (int j0 = j_w; j0 < j_hi; j0 += step) {
            const Meta mt = slab.store(ks, vs, exps + FK * w, 0, PART, valid, j0 + FK - 1 > first, NO_EXPONENT, NO_EXPONENT);
            if (j0 + step < j_hi) {
                valid = slab.load(a.kv, s.row0, kvh, j0 + step, j_hi);
                slab.pages(a.kv, table, j0 + 2 * step, s.t);
            }
            wave_sync();
            const bool masked = j0 + FK - 1 > first || mt.valid != (1 << NB) - 1;
            wide |= mt.flags & SLAB_WIDE;
            f4 sc[NB];
            float mx = -__builtin_inff();
#pragma unroll
            for (int b = 0; b < NB; b++) {
                sc[b] = f4{0.0f, 0.0f, 0.0f, 0.0f};
                const char* kr = reinterpret_cast<const char*>(ks + 16 * b * HDP);
#pragma unroll
                for (int k = 0; k < KS; k++) {
                    const h8 kf = *reinterpret_cast<const h8*>(kr + (k_off ^ (64 * k)));
                    sc[b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qh[k], sc[b], 0, 0, 0);
                    sc[b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, ql[k], sc[b], 0, 0, 0);
                    if constexpr (F32) {
                        const h8 kl = *reinterpret_cast<const h8*>(kr + (k_off ^ (64 * k)) + PART * 2);
                        sc[b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kl, qh[k], sc[b], 0, 0, 0);
                    }
                }
            }
            [[maybe_unused]] const int lift = F32 ? lift_of(a.scale, qe + mt.ke) : 0;
            if (F32 && ((mt.flags & SLAB_OTHER_K) || __builtin_amdgcn_ballot_w64(lift != 0)))
#pragma unroll
                for (int b = 0; b < NB; b++)
#pragma unroll
                    for (int t = 0; t < 4; t++)
                        sc[b][t] = __builtin_amdgcn_ldexpf(sc[b][t], exps[FK * w + 16 * b + 4 * g + t].x - mt.ke + lift);
            if (masked) {
                const int rel = last - j0 - 4 * g;
#pragma unroll
                for (int b = 0; b < NB; b++)
#pragma unroll
                    for (int t = 0; t < 4; t++)
                        sc[b][t] = (mt.valid >> b & 1) && 16 * b + t <= rel ? sc[b][t] : -__builtin_inff();
            }
#pragma unroll
            for (int b = 0; b < NB; b++)
#pragma unroll
                for (int t = 0; t < 4; t++) mx = fmaxf(mx, sc[b][t]);
            const float f = F32 ? score_factor(a.scale, qe + mt.ke - lift) : f16_f;
            mx *= f;
            mx = fmaxf(mx, other16(mx));
            mx = max32(mx);
            auto rescale = [&](float corr) {
#pragma unroll
                for (int d = 0; d < DT; d++) o[d] *= corr;
            };
            if constexpr (F32) {
                weigh_two<4 * NB>([&](int i) { return sc[i >> 2][i & 3]; }, [&](int i, float v) { sc[i >> 2][i & 3] = v; },
                                  [&](int i) { return exps[FK * w + 16 * (i >> 2) + 4 * g + (i & 3)].y; }, rescale,
                                  [](float v) { return max32(fmaxf(v, other16(v))); }, f, mx, mt.ve,
                                  (mt.flags & SLAB_OTHER_V) != 0, M, L, ref);
            } else {
                if (__builtin_amdgcn_ballot_w64(mx > M + SLACK)) {
                    const float Mn = fmaxf(M, mx);
                    const float corr = Mn == M ? 1.0f : __builtin_amdgcn_exp2f(M - Mn);
                    L *= corr;
                    rescale(corr);
                    M = Mn;
                }
                const float off = SHIFT - (M == -__builtin_inff() ? 0.0f : M);
#pragma unroll
                for (int b = 0; b < NB; b++)
#pragma unroll
                    for (int t = 0; t < 4; t++) {
                        sc[b][t] = weight(sc[b][t], f, off);
                        L += sc[b][t];
                    }
            }
            uint32_t ph[2 * NB], pl[2 * NB];
#pragma unroll
            for (int u = 0; u < 2 * NB; u++)
                split2<F32>(sc[u >> 1][(u & 1) * 2], sc[u >> 1][(u & 1) * 2 + 1], &ph[u], &pl[u]);
            const char* vr = reinterpret_cast<const char*>(vs);
            if constexpr (NB == 2) {
                const h8 p8 = __builtin_bit_cast(h8, ph), q8 = __builtin_bit_cast(h8, pl);
#pragma unroll
                for (int d = 0; d < DT; d++) {
                    const char* vd = vr + (v_off ^ (32 * d));
                    const h4 v0 = read_t(vd), v1 = read_t(vd + 32 * HDP);
                    const h8 vf = __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7);
                    o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, p8, o[d], 0, 0, 0);
                    o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, q8, o[d], 0, 0, 0);
                }
            } else {
                const h4 p4 = __builtin_bit_cast(h4, ph), q4 = __builtin_bit_cast(h4, pl);
#pragma unroll
                for (int d = 0; d < DT; d++) {
                    const char* vd = vr + (v_off ^ (32 * d));
                    const h4 vf = read_t(vd), vl = read_t(vd + PART * 2);
                    o[d] = __builtin_amdgcn_mfma_f32_16x16x16f16(vf, p4, o[d], 0, 0, 0);
                    o[d] = __builtin_amdgcn_mfma_f32_16x16x16f16(vf, q4, o[d], 0, 0, 0);
                    o[d] = __builtin_amdgcn_mfma_f32_16x16x16f16(vl, p4, o[d], 0, 0, 0);
                }
            }
            wave_sync();
        }
        L += other16(L);
        L += other32(L);
        // the wave's normalised output over its own key rows, its maximum and sum beside
        const float inv = L != 0.0f ? 1.0f / L : 0.0f;
        [[maybe_unused]] const Power unit(ref);
        float* os = reinterpret_cast<float*>(ks);
#pragma unroll
        for (int d = 0; d < DT; d++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float x = o[d][e] * inv;
                o[d][e] = F32 ? unit.times(x) : x;
            }
        if constexpr (!F32) {
            float all = 0.0f;
#pragma unroll
            for (int d = 0; d < DT; d++)
#pragma unroll
                for (int e = 0; e < 4; e++) all = fmaf(o[d][e], 0.0f, all);
            if (not_finite_of_values(all, L)) {
                wide = 1;
#pragma unroll
                for (int d = 0; d < DT; d++)
#pragma unroll
                    for (int e = 0; e < 4; e++) o[d][e] = finite_or(o[d][e], L == L);
            }
        }
        if (wide)  // rows that see a value that is not finite
            for (int j0 = j_w; j0 < j_hi; j0 += step)
                for (int j = j0; j < min(j0 + FK, j_hi); j++) {
                    const KV* v = value_row<KV>(a.kv, s.row0, table, kvh, j);
                    if (!v) continue;
#pragma unroll
                    for (int d = 0; d < DT; d++) {
                        const int dim = 16 * d + 4 * g;
                        o[d] += wide4(v + (dim < a.hd ? dim : 0), j <= last && dim < a.hd);
                    }
                }
#pragma unroll
        for (int d = 0; d < DT; d++) *reinterpret_cast<f4*>(os + c * OROW + 16 * d + 4 * g) = o[d];
        if (g == 0) {
            wml[w * 32 + c] = M;
            wml[w * 32 + 16 + c] = L;
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < pairs * (HD / 4); i += W * 64) {
        const int pi = i / (HD / 4), dim = (i % (HD / 4)) * 4;
        if (dim >= a.hd) continue;
        float Mx = -__builtin_inff(), Ls = 0.0f;
#pragma unroll
        for (int x = 0; x < W; x++)
            if (wml[x * 32 + 16 + pi] != 0.0f) Mx = fmaxf(Mx, wml[x * 32 + pi]);
        auto partial = [&](int x) {
            return *reinterpret_cast<const f4*>(reinterpret_cast<const float*>(lds + x * FK * G::KEY) + pi * OROW + dim);
        };
        float wt[W];
#pragma unroll
        for (int x = 0; x < W; x++) {
            const float l = wml[x * 32 + 16 + pi];
            wt[x] = l != 0.0f ? l * __builtin_amdgcn_exp2f(wml[x * 32 + pi] - Mx) : 0.0f;
            Ls += wt[x];
        }
        const float inv = Ls != 0.0f ? 1.0f / Ls : 0.0f;
        f4 y = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int x = 0; x < W; x++) y += wt[x] * inv * partial(x);  // weights of at most 1: large values stay in range
        if (some_not_finite(y)) y = sum_not_finite(y, W, partial);
        if (splits == 1) {
            *reinterpret_cast<f4*>(out_at(a, s, kvh, p0 + pi) + dim) = y;
        } else {
            const int64_t at = place(a, s, kvh, p0 + pi);
            float* pt = a.part + (at * a.part_splits + z) * a.hd + dim;
            put2(pt, y[0], y[1]);
            put2(pt + 2, y[2], y[3]);
            if (dim == 0) put_ml(a, at, z, Mx, Ls);
        }
    }
    return splits;
}

// The splits of a step of up to 64 sequences, a lane each.  The span of keys is the
// shortest, in steps of 64, by which all tiles' splits find room in a.tile_slots
// workgroups a KV head (one a tile does: there are as many), so that all start at
// once; by the longest kv_len alone, sequences of unlike lengths got
// fewer and longer ones.
__device__ __forceinline__ int shortest_span(const BatchArgs& a, int tiles, int keys) {
    int lo = TILE_MIN_SPAN / 64, hi = max(lo, ((int)wave_max_u32((uint32_t)keys) + 63) / 64);
    for (int mid = lo; lo < hi; mid = (lo + hi) / 2) {
        if (lanes_sum(tiles * parts_of(a, keys, 64 * mid)) <= a.tile_slots) hi = mid;
        else lo = mid + 1;
    }
    return 64 * hi;
}
// The workgroups are numbered without gaps.  Numbered over the most splits that any
// tile might have, every fourth or so had nothing to do, and with them a quarter of the
// CUs: workgroups are dealt to the parts of an XCD in turn (132 us instead of
// 100 for chunks and single rows of 16 sequences).
struct TilePlan {
    int b, tile, z, parts;  // of number `slot`; b -1: none
};
__device__ __forceinline__ TilePlan tile_plan(const BatchArgs& a, int slot) {
    const int lane = threadIdx.x & 63;
    int tiles = 0, keys = 0;
    if (lane < a.n_seq) {
        const Seq s = sequence(a, lane);
        if (s.pairs > a.few_rows) tiles = tiles_of<TILE_PAIRS>(s.pairs), keys = s.t;
    }
    const int parts = parts_of(a, keys, shortest_span(a, tiles, keys)), n = tiles * parts;
    const int before = lanes_before(n);
    const uint64_t mask = __builtin_amdgcn_ballot_w64(slot >= before && slot < before + n);
    if (mask == 0) return {-1, 0, 0, 1};
    TilePlan t;
    t.b = __builtin_amdgcn_readfirstlane((int)__builtin_ctzll(mask));
    t.parts = __builtin_amdgcn_readlane(parts, t.b);
    const int at = slot - __builtin_amdgcn_readlane(before, t.b);
    t.tile = at / t.parts;
    t.z = at - t.tile * t.parts;
    return t;
}
// A sequence's parts, for those who come by its tiles' own numbers.
__device__ __forceinline__ int planned_parts(const BatchArgs& a, const Seq& s, int b) {
    if (!a.tile_slots) return parts_of(a, s.t, a.tile_span);
    const int lane = threadIdx.x & 63;
    int tiles = 0, keys = 0;
    if (lane < a.n_seq) {
        const Seq x = sequence(a, lane);
        if (x.pairs > a.few_rows) tiles = tiles_of<TILE_PAIRS>(x.pairs), keys = x.t;
    }
    return parts_of(a, s.t, shortest_span(a, tiles, keys));
}

// KIND: which workgroups a launch has.  The two bodies in one kernel keep more
// registers than either needs, so launches that need one of them have it alone.
constexpr int TILE = 1, FEW = 2;
template <typename KV, int HD, int KIND>
__global__ __launch_bounds__((Geo<KV, HD>::W * 64), HD == 256 ? 1 : 2) void attend_kernel(BatchArgs a) {
    constexpr int W = Geo<KV, HD>::W, NT = W * 64;
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
    __shared__ Meta meta[2 * W];
    __shared__ int2 exps[2 * 64];  // of a tile's keys, twice, or of each wave's
    __shared__ float wml[W * 32];
    __shared__ int flag;
    _Float16* lds = reinterpret_cast<_Float16*>(smem);
    const int tile_blocks = a.n_kv * (a.tile_slots ? a.tile_slots : a.tiles * a.tile_splits);
    const bool tile = KIND == TILE || (KIND != FEW && (int)blockIdx.x < tile_blocks);
    int id = tile ? (int)blockIdx.x : (int)blockIdx.x - tile_blocks;
    const int kvh = id % a.n_kv;
    id /= a.n_kv;
    int z, slot, b, parts = 1;
    if (KIND != FEW && tile && a.tile_slots) {
        const TilePlan t = tile_plan(a, id);
        b = t.b, z = t.z, slot = t.tile, parts = t.parts;
    } else {
        const int most = tile ? a.tile_splits : a.few_splits;
        z = id % most, slot = id / most;
        b = tile ? sequence_of<TILE_PAIRS>(a, slot, a.group) : slot;
    }
    if (b < 0) return;
    const Seq s = sequence(a, b);
    if (s.pairs == 0 || (s.pairs > a.few_rows) != tile) return;
    const int32_t* table = a.kv.tables ? a.kv.tables + b * a.kv.table_stride : nullptr;
    if (tile) {
        if constexpr ((KIND & TILE) != 0) {
            int p0;
            if (a.tile_slots) p0 = (tiles_of<TILE_PAIRS>(s.pairs) - 1 - slot) * TILE_PAIRS;
            else p0 = tile_start(a, s, b, slot), parts = parts_of(a, s.t, a.tile_span);
            tile_rows<KV, HD>(a, s, table, b, kvh, p0, z, parts, lds, meta, exps);
        }
    } else {
        if constexpr ((KIND & FEW) != 0)
            for (int p0 = 0; p0 < s.pairs; p0 += FEW_PAIRS) {  // more than once (and then not split) only where max_rows was too small
                const int splits = few_rows<KV, HD>(a, s, table, kvh, p0, z, lds, wml, exps);
                if (splits > 1 && last_to_arrive(splits, a.counters + slot * a.n_kv + kvh, &flag))
                    join<true>(a, s, kvh, p0, min(FEW_PAIRS, s.pairs - p0), splits, reinterpret_cast<float*>(smem));
                __syncthreads();  // before the next rows take the LDS
            }
    }
}

// The tiles' splits, FEW_PAIRS pairs a workgroup, in a launch behind theirs: the
// last split to arrive would read a tile's partials (65 KB each) alone: 100 rows
// over 3300 keys took 64.9 us so, and take 31.7.
__global__ __launch_bounds__(JOIN_THREADS) void join_kernel(BatchArgs a) {
    constexpr int PER = TILE_PAIRS / FEW_PAIRS;
    __shared__ float wt[JOIN_FLOATS];
    int id = (int)blockIdx.x;
    const int kvh = id % a.n_kv;
    id /= a.n_kv;
    const int slot = id / PER, b = sequence_of<TILE_PAIRS>(a, slot, a.group);
    if (b < 0) return;
    const Seq s = sequence(a, b);
    if (s.pairs <= a.few_rows) return;
    const int p0 = tile_start(a, s, b, slot), first = p0 + id % PER * FEW_PAIRS;
    if (first >= s.pairs) return;
    const TileSplit ts = tile_split(a, s, p0, planned_parts(a, s, b));
    if (ts.splits > 1) join<false>(a, s, kvh, first, min(FEW_PAIRS, s.pairs - first), ts.splits, wt);
}

// ---- f32 rows as f16 parts, once a launch ---------------------------------------------
// Where many tiles of rows read the same f32 keys, splitting them in every
// tile (5 operations a value) cost more than the products' own work on them:
// here a workgroup splits one tile of TK keys of a KV head and writes it as LDS will
// hold it.  It moves 8 + 8 bytes an element: 9910 rows of 8 KV heads of 128 take 32 us of
// the call's 602, the products 1020 TFLOP/s.
template <int HD>
__global__ __launch_bounds__(256) void split_kernel(BatchArgs a, _Float16* images, int4* notes, int2* exps) {
    using G = Geo<Split, HD>;
    constexpr int TK = G::TK, HDP = G::HDP, CPR = HDP / 8, NP = TK * CPR / 256, PART = TK * HDP;
    static_assert(NP * 256 == TK * CPR, "whole pieces a thread");
    __shared__ uint32_t red[3][4];
    const int kvh = (int)(blockIdx.x % a.n_kv), t = (int)(blockIdx.x / a.n_kv), tid = threadIdx.x;
    const int b = sequence_of<TK>(a, t, 1);
    if (b < 0) return;
    const Seq s = sequence(a, b);
    const int j0 = (t - (int)(s.row0 / TK) - b) * TK;
    u32x4 k[NP][2], v[NP][2];
    const float* ks = reinterpret_cast<const float*>(a.kv.k) + (s.row0 + j0) * a.kv.k_position + kvh * a.kv.head;
    const float* vs = reinterpret_cast<const float*>(a.kv.v) + (s.row0 + j0) * a.kv.v_position + kvh * a.kv.head;
#pragma unroll
    for (int i = 0; i < NP; i++) {
        const int pc = tid + 256 * i, key = pc / CPR, col = pc % CPR;
        const bool in = j0 + key < s.t && col * 8 < a.hd;
#pragma unroll
        for (int p = 0; p < 2; p++) {
            k[i][p] = in ? *reinterpret_cast<const u32x4*>(ks + key * a.kv.k_position + col * 8 + 4 * p) : u32x4{0, 0, 0, 0};
            v[i][p] = in ? *reinterpret_cast<const u32x4*>(vs + key * a.kv.v_position + col * 8 + 4 * p) : u32x4{0, 0, 0, 0};
        }
    }
    uint32_t km[NP], vm[NP], kt = 0, vt = 0;
    piece_sizes(k, km, false);
    const bool wide = piece_sizes(v, vm, true);
#pragma unroll
    for (int i = 0; i < NP; i++) kt = max(kt, km[i]), vt = max(vt, vm[i]);
    kt = wave_max_u32(kt);
    vt = wave_max_u32(vt);
    if ((tid & 63) == 0) red[0][tid >> 6] = kt, red[1][tid >> 6] = vt, red[2][tid >> 6] = wide ? SLAB_WIDE : 0;
    __syncthreads();
    const int ke = hold_all(max(max(red[0][0], red[0][1]), max(red[0][2], red[0][3])), NO_EXPONENT);
    const int ve = hold_all(max(max(red[1][0], red[1][1]), max(red[1][2], red[1][3])), NO_EXPONENT);
    const int64_t im = (int64_t)t * a.n_kv + kvh;
    int ek[NP], ev[NP], flags = 0;
    if (row_exponents<CPR>(km, ke, ek)) flags |= SLAB_OTHER_K;
    if (row_exponents<CPR>(vm, ve, ev)) flags |= SLAB_OTHER_V;
#pragma unroll
    for (int i = 0; i < NP; i++)
        if (tid % CPR == 0) exps[im * TK + (tid + 256 * i) / CPR] = int2{ek[i], ev[i]};
    if (flags && (tid & 63) == 0) atomicOr(&red[2][0], flags);
    __syncthreads();
    if (tid == 0) notes[im] = int4{ke, ve, (int)(red[2][0] | red[2][1] | red[2][2] | red[2][3]), 0};
    _Float16* out = images + im * (TK * G::KEY);
#pragma unroll
    for (int i = 0; i < NP; i++) {
        const int pc = tid + 256 * i, key = pc / CPR, col = pc % CPR;
        u32x4 kh, kl, vh, vl;
        split8(k[i], ek[i], &kh, &kl);
        split8(v[i], ev[i], &vh, &vl);
        u32x4* kd = reinterpret_cast<u32x4*>(out + key * HDP + (col ^ G::k_swap(key)) * 8);
        u32x4* vd = reinterpret_cast<u32x4*>(out + 2 * PART + key * HDP + (col ^ G::v_swap(key)) * 8);
        *kd = kh;
        kd[PART / 8] = kl;
        *vd = vh;
        vd[PART / 8] = vl;
    }
}

template <typename KV, int HD, int KIND>
hipError_t launch(const BatchArgs& a, hipStream_t s) {
    using G = Geo<KV, HD>;
    constexpr size_t lds = KIND == TILE ? G::TILE_LDS : KIND == FEW ? G::FEW_LDS : G::LDS;
    const hipError_t e = hipFuncSetAttribute((const void*)attend_kernel<KV, HD, KIND>,
                                             hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    if (e != hipSuccess) return e;
    const int tile_blocks = a.tile_slots ? a.tile_slots : a.tiles * a.tile_splits;
    const unsigned blocks = (unsigned)(a.n_kv * (tile_blocks + (KIND & FEW ? a.n_seq * a.few_splits : 0)));
    static_assert(G::W * 64 == JOIN_THREADS && JOIN_FLOATS * 4 <= G::FEW_LDS, "few rows join with what they have");
    hipLaunchKernelGGL((attend_kernel<KV, HD, KIND>), dim3(blocks), dim3(G::W * 64), lds, s, a);
    if (KIND != FEW && a.tile_splits > 1)
        hipLaunchKernelGGL(join_kernel, dim3((unsigned)(a.n_kv * a.tiles * (TILE_PAIRS / FEW_PAIRS))), dim3(JOIN_THREADS), 0, s, a);
    return hipGetLastError();
}
template <typename KV, int HD>
hipError_t launch_kind(const BatchArgs& a, hipStream_t s) {
    return a.few_rows == 0 ? launch<KV, HD, TILE>(a, s) : a.tiles == 0 ? launch<KV, HD, FEW>(a, s)
                                                                       : launch<KV, HD, TILE | FEW>(a, s);
}
template <int HD>
hipError_t launch_split(const BatchArgs& a, _Float16* images, int4* notes, int2* exps, int tiles, hipStream_t s) {
    hipLaunchKernelGGL(split_kernel<HD>, dim3((unsigned)(tiles * a.n_kv)), dim3(256), 0, s, a, images, notes, exps);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? launch<Split, HD, TILE>(a, s) : e;
}
template <typename KV>
hipError_t launch_hd(const BatchArgs& a, hipStream_t s) {
    return a.hd <= 64 ? launch_kind<KV, 64>(a, s) : a.hd <= 96 ? launch_kind<KV, 96>(a, s)
         : a.hd <= 128 ? launch_kind<KV, 128>(a, s) : launch_kind<KV, 256>(a, s);
}

// A launch has fewer than 2^32 threads.
constexpr int64_t MAX_BLOCKS = (((int64_t)1 << 32) - 1) / JOIN_THREADS;
constexpr size_t PART_BYTES = (size_t)256 << 20;  // most memory of partial results
// f32 prompts are split beforehand from this many tiles a sequence on, as far
// as this much memory holds them.  Prompts of 1, 2, 4, 8, 16, 32 tiles (us), split
// beforehand: 13.4, 15.0, 19.6, 24.9, 33.6, 58.3; in every tile: 11.3, 14.3,
// 20.2, 26.2, 36.3, 69.8 (32 / 8 heads of 128).
constexpr int64_t SPLIT_MIN_TILES = 4;
constexpr size_t SPLIT_BYTES = (size_t)1 << 30;

rdl_status run(BatchArgs a, bool f16, size_t max_rows, size_t max_kv, hipStream_t s) {
    const int64_t m = a.m, rows = max_rows == 0 || (int64_t)max_rows > m ? m : (int64_t)max_rows;
    int64_t keys = a.kv.tables ? a.kv.table_stride << a.kv.shift : m;
    if (max_kv != 0 && (int64_t)max_kv < keys) keys = (int64_t)max_kv;
    keys = std::max<int64_t>(1, std::min<int64_t>(keys, INT32_MAX / 2));
    const int64_t pairs = (int64_t)a.n_seq * a.n_kv, G = a.group;
    if (pairs > (int64_t)1 << 28) return api_fail(RDL_ERR_UNSUPPORTED, "%d sequences of %d KV heads", a.n_seq, a.n_kv);
    if (m * G > INT32_MAX) return api_fail(RDL_ERR_UNSUPPORTED, "%lld rows of %d heads a KV head", (long long)m, a.group);
    while (((int64_t)1 << a.group_shift) < G) a.group_shift++;
    a.group_mul = (uint32_t)((((uint64_t)1 << 32) * (((uint64_t)1 << a.group_shift) - (uint64_t)G)) / (uint64_t)G + 1);
    // sequences of up to 16 pairs; all of them where none is expected to have more
    // (packed prompts of few rows have few keys: tiles serve them too)
    const bool only_few = rows * G <= FEW_PAIRS, only_tile = !only_few && (a.n_seq == 1 || !a.kv.tables);
    a.few_rows = only_few ? INT32_MAX : only_tile ? 0 : FEW_PAIRS;
    a.tiles = only_few ? 0 : (int)(m * G / TILE_PAIRS + a.n_seq);
    const int64_t most_parts =
        std::max<int64_t>(1, (int64_t)(PART_BYTES / ((size_t)m * a.n_heads * (a.hd + 2) * sizeof(float))));
    auto split = [&](int64_t base, int64_t target, int most, int unit, int64_t min_span, int* span, int* splits) {
        int64_t sp = std::max(min_span, keys * base / target);
        sp = (sp + unit - 1) / unit * unit;
        int64_t n = (keys + sp - 1) / sp;
        n = std::min<int64_t>({n, most_parts, most});
        sp = ((keys + n - 1) / n + unit - 1) / unit * unit;
        *splits = (int)n;
        *span = (int)std::min<int64_t>(sp, INT32_MAX / 2);
    };
    if (only_tile) a.few_span = INT32_MAX / 2, a.few_splits = 1;
    else split(pairs, FEW_TARGET, JOIN_SPLITS, 128, FEW_MIN_SPAN, &a.few_span, &a.few_splits);
    if (only_few) a.tile_span = INT32_MAX / 2, a.tile_splits = 1;
    else split((int64_t)a.tiles * a.n_kv, TILE_TARGET, JOIN_SPLITS, 64, TILE_MIN_SPAN, &a.tile_span, &a.tile_splits);
    if (a.tile_splits > 1 && a.n_seq > 1 && a.n_seq <= 64) {
        a.tile_slots = std::max(a.tiles, (int)((a.few_rows ? MIXED_TARGET : TILE_TARGET) / a.n_kv));
        a.tile_splits = (int)std::min<int64_t>({(keys + TILE_MIN_SPAN - 1) / TILE_MIN_SPAN, most_parts, JOIN_SPLITS,
                                                std::max(2 * a.tile_splits, a.few_splits)});
    }
    a.part_splits = std::max(a.few_splits, a.tile_splits);
    // (join_kernel, behind split tiles, has TILE_PAIRS / FEW_PAIRS workgroups a tile)
    const int64_t tile_blocks = a.tile_slots ? a.tile_slots : (int64_t)a.tiles * a.tile_splits;
    const int64_t blocks = a.n_kv * std::max(tile_blocks + (only_tile ? 0 : (int64_t)a.n_seq * a.few_splits),
                                             a.tile_splits > 1 ? (int64_t)a.tiles * (TILE_PAIRS / FEW_PAIRS) : 0);
    if (blocks > MAX_BLOCKS)
        return api_fail(RDL_ERR_UNSUPPORTED, "%d sequences, %lld rows: %lld workgroups", a.n_seq, (long long)m, (long long)blocks);
    // f32 prompts whose keys several tiles read: split once
    const int hdp = a.hd <= 64 ? 64 : a.hd <= 128 ? 128 : 256, tk = a.hd <= 64 ? 64 : 32;  // Geo<Split, HD>
    const int64_t tiles = m / tk + a.n_seq;
    const size_t image_bytes = (size_t)tiles * a.n_kv * tk * hdp * 8, note_bytes = (size_t)tiles * a.n_kv * (sizeof(int4) + tk * sizeof(int2));
    const bool pre = !f16 && !a.kv.tables && only_tile && m * G >= SPLIT_MIN_TILES * TILE_PAIRS * a.n_seq &&
                     image_bytes <= SPLIT_BYTES;
    const size_t part_bytes = a.part_splits > 1 ? (size_t)m * a.n_heads * a.part_splits * (a.hd + 2) * sizeof(float) : 0;
    const size_t part_room = (part_bytes + 255) & ~(size_t)255;
    CallScratch work;
    if (part_bytes || pre) {
        const rdl_status st = call_scratch(s, part_room + (pre ? image_bytes + note_bytes : 0),
                                           part_bytes && a.few_rows ? (size_t)a.n_seq * a.n_kv : 0, &work);
        if (st != RDL_OK) return st;
        a.part = reinterpret_cast<float*>(work.p);
        a.part_ml = a.part + (size_t)m * a.n_heads * a.part_splits * a.hd;
        a.counters = work.counters;
    }
    hipError_t e;
    if (pre) {
        _Float16* images = reinterpret_cast<_Float16*>(reinterpret_cast<uint8_t*>(work.p) + part_room);
        int4* notes = reinterpret_cast<int4*>(reinterpret_cast<uint8_t*>(images) + image_bytes);
        a.images = images;
        a.notes = notes;
        int2* exps = reinterpret_cast<int2*>(notes + tiles * a.n_kv);
        a.exps = exps;
        auto go = a.hd <= 64 ? launch_split<64> : a.hd <= 96 ? launch_split<96> : a.hd <= 128 ? launch_split<128> : launch_split<256>;
        e = go(a, images, notes, exps, (int)tiles, s);
    } else {
        e = f16 ? launch_hd<_Float16>(a, s) : launch_hd<float>(a, s);
    }
    const rdl_status done = call_scratch_done(s, &work);
    HIP_TRY(e);
    return done == RDL_OK ? api_ok() : done;
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
    if (rows_overlap(q, q_stride * 4, n_heads * hd * 4, out, out_stride * 4, n_heads * hd * 4, m))
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
    a->group = (int)(n_heads / n_kv);
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
    if (rdl::rows_overlap(k_dev, k_stride * elem, width * elem, out_dev, out_stride * 4, n_heads * head_dim * 4, m) ||
        rdl::rows_overlap(v_dev, v_stride * elem, width * elem, out_dev, out_stride * 4, n_heads * head_dim * 4, m))
        return api_fail(RDL_ERR_INVALID_DATA, "out overlaps k or v");
    if ((st = rdl::check_position_stride(k_stride > v_stride ? k_stride : v_stride)) != RDL_OK) return st;
    a.kv = {k_dev, v_dev, (int64_t)k_stride, (int64_t)v_stride, (int64_t)head_dim, 0, nullptr, 0, 0, 0};
    return rdl::run(a, kv_dtype == RDL_DTYPE_F16, max_rows, max_rows, (hipStream_t)stream);
}

}  // extern "C"
