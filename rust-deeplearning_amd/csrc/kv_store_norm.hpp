// kv_store_norm.hpp -- the launch behind rdl_kv_store_norm_dev, and behind
// rdl_kv_store_dev over a 4-bit pool (kv_plan.hip checks the arguments).
#pragma once

#include "kv_pool.hpp"

namespace rdl {

struct StoreNormArgs {
    PoolView pool;
    int64_t m;
    const float* q;
    int64_t q_stride;
    float* q_out;
    int64_t q_out_stride;
    int n_heads;
    const float *k, *v;
    int64_t k_stride, v_stride;
    const float *q_gamma, *k_gamma;  // NULL: no norm
    float eps;
    const int32_t *positions, *slots;
    const float *cos_t, *sin_t;
    int64_t n_positions;
    double share;  // 1 / head_dim (launch_store_norm sets it)
};
hipError_t launch_store_norm(StoreNormArgs a, hipStream_t s);

}  // namespace rdl
