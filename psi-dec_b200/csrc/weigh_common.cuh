// What the key-weight kernels share: where requests, rows and keys lie, and the numbers of a row's softmax.
#pragma once

#include "mma_common.cuh"
#include "umma_common.cuh"
#include "weigh_keys.hpp"

namespace psi {

constexpr float kInf = INFINITY;

// The request whose work holds `index`: the last one whose prefix (`which` 0: cu0, 1: cu1) is at or below it.  By a converged warp,
// 32 requests at a time: a search that halves would wait for a load in each of its steps.
template <int kWhich>
__device__ __forceinline__ uint32_t find_request(const WeighRequest* reqs, uint32_t count, uint32_t index) {
    if (count == 1) return 0;
    const uint32_t lane = threadIdx.x & 31u;
    uint32_t below = 0;
#pragma unroll 4
    for (uint32_t base = 0; base < count; base += 32) {
        const uint32_t r = base + lane;
        const uint32_t prefix = r < count ? (kWhich == 0 ? reqs[r].cu0 : reqs[r].cu1) : 0xFFFFFFFFu;
        below += __popc(__ballot_sync(0xFFFFFFFFu, r < count && prefix <= index));
    }
    return below - 1;
}

// (maximum, sum) of a row's scores in the log2 domain; an empty one is (-inf, 0).
struct Stat {
    float m, l;
    __device__ __forceinline__ void join(float m2, float l2) {
        const float top = fmaxf(m, m2);
        const float base = top == -kInf ? 0.0f : top;
        l = l * exp2f(m - base) + l2 * exp2f(m2 - base);
        m = top;
    }
    // What the second pass takes of the row: (maximum, 1 / sum), or (inf, 0) for a row that adds nothing.
    __device__ __forceinline__ float2 norm() const {
        return l > 0.0f && l < kInf && fabsf(m) < kInf ? make_float2(m, 1.0f / l) : make_float2(kInf, 0.0f);
    }
};

// The weight of a key from its product with the query row.
__device__ __forceinline__ float weight_of(float product, float scale_log2, float2 norm) {
    return norm.y > 0.0f ? fast_exp2(fmaf(product, scale_log2, -norm.x)) * norm.y : 0.0f;
}

// Query row r of a request and KV head as (flat token, head) row of q.
__device__ __forceinline__ uint64_t query_row(const WeighParams& p, const WeighRequest& rq, uint32_t head, uint32_t r) {
    return uint64_t(rq.flat_begin + r / p.group) * p.num_q_heads + head * p.group + r % p.group;
}

// Keys that row r sees.
__device__ __forceinline__ uint32_t row_limit(const WeighParams& p, const WeighRequest& rq, uint32_t r) {
    return rq.first_pos + r / p.group + 1;
}

__device__ __forceinline__ float* weight_row(const WeighParams& p, const WeighRequest& rq, uint32_t head) {
    return p.weights + (uint64_t(rq.slot) * p.geo.num_kv_heads + head) * p.stride;
}

}  // namespace psi
