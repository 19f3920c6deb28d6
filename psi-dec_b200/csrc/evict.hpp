// Launch interface of the eviction kernels (evict.cu).
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

#include "kernels.cuh"

namespace psi {

constexpr uint32_t kEvictBatch = 128;  // requests of one launch: their sizes travel as launch arguments

struct EvictRequest {
    uint32_t src, dst, length, keep;
};

struct EvictParams {
    PageGeometry geo;
    const float* weights;   // [slots][Hkv][stride]
    float* weights_out;     // the same shape, may be `weights`
    uint64_t stride;
    uint32_t* kept;         // [requests][Hkv][kept_stride]
    uint64_t kept_stride;
    uint32_t recent;
    uint32_t num_reqs;
    uint32_t unit_bytes;    // 16, 4 or 2: what a row's bytes and the arena's address are multiples of
    uint32_t in_place;      // move launch: requests whose dst is their src (1) or the others (0)
    EvictRequest reqs[kEvictBatch];
};

cudaError_t launch_evict_select(const EvictParams& p, uint32_t sms, cudaStream_t stream);
// Requests that keep their slot and requests that move to another one are two launches.
cudaError_t launch_evict_move(const EvictParams& p, uint32_t sms, cudaStream_t stream);

}  // namespace psi
