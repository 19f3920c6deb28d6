// Launch interface of the linear-attention kernels (linear_attend.cu).
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

#include "psi_cuda.h"

namespace psi {

constexpr uint32_t kLinearMaxDim = 256;
constexpr uint32_t kLinearDecays = 3;  // of each head: the decay in two f32 parts, and its logarithm

// Scalars of the device block.
enum LinearScalar : uint32_t { kLinearNumSteps = 0, kLinearScalarCount = 8 };

// A request with tokens as the kernels see it.
struct LinearRequest {
    uint32_t src, dst, fresh, q_len, flat_begin;
    uint32_t pad[3];
};
constexpr uint64_t kLinearRequestWords = sizeof(LinearRequest) / sizeof(uint32_t);

struct LinearParams {
    const uint32_t* scalars;
    const LinearRequest* reqs;
    const float* decays;     // [Hv][kLinearDecays] of the layer
    float* states;           // [slots][layers][Hv][Dk][Dv]
    const void* q;           // [T][Hk][Dk]
    const void* k;           // [T][Hk][Dk]
    const void* v;           // [T][Hv][Dv]
    void* out;               // [T][Hv][Dv]
    uint32_t layer, num_layers;
    uint32_t num_k_heads, num_v_heads, key_dim, value_dim;
    uint32_t dtype;
    float scale;
};

// The recurrent form; `most` items (requests x heads x column slices) at most, the launch's own count comes from the device.
uint32_t linear_step_slices(uint32_t value_dim);
cudaError_t launch_linear_step(const LinearParams& p, uint32_t ctas, cudaStream_t stream);

}  // namespace psi
