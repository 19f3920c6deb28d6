// Launch interface of the linear-attention kernels (linear_attend.cu).
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

#include "psi_cuda.h"

namespace psi {

constexpr uint32_t kLinearMaxDim = 256;
constexpr uint32_t kLinearChunk = 64;  // tokens of one chunk of the chunked form
// Of each head: lambda^0 .. lambda^64, rounded from 64 bits; what the rounding of lambda^64 and of lambda left.
constexpr uint32_t kLinearChunkLow = kLinearChunk + 1, kLinearStepLow = kLinearChunk + 2, kLinearDecays = kLinearChunk + 4;

// Scalars of the device block: requests of the recurrent form, runs of the chunked form, those of them whose state is carried on, and
// requests in several pieces.
enum LinearScalar : uint32_t { kLinearNumSteps = 0, kLinearNumRuns = 1, kLinearNumCarries = 2, kLinearNumScans = 3, kLinearScalarCount = 8 };

// A request of the recurrent form.
struct LinearRequest {
    uint32_t src, dst, fresh, q_len, flat_begin;
    uint32_t pad[3];
};

// A run of tokens of the chunked form: a request, or a piece of one.
constexpr uint32_t kLinearNoCarry = 0xFFFFFFFFu;
struct LinearRun {
    uint32_t src, dst, fresh;  // the request's slots; fresh: it starts from a zero state
    uint32_t keep;             // the state after the run goes to dst
    uint32_t flat_begin, tokens;
    uint32_t carry_in;         // the state before the run, or kLinearNoCarry: src's
    uint32_t carry_out;        // state pass: where the run's own part of the state goes
};
// A request of the chunked form in several pieces: `pieces` carries from `carry` on.  The state pass leaves each piece's own gain in the
// carry behind the piece's; the scan makes them the states before the pieces.
struct LinearScan {
    uint32_t src, fresh, carry, pieces, piece_chunks;  // every piece but the last has piece_chunks whole chunks
    uint32_t pad[3];
};
static_assert(sizeof(LinearScan) == sizeof(LinearRequest), "one array of the device block holds all");
constexpr uint64_t kLinearRequestWords = sizeof(LinearRequest) / sizeof(uint32_t);
static_assert(sizeof(LinearRun) == sizeof(LinearRequest), "one array of the device block holds both");

struct LinearParams {
    const uint32_t* scalars;
    const LinearRequest* reqs;  // the recurrent form's, then the runs, then the scans
    const float* decays;     // [Hv][kLinearDecays] of the layer
    float* states;           // [slots][layers][Hv][Dk][Dv]
    float* carries;          // [carry][Hv][Dk][Dv]
    const void* q;           // [T][Hk][Dk]
    const void* k;           // [T][Hk][Dk]
    const void* v;           // [T][Hv][Dv]
    void* out;               // [T][Hv][Dv]
    uint32_t* status;        // the word a bounded device-side wait writes PSI_ERR_TIMEOUT to
    uint32_t layer, num_layers;
    uint32_t num_k_heads, num_v_heads, key_dim, value_dim;
    uint32_t dtype;
    uint32_t aligned;        // chunked form: q, k and v on 16-byte boundaries
    uint32_t num_tokens;     // rows of q, k and v that may be read
    float scale;
#ifdef __CUDACC__
    __device__ __forceinline__ const LinearRun* runs() const { return reinterpret_cast<const LinearRun*>(reqs + scalars[kLinearNumSteps]); }
    __device__ __forceinline__ const LinearScan* scans() const {
        return reinterpret_cast<const LinearScan*>(reqs + scalars[kLinearNumSteps] + scalars[kLinearNumRuns]);
    }
    __device__ __forceinline__ float* state_of(uint32_t slot, uint32_t head) const {
        return states + ((uint64_t(slot) * num_layers + layer) * num_v_heads + head) * key_dim * value_dim;
    }
    __device__ __forceinline__ float* carry_of(uint32_t carry, uint32_t head) const {
        return carries + (uint64_t(carry) * num_v_heads + head) * key_dim * value_dim;
    }
#endif
};

// The recurrent form, on `ctas` CTAs that take items (requests x heads x column slices) in turn; their count comes from the device.
uint32_t linear_step_slices(uint32_t value_dim);
// Its CTAs on an SM: what their registers leave room for.
__host__ __device__ constexpr uint32_t linear_step_resident(uint32_t key_dim) { return key_dim <= 64 ? 9 : key_dim <= 128 ? 7 : 4; }
cudaError_t launch_linear_step(const LinearParams& p, uint32_t ctas, cudaStream_t stream);
// The chunked form: 16-bit types, key_dim and value_dim up to 128.
bool linear_chunk_supported(uint32_t dtype, uint32_t key_dim, uint32_t value_dim);
cudaError_t launch_linear_scan(const LinearParams& p, cudaStream_t stream);
cudaError_t launch_linear_chunk(const LinearParams& p, bool state_only, uint32_t ctas, cudaStream_t stream);

}  // namespace psi
