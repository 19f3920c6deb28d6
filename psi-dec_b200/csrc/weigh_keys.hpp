// Launch interface of the key-weight kernels (weigh_keys.cu) and the shapes that host and device agree on.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

#include "kernels.cuh"

namespace psi {

constexpr uint32_t kWeighBlock = 128;    // rows or keys of one block of the long-run kernels
constexpr uint32_t kWeighSpan = 4;       // key blocks of one second-pass item of theirs
constexpr uint32_t kWeighAnyRows = 16;   // rows and keys of one block of the CUDA-core kernels
constexpr uint32_t kWeighAnyKeys = 64;
constexpr uint32_t kWeighShortRows = 16; // query rows of a KV head up to which a run goes to the short-run kernel
constexpr uint32_t kWeighTile = 32;      // keys of one unit of the short-run kernel's shares
constexpr uint32_t kWeighPieceKeys = 1024;
constexpr uint32_t kWeighMaxPieces = 16;

// A request with tokens as the kernels see it.  Short runs first, then one entry that ends their prefix sums, then the long
// runs and one entry that ends theirs.
struct WeighRequest {
    uint32_t slot, first_pos, q_len, flat_begin;
    uint32_t keys;   // first_pos + q_len
    uint32_t cu0;    // short: tiles before this request's; long: first-pass items before
    uint32_t cu1;    // long: second-pass items before
    uint32_t unit0;  // long: (KV head, row block) units before
};
constexpr uint64_t kWeighRequestWords = sizeof(WeighRequest) / sizeof(uint32_t);

// A long run's keys are cut into pieces of 1,024 or more, at most sixteen, so that the scratch does not grow with the context.
__host__ __device__ inline uint32_t weigh_pieces(uint32_t keys) {
    const uint32_t n = keys / kWeighPieceKeys + (keys % kWeighPieceKeys != 0 ? 1u : 0u);
    return n < kWeighMaxPieces ? n : kWeighMaxPieces;
}
// Keys of one piece, in whole blocks.
__host__ __device__ inline uint32_t weigh_piece_keys(uint32_t keys, uint32_t pieces) {
    const uint32_t each = keys / pieces + (keys % pieces != 0 ? 1u : 0u);
    return (each + kWeighBlock - 1) / kWeighBlock * kWeighBlock;  // (a multiple of kWeighAnyKeys as well)
}

// Second-pass items of one KV head: spans of key blocks on the tensor cores, blocks of 64 keys on the CUDA cores.
inline uint64_t weigh_sum_items(uint32_t keys, bool tensor) {
    const uint64_t each = tensor ? kWeighBlock * kWeighSpan : kWeighAnyKeys;
    return (keys + each - 1) / each;
}

inline bool weigh_on_tensor_cores(uint32_t dtype, uint32_t head_dim) { return dtype != PSI_DTYPE_F32 && head_dim % 8 == 0; }

struct WeighParams {
    PageGeometry geo;
    const void* q;                // [T][Hq][D]
    float* weights;               // [slots][Hkv][stride]
    uint64_t stride;
    const WeighRequest* reqs;
    const uint32_t* scalars;
    uint32_t short_count, short_tiles;  // requests and tiles of the short runs, or ~0: as the device block says (captured launches)
    float2* norms;                // [max_tokens][Hq] log2-domain maximum and 1 / sum of each row; (inf, 0) for a row that adds nothing
    float2* partials;             // (m, l) by segment of the short runs, then by item of the long ones
    uint64_t long_partials_at;
    uint32_t* counters;           // arrivals by unit, zero between launches: short runs, then long ones
    uint64_t long_counters_at;
    float* scores;                // short runs: [tiles][4][score_rows][8]
    uint32_t score_rows;          // most query rows of a short run
    uint32_t group;               // q heads of a KV head
    uint32_t num_q_heads;
    uint32_t dtype;
    float scale_log2;
    __device__ __forceinline__ const WeighRequest* long_reqs() const { return reqs + scalars[kScalarWeighShort] + 1; }
    __device__ __forceinline__ float2* long_partials() const { return partials + long_partials_at; }
    __device__ __forceinline__ uint32_t* long_counters() const { return counters + long_counters_at; }
};

enum class WeighPass { kShortStatsScores, kShortStats, kShortSumScores, kShortSumAgain, kLongStats, kLongSum };
// The long runs' passes on the tcgen05 tensor cores: any head_dim that is a multiple of eight, up to 256.
cudaError_t launch_weigh_umma(const WeighParams& p, bool stats, uint32_t ctas, cudaStream_t stream);
cudaError_t launch_weigh(const WeighParams& p, WeighPass pass, uint32_t ctas, cudaStream_t stream);

}  // namespace psi
