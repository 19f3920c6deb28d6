// Launch interface of the key-weight kernels (weigh_keys.cu) and the shapes that host and device agree on.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

#include "kernels.cuh"

namespace psi {

constexpr uint32_t kWeighBlock = 128;    // rows or keys of one block of the long-run kernels
constexpr uint32_t kWeighSpan = 4;       // key blocks of one second-pass item of theirs, where its rows are cut into parts
constexpr uint32_t kWeighAnyRows = 32;   // rows and keys of one block of the CUDA-core kernels
constexpr uint32_t kWeighAnyKeys = 64;
// Query rows of a KV head up to which a run goes to the short-run kernel, whose products have 16 rows.  2 KV heads x 256, 32 requests of
// 1,024 to 8,192 keys, 16 rows: 55 us there and 99 on the long-run kernel, which also takes 99 for 24.
constexpr uint32_t kWeighShortRows = 16;
constexpr uint32_t kWeighTile = 32;      // keys of one unit of the short-run kernel's shares
constexpr uint32_t kWeighPieceBlocks = 8, kWeighMaxPieces = 16;        // of the first pass on the tensor cores, replayed
constexpr uint32_t kWeighAnyPieceKeys = 256, kWeighAnyMaxPieces = 64;  // and on the CUDA cores
// CTAs of the long-run kernels side by side: one for each SM of a B200 on the tensor cores, two on the CUDA cores.
__host__ __device__ constexpr uint32_t weigh_wave(bool tensor) { return tensor ? 148 : 296; }

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

// The entry that ends the long runs carries, for the tensor cores, the key blocks of a first-pass piece (slot) and of a second-pass
// span (first_pos); plan_weigh chooses them.
__host__ __device__ inline uint32_t weigh_blocks(uint32_t keys) { return keys / kWeighBlock + (keys % kWeighBlock != 0 ? 1u : 0u); }
__host__ __device__ inline uint32_t weigh_cut(uint32_t keys, uint32_t blocks) { return (weigh_blocks(keys) + blocks - 1) / blocks; }

// CUDA cores: a long run's keys are cut into a bounded number of pieces, so that the scratch does not grow with the context.
__host__ __device__ inline uint32_t weigh_any_pieces(uint32_t keys) {
    const uint32_t n = keys / kWeighAnyPieceKeys + (keys % kWeighAnyPieceKeys != 0 ? 1u : 0u);
    return n < kWeighAnyMaxPieces ? n : kWeighAnyMaxPieces;
}
// Keys of one piece, in whole blocks.
__host__ __device__ inline uint32_t weigh_any_piece_keys(uint32_t keys, uint32_t pieces) {
    const uint32_t each = keys / pieces + (keys % pieces != 0 ? 1u : 0u);
    return (each + kWeighAnyKeys - 1) / kWeighAnyKeys * kWeighAnyKeys;
}
__host__ __device__ inline uint32_t weigh_any_spans(uint32_t keys) { return keys / kWeighAnyKeys + (keys % kWeighAnyKeys != 0 ? 1u : 0u); }

// Into how many parts a run's rows are cut in the second pass, each an item of its own whose sums the last one adds up: where the spans
// of all KV heads are fewer than the CTAs of a wave, and a part has two row blocks left.  4/1 heads x 128, bf16, in parts and whole: 500
// tokens of 500 keys 42 and 61 us, 1,000 of 4,000 49 and 107, 2,000 of 2,000 50 and 182.
__host__ __device__ inline uint32_t weigh_row_parts(uint32_t rows, uint32_t keys, uint32_t heads, bool tensor) {
    const uint64_t spans = uint64_t(tensor ? weigh_cut(keys, kWeighSpan) : weigh_any_spans(keys)) * heads;
    if (spans >= weigh_wave(tensor)) return 1;
    const uint32_t least = tensor ? 2 * kWeighBlock : 2 * kWeighAnyRows;
    const uint32_t wanted = uint32_t((weigh_wave(tensor) + spans - 1) / spans), most = rows / least > 0 ? rows / least : 1;
    return wanted < most ? wanted : most;
}
// Row blocks of one part.
__host__ __device__ inline uint32_t weigh_part_blocks(uint32_t rows, uint32_t parts, bool tensor) {
    const uint32_t block = tensor ? kWeighBlock : kWeighAnyRows, blocks = (rows + block - 1) / block;
    return (blocks + parts - 1) / parts;
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
    float* sums;                  // second pass of long runs: [item][keys of a span], where rows are cut into parts
    uint32_t split_rows;          // they may be (not in captured launches, whose scratch does not follow the batch)
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
