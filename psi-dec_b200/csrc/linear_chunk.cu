// Linear attention over prompts on the 5th-generation tensor cores (tcgen05 / TMEM), 64 tokens at a time.
//
// With S the state before a chunk, lambda the head's decay and i, j tokens of the chunk (n of them):
//
//   o_i = scale (lambda^(i+1) q_i S + sum_{j<=i} lambda^(i-j) (q_i . k_j) v_j)
//   S'  = lambda^n S + sum_j lambda^(n-1-j) k_j^T v_j
//
// One CTA takes one value head of one request and goes through its chunks in order.  The products stand so that a thread owns one
// column v of the state and of the output (accumulator lane = v), and everything that differs by v stays inside it:
//
//   scores   [i][j] = Q K^T                    shared memory x shared memory; lanes 64-127 are not used
//   inner^T  [v][i] = V^T P^T                  V as it landed, P = lambda^(i-j) scores in shared memory, two 16-bit parts
//   outer^T  [v][i] = S^T Q^T                  S^T in TMEM, two 16-bit parts; lambda^(i+1) is applied in f32 afterwards
//   gain^T   [v][k] = (lambda^(n-1-j) V)^T K   the weighted V in 16-bit parts: bf16 three (24 bits, the lowest part in shared memory, the
//                                              others in TMEM), f16 two (22 bits)
//
// Every part is a product of its own into the same accumulator, the lowest part first; in f16 the low part is held 2^11 times as large.
// Two parts of P and S, the first towards zero, are off by 2^-15 of a value in bf16 and 2^-21 in f16, so that an output is off by its own
// rounding (one part alone: 1.4 times that; 8,192 tokens 142 us for 154).  In f16 each row of P and each column of S is scaled by a power of two first, so that
// nothing leaves f16's range; the weighted V is not scaled: below 2^-14 its parts have an absolute step of 2^-35, so that
// a state which only such values make has fewer bits than 22.  The state itself stays in f32 registers; a chunk's gain is
// added to it after an accumulation of its own, since the tensor cores' accumulation truncates.
//
// Warps 0-15: four threads for each v, a quarter of the state each: weighted V (by ldmatrix, whose fragments are what tcgen05.st takes as
// 16 x 128 bits), the state and its 16-bit parts.  Warps 16-19: outputs, in the fragments of 16 x 256 bits, which stmatrix turns into
// rows.  Warps 20 and 21: P, a row per thread.  Warp 22 issues every product but the gain, the scores a chunk ahead, so that P is made
// under the products of the chunk before.  Warp 23 brings Q, K and V into a ring of three chunks by TMA (by plain loads where a buffer
// is off its 16-byte boundaries; rows that the last box brings from behind a run are cleared by the state threads) and issues
// the gains, the longest chain from chunk to chunk, which wait for the state threads alone.  The loops are kept short: unrolled, the
// roles' code together ran out of the instruction cache and took 1.5 times as long.
// Bound by the chain of one head's chunks at 128 x 128, 2.2 us each in bf16 and 2.6 in f16, of which the state threads work for
// nearly all (without the second parts' products it is as long, without their arithmetic 6 % shorter).  One prompt of 8,192 tokens, 32
// heads, f16: 154 us in pieces (42 of bytes, 10 of products), 337 whole; three prompts of 926 to 2,185 tokens, 16/32 heads, bf16: 83 us.
// Every hand-off is an mbarrier, every wait is bounded and reports PSI_ERR_TIMEOUT through the status word, and TMEM is freed on
// every path.
#include <cstddef>

#include "launch_util.hpp"
#include "linear_attend.hpp"
#include "mma_common.cuh"
#include "umma_common.cuh"

namespace psi {

namespace {

constexpr uint32_t kC = kLinearChunk, kStages = 3;
constexpr uint32_t kGroups = 4;  // threads of a state column
constexpr uint32_t kStateThreads = kGroups * kUmmaM, kOutThreads = kUmmaM, kGroupTokens = kC / kGroups;
constexpr uint32_t kWarpOut = kStateThreads / 32, kWarpP = kWarpOut + 4, kWarpMma = kWarpP + 2, kWarpGain = kWarpMma + 1;
constexpr uint32_t kChunkThreads = (kWarpGain + 1) * 32;
constexpr uint32_t kTileBlock = kC * 128;  // bytes of 64 rows x 64 elements

// TMEM columns
constexpr uint32_t kColScores = 0, kColInner = 64, kColOuter = 128, kColGain = 192, kColState = 320, kColStateLow = 384, kColParts = 448;
constexpr uint32_t kPartColumns = kC / 2;
static_assert(kColParts + 2 * kPartColumns <= 512, "one TMEM allocation");

// Barriers: ring slots full and done by slot, the others one each, their phase the chunk's.  A parity wait cannot tell two
// completions from none: a thread waits for a phase only where the next one cannot complete without it.
constexpr uint32_t kBarFull = 0, kBarDone = kStages, kBarScores = 2 * kStages, kBarP = kBarScores + 1, kBarParts = kBarP + 1,
                   kBarGain = kBarParts + 1, kBarGainRead = kBarGain + 1, kBarState = kBarGainRead + 1, kBarOut = kBarState + 1, kNumBars = kBarOut + 1;

struct ChunkShared {
    uint64_t bars[kNumBars];
    uint32_t tmem_base, abort;
    __align__(16) float fall[kC];             // lambda^(63 - j)
    __align__(16) float last_fall[kC];        // the same of the last chunk: lambda^(n - 1 - j), 0 behind the run
    __align__(16) float rise[kC];             // lambda^(i + 1)
    // scale lambda^(63 - x), then zeros, four times, each copy an entry further on, so that a row of P reads 16 bytes at a time from
    // its own start
    __align__(16) float lag[4][2 * kC + 8];  // (the eight lanes of one phase of a read: distinct banks)
    // By chunk; P may be two chunks ahead of the outputs, the weighted V three.
    __align__(16) float p_scale[4][kC];       // f16: what the rows of P were divided by
    float column_up[4][kUmmaM];               // f16: what the columns of the state's parts were divided by
    float column_max[2][kGroups][kUmmaM];     // f16: largest magnitude of each part of a state column
    uint32_t bad_from[4][kUmmaM];             // first token of the chunk whose V is not finite in this column (64: none)
    uint32_t any_bad;                         // the item has met such a value
};

static_assert(offsetof(ChunkShared, fall) % 16 == 0 && offsetof(ChunkShared, rise) % 16 == 0 && offsetof(ChunkShared, lag) % 16 == 0 &&
                  offsetof(ChunkShared, p_scale) % 16 == 0,
              "these are read 16 bytes at a time");

template <typename T>
constexpr bool kIsHalf = std::is_same<T, __half>::value;

// The power of two that brings a largest magnitude to [2^10, 2^11), and its inverse.
__device__ __forceinline__ void range_scale(float largest, float& down, float& up) {
    int e = int(__float_as_uint(largest) >> 23) - 127 - 10;  // largest >= 0
    if (!(largest > 0.0f) || !(largest < INFINITY)) e = 0;
    e = e < -100 ? -100 : e > 100 ? 100 : e;
    down = __uint_as_float(uint32_t(127 - e) << 23);
    up = __uint_as_float(uint32_t(127 + e) << 23);
}

// x - y of two values, exact where y are x's leading bits.
__device__ __forceinline__ uint64_t rest_of(uint64_t x, float2 y) { return fma_f32x2(pack_f32x2(y.x, y.y), pack_f32x2(-1.0f, -1.0f), x); }

// Packs two values as 16-bit parts: bf16 in three (the first two towards zero, exact rests), f16 in two, the second 2^11 times as large.
template <typename T>
__device__ __forceinline__ void split_parts(uint64_t x, uint32_t (&part)[3]) {
    float2 v = unpack_f32x2(x);
    if constexpr (kIsHalf<T>) {
        part[0] = Mma<T>::pack(v.x, v.y);
        v = unpack_f32x2(mul_f32x2(rest_of(x, Mma<T>::unpack(part[0])), pack_f32x2(2048.0f, 2048.0f)));
        part[1] = Mma<T>::pack(v.x, v.y);
        part[2] = 0;
    } else {
        part[0] = Mma<T>::pack_down(v.x, v.y);
        x = rest_of(x, Mma<T>::unpack(part[0]));
        v = unpack_f32x2(x);
        part[1] = Mma<T>::pack_down(v.x, v.y);
        v = unpack_f32x2(rest_of(x, Mma<T>::unpack(part[1])));
        part[2] = Mma<T>::pack(v.x, v.y);
    }
}

// The same in two parts, the first towards zero: f16 by its leading bits, without a conversion back.  (A value below f16's normal range,
// 2^-24 of the largest beside it and less, loses what its first part rounds.)
template <typename T>
__device__ __forceinline__ void split_two(uint64_t x, uint32_t& high, uint32_t& low) {
    float2 v = unpack_f32x2(x);
    if constexpr (kIsHalf<T>) {
        const float2 lead = make_float2(__uint_as_float(__float_as_uint(v.x) & 0xFFFFE000u), __uint_as_float(__float_as_uint(v.y) & 0xFFFFE000u));
        high = Mma<T>::pack(lead.x, lead.y);
        v = unpack_f32x2(mul_f32x2(rest_of(x, lead), pack_f32x2(2048.0f, 2048.0f)));
    } else {
        high = Mma<T>::pack_down(v.x, v.y);
        v = unpack_f32x2(rest_of(x, Mma<T>::unpack(high)));
    }
    low = Mma<T>::pack(v.x, v.y);
}

// Byte offset of the 16-byte chunk `chunk` of row `row` in a tile of 64 rows: 64-element blocks one after another, each in the
// 128-byte swizzle.
__device__ __forceinline__ uint32_t tile_offset(uint32_t row, uint32_t chunk) {
    return (chunk >> 3) * kTileBlock + row * 128 + (((chunk ^ row) & 7u) << 4);
}

// 64 rows x 64 elements of one head, from `row` and element `x` on; zeros beyond the head's elements and the batch's rows.
__device__ __forceinline__ void tma_load_rows(uint32_t dst, const CUtensorMap* map, uint32_t bar, uint32_t x, uint32_t row, uint32_t head) {
    asm volatile(
        "{\n\t.reg .pred e;\n\telect.sync _|e, 0xFFFFFFFF;\n\t"
        "@e cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];\n\t}\n" ::"r"(dst),
        "l"(map), "r"(bar), "r"(x), "r"(row), "r"(head)
        : "memory");
}

__device__ __forceinline__ void tmem_store8_bits(uint32_t taddr, const uint32_t (&v)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};\n" ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]),
                 "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
                 : "memory");
}

// 16 lanes x 8 columns as fragments: register 2 b + h of lane t is row t / 4 + 8 h, column 4 b + t % 4.
__device__ __forceinline__ void tmem_store_16x128_x2(uint32_t taddr, const uint32_t (&v)[4]) {
    asm volatile("tcgen05.st.sync.aligned.16x128b.x2.b32 [%0], {%1, %2, %3, %4};\n" ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]) : "memory");
}

// 16 lanes x 32 columns as fragments: registers 4 b + 2 h + {0, 1} of lane t are row t / 4 + 8 h, columns 8 b + 2 (t % 4) + {0, 1}.
// Two of them, both under way before the wait.
__device__ __forceinline__ void tmem_load_16x256_x4(uint32_t taddr_a, uint32_t taddr_b, uint64_t (&a)[8], uint64_t (&b)[8]) {
    uint32_t r[16], q[16];
    asm volatile("tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
                   "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(taddr_a));
    asm volatile("tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n"
                 : "=r"(q[0]), "=r"(q[1]), "=r"(q[2]), "=r"(q[3]), "=r"(q[4]), "=r"(q[5]), "=r"(q[6]), "=r"(q[7]), "=r"(q[8]), "=r"(q[9]), "=r"(q[10]),
                   "=r"(q[11]), "=r"(q[12]), "=r"(q[13]), "=r"(q[14]), "=r"(q[15])
                 : "r"(taddr_b));
    asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory");
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        a[i] = pack_f32x2(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1]));
        b[i] = pack_f32x2(__uint_as_float(q[2 * i]), __uint_as_float(q[2 * i + 1]));
    }
}

__device__ __forceinline__ void stmatrix_x4_trans(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};\n" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

__device__ __forceinline__ void stmatrix_x4(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("stmatrix.sync.aligned.m8n8.x4.shared.b16 [%0], {%1, %2, %3, %4};\n" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

__device__ __forceinline__ void st_shared16(uint32_t addr, const uint32_t (&v)[4]) {
    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};\n" ::"r"(addr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]) : "memory");
}

__device__ __forceinline__ void st_shared_zero16(uint32_t addr) {
    asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};\n" ::"r"(addr), "r"(0u) : "memory");
}

template <typename T>
__device__ __forceinline__ bool not_finite_bits(uint16_t bits) {
    constexpr uint32_t kExponent = kIsHalf<T> ? 0x7C00u : 0x7F80u;
    return (bits & kExponent) == kExponent;
}

// DK: key_dim rounded up to 64 or 128.  kStateOnly: the run's state from zero, without outputs.
template <typename T, uint32_t DK, bool kStateOnly>
__global__ void __launch_bounds__(kChunkThreads, 1)
    linear_chunk_kernel(const LinearParams p, const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap k_map,
                        const __grid_constant__ CUtensorMap v_map) {
    constexpr uint32_t kBlocksK = DK / 64;
    constexpr uint32_t kQBytes = kBlocksK * kTileBlock, kVBytes = 2 * kTileBlock, kStageBytes = 2 * kQBytes + kVBytes;
    constexpr uint32_t kParts = kIsHalf<T> ? 2 : 3;
    constexpr uint32_t kRows = DK / kGroups;  // state rows of one thread
    __shared__ ChunkShared shared;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u;
    const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t smem_p = smem_base + kStages * kStageBytes, smem_out = smem_p + 4 * kTileBlock, smem_low = smem_out + 2 * kTileBlock;
    const uint32_t bar0 = smem_u32(shared.bars);
    const auto bar = [&](uint32_t which) { return bar0 + which * 8u; };
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&shared.tmem_base)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (tid == 0) {
        for (uint32_t b = 0; b < kNumBars; ++b)
            mbar_init(bar(b), b == kBarP ? 64 : b == kBarOut ? kOutThreads : b == kBarParts || b == kBarGainRead || b == kBarState ? kStateThreads : 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        shared.abort = 0;
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = shared.tmem_base;
    await_previous_kernel();
    const auto wait = [&](uint32_t which, uint32_t phase) {
        if (mbar_try(bar(which), phase & 1u)) return;
        if (*reinterpret_cast<volatile uint32_t*>(&shared.abort) == 0 && !mbar_wait(bar(which), phase & 1u)) {
            *reinterpret_cast<volatile uint32_t*>(&shared.abort) = 1;
            if (p.status != nullptr) atomicExch(p.status, uint32_t(PSI_ERR_TIMEOUT));
        }
    };
    const LinearRun* runs = p.runs();
    const uint32_t total = p.scalars[kStateOnly ? kLinearNumCarries : kLinearNumRuns] * p.num_v_heads;
    const uint32_t share = p.num_v_heads / p.num_k_heads;
    // Work: item = (run, value head).  A state pass takes the runs that another piece of their request follows; they come first.
    uint32_t done_chunks = 0;  // of the items before, the same count in every role
    if (warp == kWarpMma) {
        // ================================ scores, inner and outer products (converged warp) ===============================
        const uint32_t id_rows = umma_idesc<T>(kC, false), id_inner = umma_idesc<T>(kC, false, true);
        const auto stage_of = [&](uint32_t g) { return smem_base + g % kStages * kStageBytes; };
        // K-major operands: 8-row groups 1 KiB apart, 64-element blocks of the row 8 KiB; MN-major ones are the same memory the other
        // way round, two groups a step
        const auto row_step = [](uint32_t ks) { return ((ks >> 2) * kTileBlock + (ks & 3) * 32) / 16; };
        for (uint32_t item = blockIdx.x; item < total; item += gridDim.x) {
            const uint32_t chunks = (runs[item / p.num_v_heads].tokens + kC - 1) / kC;
            if constexpr (!kStateOnly) {
#pragma unroll 1
                for (uint32_t c = 0; c <= chunks; ++c) {
                    const uint32_t g = done_chunks + c;  // the scores run a chunk ahead of the rest
                    if (c > 0) wait(kBarP, g - 1);       // the scores before have been read, P of the chunk before is there
                    if (c < chunks) {
                        wait(kBarFull + g % kStages, g / kStages);
                        tc_fence_after();
                        const uint64_t q_rows = umma_desc(stage_of(g), 16, 1024), k_rows = umma_desc(stage_of(g) + kQBytes, 16, 1024);
                        if (elect_one()) {
#pragma unroll
                            for (uint32_t ks = 0; ks < DK / 16; ++ks) umma_ss(tmem + kColScores, q_rows + row_step(ks), k_rows + row_step(ks), id_rows, ks);
                            umma_commit_one(bar(kBarScores));
                        }
                        __syncwarp();
                    }
                    if (c > 0) {
                        const uint32_t h = g - 1;
                        wait(kBarState, h);
                        if (h > 0) wait(kBarOut, h - 1);
                        tc_fence_after();
                        const uint64_t q_rows = umma_desc(stage_of(h), 16, 1024), p_rows = umma_desc(smem_p + (h & 1u) * (2 * kTileBlock), 16, 1024),
                                       v_cols = umma_desc(stage_of(h) + 2 * kQBytes, kTileBlock, 1024);
                        if (elect_one()) {
#pragma unroll
                            for (uint32_t ks = 0; ks < DK / 16; ++ks) umma_ts(tmem + kColOuter, tmem + kColStateLow + ks * 8, q_rows + row_step(ks), id_rows, ks);
                            if (kIsHalf<T>) umma_ts_down11(tmem + kColOuter, tmem + kColState, q_rows, id_rows);
                            else umma_ts(tmem + kColOuter, tmem + kColState, q_rows, id_rows, 1u);
#pragma unroll
                            for (uint32_t ks = 1; ks < DK / 16; ++ks) umma_ts(tmem + kColOuter, tmem + kColState + ks * 8, q_rows + row_step(ks), id_rows, 1u);
#pragma unroll
                            for (uint32_t ks = 0; ks < kC / 16; ++ks)
                                umma_ss(tmem + kColInner, v_cols + ks * 2048 / 16, p_rows + kTileBlock / 16 + ks * 2, id_inner, ks);
                            if (kIsHalf<T>) umma_ss_down11(tmem + kColInner, v_cols, p_rows, id_inner);
                            else umma_ss(tmem + kColInner, v_cols, p_rows, id_inner, 1u);
#pragma unroll
                            for (uint32_t ks = 1; ks < kC / 16; ++ks) umma_ss(tmem + kColInner, v_cols + ks * 2048 / 16, p_rows + ks * 2, id_inner, 1u);
                            umma_commit_one(bar(kBarDone + h % kStages));
                        }
                        __syncwarp();
                    }
                }
            }
            done_chunks += chunks;
        }
    } else if (warp == kWarpGain) {
        // ================================ loads and gains (converged warp) ===============================================
        // The next chunk to load, in the order of the CTA's items.
        uint32_t load_item = blockIdx.x, load_t0 = 0, loaded = 0;
        const auto load_next = [&] {
            if (load_item >= total) return;
            const LinearRun run = runs[load_item / p.num_v_heads];
            const uint32_t head = load_item % p.num_v_heads, k_head = head / share, row = run.flat_begin + load_t0;
            const uint32_t slot = loaded % kStages, stage = smem_base + slot * kStageBytes, full = bar(kBarFull + slot);
            __syncwarp();
            if (p.aligned != 0) {
                if (lane == 0) mbar_expect_tx(full, (kStateOnly ? kQBytes : 2 * kQBytes) + kVBytes);
                __syncwarp();
#pragma unroll
                for (uint32_t b = 0; b < kBlocksK; ++b) {
                    tma_load_rows(stage + kQBytes + b * kTileBlock, &k_map, full, b * 64, row, k_head);
                    if constexpr (!kStateOnly) tma_load_rows(stage + b * kTileBlock, &q_map, full, b * 64, row, k_head);
                }
#pragma unroll
                for (uint32_t b = 0; b < 2; ++b) tma_load_rows(stage + 2 * kQBytes + b * kTileBlock, &v_map, full, b * 64, row, head);
            } else {
#pragma unroll 1
                for (uint32_t which = kStateOnly ? 1 : 0; which < 3; ++which) {
                    const uint16_t* base = static_cast<const uint16_t*>(which == 0 ? p.q : which == 1 ? p.k : p.v);
                    const uint32_t heads = which < 2 ? p.num_k_heads : p.num_v_heads, dim = which < 2 ? p.key_dim : p.value_dim;
                    const uint32_t chunks = which < 2 ? DK / 8 : 16;
#pragma unroll 1
                    for (uint32_t at = lane; at < kC * chunks; at += 32) {
                        const uint32_t r = at / chunks, c = at % chunks;
                        const bool live = load_t0 + r < run.tokens && c * 8u < dim;
                        const uint16_t* src = base + (uint64_t(row + r) * heads + (which < 2 ? k_head : head)) * dim + c * 8u;
                        uint32_t two[4];
#pragma unroll
                        for (int x = 0; x < 4; ++x) two[x] = live ? uint32_t(src[2 * x]) | uint32_t(src[2 * x + 1]) << 16 : 0u;
                        asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};\n" ::"r"(stage + which * kQBytes + tile_offset(r, c)), "r"(two[0]), "r"(two[1]),
                                     "r"(two[2]), "r"(two[3])
                                     : "memory");
                    }
                }
                fence_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(full);
            }
            __syncwarp();
            ++loaded;
            load_t0 += kC;
            if (load_t0 >= run.tokens) {
                load_t0 = 0;
                load_item += gridDim.x;
            }
        };
        for (uint32_t x = 0; x < kStages; ++x) load_next();
        const uint32_t id_gain = umma_idesc<T>(DK, true);
        for (uint32_t item = blockIdx.x; item < total; item += gridDim.x) {
            const uint32_t chunks = (runs[item / p.num_v_heads].tokens + kC - 1) / kC;
#pragma unroll 1
            for (uint32_t c = 0; c < chunks; ++c) {
                const uint32_t g = done_chunks + c;
                const uint64_t k_cols = umma_desc(smem_base + g % kStages * kStageBytes + kQBytes, kTileBlock, 1024);
                wait(kBarFull + g % kStages, g / kStages);
                wait(kBarParts, g);
                if (g > 0) wait(kBarGainRead, g - 1);
                tc_fence_after();
                if (elect_one()) {
                    // the lowest part first
                    if constexpr (!kIsHalf<T>) {
                        const uint64_t low = umma_desc(smem_low, 16, 1024);
#pragma unroll
                        for (uint32_t ks = 0; ks < kC / 16; ++ks) umma_ss(tmem + kColGain, low + ks * 2, k_cols + ks * 2048 / 16, id_gain, ks);
                    }
#pragma unroll
                    for (int part = 1; part >= 0; --part) {
                        const uint32_t first = tmem + kColParts + part * kPartColumns;
                        if (kIsHalf<T> && part == 0) umma_ts_down11(tmem + kColGain, first, k_cols, id_gain);
                        else umma_ts(tmem + kColGain, first, k_cols, id_gain, part == 0 || !kIsHalf<T> ? 1u : 0u);
#pragma unroll
                        for (uint32_t ks = 1; ks < kC / 16; ++ks) umma_ts(tmem + kColGain, first + ks * 8, k_cols + ks * 2048 / 16, id_gain, 1u);
                    }
                    umma_commit_one(bar(kBarGain));
                }
                __syncwarp();
                // the gain of chunk g - 1 is complete; once its other products are, its slot is free
                if (g > 0) {
                    if constexpr (!kStateOnly) wait(kBarDone + (g - 1) % kStages, (g - 1) / kStages);
                    load_next();
                }
            }
            done_chunks += chunks;
        }
        // the CTA does not go away with its own bulk copies in flight, also after an earlier wait gave up
        for (uint32_t back = 1; back <= kStages && back <= loaded; ++back) mbar_wait(bar(kBarFull + (loaded - back) % kStages), ((loaded - back) / kStages) & 1u);
    } else if (warp >= kWarpP) {
        // ================================ P: a row of scores per thread ==================================================
        if constexpr (!kStateOnly) {
            const uint32_t row = (warp - kWarpP) * 32u + lane, lane_base = ((warp - kWarpP) * 32u) << 16;
            // scale lambda^(row - j) at [j]: entry 63 - row + j of the table, from the copy where that is a multiple of four
            const float* lag = shared.lag[(kC - 1 - row) & 3u] + ((kC - 1 - row) & ~3u);
            for (uint32_t item = blockIdx.x; item < total; item += gridDim.x) {
                const uint32_t chunks = (runs[item / p.num_v_heads].tokens + kC - 1) / kC;
                asm volatile("bar.sync 6, %0;" ::"n"(kStateThreads + kOutThreads + 64) : "memory");  // the tables of this item's head are there
                for (uint32_t c = 0; c < chunks; ++c) {
                    const uint32_t g = done_chunks + c;
                    wait(kBarScores, g);
                    tc_fence_after();
                    // sixteen columns at a time, in code that stays short
                    const uint32_t end = (warp - kWarpP + 1) * 32u;  // columns that the warp's rows can see
                    const auto take = [&](uint32_t j0, float (&x)[16]) {
                        tmem_load16(tmem + kColScores + lane_base + j0, x);
#pragma unroll
                        for (uint32_t j = 0; j < 16; j += 4) {
                            const float4 w = *reinterpret_cast<const float4*>(lag + j0 + j);
                            x[j] = j0 + j <= row ? x[j] * w.x : 0.0f;
                            x[j + 1] = j0 + j + 1 <= row ? x[j + 1] * w.y : 0.0f;
                            x[j + 2] = j0 + j + 2 <= row ? x[j + 2] * w.z : 0.0f;
                            x[j + 3] = j0 + j + 3 <= row ? x[j + 3] * w.w : 0.0f;
                        }
                    };
                    float down = 1.0f, up = 1.0f;
                    if constexpr (kIsHalf<T>) {
                        float largest = 0.0f;
#pragma unroll 1
                        for (uint32_t j0 = 0; j0 < end; j0 += 16) {
                            float x[16];
                            take(j0, x);
#pragma unroll
                            for (uint32_t j = 0; j < 16; j += 2) largest = max3(largest, fabsf(x[j]), fabsf(x[j + 1]));
                        }
                        range_scale(largest, down, up);
                        shared.p_scale[g & 3u][row] = up;
                    }
                    if (g >= 2) wait(kBarDone + (g - 2) % kStages, (g - 2) / kStages);  // the product that read this half of the buffer
                    const uint32_t tile = smem_p + (g & 1u) * (2 * kTileBlock);
#pragma unroll 1
                    for (uint32_t j0 = 0; j0 < end; j0 += 16) {
                        float x[16];
                        take(j0, x);
#pragma unroll
                        for (uint32_t y = 0; y < 16; y += 8) {
                            uint32_t high[4], low[4];
#pragma unroll
                            for (uint32_t j = 0; j < 4; ++j) {
                                uint64_t two = pack_f32x2(x[y + 2 * j], x[y + 2 * j + 1]);
                                if constexpr (kIsHalf<T>) two = mul_f32x2(two, pack_f32x2(down, down));
                                split_two<T>(two, high[j], low[j]);
                            }
                            const uint32_t to = tile + tile_offset(row, (j0 + y) / 8);
                            st_shared16(to, high);
                            st_shared16(to + kTileBlock, low);
                        }
                    }
#pragma unroll 1
                    for (uint32_t x = end / 8; x < 8; ++x) {
                        st_shared_zero16(tile + tile_offset(row, x));
                        st_shared_zero16(tile + kTileBlock + tile_offset(row, x));
                    }
                    fence_async_smem();
                    tc_fence_before();
                    mbar_arrive(bar(kBarP));
                }
                done_chunks += chunks;
                asm volatile("bar.sync 5, %0;" ::"n"(kStateThreads + kOutThreads + 64) : "memory");  // the next item's tables may replace these
            }
        }
    } else if (warp >= kWarpOut) {
        // ================================ outputs ==========================================================================
        if constexpr (!kStateOnly) {
            const uint32_t rows_warp = warp - kWarpOut, lane_base = (rows_warp * 32u) << 16, thread = tid - kStateThreads;
            const uint32_t quad = lane >> 2, pair = lane & 3u;  // of a fragment: row quad (+ 8), columns 2 pair + {0, 1}
            const bool wide_out = (reinterpret_cast<uintptr_t>(p.out) & 15u) == 0;
            for (uint32_t item = blockIdx.x; item < total; item += gridDim.x) {
                const LinearRun run = runs[item / p.num_v_heads];
                const uint32_t head = item % p.num_v_heads, chunks = (run.tokens + kC - 1) / kC;
                asm volatile("bar.sync 6, %0;" ::"n"(kStateThreads + kOutThreads + 64) : "memory");
                T* const out = static_cast<T*>(p.out) + (uint64_t(run.flat_begin) * p.num_v_heads + head) * p.value_dim;
                const uint64_t stride = uint64_t(p.num_v_heads) * p.value_dim;
                for (uint32_t c = 0; c < chunks; ++c) {
                    const uint32_t g = done_chunks + c, n = min(kC, run.tokens - c * kC);
                    wait(kBarDone + g % kStages, g / kStages);
                    tc_fence_after();
                    asm volatile("bar.sync 7, %0;" ::"n"(kOutThreads) : "memory");  // the rows of the chunk before have been read
                    // [token][v] in shared memory, 16 columns v and 32 tokens at a time: lane t gives the address of row t % 8 (a token)
                    // of matrix t / 8 (8 tokens x 8 columns: two of columns, then of tokens)
                    const uint32_t tile = smem_out;
                    const bool any_bad = *reinterpret_cast<volatile uint32_t*>(&shared.any_bad) != 0;
#pragma unroll 1
                    for (uint32_t half = 0; half < 2; ++half) {
                        float up[2] = {1.0f, 1.0f};
                        if constexpr (kIsHalf<T>) {
                            up[0] = shared.column_up[g & 3u][rows_warp * 32u + half * 16 + quad];
                            up[1] = shared.column_up[g & 3u][rows_warp * 32u + half * 16 + 8 + quad];
                        }
                        const uint32_t to = tile + tile_offset(lane & 7u, rows_warp * 4 + half * 2 + ((lane >> 3) & 1u)) + (lane >> 4) * 1024;
#pragma unroll 1
                        for (uint32_t b0 = 0; b0 < 8; b0 += 4) {
                            uint64_t inner[8], outer[8];
                            const uint32_t at = tmem + lane_base + ((half * 16u) << 16) + b0 * 8;
                            tmem_load_16x256_x4(at + kColInner, at + kColOuter, inner, outer);
                            uint32_t packed[8];
#pragma unroll
                            for (uint32_t b = 0; b < 4; ++b) {
                                const uint64_t rise = *reinterpret_cast<const uint64_t*>(&shared.rise[8 * (b0 + b) + 2 * pair]);
                                uint64_t p_up = 0;
                                if constexpr (kIsHalf<T>) p_up = *reinterpret_cast<const uint64_t*>(&shared.p_scale[g & 3u][8 * (b0 + b) + 2 * pair]);
#pragma unroll
                                for (uint32_t h = 0; h < 2; ++h) {
                                    uint64_t in = inner[2 * b + h], from_state = outer[2 * b + h];
                                    if constexpr (kIsHalf<T>) {
                                        in = mul_f32x2(in, p_up);
                                        from_state = mul_f32x2(from_state, pack_f32x2(up[h], up[h]));
                                    }
                                    const float2 two = unpack_f32x2(fma_f32x2(from_state, rise, in));
                                    packed[2 * b + h] = Mma<T>::pack(two.x, two.y);
                                }
                            }
                            if (any_bad) {
#pragma unroll
                                for (uint32_t x = 0; x < 8; ++x) {
                                    const uint32_t bad = shared.bad_from[g & 3u][rows_warp * 32u + half * 16 + 8 * (x & 1u) + quad], t = 8 * (b0 + x / 2) + 2 * pair;
                                    if (t >= bad) packed[x] |= 0x7FFFu;
                                    if (t + 1 >= bad) packed[x] |= 0x7FFF0000u;
                                }
                            }
                            stmatrix_x4_trans(to + b0 * 1024, packed[0], packed[1], packed[2], packed[3]);
                            stmatrix_x4_trans(to + b0 * 1024 + 2048, packed[4], packed[5], packed[6], packed[7]);
                        }
                    }
                    if (any_bad) {
                        __syncwarp();
                        shared.bad_from[g & 3u][thread] = kC;  // (these rows are this warp's)
                    }
                    tc_fence_before();
                    mbar_arrive(bar(kBarOut));
                    asm volatile("bar.sync 7, %0;" ::"n"(kOutThreads) : "memory");
                    const uint32_t column = thread & 15u;
                    if (column * 8 < p.value_dim) {
#pragma unroll 2
                        for (uint32_t x = 0; x < kC; x += kOutThreads / 16) {
                            const uint32_t token = x + (thread >> 4);
                            uint4 value;
                            asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];\n"
                                         : "=r"(value.x), "=r"(value.y), "=r"(value.z), "=r"(value.w)
                                         : "r"(tile + tile_offset(token, column))
                                         : "memory");
                            T* to = out + (uint64_t(c) * kC + token) * stride + column * 8;
                            if (token < n) {
                                if (wide_out) {
                                    *reinterpret_cast<uint4*>(to) = value;
                                } else {
                                    const uint32_t words[4] = {value.x, value.y, value.z, value.w};
#pragma unroll
                                    for (uint32_t y = 0; y < 8; ++y) reinterpret_cast<uint16_t*>(to)[y] = uint16_t(words[y / 2] >> (16 * (y & 1u)));
                                }
                            }
                        }
                    }
                }
                done_chunks += chunks;
                asm volatile("bar.sync 5, %0;" ::"n"(kStateThreads + kOutThreads + 64) : "memory");
            }
        }
    } else {
        // ================================ a column of the state per four threads =========================================
        const uint32_t group = warp >> 2, rows_warp = warp & 3u, v = rows_warp * 32u + lane;
        const uint32_t lane_base = (rows_warp * 32u) << 16;
        const bool live = v < p.value_dim;
        const uint32_t k0 = group * kRows, token0 = group * kGroupTokens;
        const uint32_t pair = lane & 3u;  // of a fragment: tokens 2 pair + {0, 1}
        // ldmatrix: lane t gives the address of row t % 8 (a token) of matrix t / 8 (eight columns v)
        const uint32_t fetch_at = 2 * kQBytes + tile_offset(token0 + (lane & 7u), rows_warp * 4 + (lane >> 3));
        for (uint32_t item = blockIdx.x; item < total; item += gridDim.x) {
            const LinearRun run = runs[item / p.num_v_heads];
            const uint32_t head = item % p.num_v_heads;
            const float* decay = p.decays + uint64_t(head) * kLinearDecays;
            if constexpr (kStateOnly) asm volatile("bar.sync 5, %0;" ::"n"(kStateThreads) : "memory");
            if (tid < kC) {
                shared.fall[kC - 1 - tid] = decay[tid];
                shared.rise[tid] = decay[tid + 1] * p.scale;
                for (uint32_t x = 0; x < 4; ++x) {
                    shared.lag[x][tid] = tid + x < kC ? decay[kC - 1 - tid - x] * p.scale : 0.0f;
                    shared.lag[x][kC + tid] = 0.0f;  // (columns behind the row)
                }
            }
            for (uint32_t i = tid; i < 4 * kUmmaM; i += kStateThreads) shared.bad_from[i / kUmmaM][i % kUmmaM] = kC;
            if (tid == 0) shared.any_bad = 0;
            const float full_hi = decay[kC], full_lo = decay[kLinearChunkLow];
            asm volatile("bar.sync 6, %0;" ::"n"(kStateOnly ? kStateThreads : kStateThreads + kOutThreads + 64) : "memory");
            uint64_t s[kRows / 2];  // two rows of the state in each
            const float* from = kStateOnly ? nullptr : run.carry_in != kLinearNoCarry ? p.carry_of(run.carry_in, head) : run.fresh != 0 ? nullptr : p.state_of(run.src, head);
#pragma unroll
            for (uint32_t k = 0; k < kRows; k += 2) {  // (key_dim is a multiple of eight)
                const bool there = from != nullptr && live && k0 + k < p.key_dim;
                const float a = there ? from[uint64_t(k0 + k) * p.value_dim + v] : 0.0f, b = there ? from[uint64_t(k0 + k + 1) * p.value_dim + v] : 0.0f;
                s[k / 2] = pack_f32x2(a, b);
            }
            const auto put_state = [&](uint32_t g) {
                float down = 1.0f;
                if constexpr (kIsHalf<T>) {
                    float largest = 0.0f, up;
#pragma unroll
                    for (uint32_t k = 0; k < kRows / 2; ++k) {
                        const float2 two = unpack_f32x2(s[k]);
                        largest = max3(largest, fabsf(two.x), fabsf(two.y));
                    }
                    shared.column_max[g & 1u][group][v] = largest;
                    __syncwarp();
                    asm volatile("bar.sync %0, %1;" ::"r"(rows_warp + 1), "n"(32 * kGroups) : "memory");  // the other parts of these columns
#pragma unroll
                    for (uint32_t x = 0; x < kGroups; ++x) largest = fmaxf(largest, shared.column_max[g & 1u][x][v]);
                    range_scale(largest, down, up);
                    if (group == 0) shared.column_up[g & 3u][v] = up;
                }
#pragma unroll
                for (uint32_t k = 0; k < kRows / 2; k += 8) {
                    uint32_t high[8], low[8];
#pragma unroll
                    for (uint32_t x = 0; x < 8; ++x) split_two<T>(kIsHalf<T> ? mul_f32x2(s[k + x], pack_f32x2(down, down)) : s[k + x], high[x], low[x]);
                    tmem_store8_bits(tmem + kColState + lane_base + k0 / 2 + k, high);
                    tmem_store8_bits(tmem + kColStateLow + lane_base + k0 / 2 + k, low);
                }
                tmem_store_wait();
                tc_fence_before();
                mbar_arrive(bar(kBarState));
            };
            const uint32_t chunks = (run.tokens + kC - 1) / kC;
            // The state after chunk `c` of the item, whose gain is complete.
            const auto advance = [&](uint32_t c) {
                const uint32_t n = min(kC, run.tokens - c * kC);
                const float hi = n == kC ? full_hi : shared.fall[kC - 1 - n], lo = n == kC ? full_lo : 0.0f;
                const uint64_t hi2 = pack_f32x2(hi, hi), lo2 = pack_f32x2(lo, lo);
#pragma unroll
                for (uint32_t k = 0; k < kRows; k += 16) {
                    float gain[16];
                    tmem_load16(tmem + kColGain + lane_base + k0 + k, gain);
                    if (k + 16 == kRows) {
                        tc_fence_before();
                        mbar_arrive(bar(kBarGainRead));
                    }
#pragma unroll
                    for (uint32_t x = 0; x < 8; ++x)
                        s[k / 2 + x] = fma_f32x2(hi2, s[k / 2 + x], fma_f32x2(lo2, s[k / 2 + x], pack_f32x2(gain[2 * x], gain[2 * x + 1])));
                }
            };
#pragma unroll 1
            for (uint32_t c = 0; c < chunks; ++c) {
                const uint32_t g = done_chunks + c, slot = g % kStages;
                const uint32_t n = min(kC, run.tokens - c * kC);
                const uint32_t stage = smem_base + slot * kStageBytes;
                wait(kBarFull + slot, g / kStages);
                const float* weights = shared.fall;
                if (n < kC) {
                    // the last chunk: what lies behind the run is cleared, and the weights move up
                    for (uint32_t at = tid; at < (kC - n) * (DK / 8 + 16); at += kStateThreads) {
                        const uint32_t row = n + at / (DK / 8 + 16), x = at % (DK / 8 + 16);
                        st_shared_zero16(stage + (x < DK / 8 ? kQBytes + tile_offset(row, x) : 2 * kQBytes + tile_offset(row, x - DK / 8)));
                    }
                    if (tid < kC) shared.last_fall[tid] = tid < n ? shared.fall[tid + (kC - n)] : 0.0f;
                    fence_async_smem();
                    asm volatile("bar.sync 8, %0;" ::"n"(kStateThreads) : "memory");
                    weights = shared.last_fall;
                }
                // Weighted V of 32 columns and 16 tokens a warp, in parts: made while the chunk before gains, put where its parts were
                float largest = 0.0f;
                uint32_t parts[kParts][2][4];  // [part][16-row half][2 (8-token block) + 8-row half]
#pragma unroll
                for (uint32_t b = 0; b < kGroupTokens / 8; ++b) {
                    uint32_t raw[4];
                    ldmatrix_x4_trans(raw, stage + fetch_at + b * 1024);
                    const uint64_t w = *reinterpret_cast<const uint64_t*>(weights + token0 + 8 * b + 2 * pair);
#pragma unroll
                    for (uint32_t m = 0; m < 4; ++m) {
                        const float2 two = Mma<T>::unpack(raw[m]);
                        largest = max3_abs_nan(largest, two.x, two.y);
                        uint32_t split[3];
                        split_parts<T>(mul_f32x2(pack_f32x2(two.x, two.y), w), split);
#pragma unroll
                        for (uint32_t x = 0; x < kParts; ++x) parts[x][m >> 1][2 * b + (m & 1u)] = split[x];
                    }
                }
                if (!kStateOnly && !(largest < INFINITY)) shared.any_bad = 1;
                // A value that is not finite must not reach tokens before its own, whose P is zero there: it leaves the chunk's V,
                // and the outputs from its token on are no numbers.
                if (!kStateOnly && __any_sync(0xFFFFFFFFu, *reinterpret_cast<volatile uint32_t*>(&shared.any_bad) != 0)) {
                    for (uint32_t j = 0; j < kGroupTokens && token0 + j < n; ++j) {
                        const uint32_t at = stage + 2 * kQBytes + tile_offset(token0 + j, v >> 3) + (v & 7u) * 2;
                        uint16_t bits;
                        asm volatile("ld.shared.u16 %0, [%1];" : "=h"(bits) : "r"(at) : "memory");
                        if (not_finite_bits<T>(bits)) {
                            atomicMin(&shared.bad_from[g & 3u][v], token0 + j);
                            asm volatile("st.shared.u16 [%0], %1;" ::"r"(at), "h"(uint16_t(0)) : "memory");
                        }
                    }
                    fence_async_smem();
                    __syncwarp();
                }
                // The state before the first chunk.  kBarState is also what the inner product waits for before it reads V: it stands
                // behind the clearing and the removal of every chunk, the first included.
                if constexpr (!kStateOnly) {
                    if (c == 0) put_state(g);
                }
                if (c > 0) wait(kBarGain, g - 1);
                tc_fence_after();
                const uint32_t parts_at = tmem + kColParts + lane_base + token0 / 2;
#pragma unroll
                for (uint32_t x = 0; x < 2; ++x) {
                    tmem_store_16x128_x2(parts_at + x * kPartColumns, parts[x][0]);
                    tmem_store_16x128_x2(parts_at + x * kPartColumns + (16u << 16), parts[x][1]);
                }
                if constexpr (kParts == 3) {  // [v][token] in shared memory: lane t gives the address of its column v's row
#pragma unroll
                    for (uint32_t b = 0; b < kGroupTokens / 8; ++b)
                        stmatrix_x4(smem_low + tile_offset(v, token0 / 8 + b), parts[2][0][2 * b], parts[2][0][2 * b + 1], parts[2][1][2 * b], parts[2][1][2 * b + 1]);
                    fence_async_smem();
                }
                tmem_store_wait();
                tc_fence_before();
                mbar_arrive(bar(kBarParts));
                if (c > 0) advance(c - 1);
                if constexpr (!kStateOnly) {
                    if (c > 0) {
                        wait(kBarDone + (g - 1) % kStages, (g - 1) / kStages);
                        tc_fence_after();
                        put_state(g);
                    }
                }
            }
            const uint32_t last = done_chunks + chunks - 1;
            wait(kBarGain, last);
            tc_fence_after();
            advance(chunks - 1);
            float* to = kStateOnly ? p.carry_of(run.carry_out, head) : run.keep != 0 ? p.state_of(run.dst, head) : nullptr;
            if (to != nullptr && live) {
#pragma unroll
                for (uint32_t k = 0; k < kRows; k += 2) {
                    const float2 two = unpack_f32x2(s[k / 2]);
                    if (k0 + k < p.key_dim) {
                        to[uint64_t(k0 + k) * p.value_dim + v] = two.x;
                        to[uint64_t(k0 + k + 1) * p.value_dim + v] = two.y;
                    }
                }
            }
            if constexpr (!kStateOnly) wait(kBarDone + last % kStages, last / kStages);
            tc_fence_after();
            if constexpr (!kStateOnly) asm volatile("bar.sync 5, %0;" ::"n"(kStateThreads + kOutThreads + 64) : "memory");
            done_chunks += chunks;
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
}

template <typename T, uint32_t DK, bool kStateOnly>
cudaError_t launch_one(const LinearParams& params, uint32_t ctas, cudaStream_t stream) {
    // the ring, P in two parts twice, the outputs, V's lowest part (bf16)
    constexpr int kSmem = int((kStages * (2 * (DK / 64) + 2) + 4 + 2 + (kIsHalf<T> ? 0 : 2)) * kTileBlock + 1024);
    static_assert(kSmem + sizeof(ChunkShared) <= 227 * 1024);
    LinearParams p = params;
    CUtensorMap q_map{}, k_map{}, v_map{};
    p.aligned = p.aligned != 0 && make_rows_map(p.q, p.dtype, p.key_dim, p.num_k_heads, p.num_tokens, kC, &q_map) &&
                        make_rows_map(p.k, p.dtype, p.key_dim, p.num_k_heads, p.num_tokens, kC, &k_map) &&
                        make_rows_map(p.v, p.dtype, p.value_dim, p.num_v_heads, p.num_tokens, kC, &v_map)
                    ? 1u
                    : 0u;
    auto kernel = linear_chunk_kernel<T, DK, kStateOnly>;
    static std::atomic<uint64_t> done{0};
    const cudaError_t err = ensure_dynamic_smem(reinterpret_cast<const void*>(kernel), kSmem, done);
    if (err != cudaSuccess) return err;
    return launch_overlapped(kernel, dim3(ctas), dim3(kChunkThreads), kSmem, stream, p, q_map, k_map, v_map);
}

template <typename T>
cudaError_t launch_typed(const LinearParams& p, bool state_only, uint32_t ctas, cudaStream_t stream) {
    if (p.key_dim <= 64) return state_only ? launch_one<T, 64, true>(p, ctas, stream) : launch_one<T, 64, false>(p, ctas, stream);
    return state_only ? launch_one<T, 128, true>(p, ctas, stream) : launch_one<T, 128, false>(p, ctas, stream);
}

}  // namespace

bool linear_chunk_supported(uint32_t dtype, uint32_t key_dim, uint32_t value_dim) {
    return dtype != PSI_DTYPE_F32 && key_dim <= 128 && value_dim <= 128;
}

cudaError_t launch_linear_chunk(const LinearParams& p, bool state_only, uint32_t ctas, cudaStream_t stream) {
    return p.dtype == PSI_DTYPE_BF16 ? launch_typed<__nv_bfloat16>(p, state_only, ctas, stream) : launch_typed<__half>(p, state_only, ctas, stream);
}

}  // namespace psi
