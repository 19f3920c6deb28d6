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
//   inner^T  [v][i] = V^T P^T                  V as it landed, P = lambda^(i-j) scores, rounded to 16 bits, in shared memory
//   outer^T  [v][i] = S^T Q^T                  S^T rounded to 16 bits in TMEM; lambda^(i+1) is applied in f32 afterwards
//   gain^T   [v][k] = (lambda^(n-1-j) V)^T K   the weighted V in TMEM in as many 16-bit parts as make 22 bits or more (bf16 three, f16
//                                              two, the low one 2^11 times as large), a product each, so that the f32 state
//                                              loses nothing to the 16-bit operands
//
// P and S in 16 bits are two roundings of half a step of the I/O type beside the output's own: 1.4 times the error of an f32
// product that is rounded once.  In f16 each row of P and each column of S is scaled by a power of two first, so that
// nothing leaves f16's range.  The state itself stays in f32 registers; a chunk's gain is added to it after an
// accumulation of its own, since the tensor cores' accumulation truncates.
//
// Warps 0-7: two threads for each v, half of the state (and of the chunk's tokens) each: weighted V, state, output.  Warps 8 and 9: P.
// Warp 10 issues the MMAs.  Warp 11 brings Q, K and V into a ring of four chunks (cp.async; rows behind a run are zero).  (A thirteenth
// warp would cost every thread 40 registers.)
// Every hand-off is an mbarrier, every wait is bounded and reports PSI_ERR_TIMEOUT through the status word, and TMEM is freed on
// every path.
#include "launch_util.hpp"
#include "linear_attend.hpp"
#include "mma_common.cuh"
#include "umma_common.cuh"

namespace psi {

namespace {

constexpr uint32_t kC = kLinearChunk, kStages = 4;
constexpr uint32_t kWarpP = 8, kWarpMma = 10, kWarpLoad = 11, kLoadWarps = 1;
constexpr uint32_t kChunkThreads = (kWarpLoad + kLoadWarps) * 32, kStateThreads = 256;
constexpr uint32_t kLoadLag = 2;  // chunks under way in a loading warp behind the one it has just asked for

// TMEM columns
constexpr uint32_t kColScores = 0, kColInner = 0, kColOuter = 64, kColGain = 128, kColState = 256, kColParts = 320;
constexpr uint32_t kPartColumns = kC / 2, kPartBuffer = 3 * kPartColumns;
static_assert(kColParts + 2 * kPartBuffer <= 512, "one TMEM allocation");

// Barriers: ring slots full and done by slot, weighted V two taken in turn, the others one each, their phase the chunk's.  A parity
// wait cannot tell two completions from none: a thread waits for a phase only where the next one cannot complete without it.  The
// weighted V of a chunk may be there before the MMA warp has looked for the one before; two chunks ahead it cannot be, since it
// needs that chunk's gain.
constexpr uint32_t kBarFull = 0, kBarDone = kStages, kBarScores = 2 * kStages, kBarP = kBarScores + 1, kBarParts = kBarP + 1,  // (two of them)
                   kBarGain = kBarParts + 2, kBarGainRead = kBarGain + 1, kBarState = kBarGainRead + 1, kNumBars = kBarState + 1;

struct ChunkShared {
    uint64_t bars[kNumBars];
    uint32_t tmem_base, abort;
    __align__(16) float power[kC + 4];      // lambda^0 .. lambda^64
    __align__(16) float fall[kC];           // lambda^(63 - j)
    float p_scale[2][kC];                   // f16: what the rows of P were divided by, by chunk parity
    float column_max[2][2][kUmmaM];         // f16: largest magnitude of each half of a state column, by chunk parity
    // First token of each half whose V is not finite (64: none), by chunk.  The two threads of a column meet once a chunk, after
    // which one may be a chunk ahead of the other: four chunks later both have read it.
    uint32_t bad_from[4][2][kUmmaM];
};

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

// Packs two values as 16-bit parts: bf16 in three (the first two towards zero, exact rests), f16 in two, the second 2^11 times as large.
template <typename T>
__device__ __forceinline__ void split_parts(float a, float b, uint32_t (&part)[3]) {
    if constexpr (kIsHalf<T>) {
        part[0] = Mma<T>::pack(a, b);
        const float2 h = Mma<T>::unpack(part[0]);
        part[1] = Mma<T>::pack((a - h.x) * 2048.0f, (b - h.y) * 2048.0f);
        part[2] = 0;
    } else {
        part[0] = Mma<T>::pack_down(a, b);
        const float2 h = Mma<T>::unpack(part[0]);
        a -= h.x;
        b -= h.y;
        part[1] = Mma<T>::pack_down(a, b);
        const float2 m = Mma<T>::unpack(part[1]);
        part[2] = Mma<T>::pack(a - m.x, b - m.y);
    }
}

__device__ __forceinline__ float ld_shared_16bit(uint32_t addr, bool half) {
    uint16_t v;
    asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(addr) : "memory");
    return half ? __half2float(__ushort_as_half(v)) : __uint_as_float(uint32_t(v) << 16);
}

// DK: key_dim rounded up to 64 or 128.  kStateOnly: the run's state from zero, without outputs.
template <typename T, uint32_t DK, bool kStateOnly>
__global__ void __launch_bounds__(kChunkThreads, 1) linear_chunk_kernel(const LinearParams p) {
    constexpr uint32_t kBlocksK = DK / 64, kBlocksV = 2;
    constexpr uint32_t kQBytes = kC * DK * 2, kVBytes = kC * 128 * 2, kStageBytes = 2 * kQBytes + kVBytes;
    constexpr uint32_t kParts = kIsHalf<T> ? 2 : 3;
    constexpr uint32_t kHalfK = DK / 2;  // state rows of one thread
    __shared__ ChunkShared shared;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u;
    const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t smem_p = smem_base + kStages * kStageBytes;
    const uint32_t bar0 = smem_u32(shared.bars);
    const auto bar = [&](uint32_t which) { return bar0 + which * 8u; };
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&shared.tmem_base)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (tid == 0) {
        for (uint32_t b = 0; b < kStages; ++b) {
            mbar_init(bar(kBarFull + b), kLoadWarps);
            mbar_init(bar(kBarDone + b), 1);
        }
        mbar_init(bar(kBarScores), 1);
        mbar_init(bar(kBarP), 64);
        mbar_init(bar(kBarParts), kStateThreads);
        mbar_init(bar(kBarParts + 1), kStateThreads);
        mbar_init(bar(kBarGain), 1);
        mbar_init(bar(kBarGainRead), kStateThreads);
        mbar_init(bar(kBarState), kStateThreads);
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
    const uint32_t num_runs = p.scalars[kStateOnly ? kLinearNumCarries : kLinearNumRuns];
    const uint32_t total = num_runs * p.num_v_heads;
    const uint32_t share = p.num_v_heads / p.num_k_heads;
    // Work: item = (run, value head).  A state pass takes the runs that another piece of their request follows; they come first.
    uint32_t done_chunks = 0;  // of the items before, the same count in every role
    if (warp >= kWarpLoad) {
        // ================================ Q, K and V into the ring =====================================================
        const uint32_t row0 = (warp - kWarpLoad) * (kC / kLoadWarps);
        const T* q = static_cast<const T*>(p.q);
        const T* k = static_cast<const T*>(p.k);
        const T* v = static_cast<const T*>(p.v);
        uint32_t chunk = 0;
        const auto landed = [&](uint32_t c) {
            fence_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(kBarFull + c % kStages));
        };
        for (uint32_t item = blockIdx.x; item < total; item += gridDim.x) {
            const LinearRun run = runs[item / p.num_v_heads];
            const uint32_t head = item % p.num_v_heads;
            const uint64_t k_stride = uint64_t(p.num_k_heads) * p.key_dim, v_stride = uint64_t(p.num_v_heads) * p.value_dim;
            for (uint32_t t0 = 0; t0 < run.tokens; t0 += kC, ++chunk) {
                if (chunk >= kStages) wait(kBarDone + chunk % kStages, chunk / kStages - 1);
                const uint32_t stage = smem_base + chunk % kStages * kStageBytes;
                const auto copy = [&](uint32_t dst, const T* base, uint64_t stride, uint32_t dim, uint32_t chunks, uint32_t blocks) {
                    for (uint32_t at = lane; at < kC / kLoadWarps * chunks; at += 32) {
                        const uint32_t row = row0 + at / chunks, c = at % chunks;
                        const bool live = t0 + row < run.tokens && c * 8u < dim;
                        const T* src = live ? base + (run.flat_begin + t0 + row) * stride + c * 8u : base;
                        if (p.aligned != 0) {
                            cp_async_16(dst + operand_offset(blocks, row, c), src, live ? 16u : 0u);
                        } else {
                            uint32_t two[4];
#pragma unroll
                            for (int x = 0; x < 4; ++x) {
                                const uint16_t* e = reinterpret_cast<const uint16_t*>(src) + 2 * x;
                                two[x] = live ? uint32_t(e[0]) | uint32_t(e[1]) << 16 : 0u;
                            }
                            asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};\n" ::"r"(dst + operand_offset(blocks, row, c)), "r"(two[0]),
                                         "r"(two[1]), "r"(two[2]), "r"(two[3])
                                         : "memory");
                        }
                    }
                };
                if constexpr (!kStateOnly) copy(stage, q + uint64_t(head / share) * p.key_dim, k_stride, p.key_dim, DK / 8, kBlocksK);
                copy(stage + kQBytes, k + uint64_t(head / share) * p.key_dim, k_stride, p.key_dim, DK / 8, kBlocksK);
                copy(stage + 2 * kQBytes, v + uint64_t(head) * p.value_dim, v_stride, p.value_dim, 16, kBlocksV);
                cp_async_commit();
                if (chunk >= kLoadLag) {
                    cp_async_wait<kLoadLag>();
                    landed(chunk - kLoadLag);
                }
            }
        }
        cp_async_wait<0>();
        for (uint32_t c = chunk < kLoadLag ? 0 : chunk - kLoadLag; c < chunk; ++c) landed(c);
    } else if (warp == kWarpMma) {
        // ================================ MMA issue (converged warp, one elected lane) ==================================
        const uint32_t id_scores = umma_idesc<T>(kC, false), id_inner = umma_idesc<T>(kC, false, true), id_outer = umma_idesc<T>(kC, false),
                       id_gain = umma_idesc<T>(DK, true);
        for (uint32_t item = blockIdx.x; item < total; item += gridDim.x) {
            const uint32_t chunks = (runs[item / p.num_v_heads].tokens + kC - 1) / kC;
            for (uint32_t c = 0; c < chunks; ++c) {
                const uint32_t g = done_chunks + c, slot = g % kStages;
                const uint32_t stage = smem_base + slot * kStageBytes;
                // K-major: 8-row groups kBlocksK KiB apart, 64-element blocks 1 KiB; MN-major: the same memory the other way round
                const uint64_t q_rows = umma_desc(stage, 16, kBlocksK * 1024), k_rows = umma_desc(stage + kQBytes, 16, kBlocksK * 1024);
                const uint64_t k_cols = umma_desc(stage + kQBytes, 1024, kBlocksK * 1024), v_cols = umma_desc(stage + 2 * kQBytes, 1024, kBlocksV * 1024);
                wait(kBarFull + slot, g / kStages);
                wait(kBarParts + (g & 1u), g >> 1);
                if (g > 0) wait(kBarGainRead, g - 1);
                tc_fence_after();
                const uint32_t parts = tmem + kColParts + (g & 1u) * kPartBuffer;
#pragma unroll
                for (int part = int(kParts) - 1; part >= 0; --part) {  // the lowest part first
#pragma unroll
                    for (uint32_t ks = 0; ks < kC / 16; ++ks) {
                        const uint32_t a = parts + part * kPartColumns + ks * 8;
                        const uint64_t b = k_cols + ks * 2 * (kBlocksK * 1024) / 16;
                        if (kIsHalf<T> && part == 0 && ks == 0) umma_issue_ts_down11(tmem + kColGain, a, b, id_gain);
                        else umma_issue_ts(tmem + kColGain, a, b, id_gain, part < int(kParts) - 1 || ks > 0 ? 1u : 0u);
                    }
                }
                umma_commit(bar(kBarGain));
                if constexpr (!kStateOnly) {
                    wait(kBarState, g);
                    tc_fence_after();
#pragma unroll
                    for (uint32_t ks = 0; ks < DK / 16; ++ks) {
                        const uint32_t step = ((ks >> 2) * 1024 + (ks & 3) * 32) / 16;
                        umma_issue_ss(tmem + kColScores, q_rows + step, k_rows + step, id_scores, ks > 0 ? 1u : 0u);
                    }
                    umma_commit(bar(kBarScores));
#pragma unroll
                    for (uint32_t ks = 0; ks < DK / 16; ++ks) {
                        const uint32_t step = ((ks >> 2) * 1024 + (ks & 3) * 32) / 16;
                        umma_issue_ts(tmem + kColOuter, tmem + kColState + ks * 8, q_rows + step, id_outer, ks > 0 ? 1u : 0u);
                    }
                    wait(kBarP, g);
                    tc_fence_after();
                    const uint64_t p_rows = umma_desc(smem_p, 16, 1024);
#pragma unroll
                    for (uint32_t ks = 0; ks < kC / 16; ++ks)
                        umma_issue_ss(tmem + kColInner, v_cols + ks * 2 * (kBlocksV * 1024) / 16, p_rows + ks * 32 / 16, id_inner, ks > 0 ? 1u : 0u);
                }
                umma_commit(bar(kBarDone + slot));
            }
            done_chunks += chunks;
        }
    } else if (warp >= kWarpP) {
        // ================================ P: a row of scores per thread ==================================================
        if constexpr (!kStateOnly) {
            const uint32_t row = (warp - kWarpP) * 32u + lane, lane_base = ((warp - kWarpP) * 32u) << 16;
            for (uint32_t item = blockIdx.x; item < total; item += gridDim.x) {
                const uint32_t chunks = (runs[item / p.num_v_heads].tokens + kC - 1) / kC;
                for (uint32_t c = 0; c < chunks; ++c) {
                    const uint32_t g = done_chunks + c;
                    wait(kBarState, g);  // the item's table of powers is there
                    wait(kBarScores, g);
                    tc_fence_after();
                    float s[64];
                    tmem_load64(tmem + kColScores + lane_base, s);
                    float largest = 0.0f;
#pragma unroll
                    for (int j = 0; j < 64; ++j) {
                        s[j] = uint32_t(j) <= row ? s[j] * shared.power[row - j] : 0.0f;
                        if (kIsHalf<T>) largest = fmaxf(largest, fabsf(s[j]));
                    }
                    float down = 1.0f, up = 1.0f;
                    if constexpr (kIsHalf<T>) {
                        range_scale(largest, down, up);
                        shared.p_scale[g & 1u][row] = up;
                    }
#pragma unroll
                    for (uint32_t x = 0; x < 8; ++x) {
                        uint4 v;
                        v.x = Mma<T>::pack(s[8 * x] * down, s[8 * x + 1] * down);
                        v.y = Mma<T>::pack(s[8 * x + 2] * down, s[8 * x + 3] * down);
                        v.z = Mma<T>::pack(s[8 * x + 4] * down, s[8 * x + 5] * down);
                        v.w = Mma<T>::pack(s[8 * x + 6] * down, s[8 * x + 7] * down);
                        const uint32_t to = smem_p + operand_offset(1, row, x);
                        asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};\n" ::"r"(to), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
                    }
                    fence_async_smem();
                    tc_fence_before();
                    mbar_arrive(bar(kBarP));
                }
                done_chunks += chunks;
                // the table of the next item's head may replace this one once every row of this item is through
                asm volatile("bar.sync 5, 320;" ::: "memory");
            }
        }
    } else {
        // ================================ a column of the state per two threads ==========================================
        const uint32_t half = warp >> 2, rows_warp = warp & 3u, v = rows_warp * 32u + lane;
        const uint32_t lane_base = (rows_warp * 32u) << 16;
        const bool live = v < p.value_dim;
        const uint32_t k0 = half * kHalfK, token0 = half * (kC / 2);
        const auto pair_sync = [&] {
            __syncwarp();
            asm volatile("bar.sync %0, 64;" ::"r"(rows_warp + 1) : "memory");
        };
        for (uint32_t item = blockIdx.x; item < total; item += gridDim.x) {
            const LinearRun run = runs[item / p.num_v_heads];
            const uint32_t head = item % p.num_v_heads;
            const float* decay = p.decays + uint64_t(head) * kLinearDecays;
            if constexpr (kStateOnly) asm volatile("bar.sync 5, 256;" ::: "memory");
            for (uint32_t i = tid; i <= kC; i += kStateThreads) {
                shared.power[i] = decay[i];
                if (i < kC) shared.fall[kC - 1 - i] = decay[i];
            }
            const float full_hi = decay[kC], full_lo = decay[kLinearChunkLow];
            if constexpr (kStateOnly) asm volatile("bar.sync 6, 256;" ::: "memory");
            else asm volatile("bar.sync 7, 256;" ::: "memory");
            float s[kHalfK];
            const float* from = kStateOnly ? nullptr : run.carry_in != kLinearNoCarry ? p.carry_of(run.carry_in, head) : run.fresh != 0 ? nullptr : p.state_of(run.src, head);
#pragma unroll
            for (uint32_t k = 0; k < kHalfK; ++k)
                s[k] = from != nullptr && live && k0 + k < p.key_dim ? from[uint64_t(k0 + k) * p.value_dim + v] : 0.0f;
            float state_up = 1.0f;  // what the 16-bit state of the chunk under way was divided by
            const auto put_state = [&](uint32_t g) {
                float down = 1.0f;
                if constexpr (kIsHalf<T>) {
                    float largest = 0.0f;
#pragma unroll
                    for (uint32_t k = 0; k < kHalfK; ++k) largest = fmaxf(largest, fabsf(s[k]));
                    shared.column_max[g & 1u][half][v] = largest;
                    pair_sync();
                    range_scale(fmaxf(largest, shared.column_max[g & 1u][half ^ 1u][v]), down, state_up);
                } else {
                    pair_sync();  // (the other half's bad_from of the chunk before)
                }
                uint32_t packed[kHalfK / 2];
#pragma unroll
                for (uint32_t k = 0; k < kHalfK; k += 2) packed[k / 2] = Mma<T>::pack(s[k] * down, s[k + 1] * down);
                if constexpr (kHalfK == 64) tmem_store32_bits(tmem + kColState + lane_base + k0 / 2, packed);
                else tmem_store16_bits(tmem + kColState + lane_base + k0 / 2, packed);
            };
            const uint32_t chunks = (run.tokens + kC - 1) / kC;
            if constexpr (!kStateOnly) {
                put_state(done_chunks);
                tmem_store_wait();
                tc_fence_before();
                mbar_arrive(bar(kBarState));
            }
            // The state after chunk `c` of the item, whose gain is complete or about to be.
            const auto advance = [&](uint32_t c, uint32_t g) {
                const uint32_t n = min(kC, run.tokens - c * kC);
                const float hi = n == kC ? full_hi : shared.power[n], lo = n == kC ? full_lo : 0.0f;
                wait(kBarGain, g);
                tc_fence_after();
#pragma unroll
                for (uint32_t k = 0; k < kHalfK; k += 32) {
                    float gain[32];
                    tmem_load32(tmem + kColGain + lane_base + k0 + k, gain);
#pragma unroll
                    for (int x = 0; x < 32; ++x) s[k + x] = fmaf(hi, s[k + x], fmaf(lo, s[k + x], gain[x]));
                }
                tc_fence_before();
                mbar_arrive(bar(kBarGainRead));
            };
            // Outputs of chunk `c`: this thread's half of the tokens.
            float o[kC / 2];
            const auto take_output = [&](uint32_t g) {
                const float up = state_up;
#pragma unroll
                for (uint32_t i = 0; i < kC / 2; i += 16) {
                    float inner[16], outer[16];
                    tmem_load16(tmem + kColInner + lane_base + token0 + i, inner);
                    tmem_load16(tmem + kColOuter + lane_base + token0 + i, outer);
#pragma unroll
                    for (uint32_t x = 0; x < 16; ++x) {
                        const uint32_t t = token0 + i + x;
                        const float in = kIsHalf<T> ? inner[x] * shared.p_scale[g & 1u][t] : inner[x];
                        o[i + x] = fmaf(outer[x] * (kIsHalf<T> ? up : 1.0f), shared.power[t + 1], in) * p.scale;
                    }
                }
            };
            const auto store_output = [&](uint32_t c, uint32_t g) {
                const uint32_t n = min(kC, run.tokens - c * kC);
                uint32_t bad = shared.bad_from[g & 3u][0][v];
                if (half == 1) bad = min(bad, shared.bad_from[g & 3u][1][v]);
                if (!live) return;
                T* to = static_cast<T*>(p.out) + (uint64_t(run.flat_begin + c * kC + token0) * p.num_v_heads + head) * p.value_dim + v;
                const uint64_t stride = uint64_t(p.num_v_heads) * p.value_dim;
#pragma unroll
                for (uint32_t i = 0; i < kC / 2; ++i) {
                    float x = o[i];
                    if (token0 + i >= bad) x = NAN;
                    if (token0 + i < n) to[i * stride] = static_cast<T>(x);
                }
            };
            for (uint32_t c = 0; c < chunks; ++c) {
                const uint32_t g = done_chunks + c, slot = g % kStages;
                const uint32_t n = min(kC, run.tokens - c * kC);
                wait(kBarFull + slot, g / kStages);
                // weighted V of this thread's half of the tokens, in parts
                {
                    const uint32_t tile = smem_base + slot * kStageBytes + 2 * kQBytes + (token0 >> 3) * (kBlocksV * 1024) + (v >> 6) * 1024 + (v & 7u) * 2;
                    uint32_t parts[3][16];
                    float finite = 0.0f;
#pragma unroll
                    for (uint32_t j = 0; j < kC / 2; j += 2) {
                        const uint32_t at = tile + (j >> 3) * (kBlocksV * 1024);
                        const float a = ld_shared_16bit(at + (j & 7u) * 128 + ((((v >> 3) ^ j) & 7u) << 4), kIsHalf<T>);
                        const float b = ld_shared_16bit(at + ((j + 1) & 7u) * 128 + ((((v >> 3) ^ (j + 1)) & 7u) << 4), kIsHalf<T>);
                        float wa = shared.fall[token0 + j], wb = shared.fall[token0 + j + 1];
                        if (n < kC) {  // the last chunk: rows behind the run are zero
                            wa = shared.fall[min(token0 + j + (kC - n), kC - 1)];
                            wb = shared.fall[min(token0 + j + 1 + (kC - n), kC - 1)];
                        }
                        finite = fmaf(a, 0.0f, fmaf(b, 0.0f, finite));
                        uint32_t two[3];
                        split_parts<T>(a * wa, b * wb, two);
#pragma unroll
                        for (uint32_t x = 0; x < kParts; ++x) parts[x][j / 2] = two[x];
                    }
                    const uint32_t to = tmem + kColParts + (g & 1u) * kPartBuffer + lane_base + half * (kPartColumns / 2);
#pragma unroll
                    for (uint32_t x = 0; x < kParts; ++x) tmem_store16_bits(to + x * kPartColumns, parts[x]);
                    // A value that is not finite must not reach tokens before its own, whose P is zero there: it leaves the chunk's
                    // V, and the outputs from its token on are no numbers.
                    uint32_t bad = kC;
                    if (finite != finite) {
                        for (uint32_t j = 0; j < kC / 2; ++j) {
                            const uint32_t at = tile + (j >> 3) * (kBlocksV * 1024) + (j & 7u) * 128 + ((((v >> 3) ^ j) & 7u) << 4);
                            const float x = ld_shared_16bit(at, kIsHalf<T>);
                            if (!(fabsf(x) < INFINITY)) {
                                bad = min(bad, token0 + j);
                                asm volatile("st.shared.u16 [%0], %1;" ::"r"(at), "h"(uint16_t(0)) : "memory");
                            }
                        }
                        fence_async_smem();
                    }
                    shared.bad_from[g & 3u][half][v] = bad;
                    tmem_store_wait();
                    tc_fence_before();
                    mbar_arrive(bar(kBarParts + (g & 1u)));
                }
                if (c > 0) {
                    advance(c - 1, g - 1);
                    if constexpr (!kStateOnly) {
                        wait(kBarDone + (g - 1) % kStages, (g - 1) / kStages);
                        wait(kBarP, g - 1);
                        tc_fence_after();
                        take_output(g - 1);
                        put_state(g);
                        tmem_store_wait();
                        tc_fence_before();
                        mbar_arrive(bar(kBarState));
                        store_output(c - 1, g - 1);
                    }
                }
            }
            const uint32_t last = done_chunks + chunks - 1;
            advance(chunks - 1, last);
            float* to = kStateOnly ? p.carry_of(run.carry_out, head) : run.keep != 0 ? p.state_of(run.dst, head) : nullptr;
            if (to != nullptr && live) {
#pragma unroll
                for (uint32_t k = 0; k < kHalfK; ++k)
                    if (k0 + k < p.key_dim) to[uint64_t(k0 + k) * p.value_dim + v] = s[k];
            }
            wait(kBarDone + last % kStages, last / kStages);
            if constexpr (!kStateOnly) {
                wait(kBarP, last);
                pair_sync();
                tc_fence_after();
                take_output(last);
                tc_fence_before();
                store_output(chunks - 1, last);
                // the table of powers is free once the P warps and these are through
                asm volatile("bar.sync 5, 320;" ::: "memory");
            }
            done_chunks += chunks;
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
}

template <typename T, uint32_t DK, bool kStateOnly>
cudaError_t launch_one(const LinearParams& p, uint32_t ctas, cudaStream_t stream) {
    constexpr int kSmem = int(kStages * (2 * kC * DK * 2 + kC * 128 * 2) + kC * kC * 2 + 1024);
    auto kernel = linear_chunk_kernel<T, DK, kStateOnly>;
    static std::atomic<uint64_t> done{0};
    const cudaError_t err = ensure_dynamic_smem(reinterpret_cast<const void*>(kernel), kSmem, done);
    if (err != cudaSuccess) return err;
    return launch_overlapped(kernel, dim3(ctas), dim3(kChunkThreads), kSmem, stream, p);
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
