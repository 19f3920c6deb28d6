// Key weights of long query runs on the 5th-generation tensor cores (see weigh_keys.cu for the mathematics).
//
// A tile is the product of 128 query rows and 128 keys.  First pass: A = query rows, B = keys, an accumulator lane is a row, whose
// maximum and sum stay inside a thread.  Second pass: A = keys, B = query rows, a lane is a key, whose sum over the rows stays
// inside a thread, and what belongs to a row (its maximum, 1 / sum and limit) is read from shared memory.  Roles by warp, on one CTA an SM:
//   0-15   exponentials and sums; warps w, w + 4, w + 8 and w + 12 share 32 lanes, a quarter of the columns each
//   16-23  copies (cp.async from the keys' pages, any page size): key blocks into a ring, query rows into two places; they run ahead
//          of the others across blocks and items
//   24     tcgen05.mma, into four S buffers of TMEM
// Bound by the exponentials' warps: a tile's 16,384 take 1,024 cycles of the special-function unit in each pass, but the four warps of a
// scheduler go through load, maximum and exponentials in step, and a tile takes 2,000; its product takes 560 of the tensor pipe and
// its copies 650 of their warps (head_dim 128; with four copy warps, which also waited for each page ID, 2,300 bounded both passes).  Four
// prompts' ends of 4,099 to 16,384 keys, 64 tokens of 32/8 heads x 128: 101 us for both passes; eight of 4,000 to 20,000 keys, 32/4 heads x
// 256: 353.  With every warp in every role and a barrier a tile, two CTAs an SM: 104 and 486.  (A quarter of the exponentials as
// polynomials on the FMA pipe cost more issue slots than they freed.)
// Every mbarrier wait is bounded and reports PSI_ERR_TIMEOUT through the status word, and TMEM is freed on every path.
#include <type_traits>

#include "launch_util.hpp"
#include "umma_common.cuh"
#include "weigh_common.cuh"

namespace psi {

namespace {

constexpr uint32_t kRows = kWeighBlock;  // rows or keys of a block, and lanes
constexpr uint32_t kParts = 4;           // of a tile's columns
constexpr uint32_t kColumns = kRows / kParts;
constexpr uint32_t kComputeWarps = 16, kCopyWarps = 8, kComputeThreads = kComputeWarps * 32;
constexpr uint32_t kThreads = kComputeThreads + kCopyWarps * 32 + 32;
constexpr uint32_t kCopyRows = kRows / kCopyWarps;  // of a block, by one warp
constexpr uint32_t kScoreBuffers = 4, kTmemColumns = kScoreBuffers * kRows;
constexpr uint32_t kMostRing = 8;

// Of a row of kBlocks 64-element blocks: key blocks in the ring, places for query rows, and copies under way before the oldest is waited for.
__host__ __device__ constexpr uint32_t ring_blocks(uint32_t blocks) { return blocks == 1 ? 8 : blocks == 2 ? 4 : blocks == 3 ? 3 : 2; }
__host__ __device__ constexpr uint32_t row_places(uint32_t blocks) { return blocks <= 2 ? 2 : 1; }
__host__ __device__ constexpr uint32_t copies_ahead(uint32_t blocks) { return blocks <= 2 ? 3 : 2; }

struct RowNumbers {  // second pass: of a block's query rows
    __align__(16) float neg_max[kRows];
    __align__(16) float inverse[kRows];
    __align__(16) uint32_t limit[kRows];
    __align__(16) uint32_t dead[kCopyWarps];  // some of a warp's rows add nothing
};

struct UmmaWeighShared {
    uint64_t ring_full[kMostRing], ring_empty[kMostRing], score_full[kScoreBuffers], score_empty[kScoreBuffers];
    uint64_t rows_empty[2], numbers_full[2], numbers_empty[2];
    uint32_t tmem_base, abort, last_arrival;
    RowNumbers numbers[2];
    float2 stats[kParts - 1][kRows];   // what the upper parts of the columns gave, in the first pass
    float sums[2][kParts - 1][kRows];  // and in the second, of a tile and the one before
};

__device__ __forceinline__ void quad_barrier(uint32_t warp) {  // the warps that share lanes
    asm volatile("bar.sync %0, 128;" ::"r"((warp & 3u) + 1) : "memory");
}
__device__ __forceinline__ void compute_barrier() { asm volatile("bar.sync 5, %0;" ::"n"(kComputeThreads) : "memory"); }

// One item: some row blocks of a request's KV head against some of its keys.
template <bool kStats>
struct WeighItem {
    WeighRequest rq;
    uint32_t rows, head, block_begin, block_end, k_begin, k_end, pieces, unit;
    __device__ __forceinline__ WeighItem(const WeighParams& p, const WeighRequest* reqs, uint32_t count, uint32_t cut, uint32_t item) {
        rq = reqs[kStats ? find_request<0>(reqs, count, item) : find_request<1>(reqs, count, item)];
        rows = rq.q_len * p.group;
        const uint32_t blocks = (rows + kRows - 1) / kRows, cuts = weigh_cut(rq.keys, cut);
        if (kStats) {
            pieces = cuts;
            const uint32_t local = item - rq.cu0;
            unit = local / pieces;
            head = unit / blocks;
            block_begin = unit % blocks;
            block_end = block_begin + 1;
            k_begin = local % pieces * cut * kRows;
        } else {
            pieces = p.split_rows != 0 ? weigh_row_parts(rows, rq.keys, p.geo.num_kv_heads, true) : 1u;
            const uint32_t local = item - rq.cu1, each = weigh_part_blocks(rows, pieces, true);
            unit = local / pieces;
            head = unit / cuts;
            block_begin = local % pieces * each;
            block_end = min(block_begin + each, blocks);
            k_begin = unit % cuts * cut * kRows;
            // rows of tokens before the span's first key see none of it
            if (k_begin > rq.first_pos) block_begin = max(block_begin, uint32_t(uint64_t(k_begin - rq.first_pos) * p.group / kRows));
        }
        k_end = min(k_begin + cut * kRows, rq.keys);
    }
    // The item's keys that some row of the block sees end here.
    __device__ __forceinline__ uint32_t seen(const WeighParams& p, uint32_t block) const {
        return min(k_end, row_limit(p, rq, min((block + 1) * kRows, rows) - 1));
    }
    __device__ __forceinline__ uint32_t tiles(const WeighParams& p, uint32_t block) const {
        const uint32_t end = seen(p, block);
        return end > k_begin ? (end - k_begin + kRows - 1) / kRows : 0u;
    }
};

// kBlocks: 64-element blocks of a row.  kStats: first pass.
template <typename T, uint32_t kBlocks, bool kStats>
__global__ void __launch_bounds__(kThreads, 1) weigh_umma_kernel(const WeighParams p) {
    constexpr uint32_t kTileBytes = kBlocks * kRows * 128;  // a block of 128 rows: [64-element block][row][128 bytes, swizzled]
    constexpr uint32_t kRing = ring_blocks(kBlocks), kPlaces = row_places(kBlocks), kAhead = copies_ahead(kBlocks);
    static_assert(kAhead <= kRing && kRing <= kMostRing);
    __shared__ UmmaWeighShared sh;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u;
    const uint32_t smem_rows = (smem_u32(smem_raw) + 1023u) & ~1023u, smem_ring = smem_rows + kPlaces * kTileBytes;
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem_base)), "r"(kTmemColumns) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (tid == 0) {
        for (uint32_t i = 0; i < kMostRing; ++i) {
            mbar_init(smem_u32(&sh.ring_full[i]), kCopyWarps);
            mbar_init(smem_u32(&sh.ring_empty[i]), 1);
        }
        for (uint32_t i = 0; i < kScoreBuffers; ++i) {
            mbar_init(smem_u32(&sh.score_full[i]), 1);
            mbar_init(smem_u32(&sh.score_empty[i]), kComputeWarps);
        }
        for (uint32_t i = 0; i < 2; ++i) {
            mbar_init(smem_u32(&sh.rows_empty[i]), 1);
            mbar_init(smem_u32(&sh.numbers_full[i]), kCopyWarps);
            mbar_init(smem_u32(&sh.numbers_empty[i]), kComputeWarps);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        sh.abort = 0;
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sh.tmem_base;
    await_previous_kernel();
    const uint32_t count = p.scalars[kScalarWeighLong];
    const WeighRequest* reqs = p.long_reqs();
    const uint32_t total = count == 0 ? 0u : kStats ? reqs[count].cu0 : reqs[count].cu1;
    const uint32_t cut = kStats ? reqs[count].slot : reqs[count].first_pos;

    // The n-th completion of a barrier (n from 0).  Bounded; once one wait has given up, none waits any more.
    const auto wait = [&](const uint64_t& barrier, uint32_t n) {
        const uint32_t bar = smem_u32(&barrier);
        if (mbar_try(bar, n & 1u)) return;
        if (*reinterpret_cast<volatile uint32_t*>(&sh.abort) == 0 && !mbar_wait(bar, n & 1u)) {
            *reinterpret_cast<volatile uint32_t*>(&sh.abort) = 1;
            if (p.geo.fault != nullptr) atomicExch(p.geo.fault, uint32_t(PSI_ERR_TIMEOUT));
        }
    };

    // All roles go through the same items, blocks and tiles; t and b count the tiles, and the blocks with tiles, over all items.
    if (warp < kComputeWarps) {
        const uint32_t row = tid & (kRows - 1), part = tid >> 7;
        const uint32_t column0 = part * kColumns, at = tmem + (((warp & 3u) * 32u) << 16) + column0;
        const uint64_t scale2 = pack_f32x2(p.scale_log2, p.scale_log2);
        uint32_t t = 0, b = 0;
        for (uint32_t item = blockIdx.x; item < total; item += gridDim.x) {
            const WeighItem<kStats> it(p, reqs, count, cut, item);
            const auto scores = [&](float (&s)[kColumns]) {  // of tile t
                wait(sh.score_full[t % kScoreBuffers], t / kScoreBuffers);
                __syncwarp();
                tc_fence_after();
                tmem_load32(at + (t % kScoreBuffers) * kRows, s);
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&sh.score_empty[t % kScoreBuffers]));
            };
            if constexpr (kStats) {
                const uint32_t my_row = it.block_begin * kRows + row, tiles = it.tiles(p, it.block_begin);
                const uint32_t my_limit = my_row < it.rows ? min(it.k_end, row_limit(p, it.rq, my_row)) : 0u;
                Stat st{-kInf, 0.0f};
                for (uint32_t tile = 0; tile < tiles; ++tile, ++t) {
                    float s[kColumns];
                    scores(s);
                    const uint32_t key = it.k_begin + tile * kRows + column0;
                    if (key + kColumns > my_limit) {
#pragma unroll
                        for (uint32_t c = 0; c < kColumns; ++c)
                            if (key + c >= my_limit) s[c] = -kInf;
                    }
                    float tops[4] = {-kInf, -kInf, -kInf, -kInf};
#pragma unroll
                    for (uint32_t c = 0; c < kColumns; c += 2) tops[c >> 1 & 3] = max3_nan(tops[c >> 1 & 3], s[c], s[c + 1]);  // (a NaN leaves no sum)
                    float top = max3_nan(max3_nan(tops[0], tops[1], tops[2]), tops[3], tops[3]);
                    top = max3_nan(st.m, st.m, top * p.scale_log2);
                    const float base = top == -kInf ? 0.0f : top;
                    st.l *= fast_exp2(st.m - base);
                    st.m = top;
                    const uint64_t base2 = pack_f32x2(-base, -base);
                    uint64_t sum[4] = {0, 0, 0, 0};
#pragma unroll
                    for (uint32_t c = 0; c < kColumns; c += 2) {
                        const float2 x = unpack_f32x2(fma_f32x2(pack_f32x2(s[c], s[c + 1]), scale2, base2));
                        sum[c >> 1 & 3] = add_f32x2(sum[c >> 1 & 3], pack_f32x2(fast_exp2(x.x), fast_exp2(x.y)));
                    }
                    const float2 all = unpack_f32x2(add_f32x2(add_f32x2(sum[0], sum[1]), add_f32x2(sum[2], sum[3])));
                    st.l += all.x + all.y;
                }
                if (part > 0) sh.stats[part - 1][row] = make_float2(st.m, st.l);
                quad_barrier(warp);
                if (part == 0) {
#pragma unroll
                    for (uint32_t x = 0; x + 1 < kParts; ++x) st.join(sh.stats[x][row].x, sh.stats[x][row].y);
                    if (it.pieces > 1)
                        p.long_partials()[uint64_t(item) * kRows + row] = make_float2(st.m, st.l);
                    else if (my_row < it.rows)
                        p.norms[query_row(p, it.rq, it.head, my_row)] = st.norm();
                }
                quad_barrier(warp);  // (what the parts gave has been read)
                if (it.pieces > 1) {  // the last piece of the row block joins the pieces
                    __threadfence();
                    compute_barrier();
                    uint32_t* counter = p.long_counters() + it.rq.unit0 + it.unit;
                    if (tid == 0) sh.last_arrival = atomicAdd(counter, 1u) == it.pieces - 1 ? 1u : 0u;
                    compute_barrier();
                    if (sh.last_arrival != 0) {
                        __threadfence();
                        if (part == 0 && my_row < it.rows) {
                            Stat all{-kInf, 0.0f};
                            for (uint32_t o = 0; o < it.pieces; ++o) {
                                const float2 v = __ldcg(p.long_partials() + uint64_t(it.rq.cu0 + it.unit * it.pieces + o) * kRows + row);
                                all.join(v.x, v.y);
                            }
                            p.norms[query_row(p, it.rq, it.head, my_row)] = all.norm();
                        }
                        if (tid == 0) *counter = 0;
                    }
                    compute_barrier();
                }
            } else {
                // where a key's sum goes: its weight, or this part's share of it; the same thread's from block to block
                float* const sums = it.pieces > 1 ? p.sums + uint64_t(item) * (cut * kRows) - it.k_begin : weight_row(p, it.rq, it.head);
                if (it.pieces > 1 && part == 0)
                    for (uint32_t key = it.k_begin + row; key < it.k_end; key += kRows) sums[key] = 0.0f;
                for (uint32_t block = it.block_begin; block < it.block_end; ++block) {
                    const uint32_t row0 = block * kRows, tiles = it.tiles(p, block);
                    if (tiles == 0) continue;
                    const RowNumbers& numbers = sh.numbers[b & 1u];
                    wait(sh.numbers_full[b & 1u], b >> 1);
                    const uint4 dead0 = *reinterpret_cast<const uint4*>(numbers.dead), dead1 = *reinterpret_cast<const uint4*>(numbers.dead + 4);
                    const bool odd_rows = row0 + kRows > it.rows || (dead0.x | dead0.y | dead0.z | dead0.w | dead1.x | dead1.y | dead1.z | dead1.w) != 0;
                    const uint32_t first_limit = row_limit(p, it.rq, row0);
                    for (uint32_t tile = 0; tile < tiles; ++tile, ++t) {
                        const uint32_t key = it.k_begin + tile * kRows + row;
                        float before = 0.0f;
                        if (part == 0 && key < it.k_end) before = sums[key];
                        uint64_t sum[4] = {0, 0, 0, 0};
                        float s[kColumns];
                        scores(s);
                        const auto columns = [&](const auto with_mask) {
#pragma unroll
                            for (uint32_t c = 0; c < kColumns; c += 4) {
                                const ulonglong2 base = *reinterpret_cast<const ulonglong2*>(&numbers.neg_max[column0 + c]);
                                const ulonglong2 inverse = *reinterpret_cast<const ulonglong2*>(&numbers.inverse[column0 + c]);
                                float2 x = unpack_f32x2(fma_f32x2(pack_f32x2(s[c], s[c + 1]), scale2, base.x));
                                float2 y = unpack_f32x2(fma_f32x2(pack_f32x2(s[c + 2], s[c + 3]), scale2, base.y));
                                x = make_float2(fast_exp2(x.x), fast_exp2(x.y));
                                y = make_float2(fast_exp2(y.x), fast_exp2(y.y));
                                if constexpr (decltype(with_mask)::value) {
                                    const uint4 limit = *reinterpret_cast<const uint4*>(&numbers.limit[column0 + c]);
                                    const float2 i0 = unpack_f32x2(inverse.x), i1 = unpack_f32x2(inverse.y);
                                    x.x = key < limit.x && i0.x > 0.0f ? x.x : 0.0f;
                                    x.y = key < limit.y && i0.y > 0.0f ? x.y : 0.0f;
                                    y.x = key < limit.z && i1.x > 0.0f ? y.x : 0.0f;
                                    y.y = key < limit.w && i1.y > 0.0f ? y.y : 0.0f;
                                }
                                sum[c >> 2 & 1] = fma_f32x2(pack_f32x2(x.x, x.y), inverse.x, sum[c >> 2 & 1]);
                                sum[2 + (c >> 2 & 1)] = fma_f32x2(pack_f32x2(y.x, y.y), inverse.y, sum[2 + (c >> 2 & 1)]);
                            }
                        };
                        if (odd_rows || it.k_begin + (tile + 1) * kRows > first_limit)
                            columns(std::true_type{});
                        else
                            columns(std::false_type{});
                        const float2 two = unpack_f32x2(add_f32x2(add_f32x2(sum[0], sum[1]), add_f32x2(sum[2], sum[3])));
                        float all = two.x + two.y;
                        if (part > 0) sh.sums[t & 1u][part - 1][row] = all;
                        quad_barrier(warp);  // (behind it the first part reads; the place is written again two tiles on, behind the next barrier)
                        if (part == 0 && key < it.k_end) {
#pragma unroll
                            for (uint32_t x = 0; x + 1 < kParts; ++x) all += sh.sums[t & 1u][x][row];
                            sums[key] = before + all;
                        }
                    }
                    __syncwarp();
                    if (lane == 0) mbar_arrive(smem_u32(&sh.numbers_empty[b & 1u]));
                    ++b;
                }
                if (it.pieces > 1) {  // the last part of the span adds up the parts
                    __threadfence();
                    compute_barrier();
                    uint32_t* counter = p.long_counters() + it.rq.cu1 + it.unit * it.pieces;
                    if (tid == 0) sh.last_arrival = atomicAdd(counter, 1u) == it.pieces - 1 ? 1u : 0u;
                    compute_barrier();
                    if (sh.last_arrival != 0) {
                        __threadfence();
                        for (uint32_t i = tid; i < it.k_end - it.k_begin; i += kComputeThreads) {
                            float all = 0.0f;
                            for (uint32_t o = 0; o < it.pieces; ++o) all += __ldcg(p.sums + uint64_t(it.rq.cu1 + it.unit * it.pieces + o) * (cut * kRows) + i);
                            weight_row(p, it.rq, it.head)[it.k_begin + i] += all;
                        }
                        if (tid == 0) *counter = 0;
                    }
                    compute_barrier();
                }
            }
        }
    } else if (warp < kComputeWarps + kCopyWarps) {
        // A warp copies its own 16 rows of every block: two lanes find a row's offset, then kLanes lanes copy each row, a chunk of 16
        // bytes each, whose place in the swizzle stays the same from row to row (a lane's rows are a multiple of eight apart).
        constexpr uint32_t kLanes = kBlocks == 3 ? 32 : kBlocks * 8, kSide = 32 / kLanes;
        const uint32_t w = warp - kComputeWarps, chunks = p.geo.head_dim >> 3;
        const uint32_t chunk = lane % kLanes, side = lane / kLanes;
        const bool copies = chunk < kBlocks * 8, has_data = chunk < chunks;
        const uint32_t my_place = w * kCopyRows + (lane & (kCopyRows - 1));  // the row whose offset this lane finds
        const PageBounds bounds(p.geo);
        uint32_t bad = 0;
        const auto copy_rows = [&](uint32_t dst, const void* base, uint64_t offset) {  // offset: of this lane's row in elements, ~0 for zeros
            const uint16_t* from = static_cast<const uint16_t*>(base) + (has_data ? chunk * 8u : 0u);
            const uint32_t to = dst + (chunk >> 3) * (kRows * 128) + w * kCopyRows * 128;
#pragma unroll
            for (uint32_t i = 0; i < kCopyRows; i += kSide) {
                const uint32_t r = i + side;
                const uint64_t of_row = __shfl_sync(0xFFFFFFFFu, offset, r);
                const bool live = has_data && of_row != ~0ull;
                if (copies) cp_async_16(to + r * 128 + (((chunk ^ r) & 7u) << 4), from + (live ? of_row : 0u), live ? 16u : 0u);
            }
        };
        uint32_t t = 0, b = 0, landed = 0;  // tiles copied, and those of them that have been handed on
        uint32_t last_end = 0, before_last_end = 0;  // t behind the last block, and behind the one before it
        const auto hand_on = [&](uint32_t to) {  // (the copies of tiles before `to` have come back)
            fence_async_smem();
            __syncwarp();
            for (; landed < to; ++landed)
                if (lane == 0) mbar_arrive(smem_u32(&sh.ring_full[landed % kRing]));
        };
        for (uint32_t item = blockIdx.x; item < total; item += gridDim.x) {
            const WeighItem<kStats> it(p, reqs, count, cut, item);
            const uint32_t* row_ids = table_row(p.geo, it.rq.slot);
            for (uint32_t block = it.block_begin; block < it.block_end; ++block) {
                const uint32_t tiles = it.tiles(p, block);
                if (tiles == 0) continue;
                // a row's page ID is read a tile ahead, and first looked at when the tile is copied
                const auto key_of = [&](uint32_t tile) { return it.k_begin + tile * kRows + my_place; };
                const auto page_of = [&](uint32_t tile) { return key_of(tile) < it.k_end ? bounds.read(row_ids, key_of(tile) / p.geo.tokens_per_page, bad) : 0u; };
                const uint32_t my_row = block * kRows + my_place;
                const bool is_row = my_row < it.rows;
                const uint64_t at = is_row ? query_row(p, it.rq, it.head, my_row) : 0u;
                uint32_t page = page_of(0);
                // The block before last, or with one place the last, must have been handed on whole before its place is waited for.
                if (landed < (kPlaces == 1 ? last_end : before_last_end)) {
                    cp_async_wait<0>();
                    hand_on(t);
                }
                if (b >= kPlaces) wait(sh.rows_empty[b % kPlaces], b / kPlaces - 1);
                copy_rows(smem_rows + b % kPlaces * kTileBytes, p.q, is_row ? at * p.geo.head_dim : ~0ull);
                if constexpr (!kStats) {
                    // (the numbers' two places: with one place for rows, the block before last is done with as well)
                    if (b >= 2) wait(sh.numbers_empty[b & 1u], (b >> 1) - 1);
                    RowNumbers& numbers = sh.numbers[b & 1u];
                    const float2 norm = is_row ? p.norms[at] : make_float2(kInf, 0.0f);
                    numbers.neg_max[my_place] = -norm.x;
                    numbers.inverse[my_place] = norm.y;
                    numbers.limit[my_place] = is_row ? row_limit(p, it.rq, my_row) : 0u;
                    const bool dead = __any_sync(0xFFFFFFFFu, is_row && norm.y == 0.0f) != 0;
                    if (lane == 0) numbers.dead[w] = dead ? 1u : 0u;
                    __syncwarp();
                    if (lane == 0) mbar_arrive(smem_u32(&sh.numbers_full[b & 1u]));
                }
                for (uint32_t tile = 0; tile < tiles; ++tile) {
                    const uint32_t key = key_of(tile);
                    const uint64_t offset = key < it.k_end ? kv_row_offset(p.geo, page, it.head, key % p.geo.tokens_per_page) : ~0ull;
                    if (tile + 1 < tiles) page = page_of(tile + 1);
                    if (t >= kRing) wait(sh.ring_empty[t % kRing], t / kRing - 1);
                    copy_rows(smem_ring + t % kRing * kTileBytes, p.geo.pages, offset);
                    cp_async_commit();
                    ++t;
                    cp_async_wait<kAhead - 1>();
                    if (t >= kAhead) hand_on(t - kAhead + 1);
                }
                before_last_end = last_end;
                last_end = t;
                ++b;
            }
        }
        cp_async_wait<0>();
        hand_on(t);
        if (bad != 0) record_page_fault(p.geo);
    } else {
        const uint32_t idesc = umma_idesc<T>(kRows, false);
        uint32_t t = 0, b = 0;
        for (uint32_t item = blockIdx.x; item < total; item += gridDim.x) {
            const WeighItem<kStats> it(p, reqs, count, cut, item);
            for (uint32_t block = it.block_begin; block < it.block_end; ++block) {
                const uint32_t tiles = it.tiles(p, block);
                if (tiles == 0) continue;
                for (uint32_t tile = 0; tile < tiles; ++tile, ++t) {
                    wait(sh.ring_full[t % kRing], t / kRing);
                    if (t >= kScoreBuffers) wait(sh.score_empty[t % kScoreBuffers], t / kScoreBuffers - 1);
                    tc_fence_after();
                    __syncwarp();
                    if (elect_one()) {
                        const uint32_t rows_at = smem_rows + b % kPlaces * kTileBytes, ring = smem_ring + t % kRing * kTileBytes;
                        const uint64_t a_desc = umma_desc(kStats ? rows_at : ring, 16, 1024), b_desc = umma_desc(kStats ? ring : rows_at, 16, 1024);
#pragma unroll
                        for (uint32_t ks = 0; ks < kBlocks * 4; ++ks) {
                            const uint32_t step = ((ks >> 2) * (kRows * 128) + (ks & 3) * 32) / 16;
                            umma_ss(tmem + t % kScoreBuffers * kRows, a_desc + step, b_desc + step, idesc, ks);
                        }
                        umma_commit_one(smem_u32(&sh.ring_empty[t % kRing]));
                        umma_commit_one(smem_u32(&sh.score_full[t % kScoreBuffers]));
                        if (tile + 1 == tiles) umma_commit_one(smem_u32(&sh.rows_empty[b % kPlaces]));
                    }
                    __syncwarp();
                }
                ++b;
            }
        }
        // no product is under way when TMEM and shared memory go, whatever wait gave up
        if (t > 0) (void)mbar_wait(smem_u32(&sh.ring_empty[(t - 1) % kRing]), ((t - 1) / kRing) & 1u);
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemColumns) : "memory");
}

template <typename T, uint32_t kBlocks, bool kStats>
cudaError_t launch_one(const WeighParams& p, uint32_t ctas, cudaStream_t stream) {
    constexpr int kSmem = int((ring_blocks(kBlocks) + row_places(kBlocks)) * kBlocks * kRows * 128 + 1024);
    static_assert(kSmem > 114 * 1024, "one CTA an SM: each takes all of its TMEM");
    static std::atomic<uint64_t> done{0};
    const cudaError_t err = ensure_dynamic_smem(reinterpret_cast<const void*>(weigh_umma_kernel<T, kBlocks, kStats>), kSmem, done);
    if (err != cudaSuccess) return err;
    return launch_overlapped(weigh_umma_kernel<T, kBlocks, kStats>, dim3(ctas), dim3(kThreads), kSmem, stream, p);
}

template <typename T, uint32_t kBlocks>
cudaError_t launch_pass(const WeighParams& p, bool stats, uint32_t ctas, cudaStream_t stream) {
    return stats ? launch_one<T, kBlocks, true>(p, ctas, stream) : launch_one<T, kBlocks, false>(p, ctas, stream);
}

template <typename T>
cudaError_t launch_typed(const WeighParams& p, bool stats, uint32_t ctas, cudaStream_t stream) {
    switch ((p.geo.head_dim + 63) / 64) {
        case 1: return launch_pass<T, 1>(p, stats, ctas, stream);
        case 2: return launch_pass<T, 2>(p, stats, ctas, stream);
        case 3: return launch_pass<T, 3>(p, stats, ctas, stream);
        default: return launch_pass<T, 4>(p, stats, ctas, stream);
    }
}

}  // namespace

cudaError_t launch_weigh_umma(const WeighParams& p, bool stats, uint32_t ctas, cudaStream_t stream) {
    return p.dtype == PSI_DTYPE_BF16 ? launch_typed<__nv_bfloat16>(p, stats, ctas, stream) : launch_typed<__half>(p, stats, ctas, stream);
}

}  // namespace psi
