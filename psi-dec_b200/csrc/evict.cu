// Eviction from the paged cache by accumulated attention weight (psi_gqa_evict).
//
// evict_select_kernel: one to eight CTAs (a cluster) for each (request, KV head) hold the row's weights in shared memory, find the
// weight of the last kept key by a radix selection over order-preserving 32-bit keys (11, 11 and 10 bits, a histogram each, summed
// over the cluster; it ends as soon as a digit's keys belong all or not at all), then write the kept indices in ascending order with
// one ordered scan, which also brings the weights to their new places.  Counts are whole numbers, so ties and results do not
// depend on the order of the atomics.  The weights are read once; the histograms and the scan bound it: 18 us for 64 rows of 1,024 to
// 8,192 weights, 40 us for 16 rows of 65,001 to 131,072 on eight CTAs each.
// evict_move_kernel / evict_move_in_place_kernel: the kept K and V rows to the front of the destination slot: bound by the
// bytes of the rows, read and written once.  As many lanes as a row has 16-byte units take one, so that page IDs and addresses are
// worked out once for a row.  Into another slot every row is independent.  In place a row moves to a lower or
// equal index: a CTA takes one column slice of one head's K or V and goes through the rows in order, a batch in registers
// between its loads and its stores, so that nothing is overwritten that a later batch reads.  Half of 32 caches of 1,024 to 8,192
// keys, 2 heads x 256, bf16, into other slots: 52 us, 5.8 TB/s; a quarter of two of 65,001 to 131,072, 8 heads x 128, f32: 129 us, 6.2 TB/s.
// In place, selection included, the same take 183 and 521 us: the rows of a slice one batch after another, two barriers each.
// A row above 393,216 keys fits no cluster's shared memory: one CTA reads it again in each round (400,003 keys, 8 heads: 1.2 ms).
#include <cooperative_groups.h>

#include "device_common.cuh"
#include "evict.hpp"
#include "launch_util.hpp"

namespace psi {

namespace {

constexpr uint32_t kSelectThreads = 512;  // (1,024: 44 us a row of 131,072 keys on eight CTAs, 40 with 512)
constexpr uint32_t kBins = 2048;
constexpr uint32_t kMostCtas = 8;              // of a cluster
constexpr uint32_t kSliceKeys = 48 * 1024;     // of a row in one CTA's shared memory

// Order-preserving key of a weight: NaN below everything, -0 as 0.
__device__ __forceinline__ uint32_t weight_key(float w) {
    if (w != w) return 0u;
    const uint32_t bits = __float_as_uint(w + 0.0f);
    return (bits & 0x80000000u) != 0 ? ~bits : bits | 0x80000000u;
}

// Exclusive sum of `value` over the block's threads, and the block's total.
__device__ __forceinline__ uint32_t block_scan(uint32_t value, uint32_t* warp_sums, uint32_t& total) {
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
    uint32_t sum = value;
#pragma unroll
    for (int x = 1; x < 32; x <<= 1) {
        const uint32_t other = __shfl_up_sync(0xFFFFFFFFu, sum, x);
        if (lane >= uint32_t(x)) sum += other;
    }
    constexpr uint32_t kWarps = kSelectThreads / 32;
    __syncthreads();
    if (lane == 31) warp_sums[warp] = sum;
    __syncthreads();
    uint32_t sums = lane < kWarps ? warp_sums[lane] : 0u;
#pragma unroll
    for (int x = 1; x < 32; x <<= 1) {
        const uint32_t other = __shfl_up_sync(0xFFFFFFFFu, sums, x);
        if (lane >= uint32_t(x)) sums += other;
    }
    total = __shfl_sync(0xFFFFFFFFu, sums, 31);
    const uint32_t before = __shfl_sync(0xFFFFFFFFu, sums, (warp + 31u) & 31u);
    return (warp == 0 ? 0u : before) + sum - value;
}

struct SelectShared {
    uint32_t bins[kBins];
    uint32_t warp_sums[kSelectThreads / 32];
    uint32_t digit, above, count;  // of the digit that holds the last wanted key: keys above it, keys in it
    uint32_t segment;              // keys of this CTA's share of the digits, over the cluster
    uint32_t slice_above, slice_equal;
};

// grid (x: request * CTAs of a cluster + rank, y: KV head).  kHeld: the row's slice of weights fits the CTA's shared memory;
// otherwise one CTA reads it again in every pass.
template <bool kHeld>
__global__ __launch_bounds__(kSelectThreads) void evict_select_kernel(const EvictParams p) {
    namespace cg = cooperative_groups;
    cg::cluster_group cluster = cg::this_cluster();
    extern __shared__ __align__(16) float held[];
    __shared__ SelectShared sh;
    await_previous_kernel();
    const uint32_t ctas = kHeld ? cluster.num_blocks() : 1u, rank = kHeld ? cluster.block_rank() : 0u;
    const uint32_t index = blockIdx.x / ctas;
    const EvictRequest rq = p.reqs[index];
    const uint32_t head = blockIdx.y, heads = p.geo.num_kv_heads;
    const float* w = p.weights + (uint64_t(rq.src) * heads + head) * p.stride;
    float* out = p.weights_out + (uint64_t(rq.dst) * heads + head) * p.stride;
    uint32_t* kept = p.kept + (uint64_t(index) * heads + head) * p.kept_stride;
    const uint32_t recent = min(p.recent, rq.keep), pool = rq.length - recent;
    uint32_t want = rq.keep - recent;  // of the first `pool` keys
    const uint32_t slice = ((rq.length + ctas - 1) / ctas + 3u) & ~3u, begin = min(rank * slice, rq.length), end = min(begin + slice, rq.length);
    const uint32_t pool_end = max(begin, min(end, pool));
    if (kHeld) {
#pragma unroll 8
        for (uint32_t i = begin + threadIdx.x; i < end; i += kSelectThreads) held[i - begin] = w[i];
    }
    const auto weight_at = [&](uint32_t i) { return kHeld ? held[i - begin] : w[i]; };
    const auto meet = [&] {
        if (kHeld && ctas > 1) cluster.sync();
        else __syncthreads();
    };
    // `threshold`: keys above it belong, and the first `want` of those equal to it.
    uint32_t threshold = 0;
    if (want > 0 && want < pool) {
#pragma unroll 1
        for (uint32_t pass = 0; pass < 3; ++pass) {
            const uint32_t shift = pass == 0 ? 21u : pass == 1 ? 10u : 0u, digits = pass == 2 ? 1024u : 2048u, above = pass == 1 ? 21u : 10u;
            for (uint32_t i = threadIdx.x; i < kBins; i += kSelectThreads) sh.bins[i] = 0;
            __syncthreads();
            for (uint32_t base = begin; base < pool_end; base += kSelectThreads) {
                const uint32_t i = base + threadIdx.x;
                const uint32_t key = i < pool_end ? weight_key(weight_at(i)) : 0u;
                const bool counts = i < pool_end && (pass == 0 || (key >> above) == (threshold >> above));
                const uint32_t digit = (key >> shift) & (digits - 1), active = __ballot_sync(0xFFFFFFFFu, counts);
                if (counts) {
                    // where a warp's keys agree (zeros, most often) one of its lanes counts for all
                    int same = 0;
                    __match_all_sync(active, digit, &same);
                    if (!same) atomicAdd(&sh.bins[digit], 1u);
                    else if ((threadIdx.x & 31u) == uint32_t(__ffs(active)) - 1u) atomicAdd(&sh.bins[digit], uint32_t(__popc(active)));
                }
            }
            meet();
            // From the top digit down, each CTA of a cluster adds up its share of the digits; a thread holds up to four of them.
            const uint32_t per_cta = digits / ctas, per = (per_cta + kSelectThreads - 1) / kSelectThreads;
            uint32_t bin[kBins / kSelectThreads], mine = 0;
#pragma unroll
            for (uint32_t i = 0; i < kBins / kSelectThreads; ++i) {
                const uint32_t place = threadIdx.x * per + i;
                bin[i] = 0;
                if (i >= per || place >= per_cta) continue;
                const uint32_t digit = digits - 1 - (rank * per_cta + place);
                if (kHeld && ctas > 1) {
#pragma unroll
                    for (uint32_t c = 0; c < kMostCtas; ++c)
                        if (c < ctas) bin[i] += *cluster.map_shared_rank(&sh.bins[digit], c);
                } else {
                    bin[i] = sh.bins[digit];
                }
                mine += bin[i];
            }
            uint32_t total = 0;
            uint32_t before = block_scan(mine, sh.warp_sums, total);
            if (threadIdx.x == 0) sh.segment = total;
            meet();  // (the other CTAs have read these bins)
            uint32_t segments_before = 0, owner = rank;
            if (kHeld && ctas > 1) {
                uint32_t sum = 0;
                for (uint32_t c = 0; c < ctas; ++c) {
                    const uint32_t next = sum + *cluster.map_shared_rank(&sh.segment, c);
                    if (sum < want && want <= next) owner = c;
                    if (c < rank) segments_before = next;
                    sum = next;
                }
            }
            before += segments_before;
            if (owner == rank && before < want && want <= before + mine) {
#pragma unroll
                for (uint32_t i = 0; i < kBins / kSelectThreads; ++i) {
                    if (before < want && want <= before + bin[i]) {
                        sh.digit = digits - 1 - (rank * per_cta + threadIdx.x * per + i);
                        sh.above = before;
                        sh.count = bin[i];
                    }
                    before += bin[i];
                }
            }
            meet();
            const SelectShared* at = kHeld && ctas > 1 ? cluster.map_shared_rank(&sh, owner) : &sh;
            const uint32_t digit = at->digit, digit_above = at->above, digit_count = at->count;
            threshold |= digit << shift;
            want -= digit_above;
            if (want == digit_count) {  // the whole digit belongs: everything above the key below its lowest one
                threshold -= 1;      // (no underflow: a key of 0 is a NaN's, and with it all of the pool would be wanted)
                want = 0;
                break;
            }
            meet();  // (the next digit's words replace these)
        }
    } else if (want == 0) {
        threshold = 0xFFFFFFFFu;  // no weight has this key: it is a NaN's
    }  // want == pool: every key is above or equal to 0, all equal ones belong
    // One ordered scan: low half counts the keys above the threshold (recent ones among them), high half those equal to it.
    constexpr uint32_t kEach = 4;
    const auto mark_of = [&](uint32_t at, float value) {
        const uint32_t key = weight_key(value);
        return at >= end ? 0u : (at >= pool || key > threshold) ? 1u : key == threshold ? 0x10000u : 0u;
    };
    uint32_t above_before = 0, equal_before = 0;
    if (kHeld && ctas > 1) {
        // what the slices before this one hold of both kinds
        uint32_t above = 0, equal = 0;
        for (uint32_t i = begin + threadIdx.x; i < end; i += kSelectThreads) {
            const uint32_t mark = mark_of(i, held[i - begin]);
            above += mark & 1u;
            equal += mark >> 16;
        }
        uint32_t sum = 0;
        (void)block_scan(above, sh.warp_sums, sum);
        if (threadIdx.x == 0) sh.slice_above = sum;
        (void)block_scan(equal, sh.warp_sums, sum);
        if (threadIdx.x == 0) sh.slice_equal = sum;
    }
    meet();  // every CTA has its weights: they may be overwritten
    if (kHeld && ctas > 1) {
        for (uint32_t c = 0; c < rank; ++c) {
            above_before += *cluster.map_shared_rank(&sh.slice_above, c);
            equal_before += *cluster.map_shared_rank(&sh.slice_equal, c);
        }
    }
    for (uint32_t base = begin; base < end; base += kSelectThreads * kEach) {
        const uint32_t first = base + threadIdx.x * kEach;
        float value[kEach];
        uint32_t mark[kEach], mine = 0;
#pragma unroll
        for (uint32_t i = 0; i < kEach; ++i) {
            const uint32_t at = first + i;
            value[i] = at < end ? weight_at(at) : 0.0f;
            mark[i] = mark_of(at, value[i]);
            mine += mark[i];
        }
        uint32_t total = 0;
        const uint32_t before = block_scan(mine, sh.warp_sums, total);  // every thread has read its weights
        uint32_t above = above_before + (before & 0xFFFFu), equal = equal_before + (before >> 16);
#pragma unroll
        for (uint32_t i = 0; i < kEach; ++i) {
            if (mark[i] == 1u || (mark[i] != 0u && equal < want)) {
                const uint32_t to = above + min(equal, want);
                kept[to] = first + i;
                out[to] = value[i];
            }
            above += mark[i] & 1u;
            equal += mark[i] >> 16;
        }
        above_before += total & 0xFFFFu;
        equal_before += total >> 16;
    }
    // the places that came free: not before the last stores into [0, keep), which are elsewhere, nor before the last reads
    __syncthreads();
    const uint32_t free_step = (rq.length - rq.keep + ctas - 1) / ctas, free_begin = rq.keep + rank * free_step;
    const uint32_t free_end = min(free_begin + free_step, rq.length);
    for (uint32_t i = free_begin + threadIdx.x; i < free_end; i += kSelectThreads) out[i] = 0.0f;
    if (kHeld && ctas > 1) cluster.sync();  // nobody's shared memory goes before the others have read it
}

template <typename Unit>
__device__ __forceinline__ Unit* row_units(const PageGeometry& g, const PageBounds& bounds, const uint32_t* ids, uint32_t head,
                                           uint32_t token, bool value, uint32_t& bad) {
    const uint32_t page = bounds.read(ids, token / g.tokens_per_page, bad);
    const uint64_t at = kv_row_offset(g, page, head, token % g.tokens_per_page) + (value ? v_region_offset(g) : 0u);
    return reinterpret_cast<Unit*>(static_cast<unsigned char*>(const_cast<void*>(g.pages)) + at * g.elem_bytes);
}

constexpr uint32_t kMoveThreads = 256;
constexpr uint32_t kMoveEach = 4;  // rows of a lane group between its loads and its stores

// Lanes that share a row of `units` units: a power of two up to 32.
__device__ __forceinline__ uint32_t row_lanes(uint32_t units) { return units >= 32 ? 32u : units <= 1 ? 1u : 1u << (32 - __clz(units - 1)); }

// Into another slot: grid (x: stride over rows, y: KV head, z: request).
template <typename Unit>
__global__ __launch_bounds__(kMoveThreads) void evict_move_kernel(const EvictParams p) {
    await_previous_kernel();
    const EvictRequest rq = p.reqs[blockIdx.z];
    if (rq.src == rq.dst || rq.keep == 0) return;
    const uint32_t head = blockIdx.y;
    const uint32_t* kept = p.kept + (uint64_t(blockIdx.z) * p.geo.num_kv_heads + head) * p.kept_stride;
    const uint32_t* src_ids = table_row(p.geo, rq.src);
    const uint32_t* dst_ids = table_row(p.geo, rq.dst);
    const uint32_t units = p.geo.head_dim * p.geo.elem_bytes / sizeof(Unit);
    const uint32_t lanes = row_lanes(units), groups = kMoveThreads / lanes, group = threadIdx.x / lanes, lane = threadIdx.x % lanes;
    const uint64_t value_units = v_region_offset(p.geo) * p.geo.elem_bytes / sizeof(Unit);
    const PageBounds bounds(p.geo);
    uint32_t bad = 0;
    for (uint32_t base = blockIdx.x * groups * kMoveEach; base < rq.keep; base += gridDim.x * groups * kMoveEach) {
        const Unit* from[kMoveEach];
        Unit* to[kMoveEach];
#pragma unroll
        for (uint32_t i = 0; i < kMoveEach; ++i) {
            const uint32_t row = base + i * groups + group;
            from[i] = nullptr;
            to[i] = nullptr;
            if (row < rq.keep) {
                uint32_t miss = 0;
                from[i] = row_units<Unit>(p.geo, bounds, src_ids, head, kept[row], false, miss);
                to[i] = row_units<Unit>(p.geo, bounds, dst_ids, head, row, false, miss);
                if (miss != 0) to[i] = nullptr;
                bad |= miss;
            }
        }
        for (uint32_t unit = lane; unit < units; unit += lanes) {
            Unit k[kMoveEach], v[kMoveEach];
#pragma unroll
            for (uint32_t i = 0; i < kMoveEach; ++i) {
                if (to[i] != nullptr) {
                    k[i] = from[i][unit];
                    v[i] = from[i][value_units + unit];
                }
            }
#pragma unroll
            for (uint32_t i = 0; i < kMoveEach; ++i) {
                if (to[i] != nullptr) {
                    to[i][unit] = k[i];
                    to[i][value_units + unit] = v[i];
                }
            }
        }
    }
    if (bad != 0) record_page_fault(p.geo);
}

// In place: grid (x: column slice, y: 2 * KV head + (K or V), z: request).  A slice has at most 32 units.
template <typename Unit>
__global__ __launch_bounds__(kMoveThreads) void evict_move_in_place_kernel(const EvictParams p, uint32_t slice_units) {
    await_previous_kernel();
    const EvictRequest rq = p.reqs[blockIdx.z];
    if (rq.src != rq.dst || rq.keep == rq.length || rq.keep == 0) return;
    const uint32_t head = blockIdx.y >> 1;
    const bool is_value = (blockIdx.y & 1u) != 0;
    const uint32_t* kept = p.kept + (uint64_t(blockIdx.z) * p.geo.num_kv_heads + head) * p.kept_stride;
    const uint32_t* ids = table_row(p.geo, rq.src);
    const uint32_t units = p.geo.head_dim * p.geo.elem_bytes / sizeof(Unit);
    const uint32_t unit0 = blockIdx.x * slice_units, width = min(slice_units, units - unit0);
    const uint32_t lanes = row_lanes(slice_units), groups = kMoveThreads / lanes, group = threadIdx.x / lanes, lane = threadIdx.x % lanes;
    const PageBounds bounds(p.geo);
    uint32_t bad = 0;
    constexpr uint32_t kEach = 2 * kMoveEach;
    for (uint32_t base = 0; base < rq.keep; base += groups * kEach) {
        Unit value[kEach];
        Unit* to[kEach];
#pragma unroll
        for (uint32_t i = 0; i < kEach; ++i) {
            const uint32_t row = base + i * groups + group;
            to[i] = nullptr;
            const uint32_t from = row < rq.keep ? kept[row] : row;
            if (from != row && lane < width) {  // (a row before the first hole stays)
                uint32_t miss = 0;
                to[i] = row_units<Unit>(p.geo, bounds, ids, head, row, is_value, miss) + unit0 + lane;
                value[i] = row_units<Unit>(p.geo, bounds, ids, head, from, is_value, miss)[unit0 + lane];
                if (miss != 0) to[i] = nullptr;
                bad |= miss;
            }
        }
        __syncthreads();  // the batch's loads have come back before anything is stored over what they read
#pragma unroll
        for (uint32_t i = 0; i < kEach; ++i)
            if (to[i] != nullptr) *to[i] = value[i];
        __syncthreads();
    }
    if (bad != 0) record_page_fault(p.geo);
}

template <typename Unit>
cudaError_t launch_move(const EvictParams& p, uint32_t sms, cudaStream_t stream) {
    const uint32_t heads = p.geo.num_kv_heads, units = p.geo.head_dim * p.geo.elem_bytes / uint32_t(sizeof(Unit));
    if (p.in_place != 0) {
        // slices of at most 32 units, halved down to 32 bytes while the launch has fewer CTAs than two for each SM
        uint32_t slice = units < 32 ? units : 32;
        while (slice * sizeof(Unit) > 32 && uint64_t((units + slice - 1) / slice) * 2 * heads * p.num_reqs < 2 * sms) slice = (slice + 1) / 2;
        return launch_overlapped(evict_move_in_place_kernel<Unit>, dim3((units + slice - 1) / slice, 2 * heads, p.num_reqs),
                                 dim3(kMoveThreads), 0, stream, p, slice);
    }
    uint32_t most = 0;
    for (uint32_t r = 0; r < p.num_reqs; ++r)
        if (p.reqs[r].src != p.reqs[r].dst) most = p.reqs[r].keep > most ? p.reqs[r].keep : most;
    uint32_t lanes = 1;
    while (lanes < 32 && lanes < units) lanes *= 2;
    const uint32_t rows = kMoveThreads / lanes * kMoveEach;  // of one CTA at a time
    const uint32_t blocks = (most + rows - 1) / rows;
    const uint64_t ctas = uint64_t(sms) * 16;
    const uint64_t share = (ctas + uint64_t(heads) * p.num_reqs - 1) / (uint64_t(heads) * p.num_reqs);
    const uint32_t x = uint32_t(blocks < share ? (blocks > 0 ? blocks : 1) : share);
    return launch_overlapped(evict_move_kernel<Unit>, dim3(x, heads, p.num_reqs), dim3(kMoveThreads), 0, stream, p);
}

}  // namespace

cudaError_t launch_evict_select(const EvictParams& p, uint32_t sms, cudaStream_t stream) {
    uint32_t longest = 0;
    for (uint32_t r = 0; r < p.num_reqs; ++r) longest = p.reqs[r].length > longest ? p.reqs[r].length : longest;
    const uint32_t heads = p.geo.num_kv_heads;
    if (longest > kMostCtas * kSliceKeys) return launch_overlapped(evict_select_kernel<false>, dim3(p.num_reqs, heads), dim3(kSelectThreads), 0, stream, p);
    // CTAs of a row: until its slices fit, and on while there are SMs for them and 4,096 keys left to each
    uint32_t ctas = 1;
    while (ctas < kMostCtas && (uint64_t(ctas) * kSliceKeys < longest || (uint64_t(ctas) * 2 * heads * p.num_reqs <= 2ull * sms && longest / (2 * ctas) >= 4096))) ctas *= 2;
    const uint32_t slice = ((longest + ctas - 1) / ctas + 3) / 4 * 4;
    static std::atomic<uint64_t> done{0};
    cudaError_t err = ensure_dynamic_smem(reinterpret_cast<const void*>(evict_select_kernel<true>), int(kSliceKeys * sizeof(float)), done);
    if (err != cudaSuccess) return err;
    cudaLaunchAttribute attributes[2]{};
    attributes[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attributes[0].val.programmaticStreamSerializationAllowed = 1;
    attributes[1].id = cudaLaunchAttributeClusterDimension;
    attributes[1].val.clusterDim = {ctas, 1, 1};
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(p.num_reqs * ctas, heads);
    config.blockDim = dim3(kSelectThreads);
    config.dynamicSmemBytes = slice * sizeof(float);
    config.stream = stream;
    config.attrs = attributes;
    config.numAttrs = 2;
    return cudaLaunchKernelEx(&config, evict_select_kernel<true>, p);
}

cudaError_t launch_evict_move(const EvictParams& p, uint32_t sms, cudaStream_t stream) {
    if (p.unit_bytes == 16) return launch_move<uint4>(p, sms, stream);
    if (p.unit_bytes == 4) return launch_move<uint32_t>(p, sms, stream);
    return launch_move<uint16_t>(p, sms, stream);
}

}  // namespace psi
