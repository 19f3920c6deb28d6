// Eviction from the paged cache by accumulated attention weight (psi_gqa_evict).
//
// evict_select_kernel: a CTA for each (request, KV head) finds the weight of the last kept key by a radix selection over
// order-preserving 32-bit keys (11, 11 and 10 bits, a histogram each), then writes the kept indices in ascending order with one
// ordered scan, which also brings the weights to their new places.  Counts are whole numbers, so ties and results do not depend
// on the order of the atomics.
// evict_move_kernel / evict_move_in_place_kernel: the kept K and V rows to the front of the destination slot: bound by the
// bytes of the rows, read and written once.  Into another slot every row is independent.  In place a row moves to a lower or
// equal index: a CTA takes one column slice of one head's K or V and goes through the rows in order, a batch in registers
// between its loads and its stores, so that nothing is overwritten that a later batch reads.
#include "device_common.cuh"
#include "evict.hpp"
#include "launch_util.hpp"

namespace psi {

namespace {

constexpr uint32_t kSelectThreads = 512;
constexpr uint32_t kBins = 2048;

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
    __syncthreads();
    if (lane == 31) warp_sums[warp] = sum;
    __syncthreads();
    uint32_t before = 0;
    total = 0;
    for (uint32_t i = 0; i < kSelectThreads / 32; ++i) {
        const uint32_t s = warp_sums[i];
        before += i < warp ? s : 0u;
        total += s;
    }
    return before + sum - value;
}

__global__ __launch_bounds__(kSelectThreads) void evict_select_kernel(const EvictParams p) {
    __shared__ uint32_t bins[kBins];
    __shared__ uint32_t warp_sums[kSelectThreads / 32];
    __shared__ uint32_t found_digit, found_above;
    await_previous_kernel();
    const EvictRequest rq = p.reqs[blockIdx.x];
    const uint32_t head = blockIdx.y, heads = p.geo.num_kv_heads;
    const float* w = p.weights + (uint64_t(rq.src) * heads + head) * p.stride;
    float* out = p.weights_out + (uint64_t(rq.dst) * heads + head) * p.stride;
    uint32_t* kept = p.kept + (uint64_t(blockIdx.x) * heads + head) * p.kept_stride;
    const uint32_t recent = min(p.recent, rq.keep), pool = rq.length - recent;
    uint32_t want = rq.keep - recent;  // of the first `pool` keys
    // The key of the last wanted weight, digit by digit: `threshold` and how many of the keys equal to it belong.
    uint32_t threshold = 0;
    if (want > 0 && want < pool) {
        constexpr uint32_t kShift[3] = {21, 10, 0}, kDigits[3] = {2048, 2048, 1024};
        for (int pass = 0; pass < 3; ++pass) {
            for (uint32_t i = threadIdx.x; i < kBins; i += kSelectThreads) bins[i] = 0;
            __syncthreads();
            const uint32_t shift = kShift[pass], digits = kDigits[pass];
            const uint32_t above = pass == 0 ? 0u : kShift[pass - 1];
            for (uint32_t i = threadIdx.x; i < pool; i += kSelectThreads) {
                const uint32_t key = weight_key(w[i]);
                if (pass == 0 || (key >> above) == (threshold >> above)) atomicAdd(&bins[(key >> shift) & (digits - 1)], 1u);
            }
            __syncthreads();
            // thread t holds digits from the top: digits - 1 - 4 t .. down
            const uint32_t per = digits / kSelectThreads;
            uint32_t mine = 0;
            for (uint32_t i = 0; i < per; ++i) mine += bins[digits - 1 - (threadIdx.x * per + i)];
            uint32_t total = 0;
            uint32_t before = block_scan(mine, warp_sums, total);
            if (before < want && want <= before + mine) {
                for (uint32_t i = 0; i < per; ++i) {
                    const uint32_t digit = digits - 1 - (threadIdx.x * per + i);
                    if (want <= before + bins[digit]) {
                        found_digit = digit;
                        found_above = before;
                        break;
                    }
                    before += bins[digit];
                }
            }
            __syncthreads();
            threshold |= found_digit << shift;
            want -= found_above;
            __syncthreads();
        }
    } else if (want == 0) {
        threshold = 0xFFFFFFFFu;  // no weight has this key: it is a NaN's
    }  // want == pool: every key is above or equal to 0, all equal ones belong
    // One ordered scan: low half counts the keys above the threshold (recent ones among them), high half those equal to it.
    constexpr uint32_t kEach = 4;
    uint32_t above_before = 0, equal_before = 0;
    for (uint32_t base = 0; base < rq.length; base += kSelectThreads * kEach) {
        const uint32_t first = base + threadIdx.x * kEach;
        float value[kEach];
        uint32_t mark[kEach], mine = 0;
#pragma unroll
        for (uint32_t i = 0; i < kEach; ++i) {
            const uint32_t at = first + i;
            value[i] = at < rq.length ? w[at] : 0.0f;
            const uint32_t key = weight_key(value[i]);
            mark[i] = at >= rq.length ? 0u : (at >= pool || key > threshold) ? 1u : key == threshold ? 0x10000u : 0u;
            mine += mark[i];
        }
        uint32_t total = 0;
        const uint32_t before = block_scan(mine, warp_sums, total);  // every thread has read its weights
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
    __syncthreads();  // the last stores into [0, keep) and, in place, the last reads are done
    for (uint32_t i = rq.keep + threadIdx.x; i < rq.length; i += kSelectThreads) out[i] = 0.0f;
}

template <typename Unit>
__device__ __forceinline__ Unit* row_units(const PageGeometry& g, const PageBounds& bounds, const uint32_t* ids, uint32_t head,
                                           uint32_t token, bool value, uint32_t& bad) {
    const uint32_t page = bounds.read(ids, token / g.tokens_per_page, bad);
    const uint64_t at = kv_row_offset(g, page, head, token % g.tokens_per_page) + (value ? v_region_offset(g) : 0u);
    return reinterpret_cast<Unit*>(static_cast<unsigned char*>(const_cast<void*>(g.pages)) + at * g.elem_bytes);
}

constexpr uint32_t kMoveThreads = 256;
constexpr uint32_t kMoveEach = 8;

// Into another slot: grid (x: stride over row blocks, y: KV head, z: request).
template <typename Unit>
__global__ __launch_bounds__(kMoveThreads) void evict_move_kernel(const EvictParams p) {
    await_previous_kernel();
    const EvictRequest rq = p.reqs[blockIdx.z];
    if (rq.src == rq.dst || rq.keep == 0) return;
    const uint32_t head = blockIdx.y;
    const uint32_t* kept = p.kept + (uint64_t(blockIdx.z) * p.geo.num_kv_heads + head) * p.kept_stride;
    const uint32_t* src_ids = table_row(p.geo, rq.src);
    const uint32_t* dst_ids = table_row(p.geo, rq.dst);
    const uint32_t units = p.geo.head_dim * p.geo.elem_bytes / sizeof(Unit);  // of one row
    const PageBounds bounds(p.geo);
    uint32_t bad = 0;
    const uint64_t total = uint64_t(rq.keep) * 2u * units;
    const uint64_t step = uint64_t(gridDim.x) * kMoveThreads * kMoveEach;
    for (uint64_t base = uint64_t(blockIdx.x) * kMoveThreads * kMoveEach; base < total; base += step) {
        Unit value[kMoveEach];
        Unit* to[kMoveEach];
#pragma unroll
        for (uint32_t i = 0; i < kMoveEach; ++i) {
            const uint64_t at = base + i * kMoveThreads + threadIdx.x;
            to[i] = nullptr;
            if (at < total) {
                const uint32_t line = uint32_t(at / units), unit = uint32_t(at % units), row = line >> 1;
                uint32_t miss = 0;
                to[i] = row_units<Unit>(p.geo, bounds, dst_ids, head, row, (line & 1u) != 0, miss) + unit;
                value[i] = row_units<Unit>(p.geo, bounds, src_ids, head, kept[row], (line & 1u) != 0, miss)[unit];
                if (miss != 0) to[i] = nullptr;
                bad |= miss;
            }
        }
#pragma unroll
        for (uint32_t i = 0; i < kMoveEach; ++i)
            if (to[i] != nullptr) *to[i] = value[i];
    }
    if (bad != 0) record_page_fault(p.geo);
}

// In place: grid (x: column slice, y: 2 * KV head + (K or V), z: request).
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
    // the first kept row that moves: kept[i] - i does not fall
    uint32_t lo = 0, hi = rq.keep;
    while (lo < hi) {
        const uint32_t mid = (lo + hi) >> 1;
        if (kept[mid] == mid) lo = mid + 1;
        else hi = mid;
    }
    const PageBounds bounds(p.geo);
    uint32_t bad = 0;
    const uint64_t total = uint64_t(rq.keep - lo) * width;
    for (uint64_t base = 0; base < total; base += kMoveThreads * kMoveEach) {
        Unit value[kMoveEach];
        Unit* to[kMoveEach];
#pragma unroll
        for (uint32_t i = 0; i < kMoveEach; ++i) {
            const uint64_t at = base + i * kMoveThreads + threadIdx.x;
            to[i] = nullptr;
            if (at < total) {
                const uint32_t row = lo + uint32_t(at / width), unit = unit0 + uint32_t(at % width);
                uint32_t miss = 0;
                to[i] = row_units<Unit>(p.geo, bounds, ids, head, row, is_value, miss) + unit;
                value[i] = row_units<Unit>(p.geo, bounds, ids, head, kept[row], is_value, miss)[unit];
                if (miss != 0) to[i] = nullptr;
                bad |= miss;
            }
        }
        __syncthreads();  // the batch's loads have all come back: each was used above or is held in `value`
#pragma unroll
        for (uint32_t i = 0; i < kMoveEach; ++i)
            if (to[i] != nullptr) *to[i] = value[i];
        __syncthreads();
    }
    if (bad != 0) record_page_fault(p.geo);
}

template <typename Unit>
cudaError_t launch_move(const EvictParams& p, uint32_t ctas, cudaStream_t stream) {
    const uint32_t heads = p.geo.num_kv_heads, units = p.geo.head_dim * p.geo.elem_bytes / uint32_t(sizeof(Unit));
    if (p.in_place != 0) {
        // slices of at least 64 bytes, halved while the launch has fewer CTAs than asked for
        uint32_t slice = units;
        while (slice * sizeof(Unit) > 64 && (units + slice - 1) / slice * 2u * heads * p.num_reqs < ctas) slice = (slice + 1) / 2;
        return launch_overlapped(evict_move_in_place_kernel<Unit>, dim3((units + slice - 1) / slice, 2 * heads, p.num_reqs),
                                 dim3(kMoveThreads), 0, stream, p, slice);
    }
    uint32_t most = 0;
    for (uint32_t r = 0; r < p.num_reqs; ++r)
        if (p.reqs[r].src != p.reqs[r].dst) most = p.reqs[r].keep > most ? p.reqs[r].keep : most;
    const uint64_t blocks = (uint64_t(most) * 2u * units + kMoveThreads * kMoveEach - 1) / (kMoveThreads * kMoveEach);
    const uint64_t share = (uint64_t(ctas) + uint64_t(heads) * p.num_reqs - 1) / (uint64_t(heads) * p.num_reqs);
    const uint32_t x = uint32_t(blocks < share ? (blocks > 0 ? blocks : 1) : share);
    return launch_overlapped(evict_move_kernel<Unit>, dim3(x, heads, p.num_reqs), dim3(kMoveThreads), 0, stream, p);
}

}  // namespace

cudaError_t launch_evict_select(const EvictParams& p, cudaStream_t stream) {
    return launch_overlapped(evict_select_kernel, dim3(p.num_reqs, p.geo.num_kv_heads), dim3(kSelectThreads), 0, stream, p);
}

cudaError_t launch_evict_move(const EvictParams& p, uint32_t ctas, cudaStream_t stream) {
    if (p.unit_bytes == 16) return launch_move<uint4>(p, ctas, stream);
    if (p.unit_bytes == 4) return launch_move<uint32_t>(p, ctas, stream);
    return launch_move<uint16_t>(p, ctas, stream);
}

}  // namespace psi
