// Attention weight gathered by each cached key (psi_gqa_weigh_keys).
//
//   weights[slot][kv head][j] += sum over the request's query rows r (token i of the run, head of the group) of
//                                exp(scale q_r . k_j - M_r) / L_r        for j <= token_index + i
//
// with M_r and L_r the maximum and the exponential sum of row r's scores.  A row without a finite maximum or sum adds nothing.
// Two passes, since no weight is known before its row's sum is: the first finds M and 1 / L, the second adds up
// columns.  Both keep f32 scores; every key's sum is worked out by one thread group in one order, so results repeat bit for bit.
// M and 1 / L stay apart: their logarithmic sum is a number of twenty or so, whose rounding alone would be the largest error.
//
//   weigh_short_kernel   runs of up to 16 rows (decode, drafts): bound by the K bytes.  One warp is one worker with an equal
//                        share of the batch's 32-key tiles, which it streams through a ring of its own (cp.async, no barrier
//                        of the CTA; any page size), page IDs fetched a step ahead of the keys, which are two to eleven ahead of their
//                        use.  Products do not depend on the order of the columns of q and k, so a lane takes 16 consecutive
//                        bytes of a key row as the operands of two m16n8k16 steps, and the same bytes of the query rows, which
//                        stay in registers.  The first pass leaves its products in scratch, 4 bytes a row and key against
//                        2 head_dim bytes a key, so that K is read once; where there is no scratch (captured launches,
//                        very large batches) the second pass reads K again.  32 requests of 1,024 to 8,192 keys, 16/2 heads x
//                        256, bf16: 40 us, 59 % of the copy rate; 64 pairs of tokens, 4,096 to 32,768
//                        keys, 24/4 heads, f16: 390 us, 73 %; one of 777 keys: 9.7 us, two launches' latency.
//   weigh_umma_kernel    longer runs, on tcgen05 (weigh_umma.cu).
//   weigh_*_any_kernel   f32 and head dims that are no multiple of eight: the same two passes in f32 on the CUDA cores, 32 rows and 64
//                        keys a tile in shared memory, two rows and four keys a thread: bound by the reads of shared memory, six
//                        words for eight multiply-adds.
#include "mma_common.cuh"
#include "launch_util.hpp"
#include "weigh_common.cuh"

namespace psi {

namespace {

__device__ __forceinline__ uint4 ld_stream(const uint4* p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}

// 16-byte chunks of a 16-bit row that a lane holds: chunk (lane & 3) + 4 i for i < NC, zeros beyond the row.
template <int NC>
__device__ __forceinline__ void load_row(uint4 (&x)[NC], const uint4* row, uint32_t lane_chunk, uint32_t chunks) {
#pragma unroll
    for (int i = 0; i < NC; ++i) {
        const uint32_t c = lane_chunk + 4u * i;
        x[i] = c < chunks ? ld_stream(row + c) : make_uint4(0, 0, 0, 0);
    }
}

// d += A B for the two steps that one 16-byte chunk of every row makes; lo, hi: rows quad_row and quad_row + 8 of A.
template <typename T>
__device__ __forceinline__ void chunk_mma(float (&d)[4], const uint4& lo, const uint4& hi, const uint4& b) {
    const uint32_t a0[4] = {lo.x, hi.x, lo.y, hi.y}, a1[4] = {lo.z, hi.z, lo.w, hi.w};
    Mma<T>::run(d, a0, b.x, b.y);
    Mma<T>::run(d, a1, b.z, b.w);
}

// Byte offset of 16-byte chunk `chunk` of row `row` in a block of NC * 64-byte rows: the eight lanes of one phase of a 16-byte read
// (two rows, four chunks) fall into distinct banks.
template <int NC>
__device__ __forceinline__ uint32_t block_offset(uint32_t row, uint32_t chunk) {
    return row * (NC * 64u) + ((NC % 2 == 0 ? chunk ^ ((row & 1u) << 2) : chunk) << 4);
}

enum ShortMode { kStatsAndScores = 0, kStatsOnly = 1, kSumAgain = 2 };

// Steps of 16 keys that a warp's ring holds: 24 KiB a warp, 192 KiB an SM.
template <int NC>
constexpr int kRingSteps = 24 / NC;

// Requests and tiles of the short runs: with the launch where the host knows them, which spares two loads one behind the other.
struct ShortWork {
    uint32_t count, total;
    __device__ __forceinline__ explicit ShortWork(const WeighParams& p) : count(p.short_count), total(p.short_tiles) {
        if (count == 0xFFFFFFFFu) {
            count = p.scalars[kScalarWeighShort];
            total = p.reqs[count].cu0;
        }
    }
};

template <typename T, int NC, int kMode>
__global__ __launch_bounds__(256, 1) void weigh_short_kernel(const WeighParams p) {
    constexpr uint32_t kStepBytes = 16 * NC * 64;
    constexpr int kSteps = kRingSteps<NC>;
    extern __shared__ __align__(128) unsigned char smem[];
    await_previous_kernel();
    const ShortWork work(p);
    const uint32_t count = work.count, total = work.total;
    const WeighRequest* reqs = p.reqs;
    const uint32_t workers = min(gridDim.x * 8u, total);
    const uint32_t w = blockIdx.x * 8u + (threadIdx.x >> 5);
    if (w >= workers) return;
    const unsigned char* ring = smem + (threadIdx.x >> 5) * (kSteps * kStepBytes);  // this warp's
    const uint32_t ring_at = uint32_t(__cvta_generic_to_shared(ring));
    const uint32_t lane = threadIdx.x & 31u, quad_row = lane >> 2, quad_col = lane & 3u;
    const uint32_t begin = uint32_t(uint64_t(w) * total / workers), end = uint32_t(uint64_t(w + 1) * total / workers);
    const uint32_t chunks = p.geo.head_dim >> 3;
    const uint64_t policy = l2_evict_first_policy();
    const PageBounds bounds(p.geo);
    uint32_t bad = 0;
    uint32_t r_index = find_request<0>(reqs, count, begin);
    // The load cursor: a step of 16 keys, whose page IDs (of row lane % 16) are fetched a step before its keys.
    uint32_t load_step = 0, id_tile = begin, id_half = 0, id_request = r_index, id_head = 0, id_next = begin, id_begin = 0;
    const uint32_t* id_rows = nullptr;
    uint32_t id_keys = 0, page = 0, page_token = 0, page_head = 0;
    bool more = true;
    const auto fetch_ids = [&] {
        if (id_tile >= end) {
            more = false;
            return;
        }
        if (id_tile >= id_next) {  // another (request, KV head)
            while (reqs[id_request + 1].cu0 <= id_tile) ++id_request;
            const WeighRequest rq = reqs[id_request];
            const uint32_t per_head = (rq.keys + 31u) / 32u;
            id_head = (id_tile - rq.cu0) / per_head;
            id_begin = rq.cu0 + id_head * per_head;
            id_next = id_begin + per_head;
            id_keys = rq.keys;
            id_rows = table_row(p.geo, rq.slot);
        }
        const uint32_t key = min((id_tile - id_begin) * 32u + id_half * 16u + (lane & 15u), id_keys - 1u);
        page = bounds.read(id_rows, key / p.geo.tokens_per_page, bad);
        page_token = key % p.geo.tokens_per_page;
        page_head = id_head;
        if (id_half != 0) ++id_tile;
        id_half ^= 1u;
    };
    const auto load_next = [&] {
        if (more) {
            const uint64_t offset = kv_row_offset(p.geo, page, page_head, page_token);  // of row lane % 16
            const uint32_t dst = ring_at + (load_step % kSteps) * kStepBytes;
#pragma unroll
            for (int j = 0; j < 2 * NC; ++j) {
                const uint32_t at = lane + 32u * j, row = at / (NC * 4u), c = at % (NC * 4u);
                const uint64_t from = __shfl_sync(0xFFFFFFFFu, offset, row);
                const bool live = c < chunks;
                cp_async_16_hinted(dst + block_offset<NC>(row, c), static_cast<const uint16_t*>(p.geo.pages) + from + (live ? c * 8u : 0u), live ? 16u : 0u, policy);
            }
            ++load_step;
            fetch_ids();
        }
        cp_async_commit();
    };
    fetch_ids();
#pragma unroll 1
    for (int i = 0; i < kSteps - 1; ++i) load_next();
    uint32_t step = 0;
    for (uint32_t tile = begin; tile < end;) {
        while (reqs[r_index + 1].cu0 <= tile) ++r_index;
        const WeighRequest rq = reqs[r_index];
        const uint32_t per_head = (rq.keys + 31u) / 32u;
        const uint32_t head = (tile - rq.cu0) / per_head;
        const uint32_t unit_begin = rq.cu0 + head * per_head, unit_end = unit_begin + per_head;
        const uint32_t last = min(end, unit_end);
        const uint32_t rows = rq.q_len * p.group;
        uint4 q_lo[NC], q_hi[NC];
#pragma unroll
        for (int i = 0; i < NC; ++i) q_lo[i] = q_hi[i] = make_uint4(0, 0, 0, 0);
        if (quad_row < rows) load_row<NC>(q_lo, reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.q) + query_row(p, rq, head, quad_row) * p.geo.head_dim), quad_col, chunks);
        if (quad_row + 8 < rows) load_row<NC>(q_hi, reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.q) + query_row(p, rq, head, quad_row + 8) * p.geo.head_dim), quad_col, chunks);
        const bool two_halves = rows > 8;
        const uint32_t limit0 = quad_row < rows ? row_limit(p, rq, quad_row) : 0u;
        const uint32_t limit1 = quad_row + 8 < rows ? row_limit(p, rq, quad_row + 8) : 0u;
        Stat s0{-kInf, 0.0f}, s1{-kInf, 0.0f};
        float2 norm0 = make_float2(kInf, 0.0f), norm1 = norm0;
        if (kMode == kSumAgain) {
            if (quad_row < rows) norm0 = p.norms[query_row(p, rq, head, quad_row)];
            if (quad_row + 8 < rows) norm1 = p.norms[query_row(p, rq, head, quad_row + 8)];
        }
        for (; tile < last; ++tile) {
#pragma unroll 1
            for (uint32_t half = 0; half < 2; ++half, ++step) {
                const uint32_t key0 = (tile - unit_begin) * 32u + half * 16u;
                cp_async_wait<kSteps - 2>();
                __syncwarp();  // the step's keys have landed, and everyone is through with the step before it, whose place is next
                load_next();
                const unsigned char* k = ring + (step % kSteps) * kStepBytes;
                float s[2][4];  // products, -inf where a row does not see a key
#pragma unroll
                for (int t = 0; t < 2; ++t) s[t][0] = s[t][1] = s[t][2] = s[t][3] = 0.0f;
#pragma unroll
                for (int i = 0; i < NC; ++i) {
#pragma unroll
                    for (int t = 0; t < 2; ++t)
                        chunk_mma<T>(s[t], q_lo[i], q_hi[i], *reinterpret_cast<const uint4*>(k + block_offset<NC>(8u * t + quad_row, quad_col + 4u * i)));
                }
#pragma unroll
                for (int t = 0; t < 2; ++t) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const uint32_t key = key0 + 8u * t + 2u * quad_col + (e & 1);
                        s[t][e] = key < (e < 2 ? limit0 : limit1) ? s[t][e] : -kInf;
                    }
                }
                if (kMode == kSumAgain) {
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        float a = weight_of(s[t][0], p.scale_log2, norm0) + weight_of(s[t][2], p.scale_log2, norm1);
                        float b = weight_of(s[t][1], p.scale_log2, norm0) + weight_of(s[t][3], p.scale_log2, norm1);
#pragma unroll
                        for (int x = 4; x < 32; x <<= 1) {
                            a += __shfl_xor_sync(0xFFFFFFFFu, a, x);
                            b += __shfl_xor_sync(0xFFFFFFFFu, b, x);
                        }
                        const uint32_t key = key0 + 8u * t + 2u * quad_col;
                        float* row = weight_row(p, rq, head);
                        if (quad_row == 0 && key < rq.keys) row[key] += a;
                        if (quad_row == 0 && key + 1 < rq.keys) row[key + 1] += b;
                    }
                } else {
                    if (kMode == kStatsAndScores) {
                        // [8-key group][row][8 keys], as many rows as the batch's longest run has
#pragma unroll
                        for (int t = 0; t < 2; ++t) {
                            float* at = p.scores + (uint64_t(tile) * 4u + half * 2 + t) * 8u * p.score_rows + quad_row * 8u + 2u * quad_col;
                            if (quad_row < p.score_rows) *reinterpret_cast<float2*>(at) = make_float2(s[t][0], s[t][1]);
                            if (quad_row + 8 < p.score_rows) *reinterpret_cast<float2*>(at + 64) = make_float2(s[t][2], s[t][3]);
                        }
                    }
                    const float m0 = fmaxf(s0.m, fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[1][0], s[1][1])) * p.scale_log2);
                    const float base0 = m0 == -kInf ? 0.0f : m0;
                    s0.l *= fast_exp2(s0.m - base0);
                    s0.m = m0;
#pragma unroll
                    for (int t = 0; t < 2; ++t)
                        s0.l += fast_exp2(fmaf(s[t][0], p.scale_log2, -base0)) + fast_exp2(fmaf(s[t][1], p.scale_log2, -base0));
                    if (two_halves) {
                        const float m1 = fmaxf(s1.m, fmaxf(fmaxf(s[0][2], s[0][3]), fmaxf(s[1][2], s[1][3])) * p.scale_log2);
                        const float base1 = m1 == -kInf ? 0.0f : m1;
                        s1.l *= fast_exp2(s1.m - base1);
                        s1.m = m1;
#pragma unroll
                        for (int t = 0; t < 2; ++t)
                            s1.l += fast_exp2(fmaf(s[t][2], p.scale_log2, -base1)) + fast_exp2(fmaf(s[t][3], p.scale_log2, -base1));
                    }
                }
            }
        }
        if (kMode == kSumAgain) continue;
#pragma unroll
        for (int x = 1; x < 4; x <<= 1) {
            s0.join(__shfl_xor_sync(0xFFFFFFFFu, s0.m, x), __shfl_xor_sync(0xFFFFFFFFu, s0.l, x));
            s1.join(__shfl_xor_sync(0xFFFFFFFFu, s1.m, x), __shfl_xor_sync(0xFFFFFFFFu, s1.l, x));
        }
        // workers of this unit: the one that holds tile t is the last whose share begins at or before t
        const uint32_t unit = r_index * p.geo.num_kv_heads + head;
        const uint32_t first_worker = uint32_t((uint64_t(unit_begin + 1) * workers - 1) / total);
        const uint32_t last_worker = uint32_t((uint64_t(unit_end) * workers - 1) / total);
        if (first_worker == last_worker) {
            if (quad_col == 0 && quad_row < rows) p.norms[query_row(p, rq, head, quad_row)] = s0.norm();
            if (quad_col == 0 && quad_row + 8 < rows) p.norms[query_row(p, rq, head, quad_row + 8)] = s1.norm();
            continue;
        }
        // worker + unit grows from one segment of the batch to the next: a slot of its own for each
        float2* slot = p.partials + uint64_t(w + unit) * 16u;
        if (quad_col == 0) {
            slot[quad_row] = make_float2(s0.m, s0.l);
            slot[quad_row + 8] = make_float2(s1.m, s1.l);
        }
        __threadfence();
        __syncwarp();
        uint32_t arrived = 0;
        if (lane == 0) arrived = atomicAdd(p.counters + unit, 1u);
        arrived = __shfl_sync(0xFFFFFFFFu, arrived, 0);
        if (arrived == last_worker - first_worker) {
            __threadfence();
            // lanes: rows, and workers of the unit side by side; eight loads under way at a time
            const uint32_t wide = rows > 8 ? 16u : 8u, row = lane & (wide - 1), beside = 32u / wide;
            Stat s{-kInf, 0.0f};
            for (uint32_t o = first_worker + lane / wide; o <= last_worker; o += 8 * beside) {
                float2 v[8];
#pragma unroll
                for (uint32_t x = 0; x < 8; ++x)
                    v[x] = o + x * beside <= last_worker ? __ldcg(p.partials + uint64_t(o + x * beside + unit) * 16u + row) : make_float2(-kInf, 0.0f);
#pragma unroll
                for (uint32_t x = 0; x < 8; ++x) s.join(v[x].x, v[x].y);
            }
            for (uint32_t x = wide; x < 32; x <<= 1) s.join(__shfl_xor_sync(0xFFFFFFFFu, s.m, x), __shfl_xor_sync(0xFFFFFFFFu, s.l, x));
            if (lane < rows) p.norms[query_row(p, rq, head, lane)] = s.norm();
            if (lane == 0) p.counters[unit] = 0;
        }
    }
    if (bad != 0) record_page_fault(p.geo);
}

// Second pass over stored scores: a lane is a key.
__global__ __launch_bounds__(256) void weigh_scores_kernel(const WeighParams p) {
    await_previous_kernel();
    const ShortWork work(p);
    const WeighRequest* reqs = p.reqs;
    const uint32_t workers = min(gridDim.x * 8u, work.total);
    const uint32_t w = blockIdx.x * 8u + (threadIdx.x >> 5), lane = threadIdx.x & 31u;
    if (w >= workers) return;
    const uint32_t begin = uint32_t(uint64_t(w) * work.total / workers), end = uint32_t(uint64_t(w + 1) * work.total / workers);
    const uint32_t first = find_request<0>(reqs, work.count, begin);
    uint32_t r_index = first, unit_end = 0, unit_begin = 0, head = 0;
    WeighRequest rq{};
    uint32_t rows = 0;
    float2 norm = make_float2(0.0f, 0.0f);  // of row `lane`
    for (uint32_t tile = begin; tile < end; ++tile) {
        float product[kWeighShortRows];
        const float* s = p.scores + (uint64_t(tile) * 4u + (lane >> 3)) * 8u * p.score_rows + (lane & 7u);
#pragma unroll
        for (uint32_t r = 0; r < kWeighShortRows; ++r)
            if (r < p.score_rows) product[r] = __ldcs(s + r * 8u);
        if (tile >= unit_end) {  // another (request, KV head)
            while (reqs[r_index + 1].cu0 <= tile) ++r_index;
            rq = reqs[r_index];
            const uint32_t per_head = (rq.keys + 31u) / 32u;
            head = (tile - rq.cu0) / per_head;
            unit_begin = rq.cu0 + head * per_head;
            unit_end = unit_begin + per_head;
            rows = rq.q_len * p.group;
            norm = lane < rows ? p.norms[query_row(p, rq, head, lane)] : make_float2(kInf, 0.0f);
        }
        const uint32_t key = (tile - unit_begin) * 32u + lane;
        float* at = weight_row(p, rq, head) + key;
        const float before = key < rq.keys ? *at : 0.0f;
        float sum = 0.0f;
#pragma unroll
        for (uint32_t r = 0; r < kWeighShortRows; ++r) {
            const float2 of_row = make_float2(__shfl_sync(0xFFFFFFFFu, norm.x, r), __shfl_sync(0xFFFFFFFFu, norm.y, r));
            if (r < p.score_rows) sum += weight_of(product[r], p.scale_log2, of_row);
        }
        if (key < rq.keys) *at = before + sum;
    }
}

// ---- any type and head_dim: f32 products on the CUDA cores, 32 rows against 64 keys -----------------------------------------

constexpr uint32_t kAnyRows = kWeighAnyRows, kBlock = kWeighAnyKeys;
constexpr uint32_t kAnyThreads = kAnyRows / 2 * 16;  // two rows and four keys each

// Rows and keys in shared memory as f32, an odd number of 16-byte units apart, so that 16-byte reads of neighbouring keys
// fall into distinct banks; two key blocks, the next one under way while one is worked on (f32 with head_dim a multiple of four
// and 16-byte boundaries, `wide`: by cp.async; everything else element by element).
// Floats from one row to the next: an odd multiple of four.
__host__ __device__ inline uint32_t any_pitch(uint32_t head_dim) { return ((head_dim + 3) / 4 | 1u) * 4u; }

struct AnyTile {
    float* q;
    float* k[2];
    uint32_t d, pitch;
    bool wide;
    __device__ __forceinline__ AnyTile(float* smem, const WeighParams& p)
        : d(p.geo.head_dim), pitch(any_pitch(p.geo.head_dim)),
          wide(p.dtype == PSI_DTYPE_F32 && p.geo.head_dim % 4 == 0 && ((reinterpret_cast<uintptr_t>(p.q) | reinterpret_cast<uintptr_t>(p.geo.pages)) & 15u) == 0) {
        q = smem;
        k[0] = q + kAnyRows * pitch;
        k[1] = k[0] + kBlock * pitch;
        if (d % 4 != 0) {  // the elements that pad a row to a multiple of four take part in the products
            for (uint32_t row = threadIdx.x; row < kAnyRows + 2 * kBlock; row += blockDim.x)
                for (uint32_t i = d; i < pitch; ++i) smem[row * pitch + i] = 0.0f;
            __syncthreads();
        }
    }
    __device__ __forceinline__ void load_rows(float* to, const WeighParams& p, const WeighRequest& rq, uint32_t head, uint32_t row0, uint32_t rows) const {
        for (uint32_t at = threadIdx.x >> 5; at < kAnyRows; at += blockDim.x >> 5) {
            const uint32_t row = row0 + at;
            const uint64_t from = row < rows ? query_row(p, rq, head, row) * d : 0u;
            if (wide) {
                const uint32_t dst = uint32_t(__cvta_generic_to_shared(to + at * pitch));
                for (uint32_t i = 4 * (threadIdx.x & 31u); i < d; i += 128u) cp_async_16(dst + i * 4, static_cast<const float*>(p.q) + from + i, row < rows ? 16u : 0u);
            } else {
                for (uint32_t i = threadIdx.x & 31u; i < d; i += 32u) to[at * pitch + i] = row < rows ? load_as_float(p.q, from + i, p.dtype) : 0.0f;
            }
        }
    }
    __device__ __forceinline__ void load_keys(uint32_t stage, const WeighParams& p, const PageBounds& bounds, const uint32_t* row_ids, uint32_t head,
                                              uint32_t key0, uint32_t keys, uint32_t& bad) const {
        // rows at and beyond `keys` keep what they hold: those columns are masked
        const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
        constexpr uint32_t kEach = kBlock / (kAnyThreads / 32);  // of a warp
        const uint32_t mine = key0 + warp * kEach + (lane & (kEach - 1));
        uint64_t offset = 0;
        if (mine < keys) offset = kv_row_offset(p.geo, bounds.read(row_ids, mine / p.geo.tokens_per_page, bad), head, mine % p.geo.tokens_per_page);
        if (wide) {
            // as many lanes as a row has 16-byte units take one
            const uint32_t units = d / 4, lanes = units >= 32 ? 32u : units > 8 ? 16u : 8u, beside = 32u / lanes;
            for (uint32_t at = 0; at < kEach; at += beside) {
                const uint32_t r = at + lane / lanes;
                const uint64_t from = __shfl_sync(0xFFFFFFFFu, offset, r);
                const uint32_t dst = uint32_t(__cvta_generic_to_shared(k[stage] + (warp * kEach + r) * pitch));
                if (key0 + warp * kEach + r < keys)
                    for (uint32_t u = lane % lanes; u < units; u += lanes) cp_async_16(dst + u * 16, static_cast<const float*>(p.geo.pages) + from + u * 4, 16u);
            }
        } else {
            for (uint32_t r = 0; r < kEach; ++r) {
                const uint64_t from = __shfl_sync(0xFFFFFFFFu, offset, r);
                if (key0 + warp * kEach + r < keys)
                    for (uint32_t i = lane; i < d; i += 32u) k[stage][(warp * kEach + r) * pitch + i] = load_as_float(p.geo.pages, from + i, p.dtype);
            }
        }
        cp_async_commit();
    }
    // Thread t: rows 2 (t / 16) + {0, 1}, keys t % 16 + 16 {0..3}.
    __device__ __forceinline__ void product(const float* rows, uint32_t stage, float (&s)[2][4]) const {
        const float4* q0 = reinterpret_cast<const float4*>(rows + 2u * (threadIdx.x >> 4) * pitch);
        const float4* q1 = q0 + pitch / 4;
        const float4* x = reinterpret_cast<const float4*>(k[stage] + (threadIdx.x & 15u) * pitch);
#pragma unroll
        for (int a = 0; a < 2; ++a)
#pragma unroll
            for (int b = 0; b < 4; ++b) s[a][b] = 0.0f;
#pragma unroll 2
        for (uint32_t i = 0; i < (d + 3) / 4; ++i) {
            const float4 u = q0[i], v = q1[i];
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                const float4 y = x[b * 16 * (pitch / 4) + i];
                s[0][b] = fmaf(u.x, y.x, fmaf(u.y, y.y, fmaf(u.z, y.z, fmaf(u.w, y.w, s[0][b]))));
                s[1][b] = fmaf(v.x, y.x, fmaf(v.y, y.y, fmaf(v.z, y.z, fmaf(v.w, y.w, s[1][b]))));
            }
        }
    }
};

__global__ __launch_bounds__(kAnyThreads) void weigh_stats_any_kernel(const WeighParams p) {
    extern __shared__ __align__(16) float any_smem[];
    __shared__ uint32_t last_arrival;
    await_previous_kernel();
    const uint32_t count = p.scalars[kScalarWeighLong];
    if (count == 0) return;
    const WeighRequest* reqs = p.long_reqs();
    const uint32_t total = reqs[count].cu0;
    const PageBounds bounds(p.geo);
    uint32_t bad = 0;
    AnyTile tile(any_smem, p);
    const uint32_t at = 2u * (threadIdx.x >> 4), column = threadIdx.x & 15u;
    for (uint32_t item = blockIdx.x; item < total; item += gridDim.x) {
        const WeighRequest rq = reqs[find_request<0>(reqs, count, item)];
        const uint32_t pieces = weigh_any_pieces(rq.keys), rows = rq.q_len * p.group, blocks = (rows + kAnyRows - 1) / kAnyRows;
        const uint32_t local = item - rq.cu0, piece = local % pieces, unit = local / pieces;
        const uint32_t head = unit / blocks, row0 = (unit % blocks) * kAnyRows;
        const uint32_t piece_keys = weigh_any_piece_keys(rq.keys, pieces);
        const uint32_t k0 = piece * piece_keys;
        const uint32_t k1 = min(min(k0 + piece_keys, rq.keys), row_limit(p, rq, min(row0 + kAnyRows, rows) - 1));
        const uint32_t* row_ids = table_row(p.geo, rq.slot);
        Stat st[2] = {{-kInf, 0.0f}, {-kInf, 0.0f}};
        uint32_t stage = 0;
        if (k0 < k1) {
            tile.load_rows(tile.q, p, rq, head, row0, rows);
            tile.load_keys(0, p, bounds, row_ids, head, k0, k1, bad);
        }
        for (uint32_t key0 = k0; key0 < k1; key0 += kBlock, stage ^= 1u) {
            if (key0 + kBlock < k1) {
                tile.load_keys(stage ^ 1u, p, bounds, row_ids, head, key0 + kBlock, k1, bad);
                cp_async_wait<1>();
            } else {
                cp_async_wait<0>();
            }
            __syncthreads();
            float s[2][4];
            tile.product(tile.q, stage, s);
#pragma unroll
            for (int a = 0; a < 2; ++a) {
                const uint32_t row = row0 + at + a, limit = row < rows ? min(k1, row_limit(p, rq, row)) : 0u;
                float m = -kInf;
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    s[a][b] = key0 + column + 16u * b < limit ? s[a][b] : -kInf;
                    m = fmaxf(m, s[a][b]);
                }
                m = fmaxf(st[a].m, m * p.scale_log2);
                const float base = m == -kInf ? 0.0f : m;
                st[a].l *= fast_exp2(st[a].m - base);
                st[a].m = m;
#pragma unroll
                for (int b = 0; b < 4; ++b) st[a].l += fast_exp2(fmaf(s[a][b], p.scale_log2, -base));
            }
            __syncthreads();
        }
#pragma unroll
        for (int a = 0; a < 2; ++a)
#pragma unroll
            for (int x = 1; x < 16; x <<= 1)
                st[a].join(__shfl_xor_sync(0xFFFFFFFFu, st[a].m, x), __shfl_xor_sync(0xFFFFFFFFu, st[a].l, x));
        if (column == 0) {
#pragma unroll
            for (int a = 0; a < 2; ++a) {
                if (pieces == 1) {
                    if (row0 + at + a < rows) p.norms[query_row(p, rq, head, row0 + at + a)] = st[a].norm();
                } else {
                    p.long_partials()[uint64_t(item) * kAnyRows + at + a] = make_float2(st[a].m, st[a].l);
                }
            }
        }
        if (pieces > 1) {
            uint32_t* counter = p.long_counters() + rq.unit0 + unit;
            __threadfence();
            __syncthreads();
            if (threadIdx.x == 0) last_arrival = atomicAdd(counter, 1u) == pieces - 1 ? 1u : 0u;
            __syncthreads();
            if (last_arrival != 0) {
                __threadfence();
                const uint32_t row = row0 + threadIdx.x;
                if (threadIdx.x < kAnyRows && row < rows) {
                    Stat s{-kInf, 0.0f};
                    for (uint32_t o = 0; o < pieces; ++o) {
                        const float2 v = __ldcg(p.long_partials() + uint64_t(rq.cu0 + unit * pieces + o) * kAnyRows + threadIdx.x);
                        s.join(v.x, v.y);
                    }
                    p.norms[query_row(p, rq, head, row)] = s.norm();
                }
                if (threadIdx.x == 0) *counter = 0;
            }
        }
        __syncthreads();
    }
    if (bad != 0) record_page_fault(p.geo);
}

__global__ __launch_bounds__(kAnyThreads) void weigh_sum_any_kernel(const WeighParams p) {
    extern __shared__ __align__(16) float any_smem[];
    __shared__ float sums[kAnyRows / 2][kBlock];
    __shared__ float2 norms[2][kAnyRows];
    __shared__ uint32_t last_arrival;
    await_previous_kernel();
    const uint32_t count = p.scalars[kScalarWeighLong];
    if (count == 0) return;
    const WeighRequest* reqs = p.long_reqs();
    const uint32_t total = reqs[count].cu1;
    const PageBounds bounds(p.geo);
    uint32_t bad = 0;
    AnyTile tile(any_smem, p);
    float* const row_buffers[2] = {tile.q, tile.k[1]};  // the keys stay: the second key block's place holds the next rows
    const uint32_t at = 2u * (threadIdx.x >> 4), column = threadIdx.x & 15u;
    for (uint32_t item = blockIdx.x; item < total; item += gridDim.x) {
        const WeighRequest rq = reqs[find_request<1>(reqs, count, item)];
        const uint32_t all_rows = rq.q_len * p.group, spans = weigh_any_spans(rq.keys);
        const uint32_t parts = p.split_rows != 0 ? weigh_row_parts(all_rows, rq.keys, p.geo.num_kv_heads, false) : 1u;
        const uint32_t local = item - rq.cu1, part = local % parts, unit = local / parts;
        const uint32_t head = unit / spans, key0 = unit % spans * kBlock, each = weigh_part_blocks(all_rows, parts, false) * kAnyRows;
        const uint32_t rows = min((part + 1) * each, all_rows);
        const uint32_t seen_from = key0 > rq.first_pos ? (key0 - rq.first_pos) * p.group : 0u;  // rows before see none of the keys
        const uint32_t row_begin = max(part * each, seen_from);
        float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        const auto fetch = [&](uint32_t row0, uint32_t stage) {
            tile.load_rows(row_buffers[stage], p, rq, head, row0, all_rows);
            if (threadIdx.x < kAnyRows)
                norms[stage][threadIdx.x] = row0 + threadIdx.x < rows ? p.norms[query_row(p, rq, head, row0 + threadIdx.x)] : make_float2(kInf, 0.0f);
            cp_async_commit();
        };
        tile.load_keys(0, p, bounds, table_row(p.geo, rq.slot), head, key0, rq.keys, bad);
        if (row_begin < rows) fetch(row_begin, 0);
        uint32_t stage = 0;
        for (uint32_t row0 = row_begin; row0 < rows; row0 += kAnyRows, stage ^= 1u) {
            if (row0 + kAnyRows < rows) {
                fetch(row0 + kAnyRows, stage ^ 1u);
                cp_async_wait<1>();
            } else {
                cp_async_wait<0>();
            }
            __syncthreads();
            float s[2][4];
            tile.product(row_buffers[stage], 0, s);
#pragma unroll
            for (int a = 0; a < 2; ++a) {
                const uint32_t row = row0 + at + a, limit = row < rows ? row_limit(p, rq, row) : 0u;
#pragma unroll
                for (int b = 0; b < 4; ++b)
                    if (key0 + column + 16u * b < limit) sum[b] += weight_of(s[a][b], p.scale_log2, norms[stage][at + a]);
            }
            __syncthreads();
        }
        cp_async_wait<0>();
#pragma unroll
        for (int b = 0; b < 4; ++b) sums[threadIdx.x >> 4][column + 16u * b] = sum[b];
        __syncthreads();
        float all = 0.0f;
        if (threadIdx.x < kBlock) {
#pragma unroll
            for (uint32_t i = 0; i < kAnyRows / 2; ++i) all += sums[i][threadIdx.x];
        }
        const bool mine = threadIdx.x < kBlock && key0 + threadIdx.x < rq.keys;
        if (parts == 1) {
            if (mine) weight_row(p, rq, head)[key0 + threadIdx.x] += all;
        } else {  // the last part of the span adds up the parts
            if (mine) p.sums[uint64_t(item) * kBlock + threadIdx.x] = all;
            __threadfence();
            __syncthreads();
            uint32_t* counter = p.long_counters() + rq.cu1 + unit * parts;
            if (threadIdx.x == 0) last_arrival = atomicAdd(counter, 1u) == parts - 1 ? 1u : 0u;
            __syncthreads();
            if (last_arrival != 0) {
                __threadfence();
                if (mine) {
                    float whole = 0.0f;
                    for (uint32_t o = 0; o < parts; ++o) whole += __ldcg(p.sums + uint64_t(rq.cu1 + unit * parts + o) * kBlock + threadIdx.x);
                    weight_row(p, rq, head)[key0 + threadIdx.x] += whole;
                }
                if (threadIdx.x == 0) *counter = 0;
            }
        }
        __syncthreads();
    }
    if (bad != 0) record_page_fault(p.geo);
}

template <typename T, int NC, int kMode>
cudaError_t launch_short(const WeighParams& p, uint32_t ctas, cudaStream_t stream) {
    constexpr int kSmem = 8 * kRingSteps<NC> * 16 * NC * 64;
    static std::atomic<uint64_t> done{0};
    const cudaError_t err = ensure_dynamic_smem(reinterpret_cast<const void*>(weigh_short_kernel<T, NC, kMode>), kSmem, done);
    if (err != cudaSuccess) return err;
    return launch_overlapped(weigh_short_kernel<T, NC, kMode>, dim3(ctas), dim3(256), kSmem, stream, p);
}

template <typename T, int NC>
cudaError_t launch_tensor(const WeighParams& p, WeighPass pass, uint32_t ctas, cudaStream_t stream) {
    switch (pass) {
        case WeighPass::kShortStatsScores: return launch_short<T, NC, kStatsAndScores>(p, ctas, stream);
        case WeighPass::kShortStats: return launch_short<T, NC, kStatsOnly>(p, ctas, stream);
        case WeighPass::kShortSumAgain: return launch_short<T, NC, kSumAgain>(p, ctas, stream);
        default: return cudaErrorInvalidValue;
    }
}

template <typename T>
cudaError_t launch_typed(const WeighParams& p, WeighPass pass, uint32_t ctas, cudaStream_t stream) {
    const uint32_t d = p.geo.head_dim;  // 64-byte pieces of a row, rounded up to a compiled count
    if (d <= 64) return launch_tensor<T, 2>(p, pass, ctas, stream);
    if (d <= 96) return launch_tensor<T, 3>(p, pass, ctas, stream);
    if (d <= 128) return launch_tensor<T, 4>(p, pass, ctas, stream);
    if (d <= 192) return launch_tensor<T, 6>(p, pass, ctas, stream);
    return launch_tensor<T, 8>(p, pass, ctas, stream);
}

cudaError_t launch_any(const WeighParams& p, WeighPass pass, uint32_t ctas, cudaStream_t stream) {
    const int most = int((kAnyRows + 2 * kBlock) * any_pitch(256) * sizeof(float));
    const size_t smem = (kAnyRows + 2 * kBlock) * any_pitch(p.geo.head_dim) * sizeof(float);
    static std::atomic<uint64_t> stats_done{0}, sum_done{0};
    const bool stats = pass == WeighPass::kLongStats;
    const cudaError_t err = stats ? ensure_dynamic_smem(reinterpret_cast<const void*>(weigh_stats_any_kernel), most, stats_done)
                                  : ensure_dynamic_smem(reinterpret_cast<const void*>(weigh_sum_any_kernel), most, sum_done);
    if (err != cudaSuccess) return err;
    return launch_overlapped(stats ? weigh_stats_any_kernel : weigh_sum_any_kernel, dim3(ctas), dim3(kAnyThreads), smem, stream, p);
}

}  // namespace

cudaError_t launch_weigh(const WeighParams& p, WeighPass pass, uint32_t ctas, cudaStream_t stream) {
    if (pass == WeighPass::kShortSumScores) return launch_overlapped(weigh_scores_kernel, dim3(ctas), dim3(256), 0, stream, p);
    if (!weigh_on_tensor_cores(p.dtype, p.geo.head_dim)) return launch_any(p, pass, ctas, stream);
    if (pass == WeighPass::kLongStats || pass == WeighPass::kLongSum) return launch_weigh_umma(p, pass == WeighPass::kLongStats, ctas, stream);
    return p.dtype == PSI_DTYPE_BF16 ? launch_typed<__nv_bfloat16>(p, pass, ctas, stream) : launch_typed<__half>(p, pass, ctas, stream);
}

}  // namespace psi
