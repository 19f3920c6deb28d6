// Key weights of long query runs on the 5th-generation tensor cores (see weigh_keys.cu for the mathematics).
//
// A tile is the product of 128 query rows and 128 keys.  First pass: A = query rows, B = keys, an accumulator lane is a row, whose
// maximum and sum stay inside a thread.  Second pass: A = keys, B = query rows, a lane is a key, whose sum over the rows stays
// inside a thread, and what belongs to a row (its maximum, 1 / sum and limit) is read from shared memory.  The query rows
// of an item stay in shared memory, key blocks pass by in a ring of two (cp.async from their pages, any page size), and the MMA of
// a block runs under the exponentials of the block before: two S buffers in TMEM.  Threads w and w + 128 share a lane, half of the
// columns each.  Bound by issue slots: a tile's 128 x 128 exponentials take 1,024 cycles of the special-function unit in each pass and
// its product 512 of the tensor pipe (at head_dim 128), but an element takes about four instructions beside its exponential.  (A
// quarter of the exponentials as polynomials on the FMA pipe cost more slots than they freed: 68 and 80 us for the passes over
// four prompts of 4,099 to 16,384 keys, 64 tokens of 32/8 heads x 128 each.)  Two CTAs share an SM at head_dim 128 and below, so that
// one's loads and barriers run under the other's arithmetic.
// Every mbarrier wait is bounded and reports PSI_ERR_TIMEOUT through the status word, and TMEM is freed on every path.
#include <type_traits>

#include "launch_util.hpp"
#include "umma_common.cuh"
#include "weigh_common.cuh"

namespace psi {

namespace {

constexpr uint32_t kRows = kWeighBlock;     // rows or keys of a block, and lanes
constexpr uint32_t kThreads = 256;
constexpr uint32_t kTmemColumns = 2 * kRows;

struct UmmaWeighShared {
    uint64_t bars[2];
    uint32_t tmem_base, abort, last_arrival, dead_rows;
    __align__(16) float neg_max[kRows];   // second pass: of the block's rows
    __align__(16) float inverse[kRows];
    __align__(16) uint32_t limit[kRows];
    float2 half[kRows];                   // what the upper half of the columns gave
    uint64_t offsets[2][kRows];           // element offsets of the rows of a ring slot's next block
};

// kBlocks: 64-element blocks of a row.  kStats: first pass.
template <typename T, uint32_t kBlocks, bool kStats>
__global__ void __launch_bounds__(kThreads, kBlocks <= 2 ? 2 : 1) weigh_umma_kernel(const WeighParams p) {
    constexpr uint32_t kTileBytes = kBlocks * kRows * 128;  // a block of 128 rows: [64-element block][row][128 bytes, swizzled]
    constexpr uint32_t kLanes = kBlocks == 3 ? 32 : kBlocks * 8;  // threads that copy a row, a chunk each
    __shared__ UmmaWeighShared sh;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    const uint32_t tid = threadIdx.x, warp = tid >> 5;
    const uint32_t smem_rows = (smem_u32(smem_raw) + 1023u) & ~1023u, smem_ring = smem_rows + kTileBytes;
    const uint32_t bar0 = smem_u32(sh.bars);
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem_base)), "r"(kTmemColumns) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (tid == 0) {
        mbar_init(bar0, 1);
        mbar_init(bar0 + 8, 1);
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
    const uint32_t cut = kStats ? reqs[count].slot : reqs[count].first_pos, cut_keys = cut * kRows;  // of an item's keys
    const uint32_t row = tid & (kRows - 1), half = tid >> 7;
    const uint32_t lane_base = ((warp & 3u) * 32u) << 16, column0 = half * (kRows / 2);
    const PageBounds bounds(p.geo);
    uint32_t bad = 0;
    uint32_t tiles_done = 0;  // over all items: tile t has S buffer, ring slot and barrier t % 2
    const uint32_t chunks = p.geo.head_dim >> 3;
    const uint32_t idesc = umma_idesc<T>(kRows, false);

    const auto wait = [&](uint32_t tile) {
        const uint32_t bar = bar0 + (tile & 1u) * 8, parity = (tile >> 1) & 1u;
        if (mbar_try(bar, parity)) return;
        if (*reinterpret_cast<volatile uint32_t*>(&sh.abort) == 0 && !mbar_wait(bar, parity)) {
            *reinterpret_cast<volatile uint32_t*>(&sh.abort) = 1;
            if (p.geo.fault != nullptr) atomicExch(p.geo.fault, uint32_t(PSI_ERR_TIMEOUT));
        }
    };
    // Copies 128 rows whose element offsets stand in shared memory (~0: zeros) into a block.  A thread's chunk and its place in the
    // swizzle stay the same from row to row: its rows are a multiple of eight apart.
    const uint32_t copy_row = tid / kLanes, copy_chunk = tid % kLanes;
    const uint32_t copy_at = (copy_chunk >> 3) * (kRows * 128) + copy_row * 128 + (((copy_chunk ^ copy_row) & 7u) << 4);
    const bool copies = copy_chunk < kBlocks * 8, has_data = copy_chunk < chunks;
    const auto copy_block = [&](uint32_t dst, const void* base, const uint64_t* offsets) {
        if (!copies) return;
        const uint16_t* from = static_cast<const uint16_t*>(base) + (has_data ? copy_chunk * 8u : 0u);
#pragma unroll
        for (uint32_t r = 0; r < kRows; r += kThreads / kLanes) {
            const uint64_t offset = offsets[copy_row + r];
            const bool live = has_data && offset != ~0ull;
            cp_async_16(dst + copy_at + r * 128, from + (live ? offset : 0u), live ? 16u : 0u);
        }
    };

    for (uint32_t item = blockIdx.x; item < total; item += gridDim.x) {
        const uint32_t r_index = kStats ? find_request<0>(reqs, count, item) : find_request<1>(reqs, count, item);
        const WeighRequest rq = reqs[r_index];
        const uint32_t rows = rq.q_len * p.group, blocks = (rows + kRows - 1) / kRows;
        const uint32_t* row_ids = table_row(p.geo, rq.slot);
        uint32_t head, block_begin, block_end, k_begin, k_end, pieces = 1, unit = 0;
        if (kStats) {
            pieces = weigh_cut(rq.keys, cut);
            const uint32_t local = item - rq.cu0, piece = local % pieces;
            unit = local / pieces;
            head = unit / blocks;
            block_begin = unit % blocks;
            block_end = block_begin + 1;
            k_begin = piece * cut_keys;
            k_end = min(k_begin + cut_keys, rq.keys);
        } else {
            pieces = p.split_rows != 0 ? weigh_row_parts(rows, rq.keys, p.geo.num_kv_heads, true) : 1u;
            const uint32_t spans = weigh_cut(rq.keys, cut), local = item - rq.cu1, part = local % pieces, each = weigh_part_blocks(rows, pieces, true);
            unit = local / pieces;
            head = unit / spans;
            block_begin = part * each;
            block_end = min(block_begin + each, blocks);
            k_begin = unit % spans * cut_keys;
            k_end = min(k_begin + cut_keys, rq.keys);
            // rows of tokens before the span's first key see none of it
            if (k_begin > rq.first_pos) block_begin = max(block_begin, uint32_t(uint64_t(k_begin - rq.first_pos) * p.group / kRows));
            if (pieces > 1)
                for (uint32_t i = tid; i < cut_keys; i += kThreads) p.sums[uint64_t(item) * cut_keys + i] = 0.0f;
            __syncthreads();
        }
        // where a key's sum goes: its weight, or this part's share of it
        float* const sums = kStats ? nullptr : pieces > 1 ? p.sums + uint64_t(item) * cut_keys - k_begin : weight_row(p, rq, head);
        for (uint32_t block = block_begin; block < block_end; ++block) {
            const uint32_t row0 = block * kRows;
            const uint32_t seen = min(k_end, row_limit(p, rq, min(row0 + kRows, rows) - 1));  // keys that a row of the block sees end here
            const uint32_t tiles = seen > k_begin ? (seen - k_begin + kRows - 1) / kRows : 0u;
            Stat st{-kInf, 0.0f};
            const uint32_t my_row = row0 + row;
            const uint32_t my_limit = kStats && my_row < rows ? min(seen, row_limit(p, rq, my_row)) : 0u;
            const auto key_offsets = [&](uint32_t tile) {  // by the lower 128 threads, for the copy behind the next barrier
                if (half == 0) {
                    const uint32_t key = k_begin + tile * kRows + row;
                    uint64_t offset = ~0ull;
                    if (key < k_end) {
                        const uint32_t page = bounds.read(row_ids, key / p.geo.tokens_per_page, bad);
                        offset = kv_row_offset(p.geo, page, head, key % p.geo.tokens_per_page);
                    }
                    sh.offsets[tile & 1u][row] = offset;
                }
            };
            if (tiles > 0) {
                // the block's query rows, the first key block and, in the second pass, the rows' numbers
                if (half == 1) sh.offsets[1][row] = my_row < rows ? query_row(p, rq, head, my_row) * p.geo.head_dim : ~0ull;
                key_offsets(0);
                uint32_t dead = 0;
                if (!kStats && half == 1) {
                    const float2 norm = my_row < rows ? p.norms[query_row(p, rq, head, my_row)] : make_float2(kInf, 0.0f);
                    sh.neg_max[row] = -norm.x;
                    sh.inverse[row] = norm.y;
                    sh.limit[row] = my_row < rows ? row_limit(p, rq, my_row) : 0u;
                    dead = my_row < rows && norm.y == 0.0f ? 1u : 0u;
                }
                dead = __syncthreads_or(int(dead)) != 0 ? 1u : 0u;
                copy_block(smem_rows, p.q, sh.offsets[1]);
                copy_block(smem_ring + (tiles_done & 1u) * kTileBytes, p.geo.pages, sh.offsets[0]);
                cp_async_commit();
                __syncthreads();  // (the offsets have been read)
                if (tiles > 1) key_offsets(1);
                if (!kStats && tid == 0) sh.dead_rows = dead;
            }
            const auto take = [&](uint32_t tile) {
                const uint32_t key0 = k_begin + tile * kRows, t = tiles_done + tile;
                const uint32_t at = tmem + (t & 1u) * kRows + lane_base + column0;
                if constexpr (kStats) {
                    // this thread's row against 64 keys
                    float s[64];
                    tmem_load64(at, s);
                    const uint32_t key = key0 + column0;
                    if (key + 64 > my_limit) {
#pragma unroll
                        for (uint32_t c = 0; c < 64; ++c)
                            if (key + c >= my_limit) s[c] = -kInf;
                    }
                    float tops[4] = {-kInf, -kInf, -kInf, -kInf};
#pragma unroll
                    for (int c = 0; c < 64; c += 2) tops[(c >> 1) & 3] = max3_nan(tops[(c >> 1) & 3], s[c], s[c + 1]);  // (a NaN leaves no sum)
                    float top = max3_nan(max3_nan(tops[0], tops[1], tops[2]), tops[3], tops[3]);
                    top = max3_nan(st.m, st.m, top * p.scale_log2);
                    const float base = top == -kInf ? 0.0f : top;
                    st.l *= exp2_approx(st.m - base);
                    st.m = top;
                    const uint64_t scale2 = pack_f32x2(p.scale_log2, p.scale_log2), base2 = pack_f32x2(-base, -base);
                    uint64_t sum[4] = {0, 0, 0, 0};
#pragma unroll
                    for (int c = 0; c < 64; c += 2) {
                        const float2 x = unpack_f32x2(fma_f32x2(pack_f32x2(s[c], s[c + 1]), scale2, base2));
                        sum[(c >> 1) & 3] = add_f32x2(sum[(c >> 1) & 3], pack_f32x2(exp2_approx(x.x), exp2_approx(x.y)));
                    }
                    const float2 all = unpack_f32x2(add_f32x2(add_f32x2(sum[0], sum[1]), add_f32x2(sum[2], sum[3])));
                    st.l += all.x + all.y;
                } else {
                    // this thread's key against 64 rows
                    const uint32_t key = key0 + row;
                    const bool masked = key0 + kRows > row_limit(p, rq, row0) || row0 + kRows > rows || sh.dead_rows != 0;
                    const uint64_t scale2 = pack_f32x2(p.scale_log2, p.scale_log2);
                    uint64_t sum[4] = {0, 0, 0, 0};
                    const auto columns = [&](const auto with_mask) {
                        float s[64];
                        tmem_load64(at, s);
#pragma unroll
                        for (uint32_t c = 0; c < 64; c += 4) {
                            const ulonglong2 base = *reinterpret_cast<const ulonglong2*>(&sh.neg_max[column0 + c]);
                            const ulonglong2 inverse = *reinterpret_cast<const ulonglong2*>(&sh.inverse[column0 + c]);
                            float2 x = unpack_f32x2(fma_f32x2(pack_f32x2(s[c], s[c + 1]), scale2, base.x));
                            float2 y = unpack_f32x2(fma_f32x2(pack_f32x2(s[c + 2], s[c + 3]), scale2, base.y));
                            x = make_float2(exp2_approx(x.x), exp2_approx(x.y));
                            y = make_float2(exp2_approx(y.x), exp2_approx(y.y));
                            if constexpr (decltype(with_mask)::value) {
                                const uint4 limit = *reinterpret_cast<const uint4*>(&sh.limit[column0 + c]);
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
                    if (masked)
                        columns(std::true_type{});
                    else
                        columns(std::false_type{});
                    const float2 all = unpack_f32x2(add_f32x2(add_f32x2(sum[0], sum[1]), add_f32x2(sum[2], sum[3])));
                    if (half == 1) sh.half[row].x = all.x + all.y;
                    asm volatile("bar.sync %0, 64;" ::"r"((warp & 3u) + 1) : "memory");  // the warps of these lanes
                    if (half == 0 && key < k_end) sums[key] += all.x + all.y + sh.half[row].x;
                }
            };
            for (uint32_t tile = 0; tile < tiles; ++tile) {
                const uint32_t t = tiles_done + tile;
                cp_async_wait<0>();
                fence_async_smem();
                tc_fence_before();
                __syncthreads();  // the block has landed; the S buffer's last contents have been taken
                tc_fence_after();
                if (warp == 0 && elect_one()) {
                    const uint32_t ring = smem_ring + (t & 1u) * kTileBytes;
                    const uint64_t a = umma_desc(kStats ? smem_rows : ring, 16, 1024), b = umma_desc(kStats ? ring : smem_rows, 16, 1024);
#pragma unroll
                    for (uint32_t ks = 0; ks < kBlocks * 4; ++ks) {
                        const uint32_t step = ((ks >> 2) * (kRows * 128) + (ks & 3) * 32) / 16;
                        umma_ss(tmem + (t & 1u) * kRows, a + step, b + step, idesc, ks);
                    }
                    umma_commit_one(bar0 + (t & 1u) * 8);
                }
                if (tile > 0) wait(t - 1);  // its ring slot is free, its S is there
                tc_fence_after();
                if (tile + 1 < tiles) {
                    copy_block(smem_ring + ((t + 1) & 1u) * kTileBytes, p.geo.pages, sh.offsets[(tile + 1) & 1u]);
                    cp_async_commit();
                }
                if (tile + 2 < tiles) key_offsets(tile + 2);  // (its words were last read before this tile's barrier)
                if (tile > 0) take(tile - 1);
            }
            if (tiles > 0) {
                wait(tiles_done + tiles - 1);
                tc_fence_after();
                take(tiles - 1);
                tc_fence_before();
            }
            tiles_done += tiles;
            __syncthreads();  // the query rows and their numbers may be replaced
            if constexpr (kStats) {
                if (half == 1) sh.half[row] = make_float2(st.m, st.l);
                __syncthreads();
                if (half == 0) {
                    st.join(sh.half[row].x, sh.half[row].y);
                    if (pieces == 1) {
                        if (my_row < rows) p.norms[query_row(p, rq, head, my_row)] = st.norm();
                    } else {
                        p.long_partials()[uint64_t(item) * kRows + row] = make_float2(st.m, st.l);
                    }
                }
                if (pieces > 1) {
                    __threadfence();
                    __syncthreads();
                    uint32_t* counter = p.long_counters() + rq.unit0 + unit;
                    if (tid == 0) sh.last_arrival = atomicAdd(counter, 1u) == pieces - 1 ? 1u : 0u;
                    __syncthreads();
                    if (sh.last_arrival != 0) {
                        __threadfence();
                        if (half == 0 && my_row < rows) {
                            Stat all{-kInf, 0.0f};
                            for (uint32_t o = 0; o < pieces; ++o) {
                                const float2 v = __ldcg(p.long_partials() + uint64_t(rq.cu0 + unit * pieces + o) * kRows + row);
                                all.join(v.x, v.y);
                            }
                            p.norms[query_row(p, rq, head, my_row)] = all.norm();
                        }
                        if (tid == 0) *counter = 0;
                    }
                    __syncthreads();
                }
            }
        }
        if constexpr (!kStats) {
            if (pieces > 1) {  // the last part of the span adds up the parts
                __threadfence();
                __syncthreads();
                uint32_t* counter = p.long_counters() + rq.cu1 + unit * pieces;
                if (tid == 0) sh.last_arrival = atomicAdd(counter, 1u) == pieces - 1 ? 1u : 0u;
                __syncthreads();
                if (sh.last_arrival != 0) {
                    __threadfence();
                    for (uint32_t i = tid; i < k_end - k_begin; i += kThreads) {
                        float all = 0.0f;
                        for (uint32_t o = 0; o < pieces; ++o) all += __ldcg(p.sums + uint64_t(rq.cu1 + unit * pieces + o) * cut_keys + i);
                        weight_row(p, rq, head)[k_begin + i] += all;
                    }
                    if (tid == 0) *counter = 0;
                }
                __syncthreads();
            }
        }
    }
    if (bad != 0) record_page_fault(p.geo);
    tc_fence_before();
    __syncthreads();
    if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemColumns) : "memory");
}

template <typename T, uint32_t kBlocks, bool kStats>
cudaError_t launch_one(const WeighParams& p, uint32_t ctas, cudaStream_t stream) {
    constexpr int kSmem = int(3 * kBlocks * kRows * 128 + 1024);
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
