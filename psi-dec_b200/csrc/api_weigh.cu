// C ABI: attention weight gathered by cached keys, and eviction from the cache by it.
#include "api_internal.hpp"
#include "evict.hpp"
#include "weigh_keys.hpp"

using namespace psi;

namespace psi {

namespace {

using LongRun = psi_weigh_plan::LongRun;

// Into items of how many key blocks the long runs of a batch are cut, between `least` and kMostBlocks, on the tensor cores.  The CTAs
// of a wave take items in turn, so that a launch takes as many rounds as items over CTAs, rounded up, of an item each; an item
// costs kItemStart blocks beside its own.  Four prompts' ends of 4,099 to 16,384 keys, 64 tokens of 32/8 heads x 128, in whole rounds:
// 104 us for both passes, against 140 with 8 and 4 blocks an item (2.3 rounds).  Batches of many runs take many rounds of whatever
// length: theirs is fixed.
constexpr uint32_t kMostBlocks = 24, kItemStart = 1, kMostRuns = 16;

template <typename Units>
uint32_t choose_blocks(const std::vector<LongRun>& runs, uint32_t least, uint32_t otherwise, const Units& units_of) {
    if (runs.size() > kMostRuns) return std::max(least, otherwise);
    constexpr uint32_t wave = weigh_wave(true);
    uint32_t best = least;
    double least_cost = 1e300;
    for (uint32_t blocks = least; blocks <= std::max(least, kMostBlocks); ++blocks) {
        uint64_t items = 0, work = 0;
        for (const LongRun& run : runs) {
            const uint64_t cuts = (run.key_blocks + blocks - 1) / blocks;
            items += units_of(run, false) * cuts;
            work += units_of(run, true) * (run.key_blocks + cuts * kItemStart);
        }
        const double cost = items == 0 ? 0.0 : double((items + wave - 1) / wave) * double(work) / double(items);
        if (cost < least_cost) {
            least_cost = cost;
            best = blocks;
        }
    }
    return best;
}

// First pass: an item for each unit (row block, KV head) and piece, kWeighMaxPieces pieces at most.
uint32_t choose_piece(const psi_gqa* g, const std::vector<LongRun>& runs) {
    uint32_t most = 1;
    for (const LongRun& run : runs) most = std::max(most, run.key_blocks);
    const uint32_t least = (most + kWeighMaxPieces - 1) / kWeighMaxPieces;
    if (g->replay_reserved) return std::max(least, kWeighPieceBlocks);
    return choose_blocks(runs, least, kWeighPieceBlocks, [](const LongRun& run, bool) { return run.units; });
}

// Second pass: an item for each KV head and span, through all row blocks.
uint32_t choose_span(const psi_gqa* g, const std::vector<LongRun>& runs, bool parted) {
    if (g->replay_reserved || parted) return kWeighSpan;
    const uint32_t heads = g->cfg.num_kv_heads;
    return choose_blocks(runs, 1, kWeighSpan, [heads](const LongRun& run, bool work) { return work ? run.units : uint64_t(heads); });
}

}  // namespace

// The batch as the key-weight kernels see it (WeighRequest): short runs, their end, long runs, their end.  A batch whose
// counts leave 32 bits is marked, and refused by psi_gqa_weigh_keys alone.
void plan_weigh(psi_gqa* g, const uint32_t* req_slots, const uint32_t* token_indices, const uint32_t* cu_tokens, uint32_t num_reqs) {
    psi_weigh_plan& w = g->weigh;
    w.reqs.clear();
    w.num_short = w.num_long = w.max_keys = w.short_rows = 0;
    w.long_units = 0;
    w.repeated = w.too_large = w.parted = false;
    const uint32_t group = g->cfg.num_q_heads / g->cfg.num_kv_heads, heads = g->cfg.num_kv_heads;
    const bool tensor = weigh_on_tensor_cores(g->cfg.dtype, g->cfg.head_dim);
    const uint32_t block = tensor ? kWeighBlock : kWeighAnyRows;
    if (w.seen.empty()) w.seen.assign(g->cfg.layout.num_req_slots, 0);
    w.epoch += 1;
    if (w.epoch == 0) {
        std::fill(w.seen.begin(), w.seen.end(), 0u);
        w.epoch = 1;
    }
    uint64_t cu0 = 0, cu1 = 0;
    std::vector<LongRun>& long_runs = w.long_runs;
    long_runs.clear();
    for (int pass = 0; pass < 2; ++pass) {  // 0: short runs, 1: long ones
        cu0 = cu1 = 0;
        const uint32_t piece_blocks = pass == 1 ? choose_piece(g, long_runs) : 0, span_blocks = pass == 1 ? choose_span(g, long_runs, w.parted) : 0;
        for (uint32_t r = 0; r < num_reqs; ++r) {
            const uint32_t q_len = cu_tokens[r + 1] - cu_tokens[r];
            if (q_len == 0) continue;
            const uint64_t rows = uint64_t(q_len) * group;
            const uint32_t keys = token_indices[r] + q_len;
            const bool is_short = tensor && rows <= kWeighShortRows;
            const uint32_t parts = is_short || g->replay_reserved
                                       ? 1
                                       : weigh_row_parts(static_cast<uint32_t>(std::min<uint64_t>(rows, kU32Max)), keys, heads, tensor);
            const uint64_t units = (rows + block - 1) / block * heads;
            if (pass == 0) {
                if (w.seen[req_slots[r]] == w.epoch) w.repeated = true;
                w.seen[req_slots[r]] = w.epoch;
                w.max_keys = std::max(w.max_keys, keys);
                if (parts > 1) w.parted = true;
                if (!is_short && tensor) long_runs.push_back(LongRun{weigh_blocks(keys), units});
            }
            if (is_short != (pass == 0)) continue;
            w.reqs.push_back(WeighRequest{req_slots[r], token_indices[r], q_len, cu_tokens[r], keys, uint32_t(cu0), uint32_t(cu1), uint32_t(w.long_units)});
            if (is_short) {
                w.num_short += 1;
                w.short_rows = std::max(w.short_rows, uint32_t(rows));
                cu0 += (uint64_t(keys) + kWeighTile - 1) / kWeighTile * heads;
            } else {
                w.num_long += 1;
                w.long_units += units;
                cu0 += units * (tensor ? weigh_cut(keys, piece_blocks) : weigh_any_pieces(keys));
                cu1 += uint64_t(parts) * (tensor ? weigh_cut(keys, span_blocks) : weigh_any_spans(keys)) * heads;
            }
        }
        WeighRequest end{};
        end.slot = piece_blocks;
        end.first_pos = span_blocks;
        end.cu0 = uint32_t(cu0);
        end.cu1 = uint32_t(cu1);
        w.reqs.push_back(end);
        w.too_large = w.too_large || cu0 > kU32Max || cu1 > kU32Max || w.long_units > kU32Max;
        if (pass == 0) w.tiles = cu0;
    }
    w.span_keys = tensor ? w.reqs.back().first_pos * kWeighBlock : kWeighAnyKeys;
    w.stats_items = cu0;
    w.sum_items = cu1;
    require(w.captured.expired() || (!w.repeated && !w.too_large),
            "a request slot appears twice in the batch: the captured key-weight launches cannot add to its keys twice at once");
}

}  // namespace psi

namespace {

// The first call on a component: what psi_gqa_prepare does for key weights from then on, for the batch at hand.
void plan_prepared(psi_gqa* g) {
    psi_ctx* ctx = g->ctx;
    psi_weigh_plan& w = g->weigh;
    plan_weigh(g, w.batch_slots.data(), w.batch_tokens.data(), g->batch_cu.data(), static_cast<uint32_t>(w.batch_slots.size()));
    const uint32_t counts[2] = {w.num_short, w.num_long};
    static_assert(kScalarWeighLong == kScalarWeighShort + 1);
    // pageable sources: staged before the calls return
    cuda_check(cudaMemcpyAsync(static_cast<uint32_t*>(g->block.ptr) + kScalarWeighShort, counts, sizeof(counts), cudaMemcpyHostToDevice, ctx->stream),
               "cudaMemcpyAsync");
    cuda_check(cudaMemcpyAsync(static_cast<uint32_t*>(g->block.ptr) + g->off_weigh, w.reqs.data(), w.reqs.size() * sizeof(WeighRequest),
                               cudaMemcpyHostToDevice, ctx->stream),
               "cudaMemcpyAsync");
    w.wanted = w.planned = true;
}

uint64_t table_tokens(const psi_gqa* g) {
    return uint64_t(g->cfg.layout.num_blocks) * g->cfg.layout.num_page_ids_per_block * g->tokens_per_page;
}

constexpr uint64_t kMostScratch = 2ull << 30;

void run_pass(psi_gqa* g, const WeighParams& p, WeighPass pass, uint64_t ctas) {
    LaunchScope scope(g->ctx, PSI_KERNEL_CLASS_WEIGH);
    cuda_check(launch_weigh(p, pass, static_cast<uint32_t>(ctas), g->ctx->stream), "key weight launch");
}

// The largest unit of a row copy: what the rows' bytes and the arena's address are multiples of.
uint32_t copy_unit(const PageGeometry& geo) {
    const uint64_t at = reinterpret_cast<uintptr_t>(geo.pages) | (uint64_t(geo.head_dim) * geo.elem_bytes);
    return at % 16 == 0 ? 16u : at % 4 == 0 ? 4u : 2u;
}

}  // namespace

extern "C" {

int32_t psi_gqa_weigh_keys(psi_gqa* g, psi_pages* pages, psi_table* table, uint32_t layer, const void* q, float* weights,
                           uint64_t weights_stride) {
    if (g == nullptr) return PSI_ERR_INVALID_ARGUMENT;
    return guarded(g->ctx, [&] {
        psi_ctx* ctx = g->ctx;
        psi_weigh_plan& w = g->weigh;
        require(g->prepared, "GQA batch metadata must be updated before recording");
        require(q != nullptr && weights != nullptr, "q and weights must not be null");
        const bool fixed = g->replay_reserved;
        require(ctx->capturing || !stream_captured(ctx), "capture key-weight launches by psi_ctx_capture_begin: the component has to know of their graph");
        require(!ctx->capturing || fixed, "reserve replay capacity before capturing key-weight launches");
        ctx->bind();
        if (!w.planned) {
            require(!ctx->capturing,
                    "call psi_gqa_weigh_keys once after the replay reservation and before the capture: it allocates its scratch then");
            plan_prepared(g);
        }
        require(!w.repeated, "a request slot appears twice in the batch: its keys cannot gather weight from two requests at once");
        require(!w.too_large, "the batch exceeds the key-weight kernels' work counts");
        WeighParams p{};
        p.geo = page_geometry(g, pages, table, layer);
        const bool tensor = weigh_on_tensor_cores(g->cfg.dtype, g->cfg.head_dim);
        require(!tensor || ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(p.geo.pages)) & 15u) == 0,
                "q and the page arena must be 16-byte aligned");
        require((reinterpret_cast<uintptr_t>(weights) & 3u) == 0, "weights must be 4-byte aligned");
        require(reinterpret_cast<uintptr_t>(q) % dtype_bytes(g->cfg.dtype) == 0, "q must be aligned to its elements");
        require(weights_stride >= w.max_keys, "the weights' row stride must hold every key of the batch");
        require(!ctx->capturing || weights_stride >= table_tokens(g),
                "captured key-weight launches need rows of weights as long as the page table's");
        const uint32_t heads = g->cfg.num_kv_heads, group = g->cfg.num_q_heads / heads;
        const uint64_t sms = static_cast<uint64_t>(ctx->sm_count);
        const uint32_t block = tensor ? kWeighBlock : kWeighAnyRows;
        const bool can_short = tensor, can_long = !tensor || uint64_t(g->cfg.max_tokens) * group > kWeighShortRows;
        // one wave of the short-run kernel's workers
        const uint64_t short_wave = sms;
        const uint64_t short_ctas = fixed ? (can_short ? short_wave : 0) : std::min<uint64_t>(short_wave, (w.tiles + 7) / 8);
        uint64_t short_units = uint64_t(w.num_short) * heads, long_units = w.long_units, stats_items = w.stats_items;
        if (fixed) {
            short_units = can_short ? uint64_t(g->cfg.max_tokens) * heads : 0;
            const uint64_t rows = uint64_t(g->cfg.max_tokens) * group;
            long_units = can_long ? (rows / block + (tensor ? rows / (kWeighShortRows + 1) : g->cfg.max_tokens) + 1) * heads : 0;
            const uint32_t tokens = static_cast<uint32_t>(std::min<uint64_t>(table_tokens(g), kU32Max));
            stats_items = long_units * (tensor ? std::min(weigh_cut(tokens, kWeighPieceBlocks), kWeighMaxPieces) : weigh_any_pieces(tokens));
        }
        const uint64_t short_slots = (short_ctas * 8 + short_units) * 16, long_slots = stats_items * block;
        const uint64_t partial_bytes = (short_slots + long_slots) * sizeof(float2);
        // (a span's counter stands at the place of its first item)
        const uint64_t counter_words = short_units + std::max(long_units, w.parted ? w.sum_items : 0);
        const uint64_t sum_bytes = w.parted ? w.sum_items * w.span_keys * sizeof(float) : 0;
        if (ctx->capturing) {
            require(w.norms.ptr != nullptr && partial_bytes <= w.partials.bytes && counter_words * sizeof(uint32_t) <= w.counters.bytes,
                    "call psi_gqa_weigh_keys once after the replay reservation and before the capture: it allocates its scratch then");
        } else {
            require(!fixed || partial_bytes <= kMostScratch,
                    "the replay reservation needs more than 2 GiB of key-weight scratch for this max_tokens: create the component with "
                    "the largest batch the replayed steps carry");
            w.norms.ensure(ctx, uint64_t(g->cfg.max_tokens) * g->cfg.num_q_heads * sizeof(float2), false);
            // (the reservation's size is the last one)
            w.partials.ensure(ctx, partial_bytes <= w.partials.bytes || fixed ? partial_bytes : std::max<uint64_t>(partial_bytes * 3 / 2, 1 << 16), false);
            w.sums.ensure(ctx, sum_bytes > w.sums.bytes ? sum_bytes * 3 / 2 : sum_bytes, false);
            if (counter_words * sizeof(uint32_t) > w.counters.bytes) {
                w.counters.release_after(ctx);  // counters restart from zero at their new size
                w.counters.ensure(ctx, std::max<uint64_t>(counter_words * 6, 1 << 12), true);
            }
        }
        p.q = q;
        p.weights = weights;
        p.stride = weights_stride;
        p.reqs = reinterpret_cast<const WeighRequest*>(block_words(g, g->off_weigh));
        p.scalars = block_words(g, 0);
        p.norms = static_cast<float2*>(w.norms.ptr);
        p.partials = static_cast<float2*>(w.partials.ptr);
        p.long_partials_at = short_slots;
        p.counters = static_cast<uint32_t*>(w.counters.ptr);
        p.long_counters_at = short_units;
        p.sums = static_cast<float*>(w.sums.ptr);
        p.split_rows = w.parted ? 1u : 0u;
        p.group = group;
        p.short_count = fixed ? 0xFFFFFFFFu : w.num_short;
        p.short_tiles = fixed ? 0xFFFFFFFFu : static_cast<uint32_t>(w.tiles);
        p.num_q_heads = g->cfg.num_q_heads;
        p.dtype = g->cfg.dtype;
        p.scale_log2 = g->cfg.scale * 1.4426950408889634f;
        p.score_rows = w.short_rows;
        bool keep_scores = false;
        if (short_ctas > 0 && !fixed) {
            // The scores of short runs stay in scratch between the passes; beyond 2 GiB, or where the device has no room left,
            // the second pass reads the keys again instead (32 requests of 1,024 to 8,192 keys, 2 KV heads x 256, 8 rows: 51 us with
            // scratch, 73 without).
            const uint64_t bytes = w.tiles * kWeighTile * p.score_rows * sizeof(float);
            keep_scores = grow_scratch(bytes, w.scores.bytes, kMostScratch, w.scores_refused, [&](uint64_t wanted) { return w.scores.replace(ctx, wanted); });
            p.scores = static_cast<float*>(w.scores.ptr);
        }
        if (ctx->capturing) {
            std::shared_ptr<int> mark = w.captured.lock();
            if (mark == nullptr) w.captured = mark = std::make_shared<int>(0);
            ctx->capture_marks.push_back(std::move(mark));
        }
        if (short_ctas > 0) run_pass(g, p, keep_scores ? WeighPass::kShortStatsScores : WeighPass::kShortStats, short_ctas);
        const uint64_t long_wave = tensor ? sms : sms * (g->cfg.head_dim > 96 ? 2 : 4);
        const uint64_t stats_ctas = fixed ? (can_long ? long_wave : 0) : std::min<uint64_t>(long_wave, w.stats_items);
        const uint64_t sum_ctas = fixed ? stats_ctas : std::min<uint64_t>(long_wave, w.sum_items);
        if (stats_ctas > 0) run_pass(g, p, WeighPass::kLongStats, stats_ctas);
        if (short_ctas > 0) {
            const uint64_t ctas = keep_scores ? std::min<uint64_t>(sms * 8, (w.tiles + 7) / 8) : short_ctas;
            run_pass(g, p, keep_scores ? WeighPass::kShortSumScores : WeighPass::kShortSumAgain, ctas);
        }
        if (stats_ctas > 0) run_pass(g, p, WeighPass::kLongSum, sum_ctas);
    });
}

int32_t psi_gqa_evict(psi_gqa* g, psi_pages* pages, psi_table* table, uint32_t layer, const uint32_t* src_slots,
                      const uint32_t* dst_slots, const uint32_t* lengths, const uint32_t* keeps, uint32_t num_reqs, uint32_t recent,
                      const float* weights, float* weights_out, uint64_t weights_stride, uint32_t* kept, uint64_t kept_stride) {
    if (g == nullptr) return PSI_ERR_INVALID_ARGUMENT;
    return guarded(g->ctx, [&] {
        psi_ctx* ctx = g->ctx;
        require(!stream_captured(ctx), "psi_gqa_evict takes its sizes from host arrays and stays outside captured graphs");
        require(num_reqs == 0 || (src_slots != nullptr && dst_slots != nullptr && lengths != nullptr && keeps != nullptr),
                "eviction inputs must not be null");
        require(weights != nullptr && weights_out != nullptr && kept != nullptr, "weights, weights_out and kept must not be null");
        require(((reinterpret_cast<uintptr_t>(weights) | reinterpret_cast<uintptr_t>(weights_out) | reinterpret_cast<uintptr_t>(kept)) & 3u) == 0,
                "weights and kept must be 4-byte aligned");
        require(g->cfg.num_kv_heads <= 32767, "eviction launches take up to 32767 KV heads");
        EvictParams p{};
        p.geo = page_geometry(g, pages, table, layer);
        require(reinterpret_cast<uintptr_t>(p.geo.pages) % p.geo.elem_bytes == 0, "the page arena must be aligned to its elements");
        const uint64_t capacity = table_tokens(g);
        const uint32_t slots = g->cfg.layout.num_req_slots;
        std::vector<uint32_t> role(slots, 0);  // 1 + r: slot is the source of request r
        std::vector<bool> taken(slots, false);
        for (uint32_t r = 0; r < num_reqs; ++r) {
            require(src_slots[r] < slots && dst_slots[r] < slots, "GQA request page table req_slot out of range");
            require(lengths[r] <= capacity, "eviction length does not fit the request page table");
            require(lengths[r] <= weights_stride, "the weights' row stride must hold every key of the batch");
            require(keeps[r] <= lengths[r], "eviction cannot keep more keys than the request has");
            require(keeps[r] <= kept_stride, "the kept rows' stride must hold every kept key");
            require(role[src_slots[r]] == 0, "a request slot is evicted from twice in one call");
            role[src_slots[r]] = 1 + r;
        }
        for (uint32_t r = 0; r < num_reqs; ++r) {
            require(!taken[dst_slots[r]], "two requests would move to one slot");
            taken[dst_slots[r]] = true;
            require(role[dst_slots[r]] == 0 || role[dst_slots[r]] == 1 + r, "a request would move to a slot that another one is read from");
        }
        ctx->bind();
        p.weights = weights;
        p.weights_out = weights_out;
        p.stride = weights_stride;
        p.kept_stride = kept_stride;
        p.recent = recent;
        p.unit_bytes = copy_unit(p.geo);
        const uint32_t sms = static_cast<uint32_t>(ctx->sm_count);
        for (uint32_t first = 0; first < num_reqs; first += kEvictBatch) {
            p.num_reqs = std::min(kEvictBatch, num_reqs - first);
            p.kept = kept + uint64_t(first) * g->cfg.num_kv_heads * kept_stride;
            bool in_place = false, apart = false;
            for (uint32_t r = 0; r < p.num_reqs; ++r) {
                const uint32_t at = first + r;
                p.reqs[r] = EvictRequest{src_slots[at], dst_slots[at], lengths[at], keeps[at]};
                const bool same = src_slots[at] == dst_slots[at];
                in_place = in_place || (same && keeps[at] > 0 && keeps[at] < lengths[at]);
                apart = apart || (!same && keeps[at] > 0);
            }
            {
                LaunchScope scope(ctx, PSI_KERNEL_CLASS_EVICT);
                cuda_check(launch_evict_select(p, sms, ctx->stream), "eviction selection launch");
            }
            for (uint32_t way = 0; way < 2; ++way) {
                if (!(way == 0 ? apart : in_place)) continue;
                p.in_place = way;
                LaunchScope scope(ctx, PSI_KERNEL_CLASS_EVICT);
                cuda_check(launch_evict_move(p, sms, ctx->stream), "eviction move launch");
            }
        }
    });
}

}  // extern "C"
