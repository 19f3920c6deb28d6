// C ABI: linear attention with a decay for each head.
#include "api_internal.hpp"
#include "linear_attend.hpp"

using namespace psi;

struct psi_linear {
    psi_ctx* ctx = nullptr;
    psi_linear_config cfg{};
    DeviceBuffer block;        // scalars | requests, at the same place from step to step
    uint32_t* staging = nullptr;
    cudaEvent_t upload_done = nullptr;
    DeviceBuffer decays;       // [layers][Hv][kLinearDecays]
    DeviceBuffer status_word;  // u32 written by bounded device-side waits
    bool chunked = false;      // long runs take the chunked form,
    uint32_t step_tokens = 0;  // those of more tokens than this
    DeviceBuffer carries;      // [max_carries][Hv][Dk][Dv]: states between the pieces of a request
    uint32_t max_carries = 0;
    uint32_t num_steps = 0, num_runs = 0, num_carries = 0, num_scans = 0, num_tokens = 0;  // of the prepared batch
    bool prepared = false;
    std::vector<uint32_t> reads, writes;  // by slot: readers of it in the batch at hand, and whether one writes it
};

namespace {

// Runs of more tokens take the chunked form, which costs the same from 1 to 64 tokens; the recurrent form's cost grows with the tokens
// and the state.  16/32 heads, bf16, launches one behind the other, recurrent and chunked in us, for one request, 32 and 128:
//   128 x 128, 9 tokens    6.2 and 8.7,  49 and 53,  191 and 227        64 x 64, 16 tokens   5.5 and 6.0,  25 and 33,   88 and 132
//   10 tokens              7.1 and 8.7,  58 and 53,  225 and 228        24 tokens            7.1 and 6.1,  34 and 33,  125 and 133
//   16 tokens              8.3 and 8.7,  77 and 54,  300 and 228
uint32_t step_tokens(const psi_linear_config& c) { return c.key_dim <= 64 && c.value_dim <= 64 ? 16 : 9; }

// Into how many chunks the pieces of a batch's long runs are cut (0: nothing is cut).  The chunked form takes one CTA per run and head
// through its chunks in turn, so that few heads leave SMs idle; pieces side by side cost a pass for the states between them.  In units
// of a chunk's time (2.2 us at 128 x 128 in bf16, the state pass's 0.5 of it): a launch takes the longest CTA's chunks, the CTAs going
// round their items, and the scan with its two launches three.  128 x 128, bf16, cut and whole: 32 heads, 1,024 tokens 38 and 46 us,
// 8,192 tokens 157 and 284; 4 heads, 512 tokens 26 and 28, 1,024 tokens 28 and 45, 8,192 tokens 46 and 278.
uint32_t piece_chunks(const std::vector<uint32_t>& run_tokens, uint32_t heads, uint32_t sms, uint32_t max_carries) {
    uint32_t longest = 0;
    const auto chunks_of = [](uint32_t tokens) { return (tokens + kLinearChunk - 1) / kLinearChunk; };
    for (uint32_t tokens : run_tokens) longest = std::max(longest, chunks_of(tokens));
    const auto cost = [&](uint32_t length) {  // pieces of `length` chunks
        uint64_t items = 0, chunks = 0, carried = 0, carries = 0;
        for (uint32_t tokens : run_tokens) {
            const uint64_t c = chunks_of(tokens), pieces = (c + length - 1) / length;
            items += pieces * heads;
            chunks += c * heads;
            if (pieces > 1) {
                carried += (pieces - 1) * heads;
                carries += pieces;
            }
        }
        if (carries > max_carries) return 1e30;
        const auto launch = [&](uint64_t n, uint64_t work) {
            const double rounds = double((n + sms - 1) / sms);
            return std::max(std::min(rounds * length, double(work)), double(work) / sms + 0.5 * length) + rounds;
        };
        const double full = launch(items, chunks);
        return carried == 0 ? full : full + 0.5 * launch(carried, carried * length) + 3.0;
    };
    uint32_t best = 0;
    double least = cost(longest);
    for (uint32_t pieces = 2; pieces <= 32; ++pieces) {
        const uint32_t length = (longest + pieces - 1) / pieces;
        if (length < 2) break;
        const double c = cost(length);
        if (c < 0.95 * least) {
            least = c;
            best = length;
        }
    }
    return best;
}

// What the kernels know of a head's decay (kLinearDecays).
void fill_decay(float* out, float log_decay) {
    for (uint32_t i = 0; i <= kLinearChunk; ++i) out[i] = float(std::exp(double(log_decay) * i));
    out[kLinearChunkLow] = float(std::exp(double(log_decay) * kLinearChunk) - double(out[kLinearChunk]));
    out[kLinearStepLow] = float(std::exp(double(log_decay)) - double(out[1]));
    out[kLinearStepLow + 1] = 0.0f;
}

uint64_t block_capacity(const psi_linear* l) { return kLinearScalarCount + uint64_t(l->cfg.max_tokens) * kLinearRequestWords; }

}  // namespace

extern "C" {

int32_t psi_linear_create(psi_ctx* ctx, const psi_linear_config* config, psi_linear** out) {
    if (ctx == nullptr) return PSI_ERR_INVALID_ARGUMENT;
    return guarded(ctx, [&] {
        require(out != nullptr && config != nullptr, "out and config must not be null");
        *out = nullptr;
        const psi_linear_config& c = *config;
        require(c.num_k_heads > 0 && c.num_v_heads > 0, "linear attention head counts must be positive");
        require(c.num_v_heads % c.num_k_heads == 0, "linear attention v heads must be a multiple of k heads");
        require(c.num_v_heads <= 65535, "linear attention launches take up to 65535 v heads");
        require(c.key_dim > 0 && c.key_dim % 8 == 0 && c.key_dim <= kLinearMaxDim && c.value_dim > 0 && c.value_dim % 8 == 0 &&
                    c.value_dim <= kLinearMaxDim,
                "linear attention key_dim and value_dim must be multiples of 8 up to 256");
        require(c.scale > 0.0f && std::isfinite(c.scale), "linear attention scale must be positive");
        require(c.dtype <= PSI_DTYPE_F16, "unsupported linear attention dtype");
        require(c.num_req_slots > 0 && c.num_layers > 0 && c.max_tokens > 0, "linear attention slots, layers and tokens must be positive");
        require(uint64_t(c.max_tokens) * c.num_v_heads * 8 <= kU32Max, "linear attention batch exceeds the kernels' work counts");
        require(!stream_captured(ctx), "a linear attention component cannot be created during stream capture");
        ctx->bind();
        auto l = std::make_unique<psi_linear>();
        l->ctx = ctx;
        l->cfg = c;
        l->reads.assign(c.num_req_slots, 0);
        l->writes.assign(c.num_req_slots, 0);
        const uint64_t decays = uint64_t(c.num_layers) * c.num_v_heads;
        std::vector<float> none(decays * kLinearDecays);
        for (uint64_t i = 0; i < decays; ++i) fill_decay(none.data() + i * kLinearDecays, 0.0f);
        // pieces for four rounds of CTAs
        l->max_carries = std::max<uint32_t>(2, 4 * static_cast<uint32_t>(ctx->sm_count) / c.num_v_heads);
        l->step_tokens = step_tokens(c);
        l->chunked = linear_chunk_supported(c.dtype, c.key_dim, c.value_dim) && c.max_tokens > l->step_tokens;
        try {
            l->block.ensure(ctx, block_capacity(l.get()) * sizeof(uint32_t), true);
            l->status_word.ensure(ctx, sizeof(uint32_t), true);
            if (l->chunked && c.max_tokens > 2 * kLinearChunk)
                l->carries.ensure(ctx, uint64_t(l->max_carries) * c.num_v_heads * c.key_dim * c.value_dim * sizeof(float), false);
            l->decays.ensure(ctx, none.size() * sizeof(float), false);
            cuda_check(cudaMemcpyAsync(l->decays.ptr, none.data(), none.size() * sizeof(float), cudaMemcpyHostToDevice, ctx->stream),
                       "cudaMemcpyAsync");  // pageable source: staged before the call returns
            cuda_check(cudaMallocHost(reinterpret_cast<void**>(&l->staging), block_capacity(l.get()) * sizeof(uint32_t)), "cudaMallocHost");
            cuda_check(cudaEventCreateWithFlags(&l->upload_done, cudaEventDisableTiming), "cudaEventCreateWithFlags");
        } catch (...) {
            l->block.release();
            l->decays.release();
            l->status_word.release();
            l->carries.release();
            if (l->staging != nullptr) (void)cudaFreeHost(l->staging);
            throw;
        }
        *out = l.release();
    });
}

int32_t psi_linear_destroy(psi_linear* l) {
    if (l == nullptr) return PSI_OK;
    const int32_t status = guarded(l->ctx, [&] {
        l->ctx->bind();
        (void)cudaStreamSynchronize(l->ctx->stream);
        l->block.release();
        l->decays.release();
        l->status_word.release();
        l->carries.release();
        if (l->staging != nullptr) (void)cudaFreeHost(l->staging);
        if (l->upload_done != nullptr) (void)cudaEventDestroy(l->upload_done);
    });
    delete l;
    return status;
}

int32_t psi_linear_set_decay(psi_linear* l, uint32_t layer, const float* log_decay) {
    if (l == nullptr) return PSI_ERR_INVALID_ARGUMENT;
    return guarded(l->ctx, [&] {
        psi_ctx* ctx = l->ctx;
        require(log_decay != nullptr, "log_decay must not be null");
        require(layer < l->cfg.num_layers, "linear attention layer out of range");
        require(!stream_captured(ctx), "psi_linear_set_decay uploads the decays and stays outside captured graphs");
        const uint32_t heads = l->cfg.num_v_heads;
        std::vector<float> parts(uint64_t(heads) * kLinearDecays);
        for (uint32_t h = 0; h < heads; ++h) {
            require(std::isfinite(log_decay[h]) && log_decay[h] <= 0.0f, "log_decay must be finite and not positive");
            fill_decay(parts.data() + uint64_t(h) * kLinearDecays, log_decay[h]);
        }
        ctx->bind();
        cuda_check(cudaMemcpyAsync(static_cast<float*>(l->decays.ptr) + uint64_t(layer) * heads * kLinearDecays, parts.data(),
                                   parts.size() * sizeof(float), cudaMemcpyHostToDevice, ctx->stream),
                   "cudaMemcpyAsync");  // pageable source: staged before the call returns
    });
}

int32_t psi_linear_prepare(psi_linear* l, const uint32_t* req_slots, const uint32_t* out_slots, const uint32_t* token_indices,
                           const uint32_t* cu_tokens, uint32_t num_reqs) {
    if (l == nullptr) return PSI_ERR_INVALID_ARGUMENT;
    return guarded(l->ctx, [&] {
        psi_ctx* ctx = l->ctx;
        require(!stream_captured(ctx), "psi_linear_prepare uploads the step's batch and stays outside captured graphs");
        require(req_slots != nullptr && token_indices != nullptr && cu_tokens != nullptr, "metadata inputs must not be null");
        require(num_reqs > 0, "linear attention batch requires tokens");
        require(cu_tokens[0] == 0, "linear attention batch cu_tokens must start at zero");
        for (uint32_t r = 0; r < num_reqs; ++r)
            require(cu_tokens[r] <= cu_tokens[r + 1], "linear attention batch cu_tokens must be nondecreasing");
        require(cu_tokens[num_reqs] > 0, "linear attention batch requires tokens");
        require(cu_tokens[num_reqs] <= l->cfg.max_tokens, "linear attention batch exceeds the token capacity");
        const uint32_t* outs = out_slots != nullptr ? out_slots : req_slots;
        for (uint32_t r = 0; r < num_reqs; ++r)
            require(req_slots[r] < l->cfg.num_req_slots && outs[r] < l->cfg.num_req_slots, "linear attention req_slot out of range");
        l->prepared = false;
        // a slot is written by one request at most, and then read by none other
        std::fill(l->reads.begin(), l->reads.end(), 0u);
        std::fill(l->writes.begin(), l->writes.end(), 0u);
        for (uint32_t r = 0; r < num_reqs; ++r) {
            if (cu_tokens[r] == cu_tokens[r + 1]) continue;
            require(l->writes[outs[r]] == 0, "two requests would write the state of one slot");
            l->writes[outs[r]] = 1;
            if (token_indices[r] > 0) l->reads[req_slots[r]] += 1;
        }
        for (uint32_t r = 0; r < num_reqs; ++r) {
            if (cu_tokens[r] == cu_tokens[r + 1]) continue;
            const uint32_t own = outs[r] == req_slots[r] && token_indices[r] > 0 ? 1 : 0;
            require(l->reads[outs[r]] == own, "a request would write the state that another one reads");
        }
        ctx->bind();
        cuda_check(cudaEventSynchronize(l->upload_done), "cudaEventSynchronize");  // previous upload left staging
        std::fill(l->staging, l->staging + kLinearScalarCount, 0u);
        auto* reqs = reinterpret_cast<LinearRequest*>(l->staging + kLinearScalarCount);
        uint32_t n = 0;
        for (uint32_t r = 0; r < num_reqs; ++r) {
            const uint32_t q_len = cu_tokens[r + 1] - cu_tokens[r];
            if (q_len > 0 && !(l->chunked && q_len > l->step_tokens))
                reqs[n++] = LinearRequest{req_slots[r], outs[r], token_indices[r] == 0 ? 1u : 0u, q_len, cu_tokens[r], {0, 0, 0}};
        }
        l->num_steps = n;
        // the long runs in pieces: those that another one follows first, then the ends
        std::vector<uint32_t> long_runs, run_tokens;
        for (uint32_t r = 0; r < num_reqs && l->chunked; ++r) {
            if (cu_tokens[r + 1] - cu_tokens[r] <= l->step_tokens) continue;
            long_runs.push_back(r);
            run_tokens.push_back(cu_tokens[r + 1] - cu_tokens[r]);
        }
        const uint32_t chunks = l->carries.ptr == nullptr || long_runs.empty()
                                    ? 0
                                    : piece_chunks(run_tokens, l->cfg.num_v_heads, static_cast<uint32_t>(ctx->sm_count), l->max_carries);
        const uint32_t piece = chunks * kLinearChunk;  // tokens
        auto* runs = reinterpret_cast<LinearRun*>(reqs + n);
        std::vector<LinearRun> ends;
        std::vector<LinearScan> scans;
        uint32_t num_runs = 0, carry = 0;
        for (uint32_t i = 0; i < long_runs.size(); ++i) {
            const uint32_t r = long_runs[i], begin = cu_tokens[r], tokens = run_tokens[i], fresh = token_indices[r] == 0 ? 1u : 0u;
            if (piece == 0 || tokens <= piece) {
                ends.push_back(LinearRun{req_slots[r], outs[r], fresh, 1, begin, tokens, kLinearNoCarry, kLinearNoCarry});
                continue;
            }
            const uint32_t pieces = (tokens + piece - 1) / piece;
            scans.push_back(LinearScan{req_slots[r], fresh, carry, pieces, chunks, {0, 0, 0}});
            for (uint32_t x = 0; x + 1 < pieces; ++x)
                runs[num_runs++] = LinearRun{req_slots[r], outs[r], 0, 0, begin + x * piece, piece, carry + x, carry + x + 1};
            ends.push_back(LinearRun{req_slots[r], outs[r], 0, 1, begin + (pieces - 1) * piece, tokens - (pieces - 1) * piece, carry + pieces - 1, kLinearNoCarry});
            carry += pieces;
        }
        l->num_carries = num_runs;
        std::stable_sort(ends.begin(), ends.end(), [](const LinearRun& a, const LinearRun& b) { return a.tokens > b.tokens; });
        for (const LinearRun& run : ends) runs[num_runs++] = run;
        std::memcpy(runs + num_runs, scans.data(), scans.size() * sizeof(LinearScan));
        l->num_runs = num_runs;
        l->num_scans = static_cast<uint32_t>(scans.size());
        l->num_tokens = cu_tokens[num_reqs];
        l->staging[kLinearNumSteps] = n;
        l->staging[kLinearNumRuns] = num_runs;
        l->staging[kLinearNumCarries] = l->num_carries;
        l->staging[kLinearNumScans] = l->num_scans;
        cuda_check(cudaMemcpyAsync(l->block.ptr, l->staging, (kLinearScalarCount + uint64_t(n + num_runs + l->num_scans) * kLinearRequestWords) * sizeof(uint32_t),
                                   cudaMemcpyHostToDevice, ctx->stream),
                   "cudaMemcpyAsync");
        cuda_check(cudaEventRecord(l->upload_done, ctx->stream), "cudaEventRecord");
        l->prepared = true;
    });
}

int32_t psi_linear_attend(psi_linear* l, uint32_t layer, float* states, const void* q, const void* k, const void* v, void* out) {
    if (l == nullptr) return PSI_ERR_INVALID_ARGUMENT;
    return guarded(l->ctx, [&] {
        psi_ctx* ctx = l->ctx;
        require(l->prepared, "a linear attention batch must be prepared before recording");
        require(states != nullptr && q != nullptr && k != nullptr && v != nullptr && out != nullptr, "linear attention buffers must not be null");
        require(layer < l->cfg.num_layers, "linear attention layer out of range");
        require((reinterpret_cast<uintptr_t>(states) & 15u) == 0, "linear attention states must be 16-byte aligned");
        const uint32_t esz = dtype_bytes(l->cfg.dtype);
        require((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) | reinterpret_cast<uintptr_t>(out)) % esz == 0,
                "linear attention buffers must be aligned to their elements");
        ctx->bind();
        LinearParams p{};
        p.status = static_cast<uint32_t*>(l->status_word.ptr);
        p.scalars = static_cast<const uint32_t*>(l->block.ptr);
        p.reqs = reinterpret_cast<const LinearRequest*>(p.scalars + kLinearScalarCount);
        p.decays = static_cast<const float*>(l->decays.ptr) + uint64_t(layer) * l->cfg.num_v_heads * kLinearDecays;
        p.states = states;
        p.carries = static_cast<float*>(l->carries.ptr);
        p.q = q;
        p.k = k;
        p.v = v;
        p.out = out;
        p.layer = layer;
        p.num_layers = l->cfg.num_layers;
        p.num_k_heads = l->cfg.num_k_heads;
        p.num_v_heads = l->cfg.num_v_heads;
        p.key_dim = l->cfg.key_dim;
        p.value_dim = l->cfg.value_dim;
        p.dtype = l->cfg.dtype;
        p.scale = l->cfg.scale;
        // a captured launch has to be right for every later batch: its grid and its maps do not depend on this one
        const bool fixed = stream_captured(ctx);
        p.num_tokens = fixed ? l->cfg.max_tokens : l->num_tokens;
        p.aligned = ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15u) == 0 ? 1u : 0u;
        const uint64_t wave = static_cast<uint64_t>(ctx->sm_count) * linear_step_resident(l->cfg.key_dim);
        const uint64_t per_request = uint64_t(l->cfg.num_v_heads) * linear_step_slices(l->cfg.value_dim);
        const uint64_t items = (fixed ? uint64_t(l->cfg.max_tokens) : l->num_steps) * per_request;
        if (items > 0) {
            LaunchScope scope(ctx, PSI_KERNEL_CLASS_LINEAR);
            cuda_check(launch_linear_step(p, static_cast<uint32_t>(std::min(items, wave)), ctx->stream), "linear attention launch");
        }
        const uint64_t sms = static_cast<uint64_t>(ctx->sm_count);
        const auto launch_runs = [&](bool state_only, uint64_t runs) {
            const uint64_t ctas = fixed ? sms : std::min(sms, runs * l->cfg.num_v_heads);
            LaunchScope scope(ctx, PSI_KERNEL_CLASS_LINEAR);
            cuda_check(launch_linear_chunk(p, state_only, static_cast<uint32_t>(ctas), ctx->stream), "linear attention (chunk) launch");
        };
        if (l->carries.ptr != nullptr && (fixed || l->num_scans > 0)) {
            launch_runs(true, l->num_carries);
            LaunchScope scope(ctx, PSI_KERNEL_CLASS_LINEAR);
            cuda_check(launch_linear_scan(p, ctx->stream), "linear attention (scan) launch");
        }
        if (l->chunked && (fixed || l->num_runs > 0)) launch_runs(false, l->num_runs);
    });
}

int32_t psi_linear_device_status(psi_linear* l, int32_t* out) {
    if (l == nullptr || out == nullptr) return PSI_ERR_INVALID_ARGUMENT;
    return guarded(l->ctx, [&] {
        l->ctx->bind();
        cuda_check(cudaStreamSynchronize(l->ctx->stream), "cudaStreamSynchronize");
        uint32_t word = 0;
        cuda_check(cudaMemcpy(&word, l->status_word.ptr, sizeof(word), cudaMemcpyDeviceToHost), "cudaMemcpy");
        if (word != 0) cuda_check(cudaMemset(l->status_word.ptr, 0, sizeof(word)), "cudaMemset");
        *out = static_cast<int32_t>(word);
    });
}

}  // extern "C"
