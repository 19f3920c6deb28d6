// C++17 caller of GQA::weigh_keys, GQA::evict and LinearAttention: compiled without a GPU, run with one.
#include <cuda_runtime.h>

#include <cmath>
#include <cstdio>
#include <cstring>
#include <vector>

#include "psi_cuda.hpp"

namespace {

float* floats(const std::vector<float>& values) {
    void* out = nullptr;
    if (cudaMalloc(&out, values.size() * sizeof(float)) != cudaSuccess) std::abort();
    if (cudaMemcpy(out, values.data(), values.size() * sizeof(float), cudaMemcpyHostToDevice) != cudaSuccess) std::abort();
    return static_cast<float*>(out);
}

std::vector<float> host(const void* device, size_t count) {
    std::vector<float> out(count);
    if (cudaMemcpy(out.data(), device, count * sizeof(float), cudaMemcpyDeviceToHost) != cudaSuccess) std::abort();
    return out;
}

int step() {
    psi::Context ctx(0);
    const psi::GQAPageTableLayout layout{2, 1, 4, 1};
    const uint32_t d = 8, page = 4;
    psi::GQAConfig config{};
    config.num_q_heads = 2;
    config.num_kv_heads = 1;
    config.head_dim = d;
    config.scale = 1.0f;
    config.page_bytes = 2 * page * d * 4;
    config.dtype = PSI_DTYPE_F32;
    config.layout = layout;
    config.max_tokens = 16;
    psi::PageArena pages(ctx, 8, config.page_bytes);
    psi::GQARequestPageTable table(ctx, layout);
    table.write_row(0, 0, {5, 2, 7, 0});
    table.write_row(1, 0, {1, 3, 4, 6});
    psi::GQA gqa(ctx, config);
    // nine keys: K is t e_0 and the queries are e_0, so that the weights of the last token's rows are exp(t) / sum; V holds t
    std::vector<float> k(9 * d, 0.0f), v(9 * d), q(9 * 2 * d, 0.0f), out(9 * 2 * d, 0.0f);
    for (uint32_t t = 0; t < 9; ++t) {
        k[t * d] = 0.25f * float(t % 5);
        q[t * 2 * d] = 1.0f;
        for (uint32_t c = 0; c < d; ++c) v[t * d + c] = float(t);
    }
    float *dk = floats(k), *dv = floats(v), *dq = floats(q), *dout = floats(out), *dw = floats(std::vector<float>(2 * 16, 0.0f));
    float* dkept = floats(std::vector<float>(16, 0.0f));
    gqa.prepare({0}, {0}, {0, 9});
    gqa.record(pages, table, 0, dk, dv, dq, dout);
    gqa.weigh_keys(pages, table, 0, dq, dw, 16);
    if (gqa.device_status() != 0) return 2;
    const std::vector<float> weights = host(dw, 32);
    std::vector<double> want(9, 0.0);
    for (uint32_t i = 0; i < 9; ++i) {
        double sum = 0.0;
        for (uint32_t t = 0; t <= i; ++t) sum += std::exp(double(k[t * d]));
        for (uint32_t t = 0; t <= i; ++t) want[t] += std::exp(double(k[t * d])) / sum + 1.0 / double(i + 1);  // (the second head's query is zero)
    }
    for (uint32_t t = 0; t < 16; ++t)
        if (std::fabs(weights[t] - (t < 9 ? want[t] : 0.0)) > 1e-5) return 3;
    gqa.evict(pages, table, 0, {0}, {1}, {9}, {4}, 2, dw, dw, 16, reinterpret_cast<uint32_t*>(dkept), 16);
    if (gqa.device_status() != 0) return 4;
    // the two heaviest of the first seven, then 7 and 8
    std::vector<uint32_t> expect;
    for (uint32_t t = 0; t < 7; ++t) {
        uint32_t heavier = 0;
        for (uint32_t o = 0; o < 7; ++o) heavier += weights[o] > weights[t] || (weights[o] == weights[t] && o < t) ? 1u : 0u;
        if (heavier < 2) expect.push_back(t);
    }
    expect.push_back(7);
    expect.push_back(8);
    const std::vector<float> raw = host(dkept, 4), after = host(dw, 32), arena = host(pages.buffer(), 8 * 2 * page * d);
    for (uint32_t i = 0; i < 4; ++i) {
        uint32_t index = 0;
        std::memcpy(&index, &raw[i], 4);
        if (index != expect[i]) return 5;
        if (after[16 + i] != weights[index]) return 6;
        if (arena[(1 * 2 + 1) * page * d + i * d] != float(index)) return 7;  // V rows of page 1
    }
    bool refused = false;
    try {
        gqa.evict(pages, table, 0, {0}, {1}, {9}, {4, 4}, 2, dw, dw, 16, reinterpret_cast<uint32_t*>(dkept), 16);
    } catch (const psi::Error&) {
        refused = true;
    }
    if (!refused) return 8;

    psi::LinearAttention linear(ctx, psi::LinearConfig{1, 1, 8, 8, 0.5f, PSI_DTYPE_F32, 2, 1, 16});
    linear.set_decay(0, {-0.5f});
    float* states = floats(std::vector<float>(2 * 64, 7.0f));
    linear.prepare({0}, {0}, {0, 9}, {1});
    linear.attend(0, states, dk, dk, dv, dout);
    if (linear.device_status() != 0) return 9;
    const std::vector<float> got = host(dout, 9 * d), state = host(states, 128);
    double s = 0.0;
    for (uint32_t t = 0; t < 9; ++t) {
        s = std::exp(-0.5) * s + double(k[t * d]) * t;
        if (std::fabs(got[t * d + 3] - 0.5 * k[t * d] * s) > 1e-5) return 10;
    }
    if (std::fabs(state[64] - s) > 1e-5 || state[0] != 7.0f) return 11;
    for (float* x : {dk, dv, dq, dout, dw, dkept, states}) (void)cudaFree(x);
    return 0;
}

}  // namespace

int main(int argc, char**) {
    if (argc < 2) return 0;
    const int status = step();
    std::puts(status == 0 ? "step ok" : "step failed");
    return status;
}
