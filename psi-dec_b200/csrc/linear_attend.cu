// Linear attention with a decay for each head (psi_linear_attend): per value head, with lambda = exp(log_decay),
//
//   S_t = lambda S_{t-1} + k_t^T v_t        o_t = scale q_t S_t        S: f32 [Dk][Dv]
//
// (A state that is not finite stays so, as NaN after another token: the decay's low part is 0 or of the other sign.  So may its
// outputs: the rows that pad key_dim to the compiled count hold 0 v.)
// linear_step_kernel, the recurrent form: a CTA takes 32 columns of one head's state of one request into registers, goes through
// the request's tokens and writes the columns back: bound by the state's bytes, read and written once for the whole run.  A
// decay close to one that is rounded to f32 would be off by up to 2^-25 a token, and all in the same direction; it is held as two f32
// parts instead (lambda = hi + lo to 48 bits), one more multiply-add for each element and token.  Two columns an instruction (f32x2).  As
// many CTAs as are resident take items in turn, the next item's state on its way into shared memory under the one at hand, and all
// rows of up to eight tokens are requested before the first is used.  One token of 128 requests, 16/32 heads x 128: 92 us, 5.9 TB/s (91 %
// of the copy rate; 103 us before both); four to eight tokens of 32: 41 us for 21 of bytes, the arithmetic not quite under the transfers.
#include <type_traits>

#include "device_common.cuh"
#include "launch_util.hpp"
#include "linear_attend.hpp"
#include "mma_common.cuh"
#include "umma_common.cuh"

namespace psi {

namespace {

constexpr uint32_t kStepThreads = 128;
constexpr uint32_t kStepColumns = 32;                       // of the state in one CTA: eight threads of four
constexpr uint32_t kStepRowGroups = kStepThreads / 8;       // thread (group, four columns) holds rows group + 16 j
constexpr uint32_t kStepTokens = 8;                         // tokens whose rows are in shared memory at once

template <int kRows>  // of the state in one thread: key_dim <= 16 kRows
__global__ __launch_bounds__(kStepThreads, linear_step_resident(16 * kRows)) void linear_step_kernel(const LinearParams p) {
    extern __shared__ __align__(16) unsigned char next_state[];  // of the next item; a thread reads what it copied itself
    float4(*held)[kStepThreads] = reinterpret_cast<float4(*)[kStepThreads]>(next_state);
    __shared__ float2 rows[kStepTokens][kRows * 16];  // (k, q)
    __shared__ __align__(16) float v_cols[kStepTokens][kStepColumns];
    __shared__ __align__(16) float sums[kStepTokens][kStepThreads / 32][kStepColumns];
    await_previous_kernel();
    const uint32_t slices = (p.value_dim + kStepColumns - 1) / kStepColumns;
    const uint32_t total = p.scalars[kLinearNumSteps] * p.num_v_heads * slices;
    const uint32_t share = p.num_v_heads / p.num_k_heads;
    const uint32_t group = threadIdx.x >> 3, quad = threadIdx.x & 7u, warp = threadIdx.x >> 5;
    const auto fetch = [&](uint32_t item) {
        const uint32_t head = item / slices % p.num_v_heads, col = item % slices * kStepColumns + 4u * quad;
        const LinearRequest rq = p.reqs[item / slices / p.num_v_heads];
        const float* from = p.state_of(rq.src, head);
#pragma unroll
        for (int j = 0; j < kRows; ++j) {
            const uint32_t row = group + kStepRowGroups * j;
            const bool there = rq.fresh == 0 && col < p.value_dim && row < p.key_dim;  // value_dim is a multiple of eight
            cp_async_16(smem_u32(&held[j][threadIdx.x]), from + (there ? uint64_t(row) * p.value_dim + col : 0u), there ? 16u : 0u);
        }
        cp_async_commit();
    };
    if (blockIdx.x < total) fetch(blockIdx.x);
    for (uint32_t item = blockIdx.x; item < total; item += gridDim.x) {
        const uint32_t slice = item % slices, head = item / slices % p.num_v_heads;
        const LinearRequest rq = p.reqs[item / slices / p.num_v_heads];
        const uint32_t col = slice * kStepColumns + 4u * quad;
        const bool live = col < p.value_dim;
        ulonglong2 s[kRows];  // four columns, two in each word
        const float hi = p.decays[head * kLinearDecays + 1], lo = p.decays[head * kLinearDecays + kLinearStepLow];
        const uint64_t hi2 = pack_f32x2(hi, hi), lo2 = pack_f32x2(lo, lo);
        for (uint32_t t0 = 0; t0 < rq.q_len; t0 += kStepTokens) {
            const uint32_t tokens = min(kStepTokens, rq.q_len - t0);
            __syncthreads();
            // every load of the rows is under way before the first is used
            const auto stage = [&](const auto type, const auto most) {  // up to `most` tokens
                constexpr uint32_t kDtype = decltype(type)::value, kMost = decltype(most)::value;
                constexpr uint32_t kEach = (kMost * kRows * 16 + kStepThreads - 1) / kStepThreads, kEachV = (kMost * kStepColumns + kStepThreads - 1) / kStepThreads;
                float k[kEach], q[kEach], v[kEachV];
#pragma unroll
                for (uint32_t n = 0; n < kEach; ++n) {
                    const uint32_t i = threadIdx.x + n * kStepThreads, t = i / (kRows * 16u), d = i % (kRows * 16u);
                    const bool there = t < tokens && d < p.key_dim;
                    const uint64_t at = (uint64_t(rq.flat_begin + t0 + t) * p.num_k_heads + head / share) * p.key_dim + d;
                    k[n] = there ? load_as_float(p.k, at, kDtype) : 0.0f;
                    q[n] = there ? load_as_float(p.q, at, kDtype) : 0.0f;
                }
#pragma unroll
                for (uint32_t n = 0; n < kEachV; ++n) {
                    const uint32_t i = threadIdx.x + n * kStepThreads, t = i / kStepColumns, c = slice * kStepColumns + i % kStepColumns;
                    v[n] = t < tokens && c < p.value_dim ? load_as_float(p.v, (uint64_t(rq.flat_begin + t0 + t) * p.num_v_heads + head) * p.value_dim + c, kDtype) : 0.0f;
                }
#pragma unroll
                for (uint32_t n = 0; n < kEach; ++n) {
                    const uint32_t i = threadIdx.x + n * kStepThreads;
                    rows[i / (kRows * 16u)][i % (kRows * 16u)] = make_float2(k[n], q[n]);
                }
#pragma unroll
                for (uint32_t n = 0; n < kEachV; ++n) {
                    const uint32_t i = threadIdx.x + n * kStepThreads;
                    v_cols[i / kStepColumns][i % kStepColumns] = v[n];
                }
            };
            const auto stage_type = [&](const auto type) {
                if (tokens == 1) stage(type, std::integral_constant<uint32_t, 1>{});
                else stage(type, std::integral_constant<uint32_t, kStepTokens>{});
            };
            if (p.dtype == PSI_DTYPE_F32) stage_type(std::integral_constant<uint32_t, PSI_DTYPE_F32>{});
            else if (p.dtype == PSI_DTYPE_BF16) stage_type(std::integral_constant<uint32_t, PSI_DTYPE_BF16>{});
            else stage_type(std::integral_constant<uint32_t, PSI_DTYPE_F16>{});
            if (t0 == 0) {
                cp_async_wait<0>();
#pragma unroll
                for (int j = 0; j < kRows; ++j) s[j] = *reinterpret_cast<const ulonglong2*>(&held[j][threadIdx.x]);
            }
            __syncthreads();
            if (t0 == 0 && item + gridDim.x < total) fetch(item + gridDim.x);  // (what was held has been read)
            for (uint32_t t = 0; t < tokens; ++t) {
                const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(&v_cols[t][4u * quad]);
                uint64_t o_xy = 0, o_zw = 0;
#pragma unroll
                for (int j = 0; j < kRows; ++j) {
                    const float2 kq = rows[t][group + kStepRowGroups * j];
                    const uint64_t k = pack_f32x2(kq.x, kq.x), q = pack_f32x2(kq.y, kq.y);
                    s[j].x = fma_f32x2(hi2, s[j].x, fma_f32x2(lo2, s[j].x, mul_f32x2(k, v.x)));
                    s[j].y = fma_f32x2(hi2, s[j].y, fma_f32x2(lo2, s[j].y, mul_f32x2(k, v.y)));
                    o_xy = fma_f32x2(q, s[j].x, o_xy);
                    o_zw = fma_f32x2(q, s[j].y, o_zw);
                }
                // over the warp's four row groups: each keeps half of what is left of the columns, and ends with one
                const bool upper = (threadIdx.x & 16u) != 0, odd = (threadIdx.x & 8u) != 0;
                const uint64_t theirs = __shfl_xor_sync(0xFFFFFFFFu, upper ? o_xy : o_zw, 16);
                const float2 two = unpack_f32x2(add_f32x2(upper ? o_zw : o_xy, theirs));
                const float one = (odd ? two.y : two.x) + __shfl_xor_sync(0xFFFFFFFFu, odd ? two.x : two.y, 8);
                sums[t][warp][4u * quad + 2u * upper + odd] = one;
            }
            __syncthreads();
            for (uint32_t i = threadIdx.x; i < tokens * kStepColumns; i += kStepThreads) {
                const uint32_t t = i / kStepColumns, c = i % kStepColumns;
                float o = 0.0f;
#pragma unroll
                for (uint32_t x = 0; x < kStepThreads / 32; ++x) o += sums[t][x][c];
                if (slice * kStepColumns + c < p.value_dim)
                    store_from_float(p.out, (uint64_t(rq.flat_begin + t0 + t) * p.num_v_heads + head) * p.value_dim + slice * kStepColumns + c,
                                     p.dtype, o * p.scale);
            }
        }
        float* to = p.state_of(rq.dst, head);
#pragma unroll
        for (int j = 0; j < kRows; ++j) {
            const uint32_t row = group + kStepRowGroups * j;
            if (live && row < p.key_dim) *reinterpret_cast<ulonglong2*>(to + uint64_t(row) * p.value_dim + col) = s[j];
        }
    }
}

// States before the pieces of a request, from the gains of the pieces: S of piece s + 1 = lambda^(tokens of piece s) S of piece s + its gain.
// Bound by the carries' bytes, read and written once.
__global__ __launch_bounds__(256) void linear_scan_kernel(const LinearParams p) {
    await_previous_kernel();
    const uint32_t count = p.scalars[kLinearNumScans], head = blockIdx.y;
    const uint32_t elements = p.key_dim * p.value_dim / 4;
    const uint32_t at = blockIdx.x * blockDim.x + threadIdx.x;
    if (at >= elements) return;
    const float* decay = p.decays + uint64_t(head) * kLinearDecays;
    const double chunk = double(decay[kLinearChunk]) + double(decay[kLinearChunkLow]);
    for (uint32_t i = 0; i < count; ++i) {
        const LinearScan scan = p.scans()[i];
        double power = 1.0, square = chunk;
        for (uint32_t n = scan.piece_chunks; n != 0; n >>= 1, square *= square)
            if (n & 1u) power *= square;
        const float hi = float(power), lo = float(power - double(hi));
        float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (scan.fresh == 0) s = reinterpret_cast<const float4*>(p.state_of(scan.src, head))[at];
        for (uint32_t piece = 0; piece < scan.pieces; ++piece) {
            float4* carry = reinterpret_cast<float4*>(p.carry_of(scan.carry + piece, head)) + at;
            if (piece > 0) {
                const float4 gain = *carry;
                s.x = fmaf(hi, s.x, fmaf(lo, s.x, gain.x));
                s.y = fmaf(hi, s.y, fmaf(lo, s.y, gain.y));
                s.z = fmaf(hi, s.z, fmaf(lo, s.z, gain.z));
                s.w = fmaf(hi, s.w, fmaf(lo, s.w, gain.w));
            }
            *carry = s;
        }
    }
}

}  // namespace

cudaError_t launch_linear_scan(const LinearParams& p, cudaStream_t stream) {
    const uint32_t elements = p.key_dim * p.value_dim / 4;
    return launch_overlapped(linear_scan_kernel, dim3((elements + 255) / 256, p.num_v_heads), dim3(256), 0, stream, p);
}

uint32_t linear_step_slices(uint32_t value_dim) { return (value_dim + kStepColumns - 1) / kStepColumns; }

template <int kRows>
static cudaError_t launch_step(const LinearParams& p, uint32_t ctas, cudaStream_t stream) {
    constexpr int kSmem = kRows * kStepThreads * 16;
    static std::atomic<uint64_t> done{0};
    const cudaError_t err = ensure_dynamic_smem(reinterpret_cast<const void*>(linear_step_kernel<kRows>), kSmem, done);
    if (err != cudaSuccess) return err;
    return launch_overlapped(linear_step_kernel<kRows>, dim3(ctas), dim3(kStepThreads), kSmem, stream, p);
}

cudaError_t launch_linear_step(const LinearParams& p, uint32_t ctas, cudaStream_t stream) {
    if (p.key_dim <= 64) return launch_step<4>(p, ctas, stream);
    if (p.key_dim <= 128) return launch_step<8>(p, ctas, stream);
    return launch_step<16>(p, ctas, stream);
}

}  // namespace psi
