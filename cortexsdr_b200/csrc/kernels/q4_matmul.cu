// Products of activations with weights stored in 4 bits: y[t][r] = sum_c x[t][c] W[r][c] (+ bias), fp32.
//   q4_0   W = (code - 8) d, d fp16 for 32 columns
//   q4_k   W = (d sc) code - dmin mn, (sc, mn) 6 bits for 32 columns, (d, dmin) fp16 for 256
// as decodeSupportedGGUFQuantized reads them (SparseInferenceEngine.cpp:276-469).
#include <algorithm>

#include "op_common.cuh"
#include "q4_matmul.hpp"

namespace csdr {

namespace {

// Stored blocks -> the layout of Q4View. One thread per word of codes, and per row of a unit for the steps.
template <int FMT>
__global__ void __launch_bounds__(256)
q4_relay_kernel(const uint8_t* __restrict__ in, Q4View w, uint8_t* __restrict__ out, size_t n_words) {
    op_enter();
    constexpr uint32_t kCols = q4_unit_cols(FMT), kBytes = q4_unit_bytes(FMT), kWords = kCols * 2u, kBlock = FMT ? 144u : 18u;
    const size_t i = blockIdx.x * static_cast<size_t>(blockDim.x) + threadIdx.x;
    if (i >= n_words) return;
    const size_t unit = i / kWords;
    const uint32_t word = static_cast<uint32_t>(i % kWords), pair = word >> 7, lane = (word >> 2) & 31u, which = word & 3u;
    const uint32_t tile = static_cast<uint32_t>(unit / w.n_units), u = static_cast<uint32_t>(unit % w.n_units);
    const uint32_t row = tile * 16u + (lane >> 2) + (which & 1u) * 8u, group = pair * 2u + (which >> 1);
    const uint32_t col0 = u * kCols + group * 32u;
    uint8_t* to = out + unit * kBytes;
    const bool there = row < w.rows && col0 < w.cols;
    const size_t blocks = w.cols / (FMT ? 256u : 32u);
    const uint8_t* blk = in + (static_cast<size_t>(row) * blocks + (FMT ? u : col0 / 32u)) * kBlock;
    uint32_t codes = 0;
    if (there) {
        for (uint32_t n = 0; n < 8u; ++n) {
            const uint32_t c = (lane & 3u) * 8u + n;
            const uint32_t byte = FMT ? blk[16u + (group >> 1) * 32u + c] : blk[2u + c / 2u];
            codes |= ((FMT ? group & 1u : c & 1u) ? byte >> 4 : byte & 15u) << (4u * n);
        }
    }
    reinterpret_cast<uint32_t*>(to)[word] = codes;
    if (lane & 3u) return;
    // one thread per (row, group): the group's step
    const uint32_t g = lane >> 2, half = which & 1u;
    if (FMT == 0) {
        reinterpret_cast<uint16_t*>(to + 1024u)[(g * 2u + half) * 4u + group] = there ? static_cast<uint16_t>(blk[0] | blk[1] << 8) : 0;
    } else {
        uint32_t sc = 0, mn = 0;
        if (there) {
            const uint8_t* s = blk + 4;
            sc = group < 4u ? s[group] & 63u : (s[group + 4u] & 15u) | (s[group - 4u] >> 6) << 4;
            mn = group < 4u ? s[group + 4u] & 63u : (s[group + 4u] >> 4) | (s[group] >> 6) << 4;
        }
        uint8_t* m = to + 2048u + ((g * 2u + half) * 8u + group) * 2u;
        m[0] = static_cast<uint8_t>(sc);
        m[1] = static_cast<uint8_t>(mn);
        if (group == 0)
            reinterpret_cast<uint32_t*>(to + 2048u + 256u)[g * 2u + half] =
                there ? blk[0] | blk[1] << 8 | blk[2] << 16 | static_cast<uint32_t>(blk[3]) << 24 : 0u;
    }
}

// One warp per (row, token), a lane takes every 32nd run of eight columns.
template <typename T, int FMT>
__global__ void __launch_bounds__(256)
q4_matmul_kernel(Q4View w, Q4Args a) {
    op_enter();
    constexpr uint32_t kCols = q4_unit_cols(FMT), kBytes = q4_unit_bytes(FMT);
    const uint32_t lane = threadIdx.x & 31u, row = blockIdx.x * 8u + (threadIdx.x >> 5);
    const size_t t = blockIdx.y;
    if (row >= w.rows) return;
    const uint32_t g = row & 7u, half = (row >> 3) & 1u;
    const uint8_t* tile = w.base + static_cast<size_t>(row >> 4) * w.n_units * kBytes;
    const T* x = static_cast<const T*>(a.x) + t * a.x_token;
    float sum = 0.0f;
    for (uint32_t c = lane * 8u; c < w.cols; c += 256u) {
        const uint32_t u = c / kCols, group = (c % kCols) / 32u, part = (c % 32u) / 8u;
        const uint8_t* unit = tile + static_cast<size_t>(u) * kBytes;
        const uint32_t codes = reinterpret_cast<const uint32_t*>(unit)[(group >> 1) * 128u + (g * 4u + part) * 4u + (group & 1u) * 2u + half];
        float st, mn;
        if (FMT == 0) {
            st = __half2float(reinterpret_cast<const __half*>(unit + 1024u)[(g * 2u + half) * 4u + group]);
            mn = 8.0f * st;
        } else {
            const uint8_t* m = unit + 2048u + ((g * 2u + half) * 8u + group) * 2u;
            const __half2 d = reinterpret_cast<const __half2*>(unit + 2304u)[g * 2u + half];
            st = __low2float(d) * m[0];
            mn = __high2float(d) * m[1];
        }
        for (uint32_t n = 0; n < 8u; ++n)
            sum = fmaf(op_widen(x[(c + n) * a.x_col]), fmaf(static_cast<float>((codes >> (4u * n)) & 15u), st, -mn), sum);
    }
#pragma unroll
    for (uint32_t o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
    if (lane == 0) a.y[t * a.y_token + row * a.y_row] = sum + (a.bias ? a.bias[row] : 0.0f);
}

}  // namespace

void launch_q4_relay(csdr_context* ctx, const uint8_t* payload, const Q4View& w, uint8_t* out) {
    const size_t n = static_cast<size_t>((w.rows + 15u) / 16u) * w.n_units * q4_unit_cols(w.format) * 2u;
    const dim3 grid(static_cast<unsigned>((n + 255) / 256));
    LaunchScope ls(ctx, KC_Q4);
    if (w.format == 0) launch_op(ctx, q4_relay_kernel<0>, grid, 256, 0, 1, payload, w, out, n);
    else launch_op(ctx, q4_relay_kernel<1>, grid, 256, 0, 1, payload, w, out, n);
    ls.done("q4_relay_kernel");
}

void launch_q4_matmul(csdr_context* ctx, const Q4View& w, const Q4Args& a) {
    for (size_t t0 = 0; t0 < a.batch; t0 += 32768) {
        Q4Args b = a;
        b.batch = std::min<size_t>(32768, a.batch - t0);
        b.y += t0 * a.y_token;
        LaunchScope ls(ctx, KC_Q4);
        const dim3 grid((w.rows + 7u) / 8u, static_cast<unsigned>(b.batch));
        with_dtype(a.x_dtype, [&](auto* p) {
            using T = std::remove_pointer_t<decltype(p)>;
            b.x = static_cast<const T*>(a.x) + t0 * a.x_token;
            if (w.format == 0) launch_op(ctx, q4_matmul_kernel<T, 0>, grid, 256, 0, 1, w, b);
            else launch_op(ctx, q4_matmul_kernel<T, 1>, grid, 256, 0, 1, w, b);
        });
        ls.done("q4_matmul_kernel");
    }
}

}  // namespace csdr
