// Paged key/value cache held in 4 bits: appending (with the rotary embedding on the way) and reading back.
//
// A key row is rotated as the decoder rotates it (adjacent pairs, angle = position * theta^(-i / head_dim);
// apply_rope_inplace, api/cortex_sdk.cpp:1363-1423), angles and products in 64 bits: at position 10^5 an
// fp32 angle is off by 4e-3. Then each group of 64 values x of a row becomes
//   minimum = fp16(min x),  step = fp16((max x - min x) / 15),  code = clamp(rint((x - minimum) / step), 0, 15)
// against the rounded minimum and step, so that their rounding does not add to the codes' error (half a
// step). A group that holds a value that is not finite reads back as NaN; |x| past 65504 saturates.
#include <algorithm>

#include "codes4.cuh"
#include "kv_cache.hpp"
#include "op_common.cuh"

namespace csdr {

namespace {

constexpr uint32_t kWarps = 8;

// The sequence that row t belongs to: how many of first[1 ..] are at most t. All threads of the CTA.
__device__ __forceinline__ uint32_t sequence_of(const KvBatchView& b, int32_t t) {
    uint32_t below = 0;
    for (uint32_t i = 0; i < b.n_seqs; i += blockDim.x) {
        const uint32_t s = i + threadIdx.x;
        below += __syncthreads_count(s < b.n_seqs && b.first[s + 1] <= t);
    }
    return below;
}

// Where row t's token lies: its position, and its page or -1 where it has no place.
__device__ __forceinline__ bool locate(const KvView& kv, const KvBatchView& b, uint32_t t, int32_t& pos, int32_t& page) {
    const uint32_t s = sequence_of(b, static_cast<int32_t>(t));
    pos = page = -1;
    if (s >= b.n_seqs) return false;
    const int32_t first = b.first[s];
    if (static_cast<int32_t>(t) < first) return false;
    const int64_t p = static_cast<int64_t>(b.length[s]) - b.first[s + 1] + static_cast<int32_t>(t);
    if (p < 0 || (p >> kv.page_shift) >= b.pages_per_seq) return true;
    pos = static_cast<int32_t>(p);
    page = b.pages[static_cast<size_t>(s) * b.pages_per_seq + (p >> kv.page_shift)];
    if (page < 0 || static_cast<uint32_t>(page) >= kv.n_pages) page = -1;
    return true;
}

// Where the half word with values d & ~3 .. + 3 of a token lies.
template <int HD>
__device__ __forceinline__ uint32_t key_offset(uint32_t tok, uint32_t d) {
    const uint32_t o = d & 63u;
    return tok * (HD / 2) + ((o >> 4) * (HD / 32) + 2u * (d >> 6) + ((o & 15u) >> 3)) * 4u + (o & 4u) / 2u;
}
template <int HD>
__device__ __forceinline__ uint32_t value_offset(uint32_t tok, uint32_t d) {
    const uint32_t o = d & 63u;
    return 8u * HD + (tok >> 1) * HD + (o >> 3) * (HD / 8) + (d >> 6) * 8u + ((o & 7u) >> 2) * 4u + (tok & 1u) * 2u;
}
template <int HD>
__device__ __forceinline__ uint32_t meta_offset(uint32_t tok, uint32_t d, uint32_t of_values) {
    return 16u * HD + of_values * HD + ((d >> 6) * 16u + tok) * 4u;
}

template <int HD>
__device__ __forceinline__ void quantise_row(const double (&x)[HD / 32], uint8_t* block, uint32_t tok, uint32_t of_values, uint32_t lane) {
    constexpr uint32_t E = HD / 32, kLanes = 64 / E;
    double lo = x[0], hi = x[0];
    bool fine = true;
#pragma unroll
    for (uint32_t i = 0; i < E; ++i) {
        lo = fmin(lo, x[i]);
        hi = fmax(hi, x[i]);
        fine = fine && isfinite(x[i]);
    }
#pragma unroll
    for (uint32_t o = kLanes / 2; o; o >>= 1) {
        lo = fmin(lo, __shfl_xor_sync(0xFFFFFFFFu, lo, o));
        hi = fmax(hi, __shfl_xor_sync(0xFFFFFFFFu, hi, o));
        fine = __shfl_xor_sync(0xFFFFFFFFu, static_cast<int>(fine), o) && fine;
    }
    lo = fmin(fmax(lo, -65504.0), 65504.0);
    hi = fmin(fmax(hi, -65504.0), 65504.0);
    const __half mn = fine ? __float2half_rn(static_cast<float>(lo)) : __ushort_as_half(0x7FFF);
    const __half st = fine ? __float2half_rn(static_cast<float>((hi - lo) / 15.0)) : __ushort_as_half(0);
    const double m = __half2float(mn), s = __half2float(st);
    uint32_t c[E];
#pragma unroll
    for (uint32_t i = 0; i < E; ++i) c[i] = s > 0.0 ? static_cast<uint32_t>(fmin(fmax(rint((x[i] - m) / s), 0.0), 15.0)) : 0u;
    const uint32_t d = E * lane;
    uint8_t* to = block + (of_values ? value_offset<HD>(tok, d) : key_offset<HD>(tok, d));
    if constexpr (E == 2) {       // two lanes share a half word
        const uint32_t c2 = __shfl_down_sync(0xFFFFFFFFu, c[0], 1), c3 = __shfl_down_sync(0xFFFFFFFFu, c[1], 1);
        if (!(lane & 1u)) *reinterpret_cast<uint16_t*>(to) = static_cast<uint16_t>(pack_codes(c[0], c[1], c2, c3));
    } else {
#pragma unroll
        for (uint32_t i = 0; i < E; i += 4u)
            *reinterpret_cast<uint16_t*>(to + (of_values ? i : i / 2u)) = static_cast<uint16_t>(pack_codes(c[i], c[i + 1], c[i + 2], c[i + 3]));
    }
    if (lane % kLanes == 0) {
        const __half2 both = __halves2half2(mn, st);
        *reinterpret_cast<__half2*>(block + meta_offset<HD>(tok, d, of_values)) = both;
    }
}

// grid (token, slice of the heads); a warp takes a head at a time, a lane HD / 32 neighbouring values.
template <typename T, int HD>
__global__ void __launch_bounds__(kWarps * 32)
kv_append_kernel(KvView kv, KvBatchView b, KvAppend a) {
    op_enter();
    constexpr uint32_t E = HD / 32;
    const uint32_t t = blockIdx.x, lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
    int32_t pos, page;
    if (!locate(kv, b, t, pos, page)) return;
    double c[E / 2], s[E / 2];
#pragma unroll
    for (uint32_t i = 0; i < E / 2; ++i) {
        c[i] = 1.0;
        s[i] = 0.0;
        if (a.freq) sincos(static_cast<double>(pos) * a.freq[E / 2 * lane + i], &s[i], &c[i]);
    }
    const uint32_t qh = a.q ? a.q_heads : 0u, units = qh + 2u * kv.kv_heads;
    for (uint32_t u = blockIdx.y * kWarps + warp; u < units; u += gridDim.y * kWarps) {
        const bool is_q = u < qh, is_v = u >= qh + kv.kv_heads;
        const uint32_t head = is_q ? u : is_v ? u - qh - kv.kv_heads : u - qh;
        const T* src = static_cast<const T*>(is_q ? a.q : is_v ? a.v : a.k) + t * (is_q ? a.q_stride : a.kv_stride) + head * HD + E * lane;
        if (!is_q && page < 0) continue;
        double x[E];
#pragma unroll
        for (uint32_t i = 0; i < E; ++i) x[i] = op_widen(src[i]);
        if (!is_v) {
#pragma unroll
            for (uint32_t i = 0; i < E / 2; ++i) {
                const double y0 = x[2 * i] * c[i] - x[2 * i + 1] * s[i], y1 = x[2 * i] * s[i] + x[2 * i + 1] * c[i];
                x[2 * i] = y0;
                x[2 * i + 1] = y1;
            }
        }
        if (is_q) {
            T* dst = static_cast<T*>(a.q_out) + t * a.q_out_stride + head * HD + E * lane;
#pragma unroll
            for (uint32_t i = 0; i < E; ++i) dst[i] = op_narrow<T>(static_cast<float>(x[i]));
        } else {
            const uint32_t at = static_cast<uint32_t>(pos) & ((1u << kv.page_shift) - 1u);
            quantise_row<HD>(x, kv.base + kv.block_at(page, head, at), at & 15u, is_v, lane);
        }
    }
}

template <int HD>
__global__ void __launch_bounds__(kWarps * 32)
kv_read_kernel(KvView kv, KvBatchView b, float* __restrict__ k, float* __restrict__ v) {
    op_enter();
    constexpr uint32_t E = HD / 32;
    const uint32_t t = blockIdx.x, lane = threadIdx.x & 31u, warp = threadIdx.x >> 5, d = E * lane;
    int32_t pos, page;
    if (!locate(kv, b, t, pos, page)) return;
    for (uint32_t u = blockIdx.y * kWarps + warp; u < 2u * kv.kv_heads; u += gridDim.y * kWarps) {
        const uint32_t is_v = u >= kv.kv_heads, head = is_v ? u - kv.kv_heads : u;
        float* dst = (is_v ? v : k) + (static_cast<size_t>(t) * kv.kv_heads + head) * HD + d;
        uint32_t codes[E] = {};
        float st = 0.0f, mn = 0.0f;
        if (page >= 0) {
            const uint32_t at = static_cast<uint32_t>(pos) & ((1u << kv.page_shift) - 1u), tok = at & 15u;
            const uint8_t* block = kv.base + kv.block_at(page, head, at);
            const uint8_t* from = block + (is_v ? value_offset<HD>(tok, d) : key_offset<HD>(tok, d));
#pragma unroll
            for (uint32_t i = 0; i < E; ++i)
                codes[i] = unpack_code(*reinterpret_cast<const uint16_t*>(from + (is_v ? i / 4u * 4u : i / 4u * 2u)), (d + i) & 3u);
            const __half2 both = *reinterpret_cast<const __half2*>(block + meta_offset<HD>(tok, d, is_v));
            mn = __low2float(both);
            st = __high2float(both);
        }
#pragma unroll
        for (uint32_t i = 0; i < E; ++i) dst[i] = fmaf(static_cast<float>(codes[i]), st, mn);
    }
}

// Slices of a token's heads: few tokens still fill the GPU, many take whole tokens.
uint32_t slices(const csdr_context* ctx, uint32_t tokens, uint32_t units) {
    const uint32_t most = (units + kWarps - 1) / kWarps;
    return std::max(1u, std::min(most, static_cast<uint32_t>(ctx->sm_count) * 8u / std::max(1u, tokens)));
}

}  // namespace

void launch_kv_append(csdr_context* ctx, const KvView& kv, uint32_t head_dim, const KvBatchView& b, int dtype, const KvAppend& a) {
    const uint32_t units = (a.q ? a.q_heads : 0u) + 2u * kv.kv_heads;
    const dim3 grid(b.n_tokens, slices(ctx, b.n_tokens, units));
    LaunchScope ls(ctx, KC_KV_CACHE);
    with_dtype(dtype, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        if (head_dim == 64) launch_op(ctx, kv_append_kernel<T, 64>, grid, kWarps * 32, 0, 1, kv, b, a);
        else if (head_dim == 128) launch_op(ctx, kv_append_kernel<T, 128>, grid, kWarps * 32, 0, 1, kv, b, a);
        else launch_op(ctx, kv_append_kernel<T, 256>, grid, kWarps * 32, 0, 1, kv, b, a);
    });
    ls.done("kv_append_kernel");
}

void launch_kv_read(csdr_context* ctx, const KvView& kv, uint32_t head_dim, const KvBatchView& b, float* k, float* v) {
    const dim3 grid(b.n_tokens, slices(ctx, b.n_tokens, 2u * kv.kv_heads));
    LaunchScope ls(ctx, KC_KV_CACHE);
    if (head_dim == 64) launch_op(ctx, kv_read_kernel<64>, grid, kWarps * 32, 0, 1, kv, b, k, v);
    else if (head_dim == 128) launch_op(ctx, kv_read_kernel<128>, grid, kWarps * 32, 0, 1, kv, b, k, v);
    else launch_op(ctx, kv_read_kernel<256>, grid, kWarps * 32, 0, 1, kv, b, k, v);
    ls.done("kv_read_kernel");
}

}  // namespace csdr
