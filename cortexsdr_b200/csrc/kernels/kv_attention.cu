// Causal grouped-query attention over the paged 4-bit cache (kv_cache.hpp).
//   o = sum_t softmax_t(scale q . k_t) v_t,   k_t = minimum + step * code, over the tokens up to the row's own
// One warp per (token, query head), a key at a time; running maximum and sum in fp32.
#include <cfloat>

#include "kv_cache.hpp"
#include "op_common.cuh"

namespace csdr {

namespace {

constexpr uint32_t kWarps = 8;

template <typename T, int HD>
__global__ void __launch_bounds__(kWarps * 32)
kv_attention_kernel(KvView kv, KvBatchView b, KvAttend a) {
    op_enter();
    constexpr uint32_t E = HD / 32;
    const uint32_t t = blockIdx.x, lane = threadIdx.x & 31u, warp = threadIdx.x >> 5, d = E * lane;
    uint32_t s = 0;
    for (uint32_t i = 0; i < b.n_seqs; i += blockDim.x) {
        const uint32_t q = i + threadIdx.x;
        s += __syncthreads_count(q < b.n_seqs && b.first[q + 1] <= static_cast<int32_t>(t));
    }
    const uint32_t head = blockIdx.y * kWarps + warp;
    if (s >= b.n_seqs || static_cast<int32_t>(t) < b.first[s] || head >= a.q_heads) return;
    const int64_t pos = static_cast<int64_t>(b.length[s]) - b.first[s + 1] + static_cast<int32_t>(t);
    const int64_t keys = min(pos + 1, static_cast<int64_t>(b.pages_per_seq) << kv.page_shift);
    const uint32_t kvh = head / (a.q_heads / kv.kv_heads), o = d & 63u;
    const T* src = static_cast<const T*>(a.q) + t * a.q_stride + static_cast<size_t>(head) * HD + d;
    float q[E], acc[E], m = -FLT_MAX, l = 0.0f;
    bool seen = false;
#pragma unroll
    for (uint32_t i = 0; i < E; ++i) {
        q[i] = op_widen(src[i]) * a.scale;
        acc[i] = 0.0f;
    }
    for (int64_t p = 0; p < keys; ++p) {
        const int32_t page = b.pages[static_cast<size_t>(s) * b.pages_per_seq + (p >> kv.page_shift)];
        if (page < 0 || static_cast<uint32_t>(page) >= kv.n_pages) continue;
        seen = true;
        const uint32_t at = static_cast<uint32_t>(p) & ((1u << kv.page_shift) - 1u), tok = at & 15u;
        const uint8_t* block = kv.base + kv.block_at(page, kvh, at);
        const uint8_t* kr = block + tok * (HD / 2) + ((o >> 4) * (HD / 32) + 2u * (d >> 6) + ((o & 15u) >> 3)) * 4u;
        const uint8_t* vr = block + 8u * HD + (tok >> 1) * HD + (o >> 3) * (HD / 8) + (d >> 6) * 8u;
        const __half2 km = *reinterpret_cast<const __half2*>(block + 16u * HD + (tok * (HD / 64) + (d >> 6)) * 4u);
        const __half2 vm = *reinterpret_cast<const __half2*>(block + 17u * HD + (tok * (HD / 64) + (d >> 6)) * 4u);
        const uint32_t kw = *reinterpret_cast<const uint32_t*>(kr);
        float dot = 0.0f;
#pragma unroll
        for (uint32_t i = 0; i < E; ++i)
            dot = fmaf(q[i], fmaf(static_cast<float>((kw >> (4u * ((o + i) & 7u))) & 15u), __low2float(km), __high2float(km)), dot);
#pragma unroll
        for (uint32_t off = 16; off; off >>= 1) dot += __shfl_xor_sync(0xFFFFFFFFu, dot, off);
        const float top = fmaxf(m, dot), f = __expf(m - top), w = __expf(dot - top);
        m = top;
        l = l * f + w;
#pragma unroll
        for (uint32_t i = 0; i < E; ++i) {
            const uint32_t e = (o + i) & 7u;
            const uint32_t word = reinterpret_cast<const uint16_t*>(vr)[(e >> 2) * 2u + (tok & 1u)];
            acc[i] = fmaf(w, fmaf(static_cast<float>((word >> (4u * (e & 3u))) & 15u), __low2float(vm), __high2float(vm)), acc[i] * f);
        }
    }
    T* dst = static_cast<T*>(a.out) + t * a.out_stride + static_cast<size_t>(head) * HD + d;
#pragma unroll
    for (uint32_t i = 0; i < E; ++i) dst[i] = op_narrow<T>(seen ? acc[i] / l : 0.0f);
}

}  // namespace

void launch_kv_attention(csdr_context* ctx, const KvView& kv, uint32_t head_dim, const KvBatchView& b, int dtype, const KvAttend& a) {
    const dim3 grid(b.n_tokens, (a.q_heads + kWarps - 1) / kWarps);
    LaunchScope ls(ctx, KC_KV_ATTENTION);
    with_dtype(dtype, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        if (head_dim == 64) launch_op(ctx, kv_attention_kernel<T, 64>, grid, kWarps * 32, 0, 1, kv, b, a);
        else if (head_dim == 128) launch_op(ctx, kv_attention_kernel<T, 128>, grid, kWarps * 32, 0, 1, kv, b, a);
        else launch_op(ctx, kv_attention_kernel<T, 256>, grid, kWarps * 32, 0, 1, kv, b, a);
    });
    ls.done("kv_attention_kernel");
}

}  // namespace csdr
