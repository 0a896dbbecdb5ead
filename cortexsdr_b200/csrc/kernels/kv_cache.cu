// Paged key/value cache held in 4 bits: appending (with the rotary embedding on the way) and reading back.
//
// A key row is rotated as the decoder rotates it (adjacent pairs, angle = position * theta^(-i / head_dim);
// apply_rope_inplace, api/cortex_sdk.cpp:1363-1423), angles in 64 bits: at position 10^5 an fp32 angle is off by
// 4e-3. Then each group of 64 values x of a row becomes
//   minimum = fp16(min x),  step = fp16((max x - min x) / 15),  code = clamp(rint((x - minimum) / step), 0, 15)
// against the rounded minimum and step, so that their rounding does not add to the codes' error (half a
// step). A group that holds a value that is not finite reads back as NaN; |x| past 65504 saturates.
//
// What is held is that of 64-bit arithmetic, value for value: a code that falls the other way is a whole step off. The
// arithmetic is fp32 with a bound on its error; a group with a number that the bound leaves open - next to a border between
// two codes, or where minimum or step round - is done again in 64 bits (one in fifty for keys, fewer for values).
// Eight lanes have a group, eight neighbouring values each, so a warp moves 256 values at a time in 128-bit pieces. The bound
// is the bytes of q, k and v.
#include <algorithm>

#include "codes4.cuh"
#include "kv_cache.hpp"
#include "op_common.cuh"

namespace csdr {

namespace {

constexpr uint32_t kWarps = 8, kTokens = 4;      // of a CTA, the most

// Where a CTA's rows' tokens lie: rows t0 to t0 + n - 1 (n at most kTokens), by all threads. own: the row belongs to a sequence.
struct Places {
    int32_t pos[kTokens], page[kTokens];      // page: -1 for a token that has no place
    uint32_t own[kTokens];
};
__device__ __forceinline__ void locate(const KvView& kv, const KvBatchView& b, uint32_t t0, uint32_t n, Places& at) {
    // the first row's sequence: how many of first[1 ..] are at most that row
    uint32_t s = 0;
    for (uint32_t i = 0; i < b.n_seqs; i += blockDim.x) {
        const uint32_t q = i + threadIdx.x;
        s += __syncthreads_count(q < b.n_seqs && b.first[q + 1] <= static_cast<int32_t>(t0));
    }
    if (threadIdx.x < n) {
        const int32_t t = static_cast<int32_t>(t0 + threadIdx.x);
        while (s < b.n_seqs && b.first[s + 1] <= t) ++s;
        int32_t pos = -1, page = -1;
        const bool own = s < b.n_seqs && t >= b.first[s];
        if (own) {
            const int64_t p = static_cast<int64_t>(b.length[s]) - b.first[s + 1] + t;
            if (p >= 0 && (p >> kv.page_shift) < b.pages_per_seq) {
                pos = static_cast<int32_t>(p);
                page = b.pages[static_cast<size_t>(s) * b.pages_per_seq + (p >> kv.page_shift)];
                if (page < 0 || static_cast<uint32_t>(page) >= kv.n_pages) page = -1;
            } else if (p >= 0) {
                pos = static_cast<int32_t>(min(p, static_cast<int64_t>(0x7FFFFFFF)));
            }
        }
        at.pos[threadIdx.x] = pos;
        at.page[threadIdx.x] = page;
        at.own[threadIdx.x] = own;
    }
    __syncthreads();
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

// cos and sin of position * freq, to fp32's precision: the angle is reduced by multiples of pi / 2 in 64 bits (Cody
// and Waite: pi / 2 as a 33-bit head, whose multiples are exact, and the rest), then Taylor series, 1.8e-9 at pi / 4.
__device__ __forceinline__ float2 turn(int32_t pos, double freq) {
    const double a = static_cast<double>(pos) * freq, k = rint(a * 0.63661977236758134);
    const double x = fma(k, -6.077100506506192e-11, fma(k, -1.5707963267341256, a)), z = x * x;
    const double s = x * fma(z, fma(z, fma(z, fma(z, 1.0 / 362880, -1.0 / 5040), 1.0 / 120), -1.0 / 6), 1.0);
    const double c = fma(z, fma(z, fma(z, fma(z, fma(z, -1.0 / 3628800, 1.0 / 40320), -1.0 / 720), 1.0 / 24), -0.5), 1.0);
    const int q = static_cast<int>(static_cast<long long>(k) & 3);
    const double cc = q & 1 ? s : c, ss = q & 1 ? c : s;
    return make_float2(static_cast<float>(q == 1 || q == 2 ? -cc : cc), static_cast<float>(q >= 2 ? -ss : ss));
}

// Eight neighbouring elements, as they lie in memory.
template <typename T>
struct Eight {
    uint4 w[sizeof(T) / 2];
    __device__ __forceinline__ void load(const T* from, bool vec) {
        if (vec) {
#pragma unroll
            for (uint32_t i = 0; i < sizeof(T) / 2; ++i) w[i] = __ldcs(reinterpret_cast<const uint4*>(from) + i);
        } else {
            T* e = reinterpret_cast<T*>(w);
#pragma unroll
            for (uint32_t i = 0; i < 8u; ++i) e[i] = from[i];
        }
    }
    __device__ __forceinline__ float operator[](uint32_t i) const { return op_widen(reinterpret_cast<const T*>(w)[i]); }
};
template <typename T>
__device__ __forceinline__ void store8(T* to, bool vec, const float (&x)[8]) {
    Eight128<T> r;
#pragma unroll
    for (uint32_t i = 0; i < 8u; ++i) r.v[i] = op_narrow<T>(x[i]);
    if (vec) {
        r.store(to);
    } else {
#pragma unroll
        for (uint32_t i = 0; i < 8u; ++i) to[i] = r.v[i];
    }
}

template <typename F>
__device__ __forceinline__ F over_group(F v, F (*op)(F, F)) {
#pragma unroll
    for (uint32_t o = 4; o; o >>= 1) v = op(v, __shfl_xor_sync(0xFFFFFFFFu, v, o));
    return v;
}
__device__ __forceinline__ float least(float a, float b) { return fminf(a, b); }
__device__ __forceinline__ float most(float a, float b) { return fmaxf(a, b); }
__device__ __forceinline__ double least(double a, double b) { return fmin(a, b); }
__device__ __forceinline__ double most(double a, double b) { return fmax(a, b); }

// A group in 64 bits. All lanes of the warp come along.
__device__ __noinline__ void quantise_slowly(const float (&v)[8], bool rotate, int32_t pos, const double* freq, uint32_t (&c)[8], __half& mn, __half& st) {
    double x[8], lo, hi;
    bool fine = true;
#pragma unroll
    for (uint32_t i = 0; i < 8u; i += 2u) {
        double co = 1.0, si = 0.0;
        if (rotate) sincos(static_cast<double>(pos) * freq[i / 2u], &si, &co);
        x[i] = v[i] * co - v[i + 1] * si;
        x[i + 1] = v[i] * si + v[i + 1] * co;
    }
    lo = hi = x[0];
#pragma unroll
    for (uint32_t i = 0; i < 8u; ++i) {
        lo = fmin(lo, x[i]);
        hi = fmax(hi, x[i]);
        fine = fine && isfinite(x[i]);
    }
    lo = over_group<double>(lo, least);
    hi = over_group<double>(hi, most);
    fine = (__ballot_sync(0xFFFFFFFFu, fine) >> (threadIdx.x & 24u) & 0xFFu) == 0xFFu;
    lo = fmin(fmax(lo, -65504.0), 65504.0);
    hi = fmin(fmax(hi, -65504.0), 65504.0);
    mn = fine ? __float2half_rn(static_cast<float>(lo)) : __ushort_as_half(0x7FFF);
    st = fine ? __float2half_rn(static_cast<float>((hi - lo) / 15.0)) : __ushort_as_half(0);
    const double m = __half2float(mn), s = __half2float(st);
#pragma unroll
    for (uint32_t i = 0; i < 8u; ++i) c[i] = s > 0.0 ? static_cast<uint32_t>(fmin(fmax(rint((x[i] - m) / s), 0.0), 15.0)) : 0u;
}

// fp16 of every number between a and b is one and the same.
__device__ __forceinline__ bool settled(float a, float b, __half& h) {
    h = __float2half_rn(a);
    return __half_as_ushort(h) == __half_as_ushort(__float2half_rn(b));
}

// grid (tokens, slice of their groups). A warp takes four groups of a token at a time: of q (rotated only), then k, then v; the
// next four are on their way meanwhile.
template <typename T, int HD>
__global__ void __launch_bounds__(kWarps * 32)
kv_append_kernel(KvView kv, KvBatchView b, KvAppend a, uint32_t tokens) {
    op_enter();
    constexpr uint32_t G = HD / 64;
    __shared__ float2 turns[kTokens][HD / 2];
    __shared__ Places places;
    const uint32_t t0 = blockIdx.x * tokens, n_tok = min(tokens, b.n_tokens - t0);
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5, l = lane & 7u;
    locate(kv, b, t0, n_tok, places);
    if (a.freq) {
        for (uint32_t i = threadIdx.x; i < n_tok * (HD / 2); i += kWarps * 32) turns[i / (HD / 2)][i % (HD / 2)] = turn(places.pos[i / (HD / 2)], a.freq[i % (HD / 2)]);
        __syncthreads();
    }
    const uint32_t nq = (a.q ? a.q_heads : 0u) * G, nk = kv.kv_heads * G, units = nq + 2u * nk, fours = (units + 3u) / 4u;
    Eight<T> ahead;
    const uint32_t sub = lane >> 3, step = gridDim.y * kWarps;
    // a warp's place: four f of token j; the next one `step` fours on
    auto move = [&](uint32_t& j, uint32_t& f) {
        while (f >= fours && j < n_tok) {
            f -= fours;
            ++j;
        }
    };
    auto fetch = [&](uint32_t j, uint32_t f) {
        const uint32_t u = f * 4u + sub, t = t0 + j;
        if (u >= units || !places.own[j]) return;
        if (u < nq) ahead.load(static_cast<const T*>(a.q) + t * a.q_stride + u * 64u + 8u * l, a.q_vec);
        else if (places.page[j] < 0) return;
        else if (u < nq + nk) ahead.load(static_cast<const T*>(a.k) + t * a.kv_stride + (u - nq) * 64u + 8u * l, a.kv_vec);
        else ahead.load(static_cast<const T*>(a.v) + t * a.kv_stride + (u - nq - nk) * 64u + 8u * l, a.kv_vec);
    };
    const uint32_t head_bytes = (1u << (kv.page_shift - 4u)) * kv.block_bytes;      // of a page
    uint32_t j = 0, f = blockIdx.y * kWarps + warp;
    move(j, f);
    if (j < n_tok) fetch(j, f);
    while (j < n_tok) {
        const uint32_t u0 = f * 4u, u = u0 + sub, t = t0 + j, jn = j;
        const Eight<T> raw = ahead;
        f += step;
        move(j, f);
        if (j < n_tok) fetch(j, f);
        if (!places.own[jn]) continue;
        const int32_t page = places.page[jn];
        const bool is_q = u < nq, is_v = u >= nq + nk, there = u < units && (is_q || page >= 0);
        const uint32_t gr = is_q ? u : is_v ? u - nq - nk : u - nq, d = gr % G * 64u + 8u * l;
        const bool rotate = a.freq && !is_v;
        float x[8];
        uint32_t wide = 0;      // |x0| + |x1| of the pairs, as bits: a NaN counts as more than infinity
#pragma unroll
        for (uint32_t e = 0; e < 8u; ++e) x[e] = there ? raw[e] : 0.0f;
#pragma unroll
        for (uint32_t e = 0; e < 8u; e += 2u) wide = max(wide, __float_as_uint(fabsf(x[e]) + fabsf(x[e + 1])) & 0x7FFFFFFFu);
        if (rotate) {
            const float4* r = reinterpret_cast<const float4*>(&turns[jn][d / 2u]);
#pragma unroll
            for (uint32_t e = 0; e < 8u; e += 4u) {
                const float4 c = r[e / 4u];
                const float y0 = fmaf(x[e], c.x, -x[e + 1] * c.y), y1 = fmaf(x[e], c.y, x[e + 1] * c.x);
                const float y2 = fmaf(x[e + 2], c.z, -x[e + 3] * c.w), y3 = fmaf(x[e + 2], c.w, x[e + 3] * c.z);
                x[e] = y0;
                x[e + 1] = y1;
                x[e + 2] = y2;
                x[e + 3] = y3;
            }
        }
        if (there && is_q) store8(static_cast<T*>(a.q_out) + t * a.q_out_stride + gr * 64u + 8u * l, a.q_out_vec, x);
        if (u0 + 4u <= nq || page < 0) continue;       // for the whole warp
        // ---- the group: fp32, and what its error leaves open ----
        float lo = fminf(fminf(fminf(x[0], x[1]), fminf(x[2], x[3])), fminf(fminf(x[4], x[5]), fminf(x[6], x[7])));
        float hi = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
        lo = over_group<float>(lo, least);
        hi = over_group<float>(hi, most);
#pragma unroll
        for (uint32_t o = 4; o; o >>= 1) wide = max(wide, __shfl_xor_sync(0xFFFFFFFFu, wide, o));
        bool fine = wide <= 0x477FE000u || is_q;      // 65504: what saturates or is not finite goes slowly
        // rotation: cos and sin are 2^-24.9 off, a product and the sum round: 2.6 2^-24 (|x0| + |x1|)
        const float err = rotate ? __uint_as_float(wide) * 0x1p-22f : 0.0f;
        const float width = hi - lo, step15 = width * (1.0f / 15.0f), step_err = fmaf(step15, 0x1p-22f, err * 0.134f);
        __half mn, st;
        fine = (settled(lo - err, lo + err, mn) || is_q) && fine;
        fine = (settled(step15 - step_err, step15 + step_err, st) || is_q) && fine;
        const float m = __half2float(mn), s = __half2float(st);
        uint32_t c[8];
        {
            // (x - m) / s: three roundings of 2^-24 on at most 16. What lies outside 0 .. 15 by less than half a code falls to
            // the same side whatever its error
            const float by = s > 0.0f ? __frcp_rn(s) : 0.0f, open = 0.5f - fmaf(err, by, 17.0f * 0x1p-22f);
            constexpr float kWhole = 12582912.0f;      // 1.5 2^23: adding it rounds to a whole number, which its low bits are
            const f32x2 less = pack2(-m, -m), times = pack2(by, by), whole = pack2(kWhole, kWhole), back = pack2(-kWhole, -kWhole), minus = pack2(-1.0f, -1.0f);
            float off = 0.0f;
#pragma unroll
            for (uint32_t e = 0; e < 8u; e += 2u) {
                const float2 q = unpack2(mul2(add2(pack2(x[e], x[e + 1]), less), times));
                const f32x2 p = pack2(fminf(fmaxf(q.x, 0.0f), 15.0f), fminf(fmaxf(q.y, 0.0f), 15.0f));
                const f32x2 r = add2(p, whole);
                const float2 w = unpack2(fma2(add2(r, back), minus, p)), b = unpack2(r);
                off = fmaxf(off, fmaxf(fabsf(w.x), fabsf(w.y)));
                c[e] = __float_as_uint(b.x) & 15u;
                c[e + 1] = __float_as_uint(b.y) & 15u;
            }
            fine = fine && (off < open || is_q);
        }
        if (!__all_sync(0xFFFFFFFFu, fine)) {
            float v[8];
#pragma unroll
            for (uint32_t e = 0; e < 8u; ++e) v[e] = there ? raw[e] : 0.0f;
            quantise_slowly(v, rotate, places.pos[jn], a.freq ? a.freq + d / 2u : nullptr, c, mn, st);
        }
        if (there && !is_q) {
            const uint32_t at = static_cast<uint32_t>(places.pos[jn]) & ((1u << kv.page_shift) - 1u), tok = at & 15u;
            uint8_t* block = kv.base + (static_cast<size_t>(page) * kv.kv_heads + gr / G) * head_bytes + (at >> 4) * kv.block_bytes;
            const uint32_t h0 = pack_codes(c[0], c[1], c[2], c[3]), h1 = pack_codes(c[4], c[5], c[6], c[7]);
            if (is_v) {
                uint16_t* to = reinterpret_cast<uint16_t*>(block + value_offset<HD>(tok, d));
                to[0] = static_cast<uint16_t>(h0);
                to[2] = static_cast<uint16_t>(h1);
            } else {
                *reinterpret_cast<uint32_t*>(block + key_offset<HD>(tok, d)) = h0 | h1 << 16;
            }
            if (l == 0u) *reinterpret_cast<__half2*>(block + meta_offset<HD>(tok, d, is_v)) = __halves2half2(mn, st);
        }
    }
}

template <int HD>
__global__ void __launch_bounds__(kWarps * 32)
kv_read_kernel(KvView kv, KvBatchView b, float* __restrict__ k, float* __restrict__ v, bool vec, uint32_t tokens) {
    op_enter();
    constexpr uint32_t G = HD / 64;
    __shared__ Places places;
    const uint32_t t0 = blockIdx.x * tokens, n_tok = min(tokens, b.n_tokens - t0);
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5, l = lane & 7u;
    locate(kv, b, t0, n_tok, places);
    const uint32_t nk = kv.kv_heads * G, units = 2u * nk, fours = (units + 3u) / 4u;
    const uint32_t head_bytes = (1u << (kv.page_shift - 4u)) * kv.block_bytes;      // of a page
    uint32_t j = 0, f = blockIdx.y * kWarps + warp;
    for (;; f += gridDim.y * kWarps) {      // the limit is n_tok
        while (f >= fours && j < n_tok) {
            f -= fours;
            ++j;
        }
        if (j >= n_tok) break;
        const uint32_t u = f * 4u + (lane >> 3), t = t0 + j;
        if (u >= units || !places.own[j]) continue;
        const int32_t page = places.page[j];
        const uint32_t at = static_cast<uint32_t>(places.pos[j]) & ((1u << kv.page_shift) - 1u), tok = at & 15u;
        const bool is_v = u >= nk;
        const uint32_t gr = is_v ? u - nk : u, d = gr % G * 64u + 8u * l;
        float x[8];
#pragma unroll
        for (uint32_t i = 0; i < 8u; ++i) x[i] = 0.0f;
        if (page >= 0) {
            const uint8_t* block = kv.base + (static_cast<size_t>(page) * kv.kv_heads + gr / G) * head_bytes + (at >> 4) * kv.block_bytes;
            uint32_t h[2];
            if (is_v) {
                const uint16_t* from = reinterpret_cast<const uint16_t*>(block + value_offset<HD>(tok, d));
                h[0] = from[0];
                h[1] = from[2];
            } else {
                const uint32_t w = *reinterpret_cast<const uint32_t*>(block + key_offset<HD>(tok, d));
                h[0] = w & 0xFFFFu;
                h[1] = w >> 16;
            }
            const float2 both = __half22float2(*reinterpret_cast<const __half2*>(block + meta_offset<HD>(tok, d, is_v)));
#pragma unroll
            for (uint32_t i = 0; i < 8u; ++i) x[i] = fmaf(static_cast<float>(unpack_code(h[i / 4u], i & 3u)), both.y, both.x);
        }
        store8((is_v ? v : k) + (static_cast<size_t>(t) * nk + gr) * 64u + 8u * l, vec, x);
    }
}

// Few tokens: a CTA has one, or a slice of its groups, so that they fill the GPU. Many: four a CTA, whose prologue is shared.
struct Shape {
    dim3 grid;
    uint32_t tokens;
};
Shape shape_of(const csdr_context* ctx, uint32_t n_tokens, uint32_t groups) {
    const uint32_t room = static_cast<uint32_t>(ctx->sm_count) * 4u, tokens = n_tokens >= room * kTokens ? kTokens : 1u;
    const uint32_t most = (groups + kWarps * 4u - 1u) / (kWarps * 4u);
    return {dim3((n_tokens + tokens - 1u) / tokens, std::max(1u, std::min(most, room * 2u / std::max(1u, n_tokens)))), tokens};
}

}  // namespace

void launch_kv_append(csdr_context* ctx, const KvView& kv, uint32_t head_dim, const KvBatchView& b, int dtype, const KvAppend& given) {
    const size_t es = dtype == CSDR_DTYPE_F32 ? 4u : 2u;
    auto vec = [&](const void* p, size_t stride) { return (reinterpret_cast<uintptr_t>(p) | stride * es) % 16u == 0; };
    KvAppend a = given;
    a.q_vec = vec(a.q, a.q_stride);
    a.q_out_vec = vec(a.q_out, a.q_out_stride);
    a.kv_vec = vec(a.k, a.kv_stride) && vec(a.v, 0);
    const Shape s = shape_of(ctx, b.n_tokens, ((a.q ? a.q_heads : 0u) + 2u * kv.kv_heads) * (head_dim / kKvGroup));
    LaunchScope ls(ctx, KC_KV_CACHE);
    with_dtype(dtype, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        auto kern = head_dim == 64 ? kv_append_kernel<T, 64> : head_dim == 128 ? kv_append_kernel<T, 128> : kv_append_kernel<T, 256>;
        launch_op(ctx, kern, s.grid, kWarps * 32, 0, 1, kv, b, a, s.tokens);
    });
    ls.done("kv_append_kernel");
}

void launch_kv_read(csdr_context* ctx, const KvView& kv, uint32_t head_dim, const KvBatchView& b, float* k, float* v) {
    const Shape s = shape_of(ctx, b.n_tokens, 2u * kv.kv_heads * (head_dim / kKvGroup));
    const bool vec = (reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) % 16u == 0;
    LaunchScope ls(ctx, KC_KV_CACHE);
    auto kern = head_dim == 64 ? kv_read_kernel<64> : head_dim == 128 ? kv_read_kernel<128> : kv_read_kernel<256>;
    launch_op(ctx, kern, s.grid, kWarps * 32, 0, 1, kv, b, k, v, vec, s.tokens);
    ls.done("kv_read_kernel");
}

}  // namespace csdr
