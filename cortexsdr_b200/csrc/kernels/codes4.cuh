// 4-bit codes as operands of the matrix units, and what the kernels that use them share.
#pragma once

#include <cuda_fp16.h>

#include <cstdint>

namespace csdr {

// Four codes in a 16-bit half of a word, where a mask, after a shift by four bits or an exchange of the half's bytes,
// leaves each of them in bits 6 - 9.
__host__ __device__ inline uint32_t pack_codes(uint32_t c0, uint32_t c1, uint32_t c2, uint32_t c3) {
    return c0 << 6 | c1 << 2 | (c2 & 3u) << 14 | c2 >> 2 | c3 << 10;
}
__host__ __device__ inline uint32_t unpack_code(uint32_t half, uint32_t n) {
    return n == 0u ? half >> 6 & 15u : n == 1u ? half >> 2 & 15u : n == 2u ? (half >> 14 & 3u) | (half & 3u) << 2 : half >> 10 & 15u;
}

__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// With nothing to add to.
__device__ __forceinline__ void mma16816_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}

__device__ __forceinline__ float power_of_two(int n) { return __int_as_float((n + 127) << 23); }   // -126 <= n <= 127

// Eight codes of a word as four pairs of subnormal fp16: code n of either half into pair n.
// FINE: all times 2^-18. Else pairs 1 and 3 are left four bits lower, times 2^-22: two operations less, but the matrix
// units line sums up by exponents, where a subnormal counts as the smallest normal number, so four bits of the sums
// go (2e-6 of an output against 3e-7) - for results that are rounded to 16 bits.
template <bool FINE>
__device__ __forceinline__ void widen_codes(uint32_t w, uint32_t (&r)[4]) {
    const uint32_t v = __byte_perm(w, 0u, 0x2301);
    r[0] = w & 0x03C003C0u;
    r[1] = FINE ? w << 4 & 0x03C003C0u : w & 0x003C003Cu;
    r[2] = v & 0x03C003C0u;
    r[3] = FINE ? w >> 4 & 0x03C003C0u : v & 0x003C003Cu;
}
constexpr int kCodeShift = 18;
constexpr uint32_t kEights = 0x02000200u;      // code 8, twice
// Widened codes without their 8: exact.
__device__ __forceinline__ uint32_t less_eight(uint32_t codes) {
    const __half2 v = __hadd2(*reinterpret_cast<const __half2*>(&codes), __half2half2(__ushort_as_half(0x8200)));
    return *reinterpret_cast<const uint32_t*>(&v);
}

// Pairs of fp32 values, one packed operation each.
typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 pack2(float x, float y) {
    f32x2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ float2 unpack2(f32x2 v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
    f32x2 d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
    f32x2 d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
    f32x2 d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}

__device__ __forceinline__ uint32_t bits_of(__half2 h) { return *reinterpret_cast<const uint32_t*>(&h); }

// Two fp32 values as a pair of fp16 roundings and a pair of what they left.
__device__ __forceinline__ void split(f32x2 v, uint32_t& hi, uint32_t& lo) {
    const float2 x = unpack2(v);
    const __half2 h = __floats2half2_rn(x.x, x.y);
    const float2 back = __half22float2(h);
    const float2 rest = unpack2(fma2(pack2(back.x, back.y), pack2(-1.0f, -1.0f), v));
    hi = bits_of(h);
    lo = bits_of(__floats2half2_rn(rest.x, rest.y));
}

}  // namespace csdr
