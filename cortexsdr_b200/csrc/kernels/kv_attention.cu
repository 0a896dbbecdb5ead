// Causal grouped-query attention over the paged 4-bit cache (kv_cache.hpp).
//   o = sum_t softmax_t(scale q . k_t) v_t,   k_t = minimum + step * code, over the tokens up to the row's own
//
// A decode step reads every cached byte once and does 4 head_dim flops a byte for each query head of a group:
// the CUDA cores could not keep up with grouped heads, and widening codes is the other half of the work. So both products run
// on mma.m16n8k16 with the codes themselves (-8 .. 7, exact in fp16) as the second operand:
//   scores   sum over groups of step * (q . (code - 8)) + (minimum + 8 step) * (sum of q)
//   output   sum over groups of (p step) . (code - 8) + sum p (minimum + 8 step)
// Eight query rows fill the sixteen rows of a fragment: rows 0-7 are the fp16 roundings of q (or of p step), rows 8-15
// what the rounding left, so that products carry 22 bits and the sums are fp32's; the two halves of a result
// sit in one lane. A row's q is scaled by a power of two to use fp16's range, p step likewise by the
// largest step met. tcgen05 would want the codes widened into shared memory first, which costs more than the
// products here (16 of 320 issue slots a block are mma).
//
// Work is cut evenly, whatever the lengths: units are (sequence, tile of query rows, kv head), their length in 64 keys
// is known on the device, and CTA c of G takes the c-th G-th of all of it. A unit that is cut leaves partial
// (maximum, sum, output) pieces; the last CTA to arrive at it joins them, in the order of the keys. Nothing depends on the
// host knowing lengths, so a captured call follows its sequences as they grow.
#include <algorithm>
#include <cfloat>

#include "kv_cache.hpp"
#include "op_common.cuh"

namespace csdr {

namespace {

constexpr uint32_t kWarps = 4, kThreads = kWarps * 32, kBlockKeys = 64;
constexpr uint32_t kMostPerSm = 4;

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }

__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, uint32_t limit) {
    for (uint32_t spin = 0; spin < limit; ++spin) {
        uint32_t done;
        asm volatile(
            "{\n"
            ".reg .pred p;\n"
            "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
            "selp.u32 %0, 1, 0, p;\n"
            "}\n"
            : "=r"(done)
            : "r"(bar), "r"(parity)
            : "memory");
        if (done) return true;
    }
    return false;
}

__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ float power_of_two(int n) { return __int_as_float((n + 127) << 23); }   // -126 <= n <= 127

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Eight codes of a word, less 8, as four fp16 pairs, bits (4n, 4n + 16) into pair n: the code's bits below a
// leading one give 1024 + code (or 1024 + 16 code), the rest is one packed operation. Less 8, because the matrix units
// cut their sums off instead of rounding them: what has one sign drifts (1e-5 of an output over 5000 keys).
__device__ __forceinline__ uint32_t pair_or(uint32_t w, uint32_t mask) {
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, 0x64006400, 0xEA;" : "=r"(r) : "r"(w), "r"(mask));   // (w & mask) | 0x6400'6400
    return r;
}
__device__ __forceinline__ uint32_t low_code(uint32_t r) {
    const __half2 v = __hsub2(*reinterpret_cast<__half2*>(&r), __half2half2(__ushort_as_half(0x6408)));   // r - 1032
    return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t high_code(uint32_t r) {
    const __half2 v = __hfma2(*reinterpret_cast<__half2*>(&r), __half2half2(__ushort_as_half(0x2C00)), __half2half2(__ushort_as_half(0xD480)));
    return *reinterpret_cast<const uint32_t*>(&v);   // r / 16 - 72
}
__device__ __forceinline__ void widen_codes(uint32_t w, uint32_t (&r)[4]) {
    const uint32_t v = w >> 8;
    r[0] = low_code(pair_or(w, 0x000F000Fu));
    r[1] = high_code(pair_or(w, 0x00F000F0u));
    r[2] = low_code(pair_or(v, 0x000F000Fu));
    r[3] = high_code(pair_or(v, 0x00F000F0u));
}

// Two fp32 values as a pair of fp16 roundings and a pair of what they left.
__device__ __forceinline__ void split(float x, float y, uint32_t& hi, uint32_t& lo) {
    const __half2 h = __floats2half2_rn(x, y);
    const float2 back = __half22float2(h);
    const __half2 l = __floats2half2_rn(x - back.x, y - back.y);
    hi = *reinterpret_cast<const uint32_t*>(&h);
    lo = *reinterpret_cast<const uint32_t*>(&l);
}

struct AttnParams {
    KvView kv;
    KvBatchView b;
    KvAttend a;
    uint32_t group;          // query heads of a kv head
    uint32_t vec;            // q rows start on 16 bytes
    float* part;             // [CTA][2][rows][HD + 2]
    uint32_t* counters;      // [CTA]: arrivals at the unit that starts in a CTA's share and is cut
    int* status;
    uint32_t spin;
};

// A sequence as the schedule sees it.
struct Seq {
    int64_t base;            // position of its first new token
    int64_t cap;             // keys that its table can hold
    uint32_t row0, n_new, tiles;
    uint32_t pair_weight, mid_weight;
    // blocks of 64 keys that a tile of rows sees; at least one, so that rows that see nothing are written too
    template <uint32_t TILE>
    __device__ __forceinline__ int64_t keys(uint32_t tile, uint32_t group) const {
        const uint32_t last = min(n_new - 1u, static_cast<uint32_t>((static_cast<uint64_t>(TILE) * (tile + 1u) - 1u) / group));
        return min(max(base + last + 1, static_cast<int64_t>(0)), cap);
    }
    template <uint32_t TILE>
    __device__ __forceinline__ uint32_t blocks(uint32_t tile, uint32_t group) const {
        return max(1u, static_cast<uint32_t>((keys<TILE>(tile, group) + kBlockKeys - 1) / kBlockKeys));
    }
    // Causal tiles grow along a prompt: the first and the last tile make a pair, the second and the last but one,
    // whose blocks add up to nearly the same, so that a place in the work is found by a division. What a pair
    // has less than the weight is empty.
    template <uint32_t TILE>
    __device__ __forceinline__ void load(const AttnParams& p, uint32_t s) {
        const int32_t f0 = p.b.first[s], f1 = p.b.first[s + 1];
        const int64_t most = p.b.n_tokens;
        const int64_t r0 = min(max(static_cast<int64_t>(f0), static_cast<int64_t>(0)), most);
        const int64_t r1 = min(max(static_cast<int64_t>(f1), r0), most);
        row0 = static_cast<uint32_t>(r0);
        n_new = static_cast<uint32_t>(r1 - r0);
        base = static_cast<int64_t>(p.b.length[s]) - f1 + r0;
        cap = min(static_cast<int64_t>(p.b.pages_per_seq) << p.kv.page_shift, static_cast<int64_t>(0x7FFFFF00));
        tiles = static_cast<uint32_t>((static_cast<uint64_t>(n_new) * p.group + TILE - 1u) / TILE);
        pair_weight = mid_weight = 0;
        if (!tiles) return;
        const uint32_t a = blocks<TILE>(0, p.group), z = blocks<TILE>(tiles - 1u, p.group);
        // rounding to blocks and the last tile's missing rows: two blocks at most
        pair_weight = tiles == 2u ? a + z : base + n_new > cap ? 2u * z : a + z + 2u;
        if (tiles & 1u) mid_weight = blocks<TILE>(tiles / 2u, p.group);
    }
    __device__ __forceinline__ uint64_t head_weight() const { return static_cast<uint64_t>(tiles / 2u) * pair_weight + mid_weight; }
};

// One warp's eight query rows: fragments, running maxima and sums, outputs.
template <typename T, int HD>
struct Rows {
    static constexpr uint32_t W = HD / 32, G = HD / 64, NT = HD / 8;
    static constexpr bool kShared = HD > 128;      // q fragments in shared memory: the registers go to the outputs
    uint32_t q[kShared ? 1 : W * 2][4];
    float o[NT][4];
    float om[G], sum_q[G];
    float factor, m, l, escale;
    uint32_t vmax;
    int32_t limit;      // keys that this lane's row sees
    int32_t least;      // the fewest that one of the warp's rows sees, the most
    int32_t most;

    // Lane (g, t): row g of the tile, values 64 (w / 2) + 16 t + 8 (w % 2) + n of words w.
    __device__ __forceinline__ void load(const AttnParams& p, const Seq& s, uint32_t kvh, uint32_t row, uint32_t lane, uint4* shared) {
        const uint32_t t = lane & 3u, rr = row + (lane >> 2);
        const uint32_t tok = rr / p.group, head = kvh * p.group + rr % p.group;
        const bool there = tok < s.n_new;
        limit = there ? static_cast<int32_t>(min(max(s.base + tok + 1, static_cast<int64_t>(0)), s.cap)) : 0;
        least = __reduce_min_sync(0xFFFFFFFFu, there ? limit : 0x7FFFFFFF);
        most = __reduce_max_sync(0xFFFFFFFFu, limit);
        const T* src = static_cast<const T*>(p.a.q) + static_cast<size_t>(s.row0 + (there ? tok : 0u)) * p.a.q_stride + static_cast<size_t>(head) * HD;
        if (!there) src = static_cast<const T*>(p.a.q);
        float x[W][8], big = 0.0f;
#pragma unroll
        for (uint32_t w = 0; w < W; ++w) {
            const T* from = src + 64u * (w / 2u) + 16u * t + 8u * (w % 2u);
            if (p.vec) {
                constexpr uint32_t N = 16u / sizeof(T);
#pragma unroll
                for (uint32_t i = 0; i < 8u; i += N) {
                    const uint4 v = *reinterpret_cast<const uint4*>(from + i);
                    const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
                    for (uint32_t j = 0; j < N; ++j) x[w][i + j] = op_widen(e[j]);
                }
            } else {
#pragma unroll
                for (uint32_t i = 0; i < 8u; ++i) x[w][i] = op_widen(from[i]);
            }
        }
#pragma unroll
        for (uint32_t w = 0; w < W; ++w)
#pragma unroll
            for (uint32_t i = 0; i < 8u; ++i) {
                if (!there) x[w][i] = 0.0f;
                big = fmaxf(big, fabsf(x[w][i]));
            }
        big = fmaxf(big, __shfl_xor_sync(0xFFFFFFFFu, big, 1));
        big = fmaxf(big, __shfl_xor_sync(0xFFFFFFFFu, big, 2));
        // 2^e above the largest |q|: q 2^(15 - e) < 2^15, exact but for the last bits of what is 2^-24 of the largest
        const int e = big > 0.0f && big < INFINITY ? min(max(ilogbf(big) + 1, -100), 128) : 15;
        const float up = power_of_two(15 - e), k = p.a.scale * 1.4426950408889634f;
        factor = k * power_of_two(e - 15);
#pragma unroll
        for (uint32_t g = 0; g < G; ++g) sum_q[g] = 0.0f;
#pragma unroll
        for (uint32_t w = 0; w < W; ++w) {
#pragma unroll
            for (uint32_t i = 0; i < 8u; ++i) {
                sum_q[w / 2u] += x[w][i];
                x[w][i] *= up;
            }
#pragma unroll
            for (uint32_t h = 0; h < 2u; ++h) {
                uint32_t f[4];
                split(x[w][2 * h], x[w][2 * h + 4], f[0], f[1]);
                split(x[w][2 * h + 1], x[w][2 * h + 5], f[2], f[3]);
                if constexpr (kShared) {
                    shared[(w * 2u + h) * 32u + lane] = make_uint4(f[0], f[1], f[2], f[3]);
                } else {
#pragma unroll
                    for (uint32_t i = 0; i < 4u; ++i) q[w * 2u + h][i] = f[i];
                }
            }
        }
#pragma unroll
        for (uint32_t g = 0; g < G; ++g) {
            sum_q[g] += __shfl_xor_sync(0xFFFFFFFFu, sum_q[g], 1);
            sum_q[g] += __shfl_xor_sync(0xFFFFFFFFu, sum_q[g], 2);
            sum_q[g] *= k;
            om[g] = 0.0f;
        }
#pragma unroll
        for (uint32_t i = 0; i < NT; ++i)
#pragma unroll
            for (uint32_t j = 0; j < 4u; ++j) o[i][j] = 0.0f;
        m = -FLT_MAX;
        l = 0.0f;
        escale = 1.0f;
        vmax = 0;
        if constexpr (kShared) __syncwarp();
    }

    // Sixteen keys from `tok0` on, in shared memory at `block`.
    __device__ __forceinline__ void keys16(const uint8_t* block, int32_t tok0, bool valid, uint32_t lane, const uint4* shared) {
        const uint32_t g = lane >> 2, t = lane & 3u;
        float sc[4];
#pragma unroll
        for (uint32_t nt = 0; nt < 2u; ++nt) {
            uint32_t w[W];
            const uint8_t* row = block + (8u * nt + g) * (HD / 2) + t * (HD / 8);
            if constexpr (W == 2) {
                const uint2 v = *reinterpret_cast<const uint2*>(row);
                w[0] = v.x;
                w[1] = v.y;
            } else {
#pragma unroll
                for (uint32_t i = 0; i < W; i += 4u) {
                    const uint4 v = *reinterpret_cast<const uint4*>(row + 4u * i);
                    w[i] = v.x;
                    w[i + 1] = v.y;
                    w[i + 2] = v.z;
                    w[i + 3] = v.w;
                }
            }
            uint32_t meta[2 * G];
            load_meta(block + 16u * HD + (8u * nt + 2u * t) * G * 4u, meta);
            float s0 = 0.0f, s1 = 0.0f, n0 = 0.0f, n1 = 0.0f;
#pragma unroll
            for (uint32_t gq = 0; gq < G; ++gq) {
                float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (uint32_t i = 0; i < 2u; ++i) {
                    uint32_t r[4];
                    widen_codes(w[2u * gq + i], r);
#pragma unroll
                    for (uint32_t h = 0; h < 2u; ++h) {
                        if constexpr (kShared) {
                            const uint4 f = shared[((2u * gq + i) * 2u + h) * 32u + lane];
                            mma16816(acc, f.x, f.y, f.z, f.w, r[2 * h], r[2 * h + 1]);
                        } else {
                            const uint32_t* f = q[(2u * gq + i) * 2u + h];
                            mma16816(acc, f[0], f[1], f[2], f[3], r[2 * h], r[2 * h + 1]);
                        }
                    }
                }
                const float2 m0 = __half22float2(*reinterpret_cast<const __half2*>(&meta[gq]));
                const float2 m1 = __half22float2(*reinterpret_cast<const __half2*>(&meta[G + gq]));
                s0 = fmaf(m0.x, acc[0] + acc[2], s0);
                s1 = fmaf(m1.x, acc[1] + acc[3], s1);
                n0 = fmaf(fmaf(8.0f, m0.x, m0.y), sum_q[gq], n0);
                n1 = fmaf(fmaf(8.0f, m1.x, m1.y), sum_q[gq], n1);
            }
            sc[2 * nt] = fmaf(s0, factor, n0);
            sc[2 * nt + 1] = fmaf(s1, factor, n1);
        }
        uint32_t vm[2][2 * G];
        load_meta(block + 17u * HD + (2u * t) * G * 4u, vm[0]);
        load_meta(block + 17u * HD + (8u + 2u * t) * G * 4u, vm[1]);
        if (!valid || tok0 + 16 > least) {
            // keys that a row does not see weigh nothing, whatever lies there
#pragma unroll
            for (uint32_t i = 0; i < 4u; ++i) {
                const int32_t tok = tok0 + static_cast<int32_t>(8u * (i >> 1) + 2u * t + (i & 1u));
                if (!valid || tok >= limit) {
                    sc[i] = -INFINITY;
#pragma unroll
                    for (uint32_t gq = 0; gq < G; ++gq) vm[i >> 1][(i & 1u) * G + gq] = 0u;
                }
            }
        }
        float top = fmaxf(fmaxf(sc[0], sc[1]), fmaxf(sc[2], sc[3]));
        top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
        uint32_t big = 0;
#pragma unroll
        for (uint32_t i = 0; i < 2u; ++i)
#pragma unroll
            for (uint32_t j = 0; j < 2u * G; ++j) big = __vmaxu2(big, vm[i][j] & 0xFFFFu);
        big = __reduce_max_sync(0xFFFFFFFFu, big);
        if (__any_sync(0xFFFFFFFFu, top > m) || big > vmax) {
            const float next = fmaxf(m, top), f = ex2(m - next);
            m = next;
            l *= f;
#pragma unroll
            for (uint32_t gq = 0; gq < G; ++gq) om[gq] *= f;
            float both = f;
            if (big > vmax) {
                // p step 2^(14 - exponent of the largest step) < 2^15
                vmax = big;
                const float st = __half2float(__ushort_as_half(static_cast<unsigned short>(big)));
                const float next_scale = power_of_two(14 - ilogbf(st));
                both = f * (next_scale / escale);
                escale = next_scale;
            }
#pragma unroll
            for (uint32_t i = 0; i < NT; ++i)
#pragma unroll
                for (uint32_t j = 0; j < 4u; ++j) o[i][j] *= both;
        }
        float p[4], pe[4];
#pragma unroll
        for (uint32_t i = 0; i < 4u; ++i) {
            p[i] = ex2(sc[i] - m);
            pe[i] = p[i] * escale;
        }
        l += (p[0] + p[1]) + (p[2] + p[3]);
        const uint8_t* v0 = block + 8u * HD + t * HD + g * (HD / 8);
        const uint8_t* v1 = v0 + 4u * HD;
#pragma unroll
        for (uint32_t u = 0; u < G; ++u) {
            float2 s[4];
#pragma unroll
            for (uint32_t i = 0; i < 4u; ++i) {
                s[i] = __half22float2(*reinterpret_cast<const __half2*>(&vm[i >> 1][(i & 1u) * G + u]));
                om[u] = fmaf(p[i], fmaf(8.0f, s[i].x, s[i].y), om[u]);
            }
            uint32_t a0, a1, a2, a3;
            split(pe[0] * s[0].x, pe[1] * s[1].x, a0, a1);
            split(pe[2] * s[2].x, pe[3] * s[3].x, a2, a3);
            const uint2 w0 = *reinterpret_cast<const uint2*>(v0 + 8u * u), w1 = *reinterpret_cast<const uint2*>(v1 + 8u * u);
#pragma unroll
            for (uint32_t x = 0; x < 2u; ++x) {
                uint32_t r0[4], r1[4];
                widen_codes(x ? w0.y : w0.x, r0);
                widen_codes(x ? w1.y : w1.x, r1);
#pragma unroll
                for (uint32_t n = 0; n < 4u; ++n) mma16816(o[u * 8u + x * 4u + n], a0, a1, a2, a3, r0[n], r1[n]);
            }
        }
    }
    static __device__ __forceinline__ void load_meta(const uint8_t* from, uint32_t (&m)[2 * G]) {
        if constexpr (G == 1) {
            const uint2 v = *reinterpret_cast<const uint2*>(from);
            m[0] = v.x;
            m[1] = v.y;
        } else {
#pragma unroll
            for (uint32_t i = 0; i < 2u * G; i += 4u) {
                const uint4 v = *reinterpret_cast<const uint4*>(from + 4u * i);
                m[i] = v.x;
                m[i + 1] = v.y;
                m[i + 2] = v.z;
                m[i + 3] = v.w;
            }
        }
    }

    // Row g's (maximum, sum) and its output before the division, to `to`: [row][HD + 2].
    __device__ __forceinline__ void store(float* to, uint32_t lane) {
        const uint32_t g = lane >> 2, t = lane & 3u;
        l += __shfl_xor_sync(0xFFFFFFFFu, l, 1);
        l += __shfl_xor_sync(0xFFFFFFFFu, l, 2);
        float* row = to + g * (HD + 2u);
        const float down = 1.0f / escale;
#pragma unroll
        for (uint32_t u = 0; u < G; ++u) {
            om[u] += __shfl_xor_sync(0xFFFFFFFFu, om[u], 1);
            om[u] += __shfl_xor_sync(0xFFFFFFFFu, om[u], 2);
#pragma unroll
            for (uint32_t i = 0; i < 8u; ++i) {
                const float(&c)[4] = o[u * 8u + i];
                row[64u * u + 16u * t + i] = fmaf(c[0] + c[2], down, om[u]);
                row[64u * u + 16u * t + 8u + i] = fmaf(c[1] + c[3], down, om[u]);
            }
        }
        if (t == 0) {
            row[HD] = m;
            row[HD + 1] = l;
        }
    }
};

// Adds up n pieces of a row ([HD] outputs, maximum, sum), one element: the joined output, maximum and sum.
// `get` reads a float of a piece.
template <int HD, typename F>
__device__ __forceinline__ float join(uint32_t n, uint32_t d, F&& get, float& m, float& l) {
    m = -FLT_MAX;
#pragma unroll 4
    for (uint32_t i = 0; i < n; ++i) m = fmaxf(m, get(i, HD));
    float o = 0.0f;
    l = 0.0f;
#pragma unroll 4
    for (uint32_t i = 0; i < n; ++i) {
        const float f = ex2(get(i, HD) - m);
        l = fmaf(f, get(i, HD + 1), l);
        o = fmaf(f, get(i, d), o);
    }
    return o;
}

// KEYS: the four warps share a tile of eight rows and take sixteen keys of a block each (a decode step);
// else each has eight rows of a tile of 32 of its own and all see the same keys (prompts).
template <typename T, int HD, bool KEYS>
__global__ void __launch_bounds__(kThreads, HD > 128 ? 2 : 3)
kv_attention_kernel(AttnParams p) {
    constexpr uint32_t TILE = KEYS ? 8u : 32u, SB = 18u * HD;
    constexpr uint32_t kStages = KEYS ? 4u : 3u, kStageBytes = KEYS ? SB : 4u * SB;
    extern __shared__ __align__(128) uint8_t smem[];
    // stages (of each warp, or of all); then for each warp its rows to be joined (KEYS) and, before them in the
    // same place, its q fragments (head_dim 256)
    uint8_t* ring = smem;
    constexpr uint32_t kOwn = 8u * (HD + 2u) * 4u;
    static_assert(HD <= 128 || kOwn >= HD / 16 * 512u, "a warp's q fragments fit where its rows go");
    float* rows_s = reinterpret_cast<float*>(smem + (KEYS ? kWarps : 1u) * kStages * kStageBytes);
    __shared__ uint64_t bars[kWarps * kStages];
    __shared__ uint64_t scan[kWarps];
    __shared__ uint64_t found_at;
    __shared__ uint32_t found, flag, longest;
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5;
    uint4* my_q = reinterpret_cast<uint4*>(reinterpret_cast<uint8_t*>(rows_s) + warp * kOwn);
    uint8_t* my_ring = ring + (KEYS ? warp * kStages * kStageBytes : 0u);
    const uint32_t my_bar = smem_u32(&bars[KEYS ? warp * kStages : 0u]);
    if (tid == 0) {
        for (uint32_t i = 0; i < kWarps * kStages; ++i) asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(smem_u32(&bars[i])));
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        longest = 0;
    }
    __syncthreads();
    op_enter();
    asm volatile("fence.proxy.async;" ::: "memory");

    // ---- this CTA's share of the work ----
    const uint32_t per = (p.b.n_seqs + kThreads - 1u) / kThreads;
    const uint32_t s_lo = min(tid * per, p.b.n_seqs), s_hi = min(s_lo + per, p.b.n_seqs);
    uint64_t mine = 0;
    uint32_t blocks = 0;
    for (uint32_t s = s_lo; s < s_hi; ++s) {
        Seq q;
        q.load<TILE>(p, s);
        mine += q.head_weight() * p.kv.kv_heads;
        if (q.tiles) blocks = max(blocks, q.blocks<TILE>(q.tiles - 1u, p.group));
    }
    atomicMax(&longest, blocks);
    uint64_t upto = mine;
#pragma unroll
    for (uint32_t o = 1; o < 32u; o <<= 1) {
        const uint64_t v = __shfl_up_sync(0xFFFFFFFFu, upto, o);
        if (lane >= o) upto += v;
    }
    if (lane == 31u) scan[warp] = upto;
    __syncthreads();
    uint64_t total = 0, before = 0;
#pragma unroll
    for (uint32_t i = 0; i < kWarps; ++i) {
        if (i < warp) before += scan[i];
        total += scan[i];
    }
    if (!total) return;
    // Joining n pieces costs a CTA about a ninth of a block's time each: no unit is cut finer than both together take.
    const uint64_t least_blocks = 1u + static_cast<uint32_t>(sqrtf(static_cast<float>(longest) / 9.0f));
    const uint64_t ctas = min(static_cast<uint64_t>(gridDim.x), max(total / least_blocks, static_cast<uint64_t>(1)));
    if (blockIdx.x >= ctas) return;
    const uint64_t x0 = blockIdx.x * total / ctas, x1 = (blockIdx.x + 1u) * total / ctas;
    {
        uint64_t at = before + upto - mine;
        if (x0 >= at && x0 < at + mine) {
            for (uint32_t s = s_lo; s < s_hi; ++s) {
                Seq q;
                q.load<TILE>(p, s);
                const uint64_t w = q.head_weight() * p.kv.kv_heads;
                if (x0 < at + w) {
                    found = s;
                    found_at = at;
                    break;
                }
                at += w;
            }
        }
    }
    __syncthreads();
    uint32_t s = found;
    uint64_t seq_at = found_at, x = x0;
    Seq sq;
    sq.load<TILE>(p, s);
    uint32_t turn = 0;       // stages filled so far
    bool live = true;
    Rows<T, HD> rows;

    while (x < x1 && live) {
        // ---- the unit that holds place x ----
        uint64_t w = sq.head_weight() * p.kv.kv_heads;
        while (x >= seq_at + w) {
            seq_at += w;
            sq.load<TILE>(p, ++s);
            w = sq.head_weight() * p.kv.kv_heads;
        }
        const uint64_t hw = sq.head_weight(), y = x - seq_at, pairs = static_cast<uint64_t>(sq.tiles / 2u) * sq.pair_weight;
        const uint32_t kvh = static_cast<uint32_t>(y / hw);
        const uint64_t z = y % hw;
        uint32_t tile, b0;
        uint64_t next = seq_at + kvh * hw;       // where the next unit starts
        if (z < pairs) {
            const uint32_t pr = static_cast<uint32_t>(z / sq.pair_weight), o = static_cast<uint32_t>(z % sq.pair_weight);
            const uint32_t n = sq.blocks<TILE>(pr, p.group);
            next += static_cast<uint64_t>(pr) * sq.pair_weight;
            tile = pr;
            b0 = o;
            if (o >= n) {
                tile = sq.tiles - 1u - pr;
                b0 = o - n;
                next += sq.pair_weight;
                if (b0 >= sq.blocks<TILE>(tile, p.group)) {    // the empty end of a pair
                    x = next;
                    continue;
                }
            } else {
                next += n;
            }
        } else {
            tile = sq.tiles / 2u;
            b0 = static_cast<uint32_t>(z - pairs);
            next += hw;
        }
        const uint32_t n_blocks = sq.blocks<TILE>(tile, p.group);
        const uint64_t start = x - b0;
        const uint32_t b1 = static_cast<uint32_t>(min(static_cast<uint64_t>(n_blocks), static_cast<uint64_t>(b0) + (x1 - x)));
        const int32_t keys = static_cast<int32_t>(sq.keys<TILE>(tile, p.group));
        const int32_t* table = p.b.pages + static_cast<size_t>(s) * p.b.pages_per_seq;

        rows.load(p, sq, kvh, tile * TILE + (KEYS ? 0u : warp * 8u), lane, my_q);

        // ---- its keys from block b0 to b1 ----
        if constexpr (KEYS) {
            // a warp's i-th piece is keys (4 (b0 + i) + warp) * 16 and on; its page, 32 pieces at a time
            const uint32_t first = 4u * b0 + warp;
            const int32_t left = (keys + 15) / 16 - static_cast<int32_t>(first);
            const uint32_t n = left <= 0 ? 0u : min(b1 - b0, (static_cast<uint32_t>(left) + 3u) / 4u);
            int32_t page_of = -1;
            uint32_t there = 0;      // by stage: the piece has a page
            auto issue = [&](uint32_t i) {
                if ((i & 31u) == 0u) {
                    const uint32_t j = i + lane;
                    page_of = j < n ? __ldg(table + ((first + 4u * j) >> (p.kv.page_shift - 4u))) : -1;
                }
                const int32_t page = __shfl_sync(0xFFFFFFFFu, page_of, i & 31u);
                const bool ok = page >= 0 && static_cast<uint32_t>(page) < p.kv.n_pages;
                const uint32_t st = turn % kStages;
                there = ok ? there | 1u << st : there & ~(1u << st);
                if (lane == 0) {
                    const uint32_t at = ((first + 4u * i) * 16u) & ((1u << p.kv.page_shift) - 1u);
                    const uint8_t* src = p.kv.base + p.kv.block_at(ok ? page : 0, kvh, at);    // page 0 always is one
                    const uint32_t bar = my_bar + 8u * st;
                    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(SB) : "memory");
                    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                                     smem_u32(my_ring + st * SB)),
                                 "l"(src), "r"(SB), "r"(bar)
                                 : "memory");
                }
                ++turn;
            };
            const uint32_t turn0 = turn;
            for (uint32_t i = 0; i < min(n, kStages); ++i) issue(i);
            for (uint32_t i = 0; i < n; ++i) {
                const uint32_t k = turn0 + i, st = k % kStages;
                live = live && __all_sync(0xFFFFFFFFu, mbar_wait(my_bar + 8u * st, (k / kStages) & 1u, p.spin));
                if (!live) break;
                rows.keys16(my_ring + st * SB, static_cast<int32_t>((first + 4u * i) * 16u), there >> st & 1u, lane, my_q);
                __syncwarp();
                if (i + kStages < n) issue(i + kStages);
            }
            __syncwarp();
            rows.store(rows_s + warp * 8u * (HD + 2u), lane);
        } else {
            // all warps: block by block, thread 0 copies; sixteen keys without a page are left out by everyone
            const uint32_t n = b1 - b0;
            auto page_at = [&](uint32_t sub) -> int32_t {
                const int32_t page = static_cast<int32_t>(sub * 16u) < keys ? __ldg(table + (sub >> (p.kv.page_shift - 4u))) : -1;
                return page >= 0 && static_cast<uint32_t>(page) < p.kv.n_pages ? page : -1;
            };
            auto issue = [&](uint32_t i, uint32_t k) {
                const uint32_t st = k % kStages, bar = my_bar + 8u * st;
                int32_t page[4];
                uint32_t count = 0;
#pragma unroll
                for (uint32_t j = 0; j < 4u; ++j) {
                    page[j] = page_at(4u * (b0 + i) + j);
                    count += page[j] >= 0;
                }
                asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(count * SB) : "memory");
#pragma unroll
                for (uint32_t j = 0; j < 4u; ++j) {
                    if (page[j] < 0) continue;
                    const uint32_t at = ((4u * (b0 + i) + j) * 16u) & ((1u << p.kv.page_shift) - 1u);
                    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                                     smem_u32(my_ring + st * kStageBytes + j * SB)),
                                 "l"(p.kv.base + p.kv.block_at(page[j], kvh, at)), "r"(SB), "r"(bar)
                                 : "memory");
                }
            };
            if (tid == 0)
                for (uint32_t i = 0; i < min(n, kStages); ++i) issue(i, turn + i);
            for (uint32_t i = 0; i < n; ++i) {
                const uint32_t k = turn + i, st = k % kStages;
                live = live && __all_sync(0xFFFFFFFFu, mbar_wait(my_bar + 8u * st, (k / kStages) & 1u, p.spin));
                if (live) {
                    for (uint32_t j = 0; j < 4u; ++j) {
                        const int32_t tok = static_cast<int32_t>((4u * (b0 + i) + j) * 16u);
                        if (tok < rows.most) rows.keys16(my_ring + st * kStageBytes + j * SB, tok, page_at(4u * (b0 + i) + j) >= 0, lane, my_q);
                    }
                }
                live = __syncthreads_and(live);
                if (!live) break;
                if (tid == 0 && i + kStages < n) issue(i + kStages, k + kStages);
            }
            turn += n;
        }
        if constexpr (KEYS) live = __syncthreads_and(live);
        if (!live) {
            if (tid == 0) atomicExch(p.status, 1);
        }

        // ---- out, or a piece of it ----
        const bool whole = b0 == 0u && b1 == n_blocks;
        float* slot = p.part + (static_cast<size_t>(blockIdx.x) * 2u + (start >= x0 ? 1u : 0u)) * TILE * (HD + 2u);
        auto write = [&](uint32_t r, uint32_t d, float o, float l, bool seen) {
            const uint32_t rr = tile * TILE + r, tok = rr / p.group, head = kvh * p.group + rr % p.group;
            if (tok >= sq.n_new) return;
            T* dst = static_cast<T*>(p.a.out) + static_cast<size_t>(sq.row0 + tok) * p.a.out_stride + static_cast<size_t>(head) * HD + d;
            *dst = op_narrow<T>(seen ? o / l : 0.0f);
        };
        if constexpr (KEYS) {
            for (uint32_t e = tid; e < 8u * HD; e += kThreads) {
                const uint32_t r = e / HD, d = e % HD;
                float m, l;
                const float o = join<HD>(kWarps, d, [&](uint32_t i, uint32_t j) { return rows_s[(i * 8u + r) * (HD + 2u) + j]; }, m, l);
                if (whole) {
                    write(r, d, o, l, l != 0.0f);
                } else {
                    slot[r * (HD + 2u) + d] = o;
                    if (d == 0) {
                        slot[r * (HD + 2u) + HD] = m;
                        slot[r * (HD + 2u) + HD + 1u] = l;
                    }
                }
            }
            __syncthreads();
        } else if (!whole) {
            rows.store(slot + warp * 8u * (HD + 2u), lane);
        } else {
            // straight from the registers: lane (g, t) has sixteen neighbouring values of every group
            const uint32_t g = lane >> 2, t = lane & 3u;
            rows.l += __shfl_xor_sync(0xFFFFFFFFu, rows.l, 1);
            rows.l += __shfl_xor_sync(0xFFFFFFFFu, rows.l, 2);
            const float down = 1.0f / rows.escale;
#pragma unroll
            for (uint32_t u = 0; u < HD / 64; ++u) {
                rows.om[u] += __shfl_xor_sync(0xFFFFFFFFu, rows.om[u], 1);
                rows.om[u] += __shfl_xor_sync(0xFFFFFFFFu, rows.om[u], 2);
#pragma unroll
                for (uint32_t i = 0; i < 8u; ++i) {
                    const float(&c)[4] = rows.o[u * 8u + i];
                    write(warp * 8u + g, 64u * u + 16u * t + i, fmaf(c[0] + c[2], down, rows.om[u]), rows.l, rows.l != 0.0f);
                    write(warp * 8u + g, 64u * u + 16u * t + 8u + i, fmaf(c[1] + c[3], down, rows.om[u]), rows.l, rows.l != 0.0f);
                }
            }
        }
        if (!whole) {
            // CTA c has place v if floor(c total / ctas) <= v < floor((c + 1) total / ctas)
            const uint32_t c0 = static_cast<uint32_t>(((start + 1u) * ctas - 1u) / total);
            const uint32_t c1 = static_cast<uint32_t>(((start + n_blocks) * ctas - 1u) / total);
            __threadfence();
            __syncthreads();
            if (tid == 0) {
                const bool last = atomicAdd(p.counters + c0, 1u) == c1 - c0;
                if (last) p.counters[c0] = 0u;       // as the next launch finds it
                __threadfence();
                flag = last;
            }
            __syncthreads();
            if (flag) {
                for (uint32_t e = tid; e < TILE * HD; e += kThreads) {
                    const uint32_t r = e / HD, d = e % HD;
                    float m, l;
                    const float o = join<HD>(
                        c1 - c0 + 1u, d,
                        [&](uint32_t i, uint32_t j) {   // past L1: other CTAs wrote these
                            return __ldcg(p.part + ((static_cast<size_t>(c0 + i) * 2u + (i == 0u ? 1u : 0u)) * TILE + r) * (HD + 2u) + j);
                        },
                        m, l);
                    write(r, d, o, l, l != 0.0f);
                }
            }
            __syncthreads();
        }
        x = start + n_blocks < next ? next : start + n_blocks;
        if (start + n_blocks > x1) break;
    }
}

template <typename T, int HD, bool KEYS>
void launch(csdr_context* ctx, AttnParams& p) {
    constexpr size_t SB = 18u * HD;
    constexpr size_t smem = (KEYS ? kWarps * 4u * SB : 3u * 4u * SB) + (KEYS || HD > 128 ? kWarps * 8u * (HD + 2u) * 4u : 0u);
    auto kern = kv_attention_kernel<T, HD, KEYS>;
    const void* key = reinterpret_cast<const void*>(kern);
    ctx->opt_in_smem(key, smem);
    auto& fit = ctx->occupancy[key];
    if (!fit.second) {
        int n = 0;
        CSDR_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kern, kThreads, smem));
        fit = {smem, std::max(1, std::min(n, static_cast<int>(kMostPerSm)))};
    }
    launch_op(ctx, kern, dim3(static_cast<unsigned>(ctx->sm_count * fit.second)), kThreads, smem, 1, p);
}

template <typename T>
void launch_typed(csdr_context* ctx, uint32_t head_dim, bool keys, AttnParams& p) {
    if (head_dim == 64) keys ? launch<T, 64, true>(ctx, p) : launch<T, 64, false>(ctx, p);
    else if (head_dim == 128) keys ? launch<T, 128, true>(ctx, p) : launch<T, 128, false>(ctx, p);
    else keys ? launch<T, 256, true>(ctx, p) : launch<T, 256, false>(ctx, p);
}

}  // namespace

size_t kv_attention_counters(const csdr_context* ctx) { return static_cast<size_t>(ctx->sm_count) * kMostPerSm; }
size_t kv_attention_workspace(const csdr_context* ctx, uint32_t head_dim) {
    return kv_attention_counters(ctx) * (4u + 2u * 32u * (head_dim + 2u) * 4u);
}

void launch_kv_attention(csdr_context* ctx, const KvView& kv, uint32_t head_dim, const KvBatchView& b, int dtype, const KvAttend& a, void* workspace) {
    AttnParams p{};
    p.kv = kv;
    p.b = b;
    p.a = a;
    p.group = a.q_heads / kv.kv_heads;
    p.counters = static_cast<uint32_t*>(workspace);
    p.part = reinterpret_cast<float*>(p.counters + kv_attention_counters(ctx));
    p.status = ctx->status_word;
    p.spin = ctx->spin_limit_barrier;
    const size_t es = dtype == CSDR_DTYPE_F32 ? 4 : 2;
    p.vec = (reinterpret_cast<uintptr_t>(a.q) | a.q_stride * es) % 16u == 0;
    // rows of a sequence that share keys: from two tiles of eight on, warps with rows of their own
    const bool keys = static_cast<uint64_t>(b.n_tokens) * p.group < 16u * static_cast<uint64_t>(b.n_seqs);
    LaunchScope ls(ctx, KC_KV_ATTENTION);
    with_dtype(dtype, [&](auto* t) { launch_typed<std::remove_pointer_t<decltype(t)>>(ctx, head_dim, keys, p); });
    ls.done("kv_attention_kernel");
}

}  // namespace csdr
