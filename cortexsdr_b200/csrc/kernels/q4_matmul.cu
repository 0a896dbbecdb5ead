// Products of activations with weights stored in 4 bits: y[t][r] = sum_c x[t][c] W[r][c] (+ bias), fp32.
//   q4_0   W = (code - 8) d, d fp16 for 32 columns
//   q4_k   W = (d sc) code - dmin mn, (sc, mn) 6 bits for 32 columns, (d, dmin) fp16 for 256
// as decodeSupportedGGUFQuantized reads them (SparseInferenceEngine.cpp:276-469).
#include <algorithm>
#include <array>
#include <cmath>

#include <cooperative_groups.h>

#include <type_traits>

#include "codes4.cuh"
#include "op_common.cuh"
#include "q4_matmul.hpp"

namespace cg = cooperative_groups;

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
        uint32_t c[8];
        for (uint32_t n = 0; n < 8u; ++n) {
            const uint32_t col = (lane & 3u) * 8u + n;
            const uint32_t byte = FMT ? blk[16u + (group >> 1) * 32u + col] : blk[2u + col / 2u];
            c[n] = (FMT ? group & 1u : col & 1u) ? byte >> 4 : byte & 15u;
        }
        codes = pack_codes(c[0], c[1], c[2], c[3]) | pack_codes(c[4], c[5], c[6], c[7]) << 16;
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

// The product. Weights are the rows of mma.m16n8k16 (their codes as subnormals, codes4.cuh), tokens its columns: eight
// 16-bit tokens, or four fp32 ones as fp16 roundings and what these left (22 bits). Each group of 32 columns is two
// products, whose sums in fp32 then meet the group's step. The 8 of q4_0 comes off the codes (exactly: a weight of nothing adds
// nothing, however loud its activation), the minima of q4_k through the activations' own sums over the group.
//
// A one-token product must read the weights at the rate of the memory, and has no reuse to hide anything behind: a warp
// owns sixteen rows and streams its units through registers, several ahead. Few rows do not fill the GPU that way, so the
// columns are cut over the CTAs of a cluster, which add up through each other's shared memory; CTAs stay and take
// blocks of 128 rows in turn, so that activations are converted once.
constexpr uint32_t kThreads = 256, kRowsBlock = 128;

struct Q4Params {
    Q4View w;
    Q4Args a;
    uint32_t n_blocks;          // of 128 rows
    uint32_t units_rank;        // units of a row tile that a CTA of a cluster takes
    uint32_t units_staged;      // of those, units whose activations fit into shared memory at a time
    uint8_t* planes;            // activations as fragments, [token tile][unit]; null: the CTAs make them
    int* status;
    uint32_t spin;              // wait limit
    uint32_t x_vec;             // a token's columns lie one behind the other and start on 16 bytes
};

template <int FMT, int NT, bool SPLIT>
struct Q4Shape {
    static constexpr uint32_t kTokens = NT * (SPLIT ? 4u : 8u), kColumns = NT * 8u;
    static constexpr uint32_t kUnitCols = FMT ? 256u : 128u, kGroups = kUnitCols / 32u;
    // of a unit: activations as fragments [group][column][t], of q4_k the sums that meet the minima [group][column], and the powers
    // of two that products are times as large [column]
    static constexpr uint32_t kSumsAt = kGroups * kColumns * 64u, kBacksAt = kSumsAt + (FMT ? kGroups * kColumns * 4u : 0u);
    static constexpr uint32_t kStageBytes = kBacksAt + kColumns * 4u;
    // partial results of all ranks (runs of 32, so up to a run a rank more than there are), twice
    static constexpr uint32_t kSums = kRowsBlock * kTokens + 8u * 32u, kSumBytes = 2u * kSums * 4u;
};

// Eight neighbouring columns of a token as they lie in memory; what lies behind the matrix is zero.
template <typename T>
struct Eight {
    uint4 w[sizeof(T) / 2];
    __device__ __forceinline__ void load(const Q4Params& p, size_t tok, uint32_t col) {
        const T* x = static_cast<const T*>(p.a.x) + tok * p.a.x_token + static_cast<size_t>(col) * p.a.x_col;
        if (col >= p.w.cols) {       // columns come in multiples of 32
#pragma unroll
            for (uint32_t i = 0; i < sizeof(T) / 2; ++i) w[i] = make_uint4(0u, 0u, 0u, 0u);
        } else if (p.x_vec) {
#pragma unroll
            for (uint32_t i = 0; i < sizeof(T) / 2; ++i) w[i] = reinterpret_cast<const uint4*>(x)[i];
        } else {
            T* e = reinterpret_cast<T*>(w);
#pragma unroll
            for (uint32_t i = 0; i < 8u; ++i) e[i] = x[i * p.a.x_col];
        }
    }
    __device__ __forceinline__ float operator[](uint32_t i) const { return op_widen(reinterpret_cast<const T*>(w)[i]); }
};

__device__ __forceinline__ uint32_t word_of(const uint4& v, uint32_t i) { return i == 0u ? v.x : i == 1u ? v.y : i == 2u ? v.z : v.w; }
__device__ __forceinline__ float2 halves(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }

// Activations as fragments: units u0 to u1, of the n_tok tokens from tok0, one unit behind the other from `to`. A power of two
// for each token and unit brings the largest below 2^15. Sixteen lanes (32 for q4_k) have a token's columns of a unit, eight
// each: pieces t of the unit's groups. Items `first`, `first + step`, ... of whole warps.
template <typename T, int FMT, int NT>
__device__ __forceinline__ void stage(const Q4Params& p, uint32_t u0, uint32_t u1, size_t tok0, uint32_t n_tok, uint8_t* to, uint32_t first, uint32_t step) {
    constexpr bool SPLIT = std::is_same<T, float>::value, kScaled = !std::is_same<T, __half>::value;      // fp16 are operands as they come
    using S = Q4Shape<FMT, NT, SPLIT>;
    constexpr uint32_t kLanes = S::kGroups * 4u;
    const uint32_t units = u1 - u0, n = units * n_tok * kLanes;
    for (uint32_t e0 = first & ~31u; e0 < n; e0 += step) {
        const uint32_t e = e0 + (first & 31u), q = e / kLanes, piece = e & 3u;
        // neighbours: units or tokens, whichever lie closer in memory
        const uint32_t unit = p.a.x_col == 1 ? q % units : q / n_tok, tok = p.a.x_col == 1 ? q / units : q % n_tok;
        const uint32_t gr = e % kLanes / 4u;
        const bool there = e < n;
        float v[8];
        uint32_t big = 0;
        if (there) {
            Eight<T> raw;
            raw.load(p, tok0 + tok, ((u0 + unit) * S::kGroups + gr) * 32u + piece * 8u);
#pragma unroll
            for (uint32_t i = 0; i < 8u; ++i) {
                v[i] = raw[i];
                if (kScaled) big = max(big, __float_as_uint(v[i]) & 0x7FFFFFFFu);
            }
        }
        int ex = 14;
        if (kScaled) {
#pragma unroll
            for (uint32_t o = kLanes / 2u; o; o >>= 1) big = max(big, __shfl_xor_sync(0xFFFFFFFFu, big, o));
            // what is not finite stays as it is; 2^-112 counts as the smallest (from there every fp32 number is an fp16 one, or two)
            if (big != 0u && big < 0x7F800000u) ex = max(static_cast<int>(big >> 23) - 127, -112);
        }
        const float up = power_of_two(14 - ex);
        float sum_hi = 0.0f, sum_lo = 0.0f;      // for q4_k
        uint32_t hi[4], lo[4];
#pragma unroll
        for (uint32_t i = 0; i < 4u; ++i) {
            const float x = there ? v[i] * up : 0.0f, z = there ? v[i + 4] * up : 0.0f;
            if constexpr (SPLIT) {
                split(pack2(x, z), hi[i], lo[i]);
                const float2 r = halves(lo[i]), h = halves(hi[i]);
                sum_lo += r.x + r.y;
                sum_hi += h.x + h.y;
            } else {
                hi[i] = bits_of(__floats2half2_rn(x, z));
                sum_hi += x + z;      // fp16 holds them as they are
            }
        }
        if constexpr (FMT) {
            sum_hi += __shfl_xor_sync(0xFFFFFFFFu, sum_hi, 1);
            sum_hi += __shfl_xor_sync(0xFFFFFFFFu, sum_hi, 2);
        }
        if constexpr (FMT && SPLIT) {
            sum_lo += __shfl_xor_sync(0xFFFFFFFFu, sum_lo, 1);
            sum_lo += __shfl_xor_sync(0xFFFFFFFFu, sum_lo, 2);
        }
        if (there) {
            const uint32_t column = SPLIT ? tok / 4u * 8u + tok % 4u : tok, at = gr * S::kColumns + column;
            uint8_t* mine = to + static_cast<size_t>(unit) * S::kStageBytes;
            uint4* frags = reinterpret_cast<uint4*>(mine);
            frags[at * 4u + piece] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
            if constexpr (SPLIT) frags[(at + 4u) * 4u + piece] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
            if (FMT && piece == 0u) {
                float* sums = reinterpret_cast<float*>(mine + S::kSumsAt);
                sums[at] = sum_hi;
                if constexpr (SPLIT) sums[at + 4u] = sum_lo;
            }
            if (e % kLanes == 0u) {
                float* backs = reinterpret_cast<float*>(mine + S::kBacksAt);
                const float back = power_of_two(FMT ? ex - 14 : ex);      // the last 2^4 of q4_0's codes at the very end
                backs[column] = back;
                if constexpr (SPLIT) backs[column + 4u] = back;
            }
        }
    }
}

// The fragments of all units and of a launch's token tiles in global memory, for products whose CTAs would otherwise all do it.
template <typename T, int FMT, int NT>
__global__ void __launch_bounds__(kThreads)
q4_stage_kernel(Q4Params p, uint32_t units_cta) {
    op_enter();
    using S = Q4Shape<FMT, NT, std::is_same<T, float>::value>;
    const size_t tok0 = static_cast<size_t>(blockIdx.y) * S::kTokens;
    const uint32_t n_tok = static_cast<uint32_t>(min(static_cast<size_t>(S::kTokens), p.a.batch - tok0));
    const uint32_t u0 = blockIdx.x * units_cta, u1 = min(u0 + units_cta, p.w.n_units);
    stage<T, FMT, NT>(p, u0, u1, tok0, n_tok, p.planes + (static_cast<size_t>(blockIdx.y) * p.w.n_units + u0) * S::kStageBytes, threadIdx.x, kThreads);
}

// A lane's pieces of a unit: codes (pairs of groups), steps of rows g and g + 8.
template <int FMT>
struct Q4Unit {
    uint4 codes[FMT ? 4 : 2];
    uint4 steps[FMT ? 2 : 1];
    uint2 d;
    __device__ __forceinline__ void load(const uint8_t* unit, uint32_t lane) {
        const uint32_t g = lane >> 2;
#pragma unroll
        for (uint32_t i = 0; i < (FMT ? 4u : 2u); ++i) codes[i] = __ldcs(reinterpret_cast<const uint4*>(unit) + i * 32u + lane);
        if constexpr (FMT == 0) {
            steps[0] = __ldcs(reinterpret_cast<const uint4*>(unit + 1024u) + g);
        } else {
            steps[0] = __ldcs(reinterpret_cast<const uint4*>(unit + 2048u) + 2u * g);
            steps[1] = __ldcs(reinterpret_cast<const uint4*>(unit + 2048u) + 2u * g + 1u);
            d = __ldcs(reinterpret_cast<const uint2*>(unit + 2304u) + g);
        }
    }
};

template <typename T, int FMT, int NT, bool ONE>
__global__ void __launch_bounds__(kThreads, 2)
q4_matmul_kernel(Q4Params p) {
    constexpr bool SPLIT = std::is_same<T, float>::value;
    using S = Q4Shape<FMT, NT, SPLIT>;
    constexpr uint32_t kBytes = q4_unit_bytes(FMT), kAhead = FMT ? 2u : 4u;
    extern __shared__ __align__(16) uint8_t smem[];
    float* part = reinterpret_cast<float*>(smem);                             // twice
    uint8_t* xs = smem + S::kSumBytes;                                        // units
    __shared__ uint64_t bar;
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t ranks = cluster.num_blocks(), rank = cluster.block_rank();
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5, g = lane >> 2, t = lane & 3u;
    const uint32_t u_begin = min(rank * p.units_rank, p.w.n_units), u_end = min(u_begin + p.units_rank, p.w.n_units);
    const uint32_t tiles = (p.w.rows + 15u) / 16u;
    const size_t tok0 = static_cast<size_t>(blockIdx.y) * S::kTokens;
    const uint32_t n_tok = static_cast<uint32_t>(min(static_cast<size_t>(S::kTokens), p.a.batch - tok0));

    Q4Unit<FMT> ahead[kAhead];
    auto unit_at = [&](uint32_t block, uint32_t u) {
        return p.w.base + (static_cast<size_t>(block * 8u + warp) * p.w.n_units + u) * kBytes;
    };
    auto fetch_first = [&](uint32_t block, uint32_t u0, uint32_t u1) {
        if (block * 8u + warp >= tiles) return;
#pragma unroll
        for (uint32_t i = 0; i < kAhead; ++i)
            if (u0 + i < u1) ahead[i].load(unit_at(block, u0 + i), lane);
    };
    const bool staged_once = u_end - u_begin <= p.units_staged;
    // weights do not depend on what runs before
    uint32_t block = blockIdx.x / ranks;
    if (block < p.n_blocks) fetch_first(block, u_begin, min(u_end, u_begin + p.units_staged));
    // what the others write into this CTA's shared memory needs it to be there
    if (ranks > 1u) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    op_enter();

    if (p.planes) {
        if (tid == 0) {
            asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(smem_u32(&bar)));
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
            asm volatile("fence.proxy.async;" ::: "memory");
        }
        __syncthreads();
    }
    uint32_t copies = 0;
    bool live = true;
    auto bring = [&](uint32_t u0, uint32_t u1) {
        if (!p.planes) {
            stage<T, FMT, NT>(p, u0, u1, tok0, n_tok, xs, tid, kThreads);
            return;
        }
        if (tid == 0 && live) {
            const uint32_t bytes = (u1 - u0) * S::kStageBytes;
            asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(&bar)), "r"(bytes) : "memory");
            asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(xs)),
                         "l"(p.planes + (static_cast<size_t>(blockIdx.y) * p.w.n_units + u0) * S::kStageBytes), "r"(bytes), "r"(smem_u32(&bar))
                         : "memory");
        }
        if (live && !mbar_wait_first(smem_u32(&bar), copies & 1u, p.spin)) {
            live = false;
            if (warp == 0) mbar_wait(smem_u32(&bar), copies & 1u, kDrainRounds);
        }
        ++copies;
    };
    if (staged_once && u_end > u_begin) {
        bring(u_begin, u_end);
        __syncthreads();
    }

    if (ranks > 1u) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    uint32_t turn = 0;
    bool fetched = true;
    for (; block < p.n_blocks; block += gridDim.x / ranks, turn ^= 1u) {
        const bool mine = block * 8u + warp < tiles;
        float y[NT][4];
#pragma unroll
        for (uint32_t n = 0; n < NT; ++n) y[n][0] = y[n][1] = y[n][2] = y[n][3] = 0.0f;
        for (uint32_t s0 = u_begin; s0 < u_end; s0 += p.units_staged) {
            const uint32_t s1 = min(s0 + p.units_staged, u_end);
            if (!staged_once) {
                __syncthreads();
                bring(s0, s1);
                __syncthreads();
                if (!fetched) fetch_first(block, s0, s1);
                fetched = false;
            }
            if (mine) {
                for (uint32_t u = s0; u < s1; u += kAhead) {
#pragma unroll
                    for (uint32_t i = 0; i < kAhead; ++i) {
                        if (u + i >= s1) break;
                        Q4Unit<FMT>& w = ahead[i];
                        const uint8_t* staged = xs + (u + i - s0) * S::kStageBytes;
                        float z[NT][4];      // of this unit
#pragma unroll
                        for (uint32_t n = 0; n < NT; ++n) z[n][0] = z[n][1] = z[n][2] = z[n][3] = 0.0f;
                        float2 dA{}, dB{};
                        if constexpr (FMT) {
                            // 6-bit integers as subnormals come back times 2^-24
                            dA = halves(w.d.x);
                            dB = halves(w.d.y);
                            dA.x *= 0x1p42f;
                            dB.x *= 0x1p42f;
                            dA.y *= -0x1p24f;
                            dB.y *= -0x1p24f;
                        }
#pragma unroll
                        for (uint32_t gr = 0; gr < S::kGroups; ++gr) {
                            uint32_t a[4], b[4];
                            widen_codes<true>(word_of(w.codes[gr / 2u], (gr & 1u) * 2u), a);
                            widen_codes<true>(word_of(w.codes[gr / 2u], (gr & 1u) * 2u + 1u), b);
                            if constexpr (FMT == 0) {
#pragma unroll
                                for (uint32_t j = 0; j < 4u; ++j) {
                                    a[j] = less_eight(a[j]);
                                    b[j] = less_eight(b[j]);
                                }
                            }
                            float sA, sB, mA = 0.0f, mB = 0.0f;
                            if constexpr (FMT == 0) {
                                const float2 x = halves(word_of(w.steps[0], gr / 2u)), z = halves(word_of(w.steps[0], 2u + gr / 2u));
                                sA = gr & 1u ? x.y : x.x;
                                sB = gr & 1u ? z.y : z.x;
                            } else {
                                // bytes (step, minimum) of two groups in a word
                                const uint32_t x = word_of(w.steps[0], gr / 2u), z = word_of(w.steps[1], gr / 2u);
                                const float2 xs2 = halves(x & 0x00FF00FFu), xm2 = halves(x >> 8 & 0x00FF00FFu);
                                const float2 zs2 = halves(z & 0x00FF00FFu), zm2 = halves(z >> 8 & 0x00FF00FFu);
                                sA = dA.x * (gr & 1u ? xs2.y : xs2.x);
                                mA = dA.y * (gr & 1u ? xm2.y : xm2.x);
                                sB = dB.x * (gr & 1u ? zs2.y : zs2.x);
                                mB = dB.y * (gr & 1u ? zm2.y : zm2.x);
                            }
#pragma unroll
                            for (uint32_t n = 0; n < NT; ++n) {
                                const uint4 f = *(reinterpret_cast<const uint4*>(staged) + (gr * S::kColumns + n * 8u + g) * 4u + t);
                                float c[4];
                                mma16816_first(c, a[0], b[0], a[1], b[1], f.x, f.y);
                                mma16816(c, a[2], b[2], a[3], b[3], f.z, f.w);
                                if constexpr (FMT) {
                                    const float2 s = *reinterpret_cast<const float2*>(staged + S::kSumsAt + (gr * S::kColumns + n * 8u + 2u * t) * 4u);
                                    z[n][0] = fmaf(mA, s.x, z[n][0]);
                                    z[n][2] = fmaf(mB, s.x, z[n][2]);
                                    if constexpr (!ONE) {
                                        z[n][1] = fmaf(mA, s.y, z[n][1]);
                                        z[n][3] = fmaf(mB, s.y, z[n][3]);
                                    }
                                }
                                z[n][0] = fmaf(sA, c[0], z[n][0]);
                                z[n][2] = fmaf(sB, c[2], z[n][2]);
                                if constexpr (!ONE) {      // odd columns: a single token has none
                                    z[n][1] = fmaf(sA, c[1], z[n][1]);
                                    z[n][3] = fmaf(sB, c[3], z[n][3]);
                                }
                            }
                        }
#pragma unroll
                        for (uint32_t n = 0; n < NT; ++n) {
                            const float2 f = *reinterpret_cast<const float2*>(staged + S::kBacksAt + (n * 8u + 2u * t) * 4u);
                            y[n][0] = fmaf(z[n][0], f.x, y[n][0]);
                            y[n][2] = fmaf(z[n][2], f.x, y[n][2]);
                            if constexpr (!ONE) {
                                y[n][1] = fmaf(z[n][1], f.y, y[n][1]);
                                y[n][3] = fmaf(z[n][3], f.y, y[n][3]);
                            }
                        }
                        if (u + i + kAhead < s1) w.load(unit_at(block, u + i + kAhead), lane);
                    }
                }
            }
        }
        // the next block's weights are on their way while this one's results are added up
        const uint32_t next = block + gridDim.x / ranks;
        if (staged_once && next < p.n_blocks) fetch_first(next, u_begin, u_end);
        // A rank adds up every ranks-th run of 32 rows times tokens; all write into its shared memory. [turn][rank][result]
        const uint32_t n_out = kRowsBlock * n_tok, share = (n_out / 32u + ranks - 1u) / ranks * 32u;
        float* into = part + turn * S::kSums;
        if (mine) {
#pragma unroll
            for (uint32_t n = 0; n < NT; ++n) {
                if constexpr (SPLIT) {
#pragma unroll
                    for (uint32_t i = 0; i < 4u; ++i) y[n][i] += __shfl_xor_sync(0xFFFFFFFFu, y[n][i], 2);
                    if (t >= 2u) continue;
                }
                const uint32_t tok = n * (SPLIT ? 4u : 8u) + 2u * t, row = warp * 16u + g;
#pragma unroll
                for (uint32_t i = 0; i < 2u; ++i) {
                    if (tok + i >= n_tok) continue;
                    constexpr float kCodes = FMT ? 1.0f : 1u << (kCodeShift - 14);
#pragma unroll
                    for (uint32_t h = 0; h < 2u; ++h) {
                        const uint32_t e = (tok + i) * kRowsBlock + row + 8u * h, run = e / 32u, owner = run % ranks;
                        float* to = into + rank * share + run / ranks * 32u + e % 32u;
                        *cluster.map_shared_rank(to, owner) = y[n][2u * h + i] * kCodes;
                    }
                }
            }
        }
        if (ranks > 1u) cluster.sync();
        else __syncthreads();
        for (uint32_t i = tid; i < share; i += kThreads) {
            const uint32_t e = (i / 32u * ranks + rank) * 32u + i % 32u;
            if (e >= n_out) continue;
            const uint32_t tok = e / kRowsBlock;
            const size_t row = static_cast<size_t>(block) * kRowsBlock + e % kRowsBlock;
            if (row >= p.w.rows) continue;
            float sum = p.a.bias ? p.a.bias[row] : 0.0f;
            for (uint32_t r = 0; r < ranks; ++r) sum += into[r * share + i];
            p.a.y[(tok0 + tok) * p.a.y_token + row * p.a.y_row] = sum;
        }
    }
    if (!live && lane == 0) atomicExch(p.status, 1);      // results are wrong, and said to be
}

// Sizes of Q4Shape as the host has them.
struct Sizes {
    uint32_t tokens, stage_bytes, sum_bytes, groups;
    constexpr Sizes(bool split, int format, uint32_t nt)
        : tokens(nt * (split ? 4u : 8u)), stage_bytes(q4_unit_cols(format) / 32u * nt * 8u * (format ? 68u : 64u) + nt * 32u),
          sum_bytes(2u * (kRowsBlock * tokens + 8u * 32u) * 4u), groups(q4_unit_cols(format) / 32u) {}
    // units whose activations fit beside the partial results, with n CTAs an SM
    uint32_t staged(uint32_t n) const { return ((n == 2u ? 104u : 208u) * 1024u - sum_bytes) / stage_bytes; }
};

// Clusters of r CTAs that are resident at once, n CTAs an SM (GPCs do not divide by every r); none where r do not fit one.
constexpr uint32_t kNoCluster = 0xFFFFFFFFu;
uint32_t resident(csdr_context* ctx, uint32_t n, uint32_t r) {
    uint32_t& known = ctx->q4_resident[n - 1u][r - 1u];
    if (!known && r == 1u) known = static_cast<uint32_t>(ctx->sm_count) * n;
    if (!known) {
        auto kern = q4_matmul_kernel<float, 0, 1, false>;
        const size_t smem = (n == 2u ? 104u : 208u) * 1024u;
        ctx->opt_in_smem(reinterpret_cast<const void*>(kern), smem);
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3(r * static_cast<uint32_t>(ctx->sm_count));
        cfg.blockDim = dim3(kThreads);
        cfg.dynamicSmemBytes = smem;
        cudaLaunchAttribute attr{};
        attr.id = cudaLaunchAttributeClusterDimension;
        attr.val.clusterDim.x = r;
        attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
        cfg.attrs = &attr;
        cfg.numAttrs = 1;
        int clusters = 0;
        CSDR_CUDA(cudaOccupancyMaxActiveClusters(&clusters, kern, &cfg));
        known = clusters > 0 ? static_cast<uint32_t>(clusters) : kNoCluster;
    }
    return known == kNoCluster ? 0u : known;
}

// Token tiles a launch whose fragments are made ahead: what 16 MB hold.
size_t tiles_ahead(size_t tiles, size_t tile_bytes) { return std::max<size_t>(1, std::min<size_t>(tiles, (16u << 20) / tile_bytes)); }

// How a product is cut: token tiles of nt times eight operand columns, the columns of a block of 128 rows over `ranks` CTAs of a
// cluster, the row blocks over `clusters` of these in turn; `ahead`: a launch makes the activations' fragments for all.
//
// The cut with the least estimated time, microseconds. A CTA's unit of 128 columns takes 0.5, 0.8 or 1.7 for one, two or four
// eights (three times that for 256 of q4_k, whose groups are twice as many and have minima), the join of a row block 0.6, over
// a cluster 1.1; 256 items of staging 0.5 for a CTA itself, anew for every row block where they do not all fit, or 1.5 for a launch
// and 0.03 a unit; whatever does not fit the GPU at a time waits (and clusters fit less well beside what a launch in front has
// left running). Against all of its cuts the one chosen is 1.0 % off the fastest on average and 18 % at most (396 products:
// 21 weights from 256 x 256 to 151936 x 896, 1 to 1024 tokens, fp32 and bf16). One cut for a single token tile whatever the batch
// was 29 % off: 4864 x 896, 1024 fp32 tokens, 406 us, and 130 with the row blocks uncut; 256 x 256 q4_k, 16 tokens, 7.7 and 3.2
// with four tiles of four tokens instead of one.
struct Cut {
    uint32_t nt = 0, ranks = 0, units_rank = 0, units_staged = 0, clusters = 0;
    bool ahead = false;
};
Cut cut_of(csdr_context* ctx, const Q4View& w, bool split, size_t batch, bool may_stage_ahead) {
    const uint32_t blocks = (w.rows + kRowsBlock - 1u) / kRowsBlock;
    Cut best;
    float least = 0.0f;
    for (uint32_t nt = 1; nt <= 4u; nt *= 2u) {
        const Sizes sz(split, w.format, nt);
        if (nt > 1u && sz.tokens >= 2u * batch) break;
        const size_t tiles = (batch + sz.tokens - 1u) / sz.tokens;
        if (tiles > 65535u) continue;      // of a grid
        const float unit = (nt == 1u ? 0.5f : nt == 2u ? 0.8f : 1.7f) * (w.format ? 3.0f : 1.0f);
        for (uint32_t n = 2; n >= 1u; --n)
            for (uint32_t r = 1; r <= 8u && r <= w.n_units; ++r) {
                const uint32_t fit = resident(ctx, n, r);
                if (!fit) continue;
                const uint32_t units = (w.n_units + r - 1u) / r, fits = sz.staged(n);
                const uint32_t most = std::min(blocks, std::max(1u, static_cast<uint32_t>(ctx->sm_count) * n / r));
                const uint32_t fewer = std::min<uint32_t>(most, std::max<uint32_t>(1u, static_cast<uint32_t>(ctx->sm_count * n / r / tiles)));
                const float items = static_cast<float>((units * std::min<size_t>(batch, sz.tokens) * sz.groups * 4u + kThreads - 1u) / kThreads);
                // two CTAs an SM where shared memory lets them
                const uint32_t at_once = n == 2u || sz.sum_bytes + std::min(units, fits) * sz.stage_bytes <= 104u * 1024u ? resident(ctx, 2, r) : fit;
                for (uint32_t c : {most, fewer})
                    for (bool ahead : {false, true}) {
                        if (ahead && !may_stage_ahead) continue;
                        const float turns = static_cast<float>((blocks + c - 1u) / c), staging = ahead ? 0.03f * units : 0.5f * items;
                        float waves = std::max(1.0f, static_cast<float>(tiles) * c / (at_once * (ahead ? 0.95f : 1.0f)));
                        if (waves < 6.0f) waves = std::ceil(waves);
                        const float cta = 0.8f + turns * (units * unit + (r > 1u ? 1.1f : 0.6f)) + staging * (units > fits ? turns : 1.0f);
                        const float cost = (ahead ? 1.5f : 0.0f) + waves * cta;
                        if (best.nt && cost >= least) continue;
                        least = cost;
                        best = {nt, r, units, std::min(units, fits), c, ahead};
                    }
            }
    }
    return best;
}

template <typename T, int FMT, int NT, bool ONE>
void launch(csdr_context* ctx, Q4Params p, const Cut& cut) {
    using S = Q4Shape<FMT, NT, std::is_same<T, float>::value>;
    constexpr Sizes kSizes(std::is_same<T, float>::value, FMT, NT);
    static_assert(kSizes.tokens == S::kTokens && kSizes.stage_bytes == S::kStageBytes && kSizes.sum_bytes == S::kSumBytes && kSizes.groups == S::kGroups, "one size");
    p.n_blocks = (p.w.rows + kRowsBlock - 1u) / kRowsBlock;
    p.units_rank = cut.units_rank;
    p.units_staged = cut.units_staged;
    const size_t smem = S::kSumBytes + static_cast<size_t>(p.units_staged) * S::kStageBytes;
    p.x_vec = p.a.x_col == 1 && (reinterpret_cast<uintptr_t>(p.a.x) | p.a.x_token * sizeof(T)) % 16u == 0;
    auto kern = q4_matmul_kernel<T, FMT, NT, ONE>;
    ctx->opt_in_smem(reinterpret_cast<const void*>(kern), smem);
    p.status = ctx->status_word;
    p.spin = ctx->operator_spin();
    const size_t tiles = (p.a.batch + S::kTokens - 1u) / S::kTokens, tile_bytes = static_cast<size_t>(p.w.n_units) * S::kStageBytes;
    const size_t each = cut.ahead ? tiles_ahead(tiles, tile_bytes) : tiles;
    const Q4Args all = p.a;
    for (size_t t0 = 0; t0 < tiles; t0 += each) {
        const size_t n = std::min(each, tiles - t0), tok = t0 * S::kTokens;
        p.a.x = static_cast<const T*>(all.x) + tok * all.x_token;
        p.a.y = all.y + tok * all.y_token;
        p.a.batch = std::min(all.batch - tok, n * S::kTokens);
        if (cut.ahead) {
            p.planes = static_cast<uint8_t*>(ctx->scratch_get(csdr_context::kQ4Scratch, each * tile_bytes));
            constexpr uint32_t kUnits = 2;
            LaunchScope ls(ctx, KC_Q4);
            launch_op(ctx, q4_stage_kernel<T, FMT, NT>, dim3((p.w.n_units + kUnits - 1u) / kUnits, static_cast<unsigned>(n)), kThreads, 0, 1, p, kUnits);
            ls.done("q4_stage_kernel");
        }
        LaunchScope ls(ctx, KC_Q4);
        launch_op(ctx, kern, dim3(cut.clusters * cut.ranks, static_cast<unsigned>(n)), kThreads, smem, cut.ranks, p);
        ls.done("q4_matmul_kernel");
    }
}

template <typename T, int FMT>
void launch_tokens(csdr_context* ctx, const Q4Params& p) {
    constexpr bool kSplit = std::is_same<T, float>::value;
    // The same sizes are cut alike: remembered, as there are some hundred cuts to compare.
    auto remembered = [&](bool may_stage_ahead) {
        const std::array<size_t, 3> key{(static_cast<size_t>(p.w.rows) << 32) | p.w.cols, p.a.batch,
                                        static_cast<size_t>(p.w.format) | (kSplit ? 2u : 0u) | (may_stage_ahead ? 4u : 0u)};
        auto& known = ctx->q4_cuts;
        auto it = known.find(key);
        if (it == known.end()) {
            if (known.size() >= 4096u) known.clear();
            const Cut c = cut_of(ctx, p.w, kSplit, p.a.batch, may_stage_ahead);
            it = known.emplace(key, std::array<uint32_t, 6>{c.nt, c.ranks, c.units_rank, c.units_staged, c.clusters, c.ahead ? 1u : 0u}).first;
        }
        const auto& v = it->second;
        return Cut{v[0], v[1], v[2], v[3], v[4], v[5] != 0u};
    };
    Cut cut = remembered(true);
    if (cut.ahead && ctx->capturing()) {      // nothing may be allocated, and what the graph uses stays
        const Sizes sz(kSplit, FMT, cut.nt);
        const size_t tile_bytes = static_cast<size_t>(p.w.n_units) * sz.stage_bytes;
        const DevPtr& now = ctx->scratch[csdr_context::kQ4Scratch];
        if (!now || now->bytes < tiles_ahead((p.a.batch + sz.tokens - 1u) / sz.tokens, tile_bytes) * tile_bytes) cut = remembered(false);
        else if (ctx->held.empty() || ctx->held.back() != now) ctx->held.push_back(now);
    }
    if (p.a.batch == 1) launch<T, FMT, 1, true>(ctx, p, cut);
    else if (cut.nt == 1u) launch<T, FMT, 1, false>(ctx, p, cut);
    else if (cut.nt == 2u) launch<T, FMT, 2, false>(ctx, p, cut);
    else launch<T, FMT, 4, false>(ctx, p, cut);
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
    // 65535 token tiles of at least 16 are a grid's second dimension
    constexpr size_t kMost = 65535u * 16u;
    for (size_t t0 = 0; t0 < a.batch; t0 += kMost) {
        Q4Params p{};
        p.w = w;
        p.a = a;
        p.a.batch = std::min(kMost, a.batch - t0);
        p.a.x = static_cast<const uint8_t*>(a.x) + t0 * a.x_token * (a.x_dtype == CSDR_DTYPE_F32 ? 4u : 2u);
        p.a.y = a.y + t0 * a.y_token;
        with_dtype(a.x_dtype, [&](auto* t) {
            using T = std::remove_pointer_t<decltype(t)>;
            if (w.format == 0) launch_tokens<T, 0>(ctx, p);
            else launch_tokens<T, 1>(ctx, p);
        });
    }
}

}  // namespace csdr
