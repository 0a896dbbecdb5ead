// Products of activations with weights stored in 4 bits: y[t][r] = sum_c x[t][c] W[r][c] (+ bias), fp32.
//   q4_0   W = (code - 8) d, d fp16 for 32 columns
//   q4_k   W = (d sc) code - dmin mn, (sc, mn) 6 bits for 32 columns, (d, dmin) fp16 for 256
// as decodeSupportedGGUFQuantized reads them (SparseInferenceEngine.cpp:276-469).
#include <algorithm>

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
// products, whose sums in fp32 then meet the group's step; the 8 of q4_0 and the minima of q4_k come off through the
// activations' own sums over the group.
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
    uint32_t x_vec;             // a token's columns lie one behind the other and start on 16 bytes
};

template <int FMT, int NT, bool SPLIT>
struct Q4Shape {
    static constexpr uint32_t kTokens = NT * (SPLIT ? 4u : 8u), kColumns = NT * 8u;
    static constexpr uint32_t kUnitCols = FMT ? 256u : 128u, kGroups = kUnitCols / 32u;
    // activations of a unit as fragments, then the group sums that its columns need
    static constexpr uint32_t kStageBytes = kGroups * kColumns * (64u + 4u);
    static constexpr uint32_t kSumBytes = 2u * kRowsBlock * kTokens * 4u;      // partial results, twice
};

// Eight neighbouring columns of a token; what lies behind the matrix is zero.
template <typename T>
__device__ __forceinline__ void load8(const Q4Params& p, size_t tok, uint32_t col, float (&v)[8]) {
    const T* x = static_cast<const T*>(p.a.x) + tok * p.a.x_token + static_cast<size_t>(col) * p.a.x_col;
    if (p.x_vec) {       // columns come in multiples of 32
        if (col >= p.w.cols) {
#pragma unroll
            for (uint32_t i = 0; i < 8u; ++i) v[i] = 0.0f;
            return;
        }
        constexpr uint32_t N = 16u / sizeof(T);
#pragma unroll
        for (uint32_t i = 0; i < 8u; i += N) {
            const uint4 q = *reinterpret_cast<const uint4*>(x + i);
            const T* e = reinterpret_cast<const T*>(&q);
#pragma unroll
            for (uint32_t j = 0; j < N; ++j) v[i + j] = op_widen(e[j]);
        }
    } else {
#pragma unroll
        for (uint32_t i = 0; i < 8u; ++i) v[i] = col + i < p.w.cols ? op_widen(x[i * p.a.x_col]) : 0.0f;
    }
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

__device__ __forceinline__ uint32_t word_of(const uint4& v, uint32_t i) { return i == 0u ? v.x : i == 1u ? v.y : i == 2u ? v.z : v.w; }
__device__ __forceinline__ float2 halves(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }

template <typename T, int FMT, int NT>
__global__ void __launch_bounds__(kThreads, 2)
q4_matmul_kernel(Q4Params p) {
    constexpr bool SPLIT = std::is_same<T, float>::value;
    using S = Q4Shape<FMT, NT, SPLIT>;
    constexpr uint32_t kBytes = q4_unit_bytes(FMT), kAhead = FMT ? 2u : 4u;
    constexpr bool kScaled = !std::is_same<T, __half>::value;       // fp16 activations are operands as they come
    extern __shared__ __align__(16) uint8_t smem[];
    float* part = reinterpret_cast<float*>(smem);                             // [2][tokens][128 rows]
    uint8_t* xs = smem + S::kSumBytes;                                        // [unit][group][column][t] 16 bytes
    float* sums = reinterpret_cast<float*>(xs + p.units_staged * S::kGroups * S::kColumns * 64u);   // [unit][group][column]
    __shared__ uint32_t largest[S::kTokens];
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
    op_enter();

    // ---- activations: a power of two for each token brings its largest below 2^15 ----
    for (uint32_t i = tid; i < S::kTokens; i += kThreads) largest[i] = 0u;
    __syncthreads();
    if constexpr (kScaled) {
        const uint32_t c0 = u_begin * S::kUnitCols, c1 = min(u_end * S::kUnitCols, p.w.cols);
        if (p.a.x_col == 1) {       // a warp a token
            for (uint32_t tok = warp; tok < n_tok; tok += kThreads / 32u) {
                uint32_t big = 0;
#pragma unroll 4
                for (uint32_t c = c0 + lane * 8u; c < c1; c += 256u) {
                    float v[8];
                    load8<T>(p, tok0 + tok, c, v);
#pragma unroll
                    for (uint32_t i = 0; i < 8u; ++i) big = max(big, __float_as_uint(v[i]) & 0x7FFFFFFFu);
                }
                big = __reduce_max_sync(0xFFFFFFFFu, big);
                if (lane == 0) largest[tok] = big;
            }
        } else {                    // neighbouring threads have neighbouring tokens
            const uint32_t each = kThreads / n_tok, tok = tid % n_tok;
            const T* x = static_cast<const T*>(p.a.x) + (tok0 + tok) * p.a.x_token;
            uint32_t big = 0;
            if (tid / n_tok < each) {
#pragma unroll 4
                for (uint32_t c = c0 + tid / n_tok; c < c1; c += each) big = max(big, __float_as_uint(op_widen(x[static_cast<size_t>(c) * p.a.x_col])) & 0x7FFFFFFFu);
                atomicMax(&largest[tok], big);
            }
        }
    }
    __syncthreads();
    // what is not finite stays as it is; 2^-100 counts as the smallest
    auto exponent = [&](uint32_t tok) {
        if constexpr (!kScaled) return 14;
        const uint32_t b = largest[tok];
        return b == 0u || b >= 0x7F800000u ? 14 : max(static_cast<int>(b >> 23) - 127, -100);
    };
    // Columns 8 t .. 8 t + 7 of a group for one token, as one lane's operands of two products.
    auto stage = [&](uint32_t u0, uint32_t u1) {
        const uint32_t items = (u1 - u0) * S::kGroups * 4u * n_tok;
        for (uint32_t e0 = 0; e0 < items; e0 += kThreads) {
            const uint32_t e = e0 + tid;
            // neighbouring threads: the four pieces of a group, then tokens or groups, whichever lie closer
            const uint32_t piece = e & 3u, rest = e >> 2, groups = (u1 - u0) * S::kGroups;
            const uint32_t gr = p.a.x_col == 1 ? rest % groups : rest / n_tok, tok = p.a.x_col == 1 ? rest / groups : rest % n_tok;
            float v[8], sum_hi = 0.0f, sum_lo = 0.0f;
            uint32_t hi[4], lo[4];
            if (e < items) {
                const float up = power_of_two(14 - exponent(tok));
                const uint32_t col = (u0 * S::kGroups + gr) * 32u + piece * 8u;
                load8<T>(p, tok0 + tok, col, v);
#pragma unroll
                for (uint32_t i = 0; i < 8u; ++i) v[i] *= up;
#pragma unroll
                for (uint32_t i = 0; i < 4u; ++i) {
                    if constexpr (SPLIT) {
                        split(pack2(v[i], v[i + 4]), hi[i], lo[i]);
                        const float2 r = halves(lo[i]);
                        sum_lo += r.x + r.y;
                    } else {
                        hi[i] = bits_of(__floats2half2_rn(v[i], v[i + 4]));
                    }
                    const float2 r = halves(hi[i]);
                    sum_hi += r.x + r.y;
                }
            }
            sum_hi += __shfl_xor_sync(0xFFFFFFFFu, sum_hi, 1);
            sum_hi += __shfl_xor_sync(0xFFFFFFFFu, sum_hi, 2);
            if constexpr (SPLIT) {
                sum_lo += __shfl_xor_sync(0xFFFFFFFFu, sum_lo, 1);
                sum_lo += __shfl_xor_sync(0xFFFFFFFFu, sum_lo, 2);
            }
            if (e < items) {
                // q4_0: what the 8 of every code adds to the product; q4_k: the sum that the minimum meets
                constexpr float kTake = FMT ? 1.0f : -8.0f / (1u << kCodeShift);
                const uint32_t column = SPLIT ? tok / 4u * 8u + tok % 4u : tok;
                const uint32_t at = gr * S::kColumns + column;
                reinterpret_cast<uint4*>(xs)[at * 4u + piece] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                if constexpr (SPLIT) reinterpret_cast<uint4*>(xs)[(at + 4u) * 4u + piece] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                if (piece == 0u) {
                    sums[at] = sum_hi * kTake;
                    if constexpr (SPLIT) sums[at + 4u] = sum_lo * kTake;
                }
            }
        }
    };
    if (staged_once) {
        stage(u_begin, u_end);
        __syncthreads();
    }

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
                stage(s0, s1);
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
                        const uint32_t at = (u + i - s0) * S::kGroups;
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
                                const uint4 f = *(reinterpret_cast<const uint4*>(xs) + ((at + gr) * S::kColumns + n * 8u + g) * 4u + t);
                                const float2 s = *reinterpret_cast<const float2*>(sums + (at + gr) * S::kColumns + n * 8u + 2u * t);
                                float c[4];
                                if constexpr (FMT == 0) {
                                    c[0] = c[2] = s.x;
                                    c[1] = c[3] = s.y;
                                    mma16816(c, a[0], b[0], a[1], b[1], f.x, f.y);
                                } else {
                                    mma16816_first(c, a[0], b[0], a[1], b[1], f.x, f.y);
                                }
                                mma16816(c, a[2], b[2], a[3], b[3], f.z, f.w);
                                if constexpr (FMT) {
                                    y[n][0] = fmaf(mA, s.x, y[n][0]);
                                    y[n][1] = fmaf(mA, s.y, y[n][1]);
                                    y[n][2] = fmaf(mB, s.x, y[n][2]);
                                    y[n][3] = fmaf(mB, s.y, y[n][3]);
                                }
                                y[n][0] = fmaf(sA, c[0], y[n][0]);
                                y[n][1] = fmaf(sA, c[1], y[n][1]);
                                y[n][2] = fmaf(sB, c[2], y[n][2]);
                                y[n][3] = fmaf(sB, c[3], y[n][3]);
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
        float* mine_part = part + turn * S::kTokens * kRowsBlock;
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
                    const float down = power_of_two(exponent(tok + i) - 14), codes = power_of_two(FMT ? 0 : kCodeShift);
                    mine_part[(tok + i) * kRowsBlock + row] = y[n][i] * codes * down;
                    mine_part[(tok + i) * kRowsBlock + row + 8u] = y[n][2u + i] * codes * down;
                }
            }
        }
        if (ranks > 1u) cluster.sync();
        else __syncthreads();
        // a rank adds up its share
        for (uint32_t e = rank * kThreads + tid; e < kRowsBlock * n_tok; e += ranks * kThreads) {
            const uint32_t r = p.a.y_row == 1 ? e % kRowsBlock : e / n_tok, tok = p.a.y_row == 1 ? e / kRowsBlock : e % n_tok;
            const size_t row = static_cast<size_t>(block) * kRowsBlock + r;
            if (row >= p.w.rows) continue;
            float sum = p.a.bias ? p.a.bias[row] : 0.0f;
            float* at = mine_part + tok * kRowsBlock + r;
            for (uint32_t i = 0; i < ranks; ++i) sum += *cluster.map_shared_rank(at, i);
            p.a.y[(tok0 + tok) * p.a.y_token + row * p.a.y_row] = sum;
        }
    }
    if (ranks > 1u) cluster.sync();      // others may still read this CTA's shared memory
}

template <typename T, int FMT, int NT>
void launch(csdr_context* ctx, Q4Params p) {
    using S = Q4Shape<FMT, NT, std::is_same<T, float>::value>;
    p.n_blocks = (p.w.rows + kRowsBlock - 1u) / kRowsBlock;
    constexpr uint32_t kMostStaged = (96u * 1024u - S::kSumBytes) / S::kStageBytes;
    // Two CTAs an SM. Cut the columns so that the CTA with most to do has least: blocks in turn, each its units and about
    // two more for the join. A cut whose activations do not fit at a time stages them anew for every block.
    const uint32_t slots = static_cast<uint32_t>(ctx->sm_count) * 2u;
    uint32_t ranks = 1, least = UINT32_MAX;
    for (uint32_t r = 1; r <= 8u && r <= p.w.n_units; ++r) {
        const uint32_t units = (p.w.n_units + r - 1u) / r, clusters = slots / r;
        const uint32_t turns = (p.n_blocks + clusters - 1u) / clusters;
        const uint32_t cost = turns * (units * (units > kMostStaged ? 3u : 1u) + 2u);
        if (cost < least) {
            least = cost;
            ranks = r;
        }
    }
    p.units_rank = (p.w.n_units + ranks - 1u) / ranks;
    p.units_staged = std::min(p.units_rank, kMostStaged);
    const size_t smem = S::kSumBytes + static_cast<size_t>(p.units_staged) * S::kStageBytes;
    p.x_vec = p.a.x_col == 1 && (reinterpret_cast<uintptr_t>(p.a.x) | p.a.x_token * sizeof(T)) % 16u == 0;
    auto kern = q4_matmul_kernel<T, FMT, NT>;
    ctx->opt_in_smem(reinterpret_cast<const void*>(kern), smem);
    const uint32_t clusters = std::min(p.n_blocks, slots / ranks);
    const dim3 grid(clusters * ranks, static_cast<unsigned>((p.a.batch + S::kTokens - 1u) / S::kTokens));
    launch_op(ctx, kern, grid, kThreads, smem, ranks, p);
}

template <typename T, int FMT>
void launch_tokens(csdr_context* ctx, const Q4Params& p) {
    const size_t m = p.a.batch * (std::is_same<T, float>::value ? 2u : 1u);
    if (m <= 8) launch<T, FMT, 1>(ctx, p);
    else if (m <= 16) launch<T, FMT, 2>(ctx, p);
    else launch<T, FMT, 4>(ctx, p);
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
        LaunchScope ls(ctx, KC_Q4);
        with_dtype(a.x_dtype, [&](auto* t) {
            using T = std::remove_pointer_t<decltype(t)>;
            if (w.format == 0) launch_tokens<T, 0>(ctx, p);
            else launch_tokens<T, 1>(ctx, p);
        });
        ls.done("q4_matmul_kernel");
    }
}

}  // namespace csdr
