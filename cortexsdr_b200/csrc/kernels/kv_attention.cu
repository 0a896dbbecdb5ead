// Causal grouped-query attention over the paged 4-bit cache (kv_cache.hpp).
//   o = sum_t softmax_t(scale q . k_t) v_t,   k_t = minimum + step * code, over the tokens up to the row's own
//
// A decode step reads every cached byte once and does 4 head_dim flops a byte for each query head of a group: the
// CUDA cores could not keep up with grouped heads, and they have the codes to widen. So both products run on
// mma.m16n8k16 with the codes themselves as an operand: a code's bits, where they lie in a 16-bit word, are a
// subnormal fp16 (code 2^-18), which the matrix units multiply exactly; widening is an AND a pair, and some shifts.
//   scores   sum over groups of step * (q . code) + minimum * (sum of q)         q: 16 rows, eight fp16 roundings
//            of query rows and eight of what the roundings left
//   output   sum over groups of (p step) . (code - 8) + sum p (minimum + 8 step)   transposed, p step: 8 columns
// Rounding and rest carry 22 bits, sums are fp32's. A row's q is scaled by a power of two to use fp16's range, p step
// likewise by the largest step met. The matrix units cut sums off instead of rounding them, and sums of one sign drift (1e-5 of an
// output over 5000 keys): so the 8 comes off. For 16-bit outputs that is one more product a piece, of p step with eights; for
// fp32 ones it comes off every code, keys' too, and a piece's sums stand by themselves until they are added, rounded (16 sequences
// of 1024: 4.4e-7 of an output and 33.3 us, against 1.2e-6 and 31.0 as 16-bit outputs have it).
// tcgen05 wants the codes widened into shared memory first, which pays for prompts whose outputs round coarsely: bf16
// (kv_attention_tc.cu).
//
// Work is cut evenly, whatever the lengths: units are (sequence, tile of query rows, kv head), their length in 128 keys
// is known on the device, and CTA c of G takes the c-th G-th of all of it. A unit that is cut leaves partial
// (maximum, sum, output) pieces; the last CTA to arrive at it joins them, in the order of the keys. Nothing depends on the
// host knowing lengths, so a captured call follows its sequences as they grow.
#include <algorithm>
#include <type_traits>

#include "codes4.cuh"
#include "kv_attention.cuh"

namespace csdr {

namespace {

constexpr uint32_t kWarps = 4, kThreads = kWarps * 32, kPiece = 32;
static_assert(kBlockKeys == kWarps * kPiece, "a block is a piece a warp");

// A warp's query rows, 8 H of them: fragments, running maxima and sums, outputs. Lane (g, t) = (lane / 4, lane % 4) has the
// scores of rows g + 8 h for keys 2t, 2t + 1 of every eight, and the outputs of rows 8 h + 2t, + 2t + 1 for values
// 64 u + 8 g .. + 7.
// H = 1: eight rows, q and p step each as a rounding and what it left. H = 2: sixteen rows, roundings alone (16-bit q are
// exact in fp16; p step rounds to 2^-12 of itself, next to what rounding the output costs).
template <typename T, int HD, int H>
struct Rows {
    static constexpr uint32_t W = HD / 32, G = HD / 64;
    static constexpr bool kFine = std::is_same<T, float>::value;
    static constexpr bool kOnce = H == 2 || std::is_same<T, __nv_bfloat16>::value;      // bf16 rounds eight times as coarsely as p step
    static_assert(!kFine || H == 1, "sixteen rows are for 16-bit outputs");
    static constexpr float kOdd = kFine ? 1.0f : 16.0f;      // odd pairs of codes count one in kOdd
    static constexpr bool kShared = HD >= 128;     // q fragments in shared memory: the registers go to the outputs
    static constexpr uint32_t kMetaBytes = 2u * G * 16u * 16u;      // of a piece, widened
    uint32_t q[kShared ? 1 : W * 2][4];
    float o[H][G][4][4];     // tile n of a group: values 8 g + n (rows 2t, 2t + 1), 8 g + 4 + n (rows 2t, 2t + 1)
    f32x2 om[H][G], l[H];    // over even and odd keys
    float sum_q[H][G];
    float factor[H], m[H], escale;
    uint32_t vmax;           // the largest step of the values so far, as bits
    int32_t limit[H];        // keys that this lane's rows see
    int32_t least;           // the fewest that one of the warp's rows sees, the most
    int32_t most;

    // Lane (g, t): rows g + 8 h of the tile, values 64 (w / 2) + 16 t + 8 (w % 2) + n of words w. Of `parts` warps with the
    // same rows, number `part` writes its part of shared fragments.
    __device__ __forceinline__ void load(const AttnParams& p, const Seq& s, uint32_t kvh, uint32_t row, uint32_t lane, uint4* shared, uint32_t part,
                                         uint32_t parts) {
        const uint32_t t = lane & 3u;
        least = 0x7FFFFFFF;
        most = 0;
        uint32_t kept[H][H == 2 ? W * 4 : 1];      // a row's roundings, for H = 2 to be paired with the other row's
#pragma unroll
        for (uint32_t h = 0; h < H; ++h) {
            const uint32_t rr = row + 8u * h + (lane >> 2), tok = rr / p.group, head = kvh * p.group + rr % p.group;
            const bool there = tok < s.n_new;
            limit[h] = there ? static_cast<int32_t>(min(max(s.base + tok + 1, static_cast<int64_t>(0)), s.cap)) : 0;
            least = min(least, there ? limit[h] : 0x7FFFFFFF);
            most = max(most, limit[h]);
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
            // 2^e above the largest |q|: q 2^(top - e) < 2^15 (and sixteen times that), exact but for the last bits of what is
            // 2^-20 of the largest
            constexpr int kTop = kFine ? 15 : 11;
            const int e = big > 0.0f && big < INFINITY ? min(max(ilogbf(big) + 1, -110), 128) : kTop;      // 2^125 is the most that powers below go to
            // the scale's sign goes with q: the largest score / factor is the largest score
            const float up = copysignf(power_of_two(kTop - e), p.a.scale);
            factor[h] = factor_of(p.a.scale, e - kTop + kCodeShift, 100);      // scores / factor are below 2^22
#pragma unroll
            for (uint32_t g = 0; g < G; ++g) sum_q[h][g] = 0.0f;
#pragma unroll
            for (uint32_t w = 0; w < W; ++w) {
#pragma unroll
                for (uint32_t i = 0; i < 8u; ++i) {
                    x[w][i] *= up;
                    sum_q[h][w / 2u] += x[w][i];
                }
#pragma unroll
                for (uint32_t i = 0; i < 2u; ++i) {
                    if (kShared && w % parts != part) continue;
                    // values 2i, 2i + 4 meet even pairs of codes, 2i + 1, 2i + 5 odd ones
                    const f32x2 even = pack2(x[w][2 * i], x[w][2 * i + 4]), odd = pack2(x[w][2 * i + 1] * kOdd, x[w][2 * i + 5] * kOdd);
                    uint32_t f[4];
                    if constexpr (H == 1) {
                        split(even, f[0], f[1]);
                        split(odd, f[2], f[3]);
                    } else {
                        const float2 ev = unpack2(even), od = unpack2(odd);
                        kept[h][(w * 2u + i) * 2u] = bits_of(__floats2half2_rn(ev.x, ev.y));
                        kept[h][(w * 2u + i) * 2u + 1u] = bits_of(__floats2half2_rn(od.x, od.y));
                        if (h == 0u) continue;
                        f[0] = kept[0][(w * 2u + i) * 2u];
                        f[1] = kept[H - 1][(w * 2u + i) * 2u];
                        f[2] = kept[0][(w * 2u + i) * 2u + 1u];
                        f[3] = kept[H - 1][(w * 2u + i) * 2u + 1u];
                    }
                    if constexpr (kShared) {
                        shared[(w * 2u + i) * 32u + lane] = make_uint4(f[0], f[1], f[2], f[3]);
                    } else {
#pragma unroll
                        for (uint32_t j = 0; j < 4u; ++j) q[w * 2u + i][j] = f[j];
                    }
                }
            }
#pragma unroll
            for (uint32_t g = 0; g < G; ++g) {
                sum_q[h][g] += __shfl_xor_sync(0xFFFFFFFFu, sum_q[h][g], 1);
                sum_q[h][g] += __shfl_xor_sync(0xFFFFFFFFu, sum_q[h][g], 2);
                sum_q[h][g] *= power_of_two(-kCodeShift);
                om[h][g] = pack2(0.0f, 0.0f);
#pragma unroll
                for (uint32_t n = 0; n < 4u; ++n)
#pragma unroll
                    for (uint32_t j = 0; j < 4u; ++j) o[h][g][n][j] = 0.0f;
            }
            m[h] = -FLT_MAX;
            l[h] = pack2(0.0f, 0.0f);
        }
        least = __reduce_min_sync(0xFFFFFFFFu, least);
        most = __reduce_max_sync(0xFFFFFFFFu, most);
        escale = 1.0f;
        vmax = 0;
    }

    // A value of row 2t and of row 2t + 1, from the lanes that have the rows.
    static __device__ __forceinline__ float2 of_columns(float v, uint32_t lane) {
        const uint32_t from = 8u * (lane & 3u);
        return make_float2(__shfl_sync(0xFFFFFFFFu, v, from), __shfl_sync(0xFFFFFFFFu, v, from + 4u));
    }

    // 32 keys from `tok0` on, in shared memory at `block` (two blocks of sixteen); bit i of `there`: block i has a page.
    // `meta`: the warp's, for steps and minima as pairs of fp32 over neighbouring tokens.
    // edge: some row does not see all of them.
    template <bool edge>
    __device__ __forceinline__ void keys32(const uint8_t* block, int32_t tok0, uint32_t there, uint32_t lane, const uint4* shared, uint8_t* meta) {
        const uint32_t g = lane >> 2, t = lane & 3u;
        // ---- steps and minima: a lane widens a pair of tokens of the keys' groups (lanes 0-15) or of the values' ----
        uint32_t big = 0;
        {
            const uint32_t pr = lane & 15u, of_values = lane >> 4;
            const uint8_t* from = block + (pr >> 3) * (18u * HD) + (16u + of_values) * HD + (pr & 7u) * 8u;
            const float mid = kFine || of_values ? 8.0f : 0.0f;
#pragma unroll
            for (uint32_t u = 0; u < G; ++u) {
                uint2 w = *reinterpret_cast<const uint2*>(from + 64u * u);
                if (edge && of_values) {     // nothing of what lies behind the last key that is seen
                    const int32_t tok = tok0 + static_cast<int32_t>(2u * pr);
                    const bool gone = !(there >> (pr >> 3) & 1u);
                    if (gone || tok >= most) w.x = 0u;
                    if (gone || tok + 1 >= most) w.y = 0u;
                }
                const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&w.x)), b = __half22float2(*reinterpret_cast<const __half2*>(&w.y));
                const float2 c = unpack2(fma2(pack2(mid, mid), pack2(a.y, b.y), pack2(a.x, b.x)));
                *reinterpret_cast<float4*>(meta + ((of_values * G + u) * 16u + pr) * 16u) = make_float4(a.y, b.y, c.x, c.y);
                if (of_values) big = max(big, max(__float_as_uint(a.y), __float_as_uint(b.y)));
            }
        }
        __syncwarp();
        // ---- scores ----
        f32x2 sc[H][4];             // scores / factor
#pragma unroll
        for (uint32_t gq = 0; gq < G; ++gq) {
            float acc[4][4];
            uint2 w[4];
#pragma unroll
            for (uint32_t nt = 0; nt < 4u; ++nt)
                w[nt] = *reinterpret_cast<const uint2*>(block + (nt >> 1) * (18u * HD) + (8u * (nt & 1u) + g) * (HD / 2) + t * (HD / 8) + 8u * gq);
#pragma unroll
            for (uint32_t i = 0; i < 2u; ++i) {
                uint32_t f[2][4];
#pragma unroll
                for (uint32_t h = 0; h < 2u; ++h) {
                    if constexpr (kShared) {
                        const uint4 v = shared[((2u * gq + i) * 2u + h) * 32u + lane];
                        f[h][0] = v.x;
                        f[h][1] = v.y;
                        f[h][2] = v.z;
                        f[h][3] = v.w;
                    } else {
#pragma unroll
                        for (uint32_t j = 0; j < 4u; ++j) f[h][j] = q[(2u * gq + i) * 2u + h][j];
                    }
                }
#pragma unroll
                for (uint32_t nt = 0; nt < 4u; ++nt) {
                    uint32_t r[4];
                    widen_codes<kFine>(i ? w[nt].y : w[nt].x, r);
                    if constexpr (kFine) {
#pragma unroll
                        for (uint32_t n = 0; n < 4u; ++n) r[n] = less_eight(r[n]);
                    }
                    if (i == 0u) mma16816_first(acc[nt], f[0][0], f[0][1], f[0][2], f[0][3], r[0], r[1]);
                    else mma16816(acc[nt], f[0][0], f[0][1], f[0][2], f[0][3], r[0], r[1]);
                    mma16816(acc[nt], f[1][0], f[1][1], f[1][2], f[1][3], r[2], r[3]);
                }
            }
#pragma unroll
            for (uint32_t nt = 0; nt < 4u; ++nt) {
                const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(meta + (gq * 16u + 4u * nt + t) * 16u);     // steps, minima
#pragma unroll
                for (uint32_t h = 0; h < H; ++h) {
                    const f32x2 sq = pack2(sum_q[h][gq], sum_q[h][gq]);
                    const f32x2 low = gq ? fma2(v.y, sq, sc[h][nt]) : mul2(v.y, sq);
                    const f32x2 dot = H == 1 ? add2(pack2(acc[nt][0], acc[nt][1]), pack2(acc[nt][2], acc[nt][3]))
                                             : pack2(acc[nt][2 * h], acc[nt][2 * h + 1]);
                    sc[h][nt] = fma2(v.x, dot, low);
                }
            }
        }
        float top[H];
        bool grows = big > vmax;
#pragma unroll
        for (uint32_t h = 0; h < H; ++h) {
            if (edge) {
                // keys that a row does not see weigh nothing, whatever lies there
#pragma unroll
                for (uint32_t nt = 0; nt < 4u; ++nt) {
                    float2 v = unpack2(sc[h][nt]);
                    const int32_t tok = tok0 + static_cast<int32_t>(8u * nt + 2u * t);
                    const bool gone = !(there >> (nt >> 1) & 1u);
                    if (gone || tok >= limit[h]) v.x = -INFINITY;
                    if (gone || tok + 1 >= limit[h]) v.y = -INFINITY;
                    sc[h][nt] = pack2(v.x, v.y);
                }
            }
            top[h] = -INFINITY;
#pragma unroll
            for (uint32_t nt = 0; nt < 4u; ++nt) {
                const float2 v = unpack2(sc[h][nt]);
                top[h] = fmaxf(top[h], fmaxf(v.x, v.y));
            }
            top[h] = fmaxf(top[h], __shfl_xor_sync(0xFFFFFFFFu, top[h], 1));
            top[h] = fmaxf(top[h], __shfl_xor_sync(0xFFFFFFFFu, top[h], 2)) * factor[h];
            grows = grows || top[h] > m[h] + kSlack;
        }
        // The maximum follows in steps: weights may reach 2^kSlack before outputs are scaled anew
        if (__any_sync(0xFFFFFFFFu, grows)) {
            float down = 1.0f;
            big = __reduce_max_sync(0xFFFFFFFFu, big);
            if (big > vmax) {
                // weight * step < 2^(kSlack + 1 + exponent of the largest step) -> below 2^15
                vmax = big;
                const float next_scale = power_of_two(14 - static_cast<int>(kSlack) - ilogbf(__uint_as_float(big)));
                down = next_scale / escale;
                escale = next_scale;
            }
#pragma unroll
            for (uint32_t h = 0; h < H; ++h) {
                const float next = fmaxf(m[h], top[h]), f = ex2(m[h] - next);
                m[h] = next;
                l[h] = mul2(l[h], pack2(f, f));
                const float2 fc = of_columns(f, lane);
                const f32x2 both = pack2(fc.x * down, fc.y * down);
#pragma unroll
                for (uint32_t u = 0; u < G; ++u) {
                    om[h][u] = mul2(om[h][u], pack2(f, f));
#pragma unroll
                    for (uint32_t n = 0; n < 4u; ++n) scale_tile(o[h][u][n], both);
                }
            }
        }
        f32x2 p[H][4];
        const f32x2 es = pack2(escale, escale);
#pragma unroll
        for (uint32_t h = 0; h < H; ++h) {
            const f32x2 fac = pack2(factor[h], factor[h]), less = pack2(-m[h], -m[h]);
#pragma unroll
            for (uint32_t nt = 0; nt < 4u; ++nt) {
                const float2 v = unpack2(fma2(sc[h][nt], fac, less));
                p[h][nt] = pack2(ex2(v.x), ex2(v.y));
                l[h] = add2(l[h], p[h][nt]);
            }
        }
        // ---- outputs ----
#pragma unroll
        for (uint32_t u = 0; u < G; ++u) {
            uint32_t hi[H][4], lo[4];
            float eight[H][4];
#pragma unroll
            for (uint32_t nt = 0; nt < 4u; ++nt) {
                const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(meta + ((G + u) * 16u + 4u * nt + t) * 16u);     // steps, minima + 8 steps
                const f32x2 steps = mul2(v.x, es);
#pragma unroll
                for (uint32_t h = 0; h < H; ++h) {
                    f32x2 st = steps, mn = v.y;
                    if (edge) {
                        const int32_t tok = tok0 + static_cast<int32_t>(8u * nt + 2u * t);
                        float2 a = unpack2(st), b = unpack2(mn);
                        if (tok >= limit[h]) a.x = b.x = 0.0f;
                        if (tok + 1 >= limit[h]) a.y = b.y = 0.0f;
                        st = pack2(a.x, a.y);
                        mn = pack2(b.x, b.y);
                    }
                    om[h][u] = fma2(p[h][nt], mn, om[h][u]);
                    const f32x2 w = mul2(p[h][nt], st);
                    if constexpr (kOnce) {
                        const float2 x = unpack2(w);
                        hi[h][nt] = bits_of(__floats2half2_rn(x.x, x.y));
                    } else {
                        split(w, hi[h][nt], lo[nt]);
                    }
                }
            }
#pragma unroll
            for (uint32_t h = 0; h < (kFine ? 0u : H); ++h) {
                mma16816_first(eight[h], kEights, kEights, kEights, kEights, hi[h][0], hi[h][1]);
                mma16816(eight[h], kEights, kEights, kEights, kEights, hi[h][2], hi[h][3]);
                if constexpr (!kOnce) {
                    mma16816(eight[h], kEights, kEights, kEights, kEights, lo[0], lo[1]);
                    mma16816(eight[h], kEights, kEights, kEights, kEights, lo[2], lo[3]);
                }
            }
            if constexpr (kFine) {
                // a piece's sums by themselves: what is cut off is cut off them, and they are added rounded
                float z[4][4];
#pragma unroll
                for (uint32_t b = 0; b < 2u; ++b) {
                    uint32_t r[4][4];
                    values_at(block, b, u, t, g, r);
#pragma unroll
                    for (uint32_t k = 0; k < 4u; ++k)
#pragma unroll
                        for (uint32_t n = 0; n < 4u; ++n) r[k][n] = less_eight(r[k][n]);
#pragma unroll
                    for (uint32_t n = 0; n < 4u; ++n) {
                        if (b == 0u) mma16816_first(z[n], r[0][n], r[1][n], r[2][n], r[3][n], lo[2u * b], lo[2u * b + 1u]);
                        else mma16816(z[n], r[0][n], r[1][n], r[2][n], r[3][n], lo[2u * b], lo[2u * b + 1u]);
                        mma16816(z[n], r[0][n], r[1][n], r[2][n], r[3][n], hi[0][2u * b], hi[0][2u * b + 1u]);
                    }
                }
#pragma unroll
                for (uint32_t n = 0; n < 4u; ++n) {
                    const float2 x = unpack2(add2(pack2(o[0][u][n][0], o[0][u][n][1]), pack2(z[n][0], z[n][1])));
                    const float2 y = unpack2(add2(pack2(o[0][u][n][2], o[0][u][n][3]), pack2(z[n][2], z[n][3])));
                    o[0][u][n][0] = x.x;
                    o[0][u][n][1] = x.y;
                    o[0][u][n][2] = y.x;
                    o[0][u][n][3] = y.y;
                }
                continue;
            }
#pragma unroll
            for (uint32_t b = 0; b < 2u; ++b) {
                uint32_t r[4][4];
                values_at(block, b, u, t, g, r);
#pragma unroll
                for (uint32_t n = 0; n < 4u; ++n) {
#pragma unroll
                    for (uint32_t h = 0; h < H; ++h) mma16816(o[h][u][n], r[0][n], r[1][n], r[2][n], r[3][n], hi[h][2u * b], hi[h][2u * b + 1u]);
                    if constexpr (!kOnce) mma16816(o[0][u][n], r[0][n], r[1][n], r[2][n], r[3][n], lo[2u * b], lo[2u * b + 1u]);
                }
            }
#pragma unroll
            for (uint32_t n = 0; n < 4u; ++n) {
                const float times = n & 1u ? -1.0f / kOdd : -1.0f;
#pragma unroll
                for (uint32_t h = 0; h < H; ++h) add_tile(o[h][u][n], pack2(eight[h][0], eight[h][1]), pack2(times, times));
            }
        }
    }
    // Words of block b's pairs of tokens 2t, 2t + 8 as pairs of codes: values 64 u + 8 g + n and + 4 + n.
    static __device__ __forceinline__ void values_at(const uint8_t* block, uint32_t b, uint32_t u, uint32_t t, uint32_t g, uint32_t (&r)[4][4]) {
        const uint8_t* v0 = block + b * (18u * HD) + 8u * HD + t * HD + g * (HD / 8) + 8u * u;
        const uint2 w0 = *reinterpret_cast<const uint2*>(v0), w1 = *reinterpret_cast<const uint2*>(v0 + 4u * HD);
        widen_codes<kFine>(w0.x, r[0]);
        widen_codes<kFine>(w0.y, r[1]);
        widen_codes<kFine>(w1.x, r[2]);
        widen_codes<kFine>(w1.y, r[3]);
    }
    __device__ __forceinline__ void piece(const uint8_t* block, int32_t tok0, uint32_t there, uint32_t lane, const uint4* shared, uint8_t* meta) {
        if (there != 3u || tok0 + 32 > least) keys32<true>(block, tok0, there, lane, shared, meta);
        else keys32<false>(block, tok0, there, lane, shared, meta);
    }
    static __device__ __forceinline__ void scale_tile(float (&c)[4], f32x2 f) {
        const float2 a = unpack2(mul2(pack2(c[0], c[1]), f)), b = unpack2(mul2(pack2(c[2], c[3]), f));
        c[0] = a.x;
        c[1] = a.y;
        c[2] = b.x;
        c[3] = b.y;
    }
    static __device__ __forceinline__ void add_tile(float (&c)[4], f32x2 e, f32x2 k) {
        const float2 a = unpack2(fma2(e, k, pack2(c[0], c[1]))), b = unpack2(fma2(e, k, pack2(c[2], c[3])));
        c[0] = a.x;
        c[1] = a.y;
        c[2] = b.x;
        c[3] = b.y;
    }

    // Calls out(row, value of the head, eight values, sum) with the outputs before the division, for rows 8 h + 2t and + 2t + 1,
    // and row(row, maximum, sum) once for each row.
    template <typename Out, typename Row>
    __device__ __forceinline__ void finish(uint32_t lane, Out&& out, Row&& row) {
        const uint32_t g = lane >> 2, t = lane & 3u;
        auto all = [](f32x2 v) {
            const float2 e = unpack2(v);
            float x = e.x + e.y;
            x += __shfl_xor_sync(0xFFFFFFFFu, x, 1);
            return x + __shfl_xor_sync(0xFFFFFFFFu, x, 2);
        };
        const float down = power_of_two(kCodeShift) / escale;
#pragma unroll
        for (uint32_t h = 0; h < H; ++h) {
            const float sum = all(l[h]);
            const float2 sums = of_columns(sum, lane);
            if (t == 0) row(8u * h + g, m[h], sum);
#pragma unroll
            for (uint32_t u = 0; u < G; ++u) {
                const float2 mins = of_columns(all(om[h][u]), lane);
                float v[2][8];
#pragma unroll
                for (uint32_t n = 0; n < 4u; ++n) {
                    const float d = n & 1u ? down * kOdd : down;
                    v[0][n] = fmaf(o[h][u][n][0], d, mins.x);
                    v[1][n] = fmaf(o[h][u][n][1], d, mins.y);
                    v[0][4 + n] = fmaf(o[h][u][n][2], d, mins.x);
                    v[1][4 + n] = fmaf(o[h][u][n][3], d, mins.y);
                }
                out(8u * h + 2u * t, 64u * u + 8u * g, v[0], sums.x);
                out(8u * h + 2u * t + 1u, 64u * u + 8u * g, v[1], sums.y);
            }
        }
    }
    // Row r's output before the division, maximum and sum, to `to`: [row][HD + 4].
    __device__ __forceinline__ void store(float* to, uint32_t lane) {
        finish(
            lane,
            [&](uint32_t r, uint32_t d, const float(&v)[8], float) {
                float4* at = reinterpret_cast<float4*>(to + r * kPitch<HD> + d);
                at[0] = make_float4(v[0], v[1], v[2], v[3]);
                at[1] = make_float4(v[4], v[5], v[6], v[7]);
            },
            [&](uint32_t r, float top, float sum) {
                *reinterpret_cast<float2*>(to + r * kPitch<HD> + HD) = make_float2(top, sum);
            });
    }
};

// CTAs an SM: what the registers of the outputs leave room for.
template <int HD, int H>
__host__ __device__ constexpr int ctas() { return HD > 128 ? 2 : HD * H > 128 ? 3 : 4; }
// Stages of 32 keys that a warp (KEYS) or the CTA keeps on their way.
template <int HD, bool KEYS>
__host__ __device__ constexpr uint32_t stages() { return !KEYS || HD == 64 ? 4u : 2u; }
template <int HD, bool KEYS>
constexpr size_t smem_bytes() {
    return (KEYS ? kWarps : 1u) * stages<HD, KEYS>() * 36u * HD + kWarps * 2u * (HD / 64u) * 256u +
           (HD >= 128 ? (KEYS ? 1u : kWarps) * (HD / 16u) * 512u : 0u);
}

// KEYS: the four warps share a tile of eight rows and take 32 keys of a block each (a decode step); else each has 8 H
// rows of its own and all see the same keys (prompts).
template <typename T, int HD, bool KEYS, int H>
__global__ void __launch_bounds__(kThreads, ctas<HD, H>())
kv_attention_kernel(AttnParams p) {
    constexpr uint32_t TILE = KEYS ? 8u : 32u * H, SB = 18u * HD;      // SB: a block of sixteen tokens
    using Warp = Rows<T, HD, H>;
    constexpr uint32_t kStages = stages<HD, KEYS>(), kStageBytes = 2u * SB;
    extern __shared__ __align__(128) uint8_t smem[];
    // stages (of each warp, or of all); for each warp, widened steps and minima; q fragments (head_dim 128 and 256). Rows to be
    // joined (KEYS) lie where the warp's stages were
    uint8_t* ring = smem;
    uint8_t* meta_s = smem + (KEYS ? kWarps : 1u) * kStages * kStageBytes;
    __shared__ uint64_t bars[kWarps * kStages];
    __shared__ uint64_t empty[kStages];      // where the warps share stages: all are through with one
    __shared__ uint32_t there_s[kStages];
    __shared__ ScheduleShared<kThreads> sched;
    __shared__ uint32_t flag;
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5;
    uint8_t* my_meta = meta_s + warp * Warp::kMetaBytes;
    uint4* my_q = reinterpret_cast<uint4*>(meta_s + kWarps * Warp::kMetaBytes + (KEYS ? 0u : warp) * (HD / 16u) * 512u);
    uint8_t* my_ring = ring + (KEYS ? warp * kStages * kStageBytes : 0u);
    static_assert(!KEYS || kStages * kStageBytes >= 8u * kPitch<HD> * 4u, "a warp's rows fit into its stages");
    auto rows_of = [&](uint32_t w) { return reinterpret_cast<float*>(ring + w * kStages * kStageBytes); };
    const uint32_t my_bar = smem_u32(&bars[KEYS ? warp * kStages : 0u]);
    if (tid == 0) {
        for (uint32_t i = 0; i < kWarps * kStages; ++i) asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(smem_u32(&bars[i])));
        for (uint32_t i = 0; i < kStages; ++i) asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(&empty[i])), "r"(kWarps));
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        sched.longest = sched.n_units = 0;
    }
    __syncthreads();
    op_enter();
    asm volatile("fence.proxy.async;" ::: "memory");

    Schedule<TILE, kThreads> sch;
    if (!sch.begin(p, sched)) return;
    const uint64_t x1 = sch.x1;
    uint64_t x = sch.x0;
    uint32_t turn = 0;       // stages filled so far
    bool live = true;
    Warp rows;

    // Two blocks of sixteen tokens, one copy where they lie one behind the other; a block without a page is left out.
    const uint32_t in_page = (1u << (p.kv.page_shift - 4u)) - 1u;
    const size_t page_bytes = p.kv.block_at(1u, 0u, 0u);
    const uint8_t* head_base = nullptr;      // of the unit's kv head
    auto fetch = [&](uint8_t* to, uint32_t bar, uint32_t sub, int32_t pg0, int32_t pg1) {
        const bool one = pg0 == pg1 && in_page != 0u;
        const uint32_t first = one && pg0 >= 0 ? 2u * SB : pg0 >= 0 ? SB : 0u, second = !one && pg1 >= 0 ? SB : 0u;
        asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(first + second) : "memory");
        auto copy = [&](uint32_t at, int32_t page, uint32_t block, uint32_t size) {
            asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(to) + at),
                         "l"(head_base + static_cast<uint32_t>(page) * page_bytes + (block & in_page) * SB), "r"(size), "r"(bar)
                         : "memory");
        };
        if (first) copy(0u, pg0, sub, first);
        if (second) copy(SB, pg1, sub + 1u, second);
    };

    while (x < x1) {      // without the keys once a wait has run out: who joins a unit counts on everyone
        Unit un;
        if (!sch.at(p, x, un)) {
            x = un.next;
            continue;
        }
        const Seq& sq = sch.sq;
        const uint32_t kvh = un.kvh, tile = un.tile, b0 = un.b0, b1 = un.b1, n_blocks = un.n_blocks;
        const uint64_t start = un.start, next = un.next;
        const int32_t keys = un.keys;
        head_base = p.kv.base + p.kv.block_at(0u, kvh, 0u);
        const int32_t* table = p.b.pages + static_cast<size_t>(sch.s) * p.b.pages_per_seq;

        // ---- its keys from block b0 to b1, in pieces of 32 ----
        const uint32_t subs = static_cast<uint32_t>(keys + 15) / 16u;      // blocks of sixteen that exist
        if constexpr (KEYS) {
            // a warp's i-th piece is number 4 (b0 + i) + warp; the pages of sixteen pieces at a time, a lane a block
            const uint32_t first = 4u * b0 + warp;
            const uint32_t n = !live || 2u * first >= subs ? 0u : min(b1 - b0, (subs - 2u * first + 7u) / 8u);
            int32_t page_of = -1;
            uint32_t there = 0;      // two bits a stage: the piece's blocks have pages
            auto issue = [&](uint32_t i) {
                if ((i & 15u) == 0u) {
                    const uint32_t sub = 2u * (first + 4u * (i + (lane >> 1))) + (lane & 1u);
                    page_of = sub < subs ? table[sub >> (p.kv.page_shift - 4u)] : -1;
                    if (static_cast<uint32_t>(page_of) >= p.kv.n_pages) page_of = -1;
                }
                const int32_t pg0 = __shfl_sync(0xFFFFFFFFu, page_of, 2u * (i & 15u)), pg1 = __shfl_sync(0xFFFFFFFFu, page_of, 2u * (i & 15u) + 1u);
                const uint32_t st = turn % kStages, have = (pg0 >= 0 ? 1u : 0u) | (pg1 >= 0 ? 2u : 0u);
                there = (there & ~(3u << 2u * st)) | have << 2u * st;
                if (lane == 0) fetch(my_ring + st * kStageBytes, my_bar + 8u * st, 2u * (first + 4u * i), pg0, pg1);
                ++turn;
            };
            const uint32_t turn0 = turn;
            for (uint32_t i = 0; i < min(n, kStages); ++i) issue(i);
            rows.load(p, sq, kvh, tile * TILE, lane, my_q, warp, kWarps);
            if constexpr (Warp::kShared) __syncthreads();
            for (uint32_t i = 0; i < n; ++i) {
                const uint32_t k = turn0 + i, st = k % kStages;
                live = mbar_wait_first(my_bar + 8u * st, (k / kStages) & 1u, p.spin);
                if (!live) {
                    for (uint32_t j = k; j < turn; ++j) mbar_wait(my_bar + 8u * (j % kStages), (j / kStages) & 1u, kDrainRounds);
                    break;
                }
                rows.piece(my_ring + st * kStageBytes, static_cast<int32_t>((first + 4u * i) * kPiece), there >> 2u * st & 3u, lane, my_q, my_meta);
                __syncwarp();
                if (i + kStages < n) issue(i + kStages);
            }
            __syncwarp();
            rows.store(rows_of(warp), lane);
        } else {
            // All warps see every piece. Warp 0 copies: a stage when all are through with it, one piece behind their work
            const uint32_t first = 4u * b0, n = live ? min(4u * (b1 - b0), (max(subs, 2u * first) - 2u * first + 1u) / 2u) : 0u, turn0 = turn;
            uint32_t issued = 0;
            int32_t page_of = -1;
            auto issue = [&](uint32_t i) {
                if ((i & 15u) == 0u) {
                    const uint32_t sub = 2u * (first + i) + lane;
                    page_of = sub < subs ? table[sub >> (p.kv.page_shift - 4u)] : -1;
                    if (static_cast<uint32_t>(page_of) >= p.kv.n_pages) page_of = -1;
                }
                const int32_t pg0 = __shfl_sync(0xFFFFFFFFu, page_of, 2u * (i & 15u)), pg1 = __shfl_sync(0xFFFFFFFFu, page_of, 2u * (i & 15u) + 1u);
                const uint32_t k = turn0 + i, st = k % kStages;
                if (k >= kStages) live = live && mbar_wait(smem_u32(&empty[st]), (k / kStages - 1u) & 1u, p.spin);
                if (!live) return;
                ++issued;
                if (lane == 0) {
                    there_s[st] = (pg0 >= 0 ? 1u : 0u) | (pg1 >= 0 ? 2u : 0u);
                    fetch(my_ring + st * kStageBytes, my_bar + 8u * st, 2u * (first + i), pg0, pg1);
                }
            };
            if (warp == 0)
                for (uint32_t i = 0; i < min(n, kStages); ++i) issue(i);
            rows.load(p, sq, kvh, tile * TILE + warp * 8u * H, lane, my_q, 0u, 1u);
            __syncwarp();
            for (uint32_t i = 0; i < n && live; ++i) {
                const uint32_t k = turn0 + i, st = k % kStages;
                live = mbar_wait_first(my_bar + 8u * st, (k / kStages) & 1u, p.spin);
                if (!live) break;
                const int32_t tok = static_cast<int32_t>(kPiece * (first + i));
                if (tok < rows.most) rows.piece(my_ring + st * kStageBytes, tok, there_s[st], lane, my_q, my_meta);
                __syncwarp();
                if (lane == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(&empty[st])) : "memory");
                if (warp == 0 && i >= 1u && i - 1u + kStages < n) issue(i - 1u + kStages);
            }
            if (!live)      // warp 0 has copied
                for (uint32_t j = max(issued, kStages) - kStages; j < issued; ++j)
                    mbar_wait(my_bar + 8u * ((turn0 + j) % kStages), ((turn0 + j) / kStages) & 1u, kDrainRounds);
            turn += n;
        }
        live = __syncthreads_and(live);
        if (!live) {
            if (tid == 0) atomicExch(p.status, 1);
        }

        // ---- out, or a piece of it ----
        const bool whole = b0 == 0u && b1 == n_blocks;
        float* slot = p.part + (static_cast<size_t>(blockIdx.x) * 2u + (start >= sch.x0 ? 1u : 0u)) * TILE * kPitch<HD>;
        auto write = [&](uint32_t r, uint32_t d, const float(&o)[8], float l) {
            const uint32_t rr = tile * TILE + r, tok = rr / p.group, head = kvh * p.group + rr % p.group;
            if (tok >= sq.n_new) return;
            T* dst = static_cast<T*>(p.a.out) + static_cast<size_t>(sq.row0 + tok) * p.a.out_stride + static_cast<size_t>(head) * HD + d;
            store_row(dst, o, l != 0.0f ? 1.0f / l : 0.0f, p.vec_out);      // rows that saw nothing: zeros
        };
        if constexpr (KEYS) {
            for (uint32_t e = tid; e < HD; e += kThreads) {
                const uint32_t r = e / (HD / 8u), d = e % (HD / 8u) * 8u;
                float o[8], m, l;
                join<HD>(kWarps, d, [&](uint32_t i, uint32_t j) { return *reinterpret_cast<const float4*>(rows_of(i) + r * kPitch<HD> + j); }, o, m, l);
                if (whole) {
                    write(r, d, o, l);
                } else {
                    float4* to = reinterpret_cast<float4*>(slot + r * kPitch<HD> + d);
                    to[0] = make_float4(o[0], o[1], o[2], o[3]);
                    to[1] = make_float4(o[4], o[5], o[6], o[7]);
                    if (d == 0) *reinterpret_cast<float4*>(slot + r * kPitch<HD> + HD) = make_float4(m, l, 0.0f, 0.0f);
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");     // the stages are copied into again
            __syncthreads();
        } else if (!whole) {
            rows.store(slot + warp * 8u * H * kPitch<HD>, lane);
        } else {
            rows.finish(
                lane, [&](uint32_t r, uint32_t d, const float(&v)[8], float sum) { write(warp * 8u * H + r, d, v, sum); }, [](uint32_t, float, float) {});
        }
        if (!whole) {
            const uint32_t c0 = sch.holder(start), c1 = sch.holder(start + n_blocks - 1u);
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
                for (uint32_t e = tid; e < TILE * HD / 8u; e += kThreads) {
                    const uint32_t r = e / (HD / 8u), d = e % (HD / 8u) * 8u;
                    float o[8], m, l;
                    join<HD>(
                        c1 - c0 + 1u, d,
                        [&](uint32_t i, uint32_t j) {   // past L1: other CTAs wrote these
                            return __ldcg(reinterpret_cast<const float4*>(
                                p.part + ((static_cast<size_t>(c0 + i) * 2u + (i == 0u ? 1u : 0u)) * TILE + r) * kPitch<HD> + j));
                        },
                        o, m, l);
                    write(r, d, o, l);
                }
            }
            __syncthreads();
        }
        x = start + n_blocks < next ? next : start + n_blocks;
        if (start + n_blocks > x1) break;
    }
}

template <typename T, int HD, bool KEYS, int H>
void launch(csdr_context* ctx, AttnParams& p) {
    constexpr size_t smem = smem_bytes<HD, KEYS>();
    auto kern = kv_attention_kernel<T, HD, KEYS, H>;
    const void* key = reinterpret_cast<const void*>(kern);
    ctx->opt_in_smem(key, smem);
    auto& fit = ctx->occupancy[key];
    if (!fit.second) {
        int n = 0;
        CSDR_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kern, kThreads, smem));
        fit = {smem, std::max(1, std::min(n, ctas<HD, H>()))};
    }
    launch_op(ctx, kern, dim3(static_cast<unsigned>(ctx->sm_count * fit.second)), kThreads, smem, 1, p);
}

template <typename T, int HD>
void launch_rows(csdr_context* ctx, uint64_t rows, AttnParams& p) {
    // query rows of a sequence and kv head, on average. Few: the warps share eight rows and have keys of their own, so that a
    // tile's keys are spread over four warps. Many: each has rows of its own and keys are shared. 4 sequences of 2048, 8 kv heads
    // of 128, us for 64, 128, 512, 2048 rows:
    //   fp32   49, 72, 203, 680 and 51, 81, 212, 647 (heads of 256: 74, 119, 388, 1358 and 96, 141, 401, 1286)
    //   fp16   43, 64, 177, 585 and 57, 75, 147, 363
    //   bf16   41, 58, 160, 526 and, on tcgen05, 51, 53, 76, 164 (fp16 outputs are eight times as fine and keep their codes)
    // One form for all sequences of a call, whatever they have: a captured call does not know. Single tokens beside a prompt cost
    // more than in a call of their own: 31 over 8192 keys and 2048 rows of a prompt 515 (fp32), 543 (fp16), 364 (bf16), as two calls
    // 486, 309, 191; 31 over 1024 and 512 rows of a prompt 74, 61, 57, as two calls 85, 83, 72.
    constexpr bool kWide = std::is_same<T, float>::value || HD > 128;
    if (rows < (kWide ? 1024u : std::is_same<T, __half>::value ? 192u : 96u)) {
        launch<T, HD, true, 1>(ctx, p);
    } else if constexpr (kWide) {
        launch<T, HD, false, 1>(ctx, p);
    } else if constexpr (std::is_same<T, __half>::value) {
        launch<T, HD, false, 2>(ctx, p);
    } else {
        launch_kv_attention_tc(ctx, HD, p);
    }
}

}  // namespace

size_t kv_attention_counters(const csdr_context* ctx) { return static_cast<size_t>(ctx->sm_count) * 4u; }
size_t kv_attention_workspace(const csdr_context* ctx, uint32_t head_dim) {
    // two pieces of a tile of at most 64 rows (32 for the widest heads) a CTA, at most four CTAs an SM; or 128 rows and two CTAs
    return kv_attention_counters(ctx) * (4u + 2u * (head_dim > 128u ? 32u : 64u) * (head_dim + 4u) * 4u);
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
    p.spin = ctx->operator_spin();
    const size_t es = dtype == CSDR_DTYPE_F32 ? 4 : 2;
    p.vec = (reinterpret_cast<uintptr_t>(a.q) | a.q_stride * es) % 16u == 0;
    p.vec_out = (reinterpret_cast<uintptr_t>(a.out) | a.out_stride * es) % 16u == 0;
    const uint64_t all_rows = static_cast<uint64_t>(b.n_tokens) * p.group, rows = all_rows / b.n_seqs;
    if (all_rows > 0xFFFFFF00u) throw Error(CSDR_ERR_LIMIT, "attention: more query rows of a kv head than 2^32");
    LaunchScope ls(ctx, KC_KV_ATTENTION);
    with_dtype(dtype, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        if (head_dim == 64) launch_rows<T, 64>(ctx, rows, p);
        else if (head_dim == 128) launch_rows<T, 128>(ctx, rows, p);
        else launch_rows<T, 256>(ctx, rows, p);
    });
    ls.done("kv_attention_kernel");
}

}  // namespace csdr
