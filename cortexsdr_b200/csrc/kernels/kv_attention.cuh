// What the attention kernels over the paged 4-bit cache share: how the work is cut, and how pieces of it are joined.
#pragma once

#include <cfloat>

#include "kv_cache.hpp"
#include "op_common.cuh"

namespace csdr {

constexpr uint32_t kBlockKeys = 128;     // keys of a place in the schedule
constexpr float kSlack = 6.0f;
template <int HD>
constexpr uint32_t kPitch = HD + 4;      // of a row of outputs with its maximum and sum

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// |scale| log2 e 2^n, what a row's products are multiplied by to be exponents of two. At least a normal number (nothing that is
// smaller tells keys apart), and at most 2^most, so that no score passes fp32: there the least difference of two products decides.
__device__ __forceinline__ float factor_of(float scale, int n, int most) {
    const int first = min(n, 127);
    const float f = fabsf(scale) * __int_as_float((first + 127) << 23) * (1.4426950408889634f * __int_as_float((n - first + 127) << 23));
    return fminf(fmaxf(f, FLT_MIN), __int_as_float((most + 127) << 23));
}

struct AttnParams {
    KvView kv;
    KvBatchView b;
    KvAttend a;
    uint32_t group;          // query heads of a kv head
    uint32_t vec, vec_out;   // rows of q, of the result start on 16 bytes
    float* part;             // [CTA][2][rows][HD + 4]
    uint32_t* counters;      // [CTA]: arrivals at the unit that starts in a CTA's share and is cut
    int* status;
    uint32_t spin;
};

__device__ __forceinline__ uint64_t quotient(uint64_t a, uint64_t b) {
    return (a | b) >> 32 ? a / b : static_cast<uint32_t>(a) / static_cast<uint32_t>(b);
}

// A sequence as the schedule sees it.
struct Seq {
    int64_t base;            // position of its first new token
    int64_t cap;             // keys that its table can hold
    uint32_t row0, n_new, tiles;
    uint32_t pair_weight, mid_weight;
    // blocks of 128 keys that a tile of rows sees; at least one, so that rows that see nothing are written too
    template <uint32_t TILE>
    __device__ __forceinline__ int64_t keys(uint32_t tile, uint32_t group) const {
        // TILE (tiles + 1) fits 32 bits (launch_kv_attention)
        const uint32_t last = tile + 1u == tiles ? n_new - 1u : (TILE * (tile + 1u) - 1u) / group;
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
        tiles = (n_new * p.group + TILE - 1u) / TILE;
        pair_weight = mid_weight = 0;
        if (!tiles) return;
        if (tiles == 1u) {
            mid_weight = blocks<TILE>(0, p.group);
            return;
        }
        const uint32_t a = blocks<TILE>(0, p.group), z = blocks<TILE>(tiles - 1u, p.group);
        // rounding to blocks and the last tile's missing rows: two blocks at most
        pair_weight = tiles == 2u ? a + z : base + n_new > cap ? 2u * z : a + z + 2u;
        if (tiles & 1u) mid_weight = blocks<TILE>(tiles / 2u, p.group);
    }
    // As lane `from` of the warp has it.
    __device__ __forceinline__ Seq of_lane(uint32_t from) const {
        Seq q;
        q.base = __shfl_sync(0xFFFFFFFFu, base, from);
        q.cap = __shfl_sync(0xFFFFFFFFu, cap, from);
        q.row0 = __shfl_sync(0xFFFFFFFFu, row0, from);
        q.n_new = __shfl_sync(0xFFFFFFFFu, n_new, from);
        q.tiles = __shfl_sync(0xFFFFFFFFu, tiles, from);
        q.pair_weight = __shfl_sync(0xFFFFFFFFu, pair_weight, from);
        q.mid_weight = __shfl_sync(0xFFFFFFFFu, mid_weight, from);
        return q;
    }
    __device__ __forceinline__ uint64_t head_weight() const { return static_cast<uint64_t>(tiles / 2u) * pair_weight + mid_weight; }
};

// Joins n pieces of a row (outputs, maximum, sum), eight values of it. `get` reads four floats of a piece.
template <int HD, typename F>
__device__ __forceinline__ void join(uint32_t n, uint32_t d, F&& get, float (&o)[8], float& m, float& l) {
    m = -FLT_MAX;
    l = 0.0f;
#pragma unroll
    for (uint32_t j = 0; j < 8u; ++j) o[j] = 0.0f;
#pragma unroll 4
    for (uint32_t i = 0; i < n; ++i) m = fmaxf(m, get(i, HD).x);
#pragma unroll 4
    for (uint32_t i = 0; i < n; ++i) {
        const float4 st = get(i, HD), a = get(i, d), b = get(i, d + 4u);
        const float f = ex2(st.x - m);
        l = fmaf(f, st.y, l);
        o[0] = fmaf(f, a.x, o[0]);
        o[1] = fmaf(f, a.y, o[1]);
        o[2] = fmaf(f, a.z, o[2]);
        o[3] = fmaf(f, a.w, o[3]);
        o[4] = fmaf(f, b.x, o[4]);
        o[5] = fmaf(f, b.y, o[5]);
        o[6] = fmaf(f, b.z, o[6]);
        o[7] = fmaf(f, b.w, o[7]);
    }
}

// Eight results, as one or two 128-bit pieces where rows start on 16 bytes.
template <typename T>
__device__ __forceinline__ void store_row(T* to, const float (&v)[8], float by, bool vec) {
    Eight128<T> r;
#pragma unroll
    for (uint32_t i = 0; i < 8u; ++i) r.v[i] = op_narrow<T>(v[i] * by);
    if (vec) {
        r.store(to);
    } else {
#pragma unroll
        for (uint32_t i = 0; i < 8u; ++i) to[i] = r.v[i];
    }
}

// This CTA's share of the work, and the unit that lies at a place of it.
template <uint32_t THREADS>
struct ScheduleShared {
    uint64_t scan[THREADS / 32u], found_at;
    uint32_t found, longest, n_units;      // the last two start at zero
};
struct Unit {
    uint64_t start, next;      // its first place, where the next unit starts
    uint32_t kvh, tile, b0, b1, n_blocks;
    int32_t keys;
};
template <uint32_t TILE, uint32_t THREADS>
struct Schedule {
    uint64_t total, x0, x1, ctas;      // places x0 to x1 - 1
    uint64_t seq_at;                   // first place of sequence s
    uint32_t s;
    Seq sq;

    __device__ __forceinline__ void share(uint32_t longest_unit, uint32_t units) {
        // Joining n pieces costs a CTA about a sixteenth of a block's time each: no unit is cut finer than both together take.
        const uint64_t least_blocks = 1u + static_cast<uint32_t>(sqrtf(static_cast<float>(longest_unit) / 16.0f));
        ctas = min(static_cast<uint64_t>(gridDim.x), max(quotient(total, least_blocks), static_cast<uint64_t>(1)));
        // Units that are all as long, one a CTA, where sharing them evenly would save less than the joins cost (two blocks' time;
        // 16 sequences of 1024 with 32 heads: 39.7 -> 33.9 us)
        if (units <= gridDim.x && total == static_cast<uint64_t>(units) * longest_unit && longest_unit <= quotient(total, ctas) + 2u) {
            ctas = units;
            x0 = static_cast<uint64_t>(blockIdx.x) * longest_unit;
            x1 = x0 + longest_unit;
        } else {
            x0 = quotient(blockIdx.x * total, ctas);
            x1 = quotient((blockIdx.x + 1u) * total, ctas);
        }
    }
    static __device__ __forceinline__ uint64_t scan_up(uint64_t v, uint32_t lane) {
#pragma unroll
        for (uint32_t o = 1; o < 32u; o <<= 1) {
            const uint64_t w = __shfl_up_sync(0xFFFFFFFFu, v, o);
            if (lane >= o) v += w;
        }
        return v;
    }
    // All threads of the CTA. False: nothing for it.
    __device__ __forceinline__ bool begin(const AttnParams& p, ScheduleShared<THREADS>& sh) {
        const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5;
        if (p.b.n_seqs <= 32u) {
            // every warp for itself, a lane a sequence
            Seq q{};
            if (lane < p.b.n_seqs) q.load<TILE>(p, lane);
            const uint64_t w = q.head_weight() * p.kv.kv_heads, upto = scan_up(w, lane);
            total = __shfl_sync(0xFFFFFFFFu, upto, 31);
            if (!total) return false;
            share(__reduce_max_sync(0xFFFFFFFFu, q.tiles ? q.blocks<TILE>(q.tiles - 1u, p.group) : 0u),
                  __reduce_add_sync(0xFFFFFFFFu, q.tiles * p.kv.kv_heads));
            if (blockIdx.x >= ctas) return false;
            s = __ffs(__ballot_sync(0xFFFFFFFFu, x0 >= upto - w && x0 < upto)) - 1u;
            seq_at = __shfl_sync(0xFFFFFFFFu, upto - w, s);
            sq = q.of_lane(s);
            return true;
        }
        const uint32_t per = (p.b.n_seqs + THREADS - 1u) / THREADS;
        const uint32_t s_lo = min(tid * per, p.b.n_seqs), s_hi = min(s_lo + per, p.b.n_seqs);
        uint64_t mine = 0;
        uint32_t blocks = 0, units = 0;
        for (uint32_t i = s_lo; i < s_hi; ++i) {
            Seq q;
            q.load<TILE>(p, i);
            mine += q.head_weight() * p.kv.kv_heads;
            if (q.tiles) blocks = max(blocks, q.blocks<TILE>(q.tiles - 1u, p.group));
            units += q.tiles * p.kv.kv_heads;
        }
        atomicMax(&sh.longest, blocks);
        atomicAdd(&sh.n_units, units);
        const uint64_t upto = scan_up(mine, lane);
        if (lane == 31u) sh.scan[warp] = upto;
        __syncthreads();
        uint64_t before = 0;
        total = 0;
#pragma unroll
        for (uint32_t i = 0; i < THREADS / 32u; ++i) {
            if (i < warp) before += sh.scan[i];
            total += sh.scan[i];
        }
        if (!total) return false;
        share(sh.longest, sh.n_units);
        if (blockIdx.x >= ctas) return false;
        uint64_t at = before + upto - mine;
        if (x0 >= at && x0 < at + mine) {
            for (uint32_t i = s_lo; i < s_hi; ++i) {
                Seq q;
                q.load<TILE>(p, i);
                const uint64_t w = q.head_weight() * p.kv.kv_heads;
                if (x0 < at + w) {
                    sh.found = i;
                    sh.found_at = at;
                    break;
                }
                at += w;
            }
        }
        __syncthreads();
        s = sh.found;
        seq_at = sh.found_at;
        sq.load<TILE>(p, s);
        return true;
    }
    // The unit that holds place x, which does not fall from call to call. False: an empty place, the next unit starts at `next`.
    __device__ __forceinline__ bool at(const AttnParams& p, uint64_t x, Unit& u) {
        uint64_t w = sq.head_weight() * p.kv.kv_heads;
        while (x >= seq_at + w) {
            seq_at += w;
            sq.load<TILE>(p, ++s);
            w = sq.head_weight() * p.kv.kv_heads;
        }
        const uint64_t hw = sq.head_weight(), y = x - seq_at, pairs = static_cast<uint64_t>(sq.tiles / 2u) * sq.pair_weight;
        u.kvh = static_cast<uint32_t>(quotient(y, hw));
        const uint64_t z = y - u.kvh * hw;
        u.next = seq_at + u.kvh * hw;
        if (sq.tiles == 1u) {
            u.tile = 0u;
            u.b0 = static_cast<uint32_t>(z);
            u.next += hw;
        } else if (z < pairs) {
            const uint32_t pr = static_cast<uint32_t>(quotient(z, sq.pair_weight)), o = static_cast<uint32_t>(z - static_cast<uint64_t>(pr) * sq.pair_weight);
            const uint32_t n = sq.blocks<TILE>(pr, p.group);
            u.next += static_cast<uint64_t>(pr) * sq.pair_weight;
            u.tile = pr;
            u.b0 = o;
            if (o >= n) {
                u.tile = sq.tiles - 1u - pr;
                u.b0 = o - n;
                u.next += sq.pair_weight;
                if (u.b0 >= sq.blocks<TILE>(u.tile, p.group)) return false;    // the empty end of a pair
            } else {
                u.next += n;
            }
        } else {
            u.tile = sq.tiles / 2u;
            u.b0 = static_cast<uint32_t>(z - pairs);
            u.next += hw;
        }
        u.n_blocks = sq.blocks<TILE>(u.tile, p.group);
        u.start = x - u.b0;
        u.b1 = static_cast<uint32_t>(min(static_cast<uint64_t>(u.n_blocks), static_cast<uint64_t>(u.b0) + (x1 - x)));
        u.keys = static_cast<int32_t>(sq.keys<TILE>(u.tile, p.group));
        return true;
    }
    // CTAs whose shares a unit lies in: CTA c has place v if floor(c total / ctas) <= v < floor((c + 1) total / ctas)
    __device__ __forceinline__ uint32_t holder(uint64_t place) const { return static_cast<uint32_t>(quotient((place + 1u) * ctas - 1u, total)); }
};

// bf16, heads of 64 or 128, many query rows a sequence (kv_attention_tc.cu).
void launch_kv_attention_tc(csdr_context* ctx, uint32_t head_dim, AttnParams& p);

}  // namespace csdr
