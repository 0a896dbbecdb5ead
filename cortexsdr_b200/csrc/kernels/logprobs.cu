// Log probabilities of given tokens, the entropy and the top alternatives of rows of logits:
//   M = max x, S = sum exp(x - M):  logprob(i) = x_i - M - log S,  entropy = log S - sum exp(x - M) (x - M) / S
// The alternatives are ordered by logit, equal ones by index. A row whose softmax is not defined (a NaN or
// +infinity among the logits, or nothing above -infinity) answers NaN, and -1 for the ids.
//
// One pass over the logits. A thread keeps the maximum, the sum and the weighted sum of what it has seen, scaled anew
// when the maximum grows. A logit may be among the alternatives only if it reaches a bound that the k-th best cannot be below:
// the least, over the CTA's W warps, of the ceil(k / W)-th greatest of the lanes' maxima so far, taken after the first
// round and whenever the logits seen have doubled. What reaches it is put aside, some hundred pieces of a row,
// and ranked at the end (2048 rows of 151936 in bf16: 101 us without alternatives, 132 with 20, 156 with lists kept in order on the
// way; in a long run of calls 140 to 146, where the power cap holds the clock at 1.87 GHz). A row where more do than there is room
// for (rising order) is read again with the bound it ended with, into sorted lists. Keys are (logit, index), so results do not depend
// on who comes first. Few rows are cut over the CTAs of a cluster, whose leader joins them. What bounds it: the logits' bytes, and
// behind them the exponentials (one a logit, sixteen a clock and SM: 0.7 of the memory's time for 16-bit logits).
#include <cooperative_groups.h>

#include <algorithm>
#include <cfloat>

#include "codes4.cuh"
#include "logprobs.hpp"
#include "op_common.cuh"

namespace cg = cooperative_groups;

namespace csdr {

namespace {

constexpr uint32_t kRound = 4;     // 128-bit loads a thread has under way
typedef unsigned long long u64;

// Orders as the logits do; above zero for every logit.
__device__ __forceinline__ uint32_t order_of(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);   // -0 counts as 0
    return b ^ (static_cast<uint32_t>(static_cast<int32_t>(b) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float logit_of(uint32_t order) {
    return __uint_as_float(order & 0x80000000u ? order ^ 0x80000000u : ~order);
}
// Equal logits: the lower index is the greater key.
__device__ __forceinline__ u64 key_of(float x, uint32_t i) { return static_cast<u64>(order_of(x)) << 32 | (0xFFFFFFFFu - i); }

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
constexpr float kLog2e = 1.4426950408889634f;

// Maximum, sum of p = exp(x - maximum), sum of p log2 p.
struct Sums {
    float m = -FLT_MAX, s = 0.0f, e = 0.0f;
    __device__ __forceinline__ void raise(float top) {
        const float d = fmaxf((m - top) * kLog2e, -1000.0f), f = ex2(d);      // an empty sum has no distance
        e = f * fmaf(d, s, e);
        s *= f;
        m = top;
    }
    // Of the warp's lanes together, in every lane.
    __device__ __forceinline__ void over_lanes() {
        raise(logit_of(__reduce_max_sync(0xFFFFFFFFu, order_of(m))));
#pragma unroll
        for (uint32_t o = 16; o; o >>= 1) {
            s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
            e += __shfl_xor_sync(0xFFFFFFFFu, e, o);
        }
    }
    // One logit, not above the maximum. (x - m is exact near the maximum; products with log2 e are not)
    __device__ __forceinline__ void one(float x) {
        const float d = (x - m) * kLog2e, p = ex2(d);
        s += p;
        e = fmaf(p, fmaxf(d, -1000.0f), e);
    }
};

// A 128-bit piece: pairs of logits, and the greatest.
template <typename T>
struct Vec;
template <>
struct Vec<float> {
    static constexpr uint32_t N = 4;
    uint4 w;
    __device__ __forceinline__ float2 pair(uint32_t i) const {
        return i ? make_float2(__uint_as_float(w.z), __uint_as_float(w.w)) : make_float2(__uint_as_float(w.x), __uint_as_float(w.y));
    }
    __device__ __forceinline__ float top() const {
        return fmaxf(fmaxf(__uint_as_float(w.x), __uint_as_float(w.y)), fmaxf(__uint_as_float(w.z), __uint_as_float(w.w)));
    }
};
__device__ __forceinline__ uint32_t word_of(const uint4& w, uint32_t i) { return i == 0u ? w.x : i == 1u ? w.y : i == 2u ? w.z : w.w; }
template <>
struct Vec<__nv_bfloat16> {
    static constexpr uint32_t N = 8;
    uint4 w;
    __device__ __forceinline__ float2 pair(uint32_t i) const {
        const uint32_t p = word_of(w, i);
        return make_float2(__uint_as_float(p << 16), __uint_as_float(p & 0xFFFF0000u));
    }
    __device__ __forceinline__ float top() const {
        auto h = [&](uint32_t i) { const uint32_t p = word_of(w, i); return *reinterpret_cast<const __nv_bfloat162*>(&p); };
        const __nv_bfloat162 m = __hmax2(__hmax2(h(0), h(1)), __hmax2(h(2), h(3)));
        return fmaxf(__low2float(m), __high2float(m));
    }
};
template <>
struct Vec<__half> {
    static constexpr uint32_t N = 8;
    uint4 w;
    __device__ __forceinline__ float2 pair(uint32_t i) const {
        const uint32_t p = word_of(w, i);
        return __half22float2(*reinterpret_cast<const __half2*>(&p));
    }
    __device__ __forceinline__ float top() const {
        auto h = [&](uint32_t i) { const uint32_t p = word_of(w, i); return *reinterpret_cast<const __half2*>(&p); };
        const __half2 m = __hmax2(__hmax2(h(0), h(1)), __hmax2(h(2), h(3)));
        return fmaxf(__low2float(m), __high2float(m));
    }
};

// The warp's list: lane i has the i-th greatest key, zero where there is none.
__device__ __forceinline__ void insert(u64& list, u64 key, uint32_t lane) {
    const uint32_t at = __popc(__ballot_sync(0xFFFFFFFFu, list > key));
    const u64 before = __shfl_up_sync(0xFFFFFFFFu, list, 1);
    list = lane < at ? list : lane == at ? key : before;
}

// The j-th greatest (from 0) of the lanes' values.
__device__ __forceinline__ uint32_t nth_greatest(uint32_t v, uint32_t j) {
    uint32_t top = 0;
#pragma unroll 1
    for (uint32_t i = 0; i <= j; ++i) {
        top = __reduce_max_sync(0xFFFFFFFFu, v);
        const uint32_t who = __ffs(__ballot_sync(0xFFFFFFFFu, v == top)) - 1u;      // one of equal ones
        if ((threadIdx.x & 31u) == who) v = 0u;
    }
    return top;
}

constexpr uint32_t kAside = 640, kMostKeys = 16 * kMaxTop;
template <uint32_t kWarps>
struct Shared {
    Sums sums[kWarps];
    Sums joined;                 // of this CTA
    uint32_t bound[kWarps];      // each warp's: an order that so many of its logits reach
    uint4 piece[kAside];         // pieces with a logit that reached the bound, and which ones
    uint32_t aside[kAside];
    u64 keys[kMostKeys];         // logits that reach the last bound; in a second reading, the warps' lists
    u64 best[kMaxTop];           // of this CTA; the leader's: of the row
    Sums parts[8];               // the leader's: of every CTA of the cluster
    u64 offered[8 * kMaxTop];
    uint32_t n_aside, n_keys;
};

// The best k of n keys in `from`, in order: a key's place is the number of greater ones (keys differ, but for zeros, which
// stand for none). Not inlined: what runs once a row is mostly waiting for its own instructions.
template <uint32_t kThreads>
__device__ __noinline__ void best_of(const u64* from, uint32_t n, u64* to, uint32_t k) {
    // four lanes a key; a warp's lanes stay together
    for (uint32_t i0 = 0; i0 < n; i0 += kThreads / 4u) {
        const uint32_t i = i0 + threadIdx.x / 4u;
        const u64 key = i < n ? from[i] : 0u;
        uint32_t at = 0;
#pragma unroll 8
        for (uint32_t j = threadIdx.x & 3u; j < n; j += 4u) at += from[j] > key;
        at += __shfl_xor_sync(0xFFFFFFFFu, at, 1);
        at += __shfl_xor_sync(0xFFFFFFFFu, at, 2);
        if (!(threadIdx.x & 3u) && at < k && key) to[at] = key;
    }
}

template <typename T, bool TOP, uint32_t kThreads>
__global__ void __launch_bounds__(kThreads, 1024 / kThreads)
logprob_kernel(LogprobArgs a) {
    constexpr uint32_t kWarps = kThreads / 32;
    __shared__ Shared<kWarps> sh;
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t ranks = cluster.num_blocks(), rank = cluster.block_rank();
    const uint32_t row = blockIdx.x / ranks, tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5;
    if (threadIdx.x == 0) sh.n_aside = sh.n_keys = 0;
    if (TOP && threadIdx.x < kMaxTop) sh.best[threadIdx.x] = 0;
    // what the others write into the leader's shared memory needs it to be there
    if (ranks > 1u) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    op_enter();
    const T* x = static_cast<const T*>(a.logits) + row * a.stride;
    constexpr uint32_t N = Vec<T>::N;
    // elements in front of the first 16-byte boundary, 128-bit pieces, elements behind the last
    const uint32_t head = min(a.vocab, static_cast<uint32_t>((16u - (reinterpret_cast<uintptr_t>(x) & 15u)) & 15u) / static_cast<uint32_t>(sizeof(T)));
    const uint32_t n_vec = (a.vocab - head) / N, per = (n_vec + ranks - 1u) / ranks;
    const uint32_t v0 = min(rank * per, n_vec), v1 = min(v0 + per, n_vec), tail = head + n_vec * N;
    const uint4* vec = reinterpret_cast<const uint4*>(x + head);

    Sums mine;
    u64 list = 0;
    const uint32_t k = a.top, share = TOP ? (k + kWarps - 1u) / kWarps : 0u;       // a warp's part of a bound
    uint32_t bound = 0;          // as an order; what does not reach it is no alternative
    float reach = -INFINITY;     // the same as a logit
    auto consider = [&](float v, uint32_t i, bool there) {
        uint32_t who = __ballot_sync(0xFFFFFFFFu, there && !(v < reach));
        while (who) {
            const uint32_t from = __ffs(who) - 1u;
            who &= who - 1u;
            const u64 key = __shfl_sync(0xFFFFFFFFu, key_of(v, i), from);
            if (key > __shfl_sync(0xFFFFFFFFu, list, k - 1u)) insert(list, key, lane);
        }
    };
    auto new_bound = [&]() {
        // lanes read the warps' bounds; those that are stale are lower, which only lets more through
        const uint32_t b = lane < kWarps ? *reinterpret_cast<volatile uint32_t*>(&sh.bound[lane]) : 0xFFFFFFFFu;
        bound = max(bound, __reduce_min_sync(0xFFFFFFFFu, b));
        reach = bound ? logit_of(bound) : -INFINITY;
    };
    Vec<T> w[kRound], ahead[kRound];
    // The pieces of the lanes in `who`, one lane's after the other: its logits spread over the lanes.
    auto consider_pieces = [&](uint32_t who, const Vec<T>& v, uint32_t i) {
        while (who) {
            const uint32_t from = __ffs(who) - 1u;
            who &= who - 1u;
            Vec<T> one;
            one.w.x = __shfl_sync(0xFFFFFFFFu, v.w.x, from);
            one.w.y = __shfl_sync(0xFFFFFFFFu, v.w.y, from);
            one.w.z = __shfl_sync(0xFFFFFFFFu, v.w.z, from);
            one.w.w = __shfl_sync(0xFFFFFFFFu, v.w.w, from);
            const uint32_t at = head + __shfl_sync(0xFFFFFFFFu, i, from) * N + lane;
            const uint32_t pr = lane / 2u % (N / 2u);
            const float2 f = pr < 2u ? (pr & 1u ? one.pair(1) : one.pair(0)) : (pr & 1u ? one.pair(N / 2u - 1u) : one.pair(N / 2u - 2u));
            consider(lane & 1u ? f.y : f.x, at, lane < N);
        }
    };
    auto fetch = [&](uint32_t base) {
#pragma unroll
        for (uint32_t j = 0; j < kRound; ++j) {
            const uint32_t i = base + j * kThreads + tid;
            if (i < v1) ahead[j].w = __ldcs(vec + i);
        }
    };
    fetch(v0);
    bool first = true, fresh = true;
    uint32_t round = 1;
    float lane_top = -INFINITY;
    // so many lanes of the warp have a logit of at least its bound
    auto publish = [&]() {
        const uint32_t b = nth_greatest(order_of(lane_top), share - 1u);
        if (lane == 0) *reinterpret_cast<volatile uint32_t*>(&sh.bound[warp]) = b;
    };
    auto put_aside = [&](const Vec<T>& v, uint32_t piece) {
        const uint32_t at = atomicAdd(&sh.n_aside, 1u);
        if (at < kAside) {
            sh.aside[at] = piece;
            sh.piece[at] = v.w;
        }
    };
    for (uint32_t base = v0; base < v1 || first; base += kThreads * kRound) {
        float top[kRound], most_there = -INFINITY;
#pragma unroll
        for (uint32_t j = 0; j < kRound; ++j) {
            w[j] = ahead[j];
            top[j] = base + j * kThreads + tid < v1 ? w[j].top() : -INFINITY;
            most_there = fmaxf(most_there, top[j]);
        }
        const float most = fmaxf(most_there, -FLT_MAX);
        if (base + kThreads * kRound < v1) fetch(base + kThreads * kRound);
        if (TOP) {
            lane_top = fmaxf(lane_top, most_there);
            if (first) {
                publish();
                __syncthreads();
            }
            if (fresh) new_bound();
            fresh = first;
            if ((round & (round - 1u)) == 0u) {
                if (!first) publish();
                fresh = true;
            }
            ++round;
        }
        if (most > mine.m) mine.raise(most);
        const f32x2 less = pack2(-mine.m, -mine.m), log2e = pack2(kLog2e, kLog2e);
        f32x2 s2 = pack2(0.0f, 0.0f), e2 = s2;
#pragma unroll
        for (uint32_t j = 0; j < kRound; ++j) {
            if (base + j * kThreads + tid >= v1) break;
#pragma unroll
            for (uint32_t i = 0; i < Vec<T>::N / 2u; ++i) {
                const float2 v = w[j].pair(i);
                const f32x2 d = mul2(add2(pack2(v.x, v.y), less), log2e);
                const float2 y = unpack2(d);
                const f32x2 q = pack2(ex2(y.x), ex2(y.y));
                s2 = add2(s2, q);
                e2 = fma2(q, d, e2);
            }
        }
        {
            const float2 sv = unpack2(s2), ev = unpack2(e2);
            float e = ev.x + ev.y;
            if (e != e) {        // a -infinity, which counts as nothing (or a NaN, which the sum has too)
                e = 0.0f;
#pragma unroll
                for (uint32_t j = 0; j < kRound; ++j) {
                    if (base + j * kThreads + tid >= v1) break;
#pragma unroll
                    for (uint32_t i = 0; i < Vec<T>::N / 2u; ++i) {
                        const float2 v = w[j].pair(i);
                        const float dx = fmaxf((v.x - mine.m) * kLog2e, -1000.0f), dy = fmaxf((v.y - mine.m) * kLog2e, -1000.0f);
                        e = fmaf(ex2(dx), dx, fmaf(ex2(dy), dy, e));
                    }
                }
            }
            mine.s += sv.x + sv.y;
            mine.e += e;
        }
        if (TOP) {
#pragma unroll
            for (uint32_t j = 0; j < kRound; ++j) {
                const uint32_t i = base + j * kThreads + tid;
                if (i < v1 && !(top[j] < reach)) put_aside(w[j], i);
            }
        }
        first = false;
    }
    // what does not fill a piece
    if (rank == ranks - 1u && warp == 0) {
        const uint32_t loose = head + (a.vocab - tail);      // less than 2 N: at most one a lane
        const uint32_t i = lane < head ? lane : tail + lane - head;
        const bool there = lane < loose;
        const float v = there ? op_widen(x[i]) : 0.0f;
        if (there) {
            if (v > mine.m) mine.raise(v);
            mine.one(v);
        }
    }
    if (TOP) publish();
    // ---- the CTA's sums and best ----
    mine.over_lanes();
    if (lane == 0) sh.sums[warp] = mine;
    __syncthreads();
    if (warp == 0) {
        Sums all;
        if (lane < kWarps) all = sh.sums[lane];
        all.over_lanes();
        if (lane == 0) sh.joined = all;
    }
    auto rank_keys = [&](const u64* from, uint32_t n, u64* to) { best_of<kThreads>(from, n, to, k); };
    if (TOP) {
        new_bound();
        const uint32_t n = sh.n_aside;
        auto offer = [&](float v, uint32_t i) {
            if (v < reach) return;
            const uint32_t at = atomicAdd(&sh.n_keys, 1u);
            if (at < kMostKeys) sh.keys[at] = key_of(v, i);
        };
        const uint32_t loose = rank == ranks - 1u ? head + (a.vocab - tail) : 0u;
        if (n <= kAside) {
#pragma unroll 1
            for (uint32_t e = tid; e < n * N; e += kThreads) {
                offer(op_widen(reinterpret_cast<const T*>(sh.piece)[e]), head + sh.aside[e / N] * N + e % N);
            }
            if (tid < loose) {
                const uint32_t i = tid < head ? tid : tail + tid - head;
                offer(op_widen(x[i]), i);
            }
            __syncthreads();
        }
        if (n > kAside || sh.n_keys > kMostKeys) {      // again, each warp into a list
            __syncthreads();
            if (tid == 0) sh.n_keys = 0;
            __syncthreads();
#pragma unroll 1
            for (uint32_t base = v0; base < v1; base += kThreads) {
                const uint32_t i = base + tid;
                Vec<T> v;
                v.w = make_uint4(0u, 0u, 0u, 0u);
                if (i < v1) v.w = vec[i];
                // a full list takes what is greater: an equal logit has the higher index
                const u64 least = __shfl_sync(0xFFFFFFFFu, list, k - 1u);
                const bool enters = least ? v.top() > logit_of(static_cast<uint32_t>(least >> 32)) : !(v.top() < reach);
                const uint32_t who = __ballot_sync(0xFFFFFFFFu, i < v1 && enters);
                if (who) consider_pieces(who, v, i);
            }
            if (warp == 0 && loose) {
                const uint32_t i = lane < head ? lane : tail + lane - head;
                consider(lane < loose ? op_widen(x[i]) : 0.0f, i, lane < loose);
            }
            if (lane < k && list != 0u) sh.keys[atomicAdd(&sh.n_keys, 1u)] = list;
        }
        __syncthreads();
        rank_keys(sh.keys, sh.n_keys, sh.best);
    }
    if (ranks > 1u) {
        asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
        __syncthreads();
        if (tid == 0) *cluster.map_shared_rank(&sh.parts[rank], 0) = sh.joined;
        if (TOP && tid < k) cluster.map_shared_rank(sh.offered, 0)[rank * k + tid] = sh.best[tid];
        cluster.sync();
    } else {
        __syncthreads();
    }
    if (rank == 0) {
        Sums all = sh.joined;
        if (ranks > 1u) {
            all = Sums{};
            if (lane < ranks) all = sh.parts[lane];
            all.over_lanes();
            if (TOP) {
                rank_keys(sh.offered, ranks * k, sh.best);
                __syncthreads();
            }
        }
        const bool fine = all.s > 0.0f;      // a NaN is not
        const float ls = logf(all.s);
        if (tid == 0) {
            if (a.logprob) {
                const int32_t t = a.targets[row];
                a.logprob[row] = fine && t >= 0 && static_cast<uint32_t>(t) < a.vocab ? op_widen(x[t]) - all.m - ls : NAN;
            }
            if (a.entropy) a.entropy[row] = fine ? ls - all.e / all.s * 0.6931471805599453f : NAN;
        }
        if (TOP && tid < k) {
            const u64 key = sh.best[tid];
            const size_t at = static_cast<size_t>(row) * k + tid;
            a.top_ids[at] = fine ? static_cast<int32_t>(0xFFFFFFFFu - static_cast<uint32_t>(key)) : -1;
            a.top_logprobs[at] = fine ? logit_of(static_cast<uint32_t>(key >> 32)) - all.m - ls : NAN;
        }
    }
}

}  // namespace

void launch_logprobs(csdr_context* ctx, int dtype, const LogprobArgs& a) {
    LaunchScope ls(ctx, KC_LOGPROB);
    with_dtype(dtype, [&](auto* p) {
        using T = std::remove_pointer_t<decltype(p)>;
        // Few rows are cut over two, four or eight CTAs of 512 threads, while every CTA has an SM of its own; up to a row an SM in
        // two, where a part is worth a second CTA on the SM, which is eight loads a thread; more rows are not cut and go by four
        // CTAs of 256 an SM (three: 140 us instead of 133 for 2048 rows of 151936 in bf16). Rows of fp32 logits, us uncut and in
        // two, four, eight parts:
        //   of 151936   10 rows 13.4, 7.6, 5.5, 5.1;  37: 13.6, 7.7, 7.7, 8.0;  74: 27, 11, 13, 15;  148: 29.5, 16.9, 23, 26;
        //               296: 35, 32, 39, 50;  592: 55, 62, 71, 93 (bf16, 20 alternatives: 148 rows 22, 19, 30, 46; 296: 28, 35, 52, 84)
        //   of 32000    10 rows 4.6, 4.3, 3.6, 3.7;  74: 4.9, 4.3, 6.2, 8.2;  148: 5.1, 5.1, 8.7, 13 (bf16, 20 alternatives: 9.1, 10.3)
        uint32_t ranks = 1;
        while (ranks < 8u && static_cast<uint64_t>(a.rows) * ranks * 2u <= static_cast<uint64_t>(ctx->sm_count) &&
               a.vocab / (ranks * 2u) >= 512u * Vec<T>::N)
            ranks *= 2u;
        if (ranks == 1u && a.rows <= static_cast<uint32_t>(ctx->sm_count) && a.vocab / 2u >= 8u * 512u * Vec<T>::N) ranks = 2;
        const dim3 grid(a.rows * ranks);
        if (ranks == 1u) {
            if (a.top) launch_op(ctx, logprob_kernel<T, true, 256>, grid, 256, 0, 1, a);
            else launch_op(ctx, logprob_kernel<T, false, 256>, grid, 256, 0, 1, a);
        } else {
            if (a.top) launch_op(ctx, logprob_kernel<T, true, 512>, grid, 512, 0, ranks, a);
            else launch_op(ctx, logprob_kernel<T, false, 512>, grid, 512, 0, ranks, a);
        }
    });
    ls.done("logprob_kernel");
}

}  // namespace csdr
