// Log probabilities of given tokens, the entropy and the top alternatives of rows of logits:
//   M = max x, S = sum exp(x - M):  logprob(i) = x_i - M - log S,  entropy = log S - sum exp(x - M) (x - M) / S
// The alternatives are ordered by logit, equal ones by index. A row whose softmax is not defined (a NaN or
// +infinity among the logits, or nothing above -infinity) answers NaN, and -1 for the ids.
//
// One pass over the logits. A thread keeps the maximum, the sum and the weighted sum of what it has seen, scaled anew
// when the maximum grows. For the alternatives a warp keeps a sorted list of the best it has met, a key a lane; a logit
// is looked at only if it reaches a bound that the k-th best of the row cannot be below: the least, over the CTA's
// W warps, of the warps' ceil(k / W)-th best so far (in the first round: of the lanes' maxima, before any is in a
// list). Some hundred logits of a row reach it; a row in rising order, where all do, is slow and right.
// Keys are (logit, index), so neither lists nor results depend on who comes first. Few rows are cut over the CTAs of a
// cluster, whose leader joins them. What bounds it: the logits' bytes; exponentials and comparisons come to eight
// operations a 16-bit logit, some 0.8 of the issue slots at the memory's rate.
#include <cooperative_groups.h>

#include <algorithm>
#include <cfloat>

#include "logprobs.hpp"
#include "op_common.cuh"

namespace cg = cooperative_groups;

namespace csdr {

namespace {

constexpr uint32_t kThreads = 512, kWarps = kThreads / 32, kRound = 4;     // 128-bit loads a thread has under way
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

// Maximum, sum of exp(x - maximum), sum of exp(x - maximum) (x - maximum).
struct Sums {
    float m = -FLT_MAX, s = 0.0f, e = 0.0f;
    __device__ __forceinline__ void raise(float top) {
        const float d = fmaxf(m - top, -1000.0f), f = ex2(d * kLog2e);      // an empty sum has no distance
        e = f * fmaf(d, s, e);
        s *= f;
        m = top;
    }
    __device__ __forceinline__ void add(const Sums& o) {
        Sums b = o;
        const float top = fmaxf(m, b.m);
        raise(top);
        b.raise(top);
        s += b.s;
        e += b.e;
    }
};

template <typename T>
struct Vec {
    static constexpr uint32_t N = 16u / sizeof(T);
    uint4 w;
    __device__ __forceinline__ float operator[](uint32_t i) const;
};
template <>
__device__ __forceinline__ float Vec<float>::operator[](uint32_t i) const {
    return __uint_as_float(i == 0u ? w.x : i == 1u ? w.y : i == 2u ? w.z : w.w);
}
template <>
__device__ __forceinline__ float Vec<__nv_bfloat16>::operator[](uint32_t i) const {
    const uint32_t p = i / 2u == 0u ? w.x : i / 2u == 1u ? w.y : i / 2u == 2u ? w.z : w.w;
    return __uint_as_float(i & 1u ? p & 0xFFFF0000u : p << 16);
}
template <>
__device__ __forceinline__ float Vec<__half>::operator[](uint32_t i) const {
    const uint32_t p = i / 2u == 0u ? w.x : i / 2u == 1u ? w.y : i / 2u == 2u ? w.z : w.w;
    return __half2float(__ushort_as_half(static_cast<unsigned short>(i & 1u ? p >> 16 : p)));
}

// The warp's list: lane i has the i-th greatest key, zero where there is none.
__device__ __forceinline__ void insert(u64& list, u64 key, uint32_t lane) {
    const uint32_t at = __popc(__ballot_sync(0xFFFFFFFFu, list > key));
    const u64 before = __shfl_up_sync(0xFFFFFFFFu, list, 1);
    list = lane < at ? list : lane == at ? key : before;
}

// The j-th greatest (from 0) of the lanes' values.
__device__ __forceinline__ uint32_t nth_greatest(uint32_t v, uint32_t j) {
    uint32_t top = 0;
    for (uint32_t i = 0; i <= j; ++i) {
        top = __reduce_max_sync(0xFFFFFFFFu, v);
        const uint32_t who = __ffs(__ballot_sync(0xFFFFFFFFu, v == top)) - 1u;      // one of equal ones
        if ((threadIdx.x & 31u) == who) v = 0u;
    }
    return top;
}

struct Shared {
    Sums sums[kWarps];
    Sums joined;                 // of this CTA
    uint32_t bound[kWarps];      // each warp's: an order that so many of its logits reach
    u64 keys[kWarps * kMaxTop];
    u64 best[kMaxTop];           // of this CTA
    uint32_t count;
};

template <typename T, bool TOP>
__global__ void __launch_bounds__(kThreads, 2)
logprob_kernel(LogprobArgs a) {
    __shared__ Shared sh;
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t ranks = cluster.num_blocks(), rank = cluster.block_rank();
    const uint32_t row = blockIdx.x / ranks, tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5;
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
    bool first = true;
    for (uint32_t base = v0; base < v1 || first; base += kThreads * kRound) {
        Vec<T> w[kRound];
        float top[kRound], most = -FLT_MAX;
#pragma unroll
        for (uint32_t j = 0; j < kRound; ++j) {
            const uint32_t i = base + j * kThreads + tid;
            if (i < v1) w[j].w = __ldcs(vec + i);
        }
#pragma unroll
        for (uint32_t j = 0; j < kRound; ++j) {
            top[j] = -INFINITY;
            if (base + j * kThreads + tid < v1) {
#pragma unroll
                for (uint32_t e = 0; e < N; ++e) top[j] = fmaxf(top[j], w[j][e]);
            }
            most = fmaxf(most, top[j]);
        }
        if (TOP) {
            if (first) {
                // so many lanes have a logit of at least this
                const uint32_t b = nth_greatest(order_of(fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]))), share - 1u);
                if (lane == 0) sh.bound[warp] = b;
                __syncthreads();
            }
            new_bound();
        }
        if (most > mine.m) mine.raise(most);
        const float m = mine.m;
#pragma unroll
        for (uint32_t j = 0; j < kRound; ++j) {
            const uint32_t i = base + j * kThreads + tid;
            const bool there = i < v1;
            if (there) {
#pragma unroll
                for (uint32_t e = 0; e < N; ++e) {
                    const float d = w[j][e] - m, p = ex2(d * kLog2e);
                    mine.s += p;
                    mine.e = fmaf(p, fmaxf(d, -1000.0f), mine.e);     // exp(-infinity) counts as nothing
                }
            }
            if (TOP && __any_sync(0xFFFFFFFFu, there && !(top[j] < reach))) {
#pragma unroll
                for (uint32_t e = 0; e < N; ++e) consider(w[j][e], head + i * N + e, there);
            }
        }
        if (TOP) {
            const uint32_t b = static_cast<uint32_t>(__shfl_sync(0xFFFFFFFFu, list, share - 1u) >> 32);
            if (lane == 0 && b > sh.bound[warp]) sh.bound[warp] = b;
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
            const float d = v - mine.m, p = ex2(d * kLog2e);
            mine.s += p;
            mine.e = fmaf(p, fmaxf(d, -1000.0f), mine.e);
        }
        if (TOP) consider(v, i, there);
    }
    // ---- the CTA's sums and best ----
#pragma unroll
    for (uint32_t o = 16; o; o >>= 1) {
        Sums b;
        b.m = __shfl_xor_sync(0xFFFFFFFFu, mine.m, o);
        b.s = __shfl_xor_sync(0xFFFFFFFFu, mine.s, o);
        b.e = __shfl_xor_sync(0xFFFFFFFFu, mine.e, o);
        mine.add(b);
    }
    if (lane == 0) sh.sums[warp] = mine;
    if (tid == 0) sh.count = 0;
    __syncthreads();
    if (tid == 0) {
        Sums all = sh.sums[0];
        for (uint32_t i = 1; i < kWarps; ++i) all.add(sh.sums[i]);
        sh.joined = all;
    }
    // The best of n keys in `from`, in order: a key's place is the number of greater ones (keys differ).
    auto rank_keys = [&](const u64* from, uint32_t n, u64* to) {
        for (uint32_t i = tid; i < n; i += kThreads) {
            const u64 key = from[i];
            uint32_t at = 0;
            for (uint32_t j = 0; j < n && at < k; ++j) at += from[j] > key;
            if (at < k) to[at] = key;
        }
    };
    if (TOP) {
        new_bound();
        const bool keep = lane < k && list != 0u && static_cast<uint32_t>(list >> 32) >= bound;
        const uint32_t who = __ballot_sync(0xFFFFFFFFu, keep);
        uint32_t at = 0;
        if (lane == 0 && who) at = atomicAdd(&sh.count, __popc(who));
        at = __shfl_sync(0xFFFFFFFFu, at, 0);
        if (keep) sh.keys[at + __popc(who & ((1u << lane) - 1u))] = list;
        if (tid < kMaxTop) sh.best[tid] = 0;
        __syncthreads();
        rank_keys(sh.keys, sh.count, sh.best);
    }
    if (ranks > 1u) cluster.sync();
    else __syncthreads();
    if (rank == 0) {
        Sums all = sh.joined;
        if (ranks > 1u) {
            for (uint32_t r = 1; r < ranks; ++r) all.add(*cluster.map_shared_rank(&sh.joined, r));
            if (TOP) {
                for (uint32_t i = tid; i < ranks * k; i += kThreads) sh.keys[i] = cluster.map_shared_rank(sh.best, i / k)[i % k];
                __syncthreads();
                // a CTA with fewer than k logits leaves zeros, which rank behind every key
                rank_keys(sh.keys, ranks * k, sh.best);
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
            if (a.entropy) a.entropy[row] = fine ? ls - all.e / all.s : NAN;
        }
        if (TOP && tid < k) {
            const u64 key = sh.best[tid];
            const size_t at = static_cast<size_t>(row) * k + tid;
            a.top_ids[at] = fine ? static_cast<int32_t>(0xFFFFFFFFu - static_cast<uint32_t>(key)) : -1;
            a.top_logprobs[at] = fine ? logit_of(static_cast<uint32_t>(key >> 32)) - all.m - ls : NAN;
        }
    }
    if (ranks > 1u) cluster.sync();      // the leader may still read this CTA's shared memory
}

}  // namespace

void launch_logprobs(csdr_context* ctx, int dtype, const LogprobArgs& a) {
    LaunchScope ls(ctx, KC_LOGPROB);
    with_dtype(dtype, [&](auto* p) {
        using T = std::remove_pointer_t<decltype(p)>;
        // two CTAs an SM; a row is cut while that leaves some idle and its parts are longer than a round
        uint32_t ranks = 1;
        while (ranks < 8u && static_cast<uint64_t>(a.rows) * ranks * 2u <= static_cast<uint64_t>(ctx->sm_count) * 2u &&
               a.vocab / (ranks * 2u) >= kThreads * Vec<T>::N)
            ranks *= 2u;
        const dim3 grid(a.rows * ranks);
        if (a.top) launch_op(ctx, logprob_kernel<T, true>, grid, kThreads, 0, ranks, a);
        else launch_op(ctx, logprob_kernel<T, false>, grid, kThreads, 0, ranks, a);
    });
    ls.done("logprob_kernel");
}

}  // namespace csdr
