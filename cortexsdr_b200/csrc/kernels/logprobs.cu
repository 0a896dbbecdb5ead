// Log probabilities of given tokens, the entropy and the top alternatives of rows of logits:
//   M = max x, S = sum exp(x - M):  logprob(i) = x_i - M - log S,  entropy = log S - sum exp(x - M) (x - M) / S
// The alternatives are ordered by logit, equal ones by index. A row whose softmax is not defined (a NaN or
// +infinity among the logits, or nothing above -infinity) answers NaN, and -1 for the ids.
#include <cfloat>

#include "logprobs.hpp"
#include "op_common.cuh"

namespace csdr {

namespace {

constexpr uint32_t kThreads = 256;

// Orders as the logits do, equal logits by index, lowest first; above zero for every logit.
__device__ __forceinline__ unsigned long long key_of(float x, uint32_t i) {
    const uint32_t b = __float_as_uint(x + 0.0f);   // -0 counts as 0
    const uint32_t o = b ^ (static_cast<uint32_t>(static_cast<int32_t>(b) >> 31) | 0x80000000u);
    return static_cast<unsigned long long>(o) << 32 | (0xFFFFFFFFu - i);
}

template <typename R>
__device__ __forceinline__ R block_reduce(R v, R* buf, R (*op)(R, R)) {
    buf[threadIdx.x] = v;
    __syncthreads();
    for (uint32_t o = kThreads / 2; o; o >>= 1) {
        if (threadIdx.x < o) buf[threadIdx.x] = op(buf[threadIdx.x], buf[threadIdx.x + o]);
        __syncthreads();
    }
    v = buf[0];
    __syncthreads();
    return v;
}
__device__ float max_of(float a, float b) { return fmaxf(a, b); }
__device__ float sum_of(float a, float b) { return a + b; }
__device__ unsigned long long key_max(unsigned long long a, unsigned long long b) { return a > b ? a : b; }

template <typename T>
__global__ void __launch_bounds__(kThreads)
logprob_kernel(LogprobArgs a) {
    op_enter();
    __shared__ float fbuf[kThreads];
    __shared__ unsigned long long kbuf[kThreads];
    const uint32_t row = blockIdx.x;
    const T* x = static_cast<const T*>(a.logits) + row * a.stride;
    float m = -FLT_MAX;
    for (uint32_t i = threadIdx.x; i < a.vocab; i += kThreads) m = fmaxf(m, op_widen(x[i]));
    m = block_reduce(m, fbuf, max_of);
    float s = 0.0f, e = 0.0f;
    for (uint32_t i = threadIdx.x; i < a.vocab; i += kThreads) {
        const float d = op_widen(x[i]) - m, p = expf(d);
        s += p;
        e = fmaf(p, fmaxf(d, -1000.0f), e);
    }
    s = block_reduce(s, fbuf, sum_of);
    e = block_reduce(e, fbuf, sum_of);
    const bool fine = s > 0.0f;      // a NaN is not
    const float ls = logf(s);
    if (threadIdx.x == 0) {
        if (a.logprob) {
            const int32_t t = a.targets[row];
            a.logprob[row] = fine && t >= 0 && static_cast<uint32_t>(t) < a.vocab ? op_widen(x[t]) - m - ls : NAN;
        }
        if (a.entropy) a.entropy[row] = fine ? ls - e / s : NAN;
    }
    unsigned long long last = ~0ull;
    for (uint32_t k = 0; k < a.top; ++k) {
        unsigned long long best = 0;
        for (uint32_t i = threadIdx.x; i < a.vocab; i += kThreads) {
            const unsigned long long key = key_of(op_widen(x[i]), i);
            if (key < last && key > best) best = key;
        }
        last = block_reduce(best, kbuf, key_max);
        if (threadIdx.x == 0) {
            const uint32_t i = 0xFFFFFFFFu - static_cast<uint32_t>(last);
            a.top_ids[static_cast<size_t>(row) * a.top + k] = fine ? static_cast<int32_t>(i) : -1;
            a.top_logprobs[static_cast<size_t>(row) * a.top + k] = fine ? op_widen(x[i]) - m - ls : NAN;
        }
    }
}

}  // namespace

void launch_logprobs(csdr_context* ctx, int dtype, const LogprobArgs& a) {
    LaunchScope ls(ctx, KC_LOGPROB);
    with_dtype(dtype, [&](auto* p) {
        using T = std::remove_pointer_t<decltype(p)>;
        launch_op(ctx, logprob_kernel<T>, dim3(a.rows), kThreads, 0, 1, a);
    });
    ls.done("logprob_kernel");
}

}  // namespace csdr
