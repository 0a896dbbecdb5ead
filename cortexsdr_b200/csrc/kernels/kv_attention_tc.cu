// Causal grouped-query attention over the paged 4-bit cache for prompts of bf16 rows: 128 query rows at a time against
// blocks of 64 keys, both products on tcgen05.
//
// Codes are widened to fp16 values minimum + step * code, one rounding (2^-11 of the value, at most 65504), once for 128 rows
// (kv_attention.cu, which keeps the codes as they are, widens them for sixteen). Query rows are scaled by a power of two to
// fp16's range (exactly); weights round to fp16, relative to the row's largest; scores, sums and outputs are fp32.
//
// Four warps have a row a thread: scores out of TMEM, the running maximum and sum, weights into shared memory. Four widen the
// next block meanwhile, and one of them issues the products: a block's scores before the outputs of the one in front of it, so
// that the matrix unit does not wait for the exponentials (a warp of its own for that would leave every thread 96 registers
// instead of 128). Two CTAs an SM fill what is left. Work is cut as there (kv_attention.cuh).
//
// 3 sequences of up to 2048 with 512 new tokens, 32 query heads over 8 of 128: 114 us, 332 TFLOP/s (by warps 245 us). The products
// are 42 of it (one of 64 columns takes 75 cycles, of 128 columns 121: 1080 a block); a warp widens its part of a block in 1400
// cycles and has a row's weights in 960. A block passes through the three one after the other, and two CTAs overlap them only
// in part: a CTA has a block every 7200 cycles (31 blocks each at 1.965 GHz), of which these are 3440. The rest are the waits
// between the roles, and what 128 registers a thread do not hold (heads of 128: 560 bytes of spills, 640 of reloads). Tried and
// slower: 256 rows a CTA (129 us: one CTA's phases have nobody beside them), keys published before values (122 us).
#include "codes4.cuh"
#include "kv_attention.cuh"

namespace csdr {

namespace {

constexpr uint32_t kRows = 128, kKeys = 64, kThreads = 256;      // warps 0 - 3 rows, 4 - 7 keys and values, 7 products too
constexpr uint32_t kTmemColumns = 256, kTmemOut = 2u * kKeys;    // two blocks of scores, then the outputs
constexpr uint32_t kPanel = 64;                                  // values of a 128-byte row of an operand

struct Control {
    uint64_t kv_full[2], pv_done[2], s_full[2], p_full, q_full, drained;
    uint32_t tmem, flag, failed;
    uint16_t odd[2][2][4];      // tokens whose values are NaN, a bit each: [buffer][group][block of sixteen]
    uint8_t there[2][4];        // blocks of sixteen that have a page
    ScheduleShared<kThreads> sched;
};

// Operands lie as 128-byte rows (64 values), sixteen-byte pieces exchanged within groups of eight rows (128-byte swizzle).
template <int HD>
struct Layout {
    static constexpr uint32_t kPanels = HD / kPanel;
    static constexpr uint32_t kQ = 0, kP = kPanels * kRows * 128u, kKv = kP + kRows * 128u;
    static constexpr uint32_t kOperand = kPanels * kKeys * 128u;                          // keys or values of a block
    static constexpr uint32_t kControl = kKv + 4u * kOperand, kBytes = kControl + sizeof(Control);
    static __device__ __forceinline__ uint32_t keys(uint32_t buffer) { return kKv + buffer * 2u * kOperand; }
    static __device__ __forceinline__ uint32_t values(uint32_t buffer) { return keys(buffer) + kOperand; }
};
__device__ __forceinline__ uint32_t piece_at(uint32_t row, uint32_t piece) { return row * 128u + ((piece ^ (row & 7u)) << 4); }

// Shared-memory descriptors as their two halves: groups of eight rows 1024 bytes apart; `leading` bytes to the next panel
// where rows are the reduction (values).
__device__ __forceinline__ uint32_t desc_lo(uint32_t addr, uint32_t leading) { return ((addr & 0x3FFFFu) >> 4) | (leading >> 4) << 16; }
constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);
// kind::f16: D fp32, A and B fp16, A K-major, M = 128.
__host__ __device__ constexpr uint32_t idesc(uint32_t n, bool b_rows_reduce) { return (1u << 4) | (b_rows_reduce ? 1u << 16 : 0u) | (n >> 3) << 17 | (kRows >> 4) << 24; }

// Issued by one lane, with the whole warp going along.
__device__ __forceinline__ void mma(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t id, bool accumulate, uint32_t leader) {
    asm volatile(
        "{\n"
        ".reg .pred p, q;\n"
        ".reg .b64 a, b;\n"
        "setp.ne.b32 p, %5, 0;\n"
        "setp.ne.b32 q, %6, 0;\n"
        "mov.b64 a, {%1, %4};\n"
        "mov.b64 b, {%2, %4};\n"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n"
        "}\n" ::"r"(d),
        "r"(a_lo), "r"(b_lo), "r"(id), "r"(kDescHi), "r"(static_cast<uint32_t>(accumulate)), "r"(leader)
        : "memory");
}
__device__ __forceinline__ void commit(uint32_t bar, uint32_t leader) {
    asm volatile(
        "{\n"
        ".reg .pred q;\n"
        "setp.ne.b32 q, %1, 0;\n"
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n"
        "}\n" ::"r"(bar),
        "r"(leader)
        : "memory");
}
__device__ __forceinline__ void before_sync() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void after_sync() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_loaded() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_ld32(uint32_t at, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(at)
        : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t at, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(at)
        : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t at, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(at),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}

__device__ __forceinline__ void arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
// What this warp wrote into shared memory is for the matrix unit.
__device__ __forceinline__ void publish(uint32_t bar, uint32_t lane) {
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    before_sync();
    __syncwarp();
    if (lane == 0u) arrive(bar);
}

// Eight codes of a word as four pairs of fp16 values: code n of the low half, of the high half.
__device__ __forceinline__ void values_of(uint32_t w, uint32_t steps, uint32_t minima, uint32_t (&r)[4]) {
    const uint32_t v = __byte_perm(w, 0u, 0x2301);
    // bits 6 - 9 under the exponent of 16: 16 + code
    r[0] = (w & 0x03C003C0u) | 0x4C004C00u;
    r[1] = (w << 4 & 0x03C003C0u) | 0x4C004C00u;
    r[2] = (v & 0x03C003C0u) | 0x4C004C00u;
    r[3] = (w >> 4 & 0x03C003C0u) | 0x4C004C00u;
    const __half2 s = *reinterpret_cast<const __half2*>(&steps), m = *reinterpret_cast<const __half2*>(&minima);
#pragma unroll
    for (uint32_t i = 0; i < 4u; ++i) {
        const __half2 c = __hadd2(*reinterpret_cast<const __half2*>(&r[i]), __half2half2(__ushort_as_half(0xCC00)));      // - 16
        r[i] = bits_of(__hmin2_nan(__hfma2(c, s, m), __half2half2(__ushort_as_half(0x7BFF))));
    }
}
__device__ __forceinline__ bool half_is_nan(uint32_t h) { return (h & 0x7FFFu) > 0x7C00u; }

// What a lane takes of a block of sixteen tokens, as it lies in the cache. Piece j: 16 bytes of codes.
template <int HD>
struct Raw {
    static constexpr uint32_t N = HD / 64u, G = HD / 64u;
    uint4 k[N], v[N];
    uint32_t km[N][G];
    uint2 vm[N][G];
    static __device__ __forceinline__ uint32_t key_of(uint32_t i) { return i / (HD / 32u); }
    static __device__ __forceinline__ uint32_t pair_of(uint32_t i) { return i / (HD / 16u); }
    __device__ __forceinline__ void load(const uint8_t* block, bool there, uint32_t lane) {
#pragma unroll
        for (uint32_t j = 0; j < N; ++j) {
            const uint32_t i = lane + 32u * j;
            k[j] = v[j] = make_uint4(0u, 0u, 0u, 0u);
            if (there) {
                k[j] = reinterpret_cast<const uint4*>(block)[i];
                v[j] = reinterpret_cast<const uint4*>(block + 8u * HD)[i];
            }
#pragma unroll
            for (uint32_t u = 0; u < G; ++u) {
                km[j][u] = 0u;
                vm[j][u] = make_uint2(0u, 0u);
                if (there) {
                    km[j][u] = reinterpret_cast<const uint32_t*>(block + 16u * HD)[u * 16u + key_of(i)];
                    vm[j][u] = reinterpret_cast<const uint2*>(block + 17u * HD)[u * 8u + pair_of(i)];
                }
            }
        }
    }
};

template <int HD>
__global__ void __launch_bounds__(kThreads, 2)
kv_attention_tc_kernel(AttnParams p) {
    using T = __nv_bfloat16;
    using L = Layout<HD>;
    constexpr uint32_t SB = 18u * HD, G = HD / 64u;
    extern __shared__ __align__(1024) uint8_t smem[];
    Control& ctl = *reinterpret_cast<Control*>(smem + L::kControl);
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5;
    if (tid == 0) {
        for (uint32_t i = 0; i < 2u; ++i) {
            asm volatile("mbarrier.init.shared::cta.b64 [%0], 4;" ::"r"(smem_u32(&ctl.kv_full[i])));
            asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(smem_u32(&ctl.pv_done[i])));
            asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(smem_u32(&ctl.s_full[i])));
        }
        asm volatile("mbarrier.init.shared::cta.b64 [%0], 4;" ::"r"(smem_u32(&ctl.p_full)));
        asm volatile("mbarrier.init.shared::cta.b64 [%0], 4;" ::"r"(smem_u32(&ctl.q_full)));
        asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(smem_u32(&ctl.drained)));
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        ctl.sched.longest = ctl.sched.n_units = ctl.failed = 0;
    }
    __syncthreads();
    asm volatile("griddepcontrol.wait;" ::: "memory");
    Schedule<kRows, kThreads> sch;
    if (!sch.begin(p, ctl.sched)) return;
    // The kernel behind starts only when every CTA has its columns: one that took them first would keep them until this one ends
    if (warp == 7u) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&ctl.tmem)), "n"(kTmemColumns) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    before_sync();
    __syncthreads();
    after_sync();
    asm volatile("griddepcontrol.launch_dependents;");
    const uint32_t tmem = ctl.tmem, smem0 = smem_u32(smem);
    auto bar = [&](const uint64_t& b) { return smem_u32(&b); };

    uint64_t x = sch.x0;
    const uint64_t x1 = sch.x1;
    uint32_t k0 = 0;             // blocks of 64 keys before this unit
    bool live = true;
    // The CTA's units one after the other, by each of the three roles for itself: body(unit, its blocks of 64 keys).
    auto for_units = [&](auto&& body) {
        while (x < x1) {
            Unit un;
            if (!sch.at(p, x, un)) {
                x = un.next;
                continue;
            }
            const int32_t last = min(static_cast<int32_t>(min(un.b1, 0xFFFFFFu) * kBlockKeys), un.keys), from = static_cast<int32_t>(un.b0 * kBlockKeys);
            const uint32_t n = last > from ? static_cast<uint32_t>(last - from + static_cast<int32_t>(kKeys) - 1) / kKeys : 0u;
            body(un, n);
            k0 += n;
            x = un.start + un.n_blocks < un.next ? un.next : un.start + un.n_blocks;
            if (un.start + un.n_blocks > x1) break;
        }
    };

    if (warp < 4u) {
        // ---- rows ----
        const uint32_t lane_at = tmem + ((warp * 32u) << 16);
        for_units([&](const Unit& un, uint32_t n) {
            const Seq& sq = sch.sq;
            const uint32_t rr = un.tile * kRows + tid, tok = rr / p.group, head = un.kvh * p.group + rr % p.group;
            const bool there = tok < sq.n_new;
            const int32_t limit = there ? static_cast<int32_t>(min(max(sq.base + tok + 1, static_cast<int64_t>(0)), sq.cap)) : 0;
            const int32_t least = __reduce_min_sync(0xFFFFFFFFu, there ? limit : 0x7FFFFFFF);
            const bool whole = un.b0 == 0u && un.b1 == un.n_blocks;
            float m = -FLT_MAX, l = 0.0f, factor = 1.0f;
            uint32_t bad = 0;          // groups of values that a NaN that this row sees has spoilt
            if (n && live) {
                uint4 raw[HD / 8];
                const T* src = static_cast<const T*>(p.a.q) + static_cast<size_t>(sq.row0 + (there ? tok : 0u)) * p.a.q_stride + static_cast<size_t>(head) * HD;
#pragma unroll
                for (uint32_t c = 0; c < HD / 8u; ++c) {
                    raw[c] = make_uint4(0u, 0u, 0u, 0u);
                    if (!there) continue;
                    if (p.vec) {
                        raw[c] = *(reinterpret_cast<const uint4*>(src) + c);
                    } else {
                        T* e = reinterpret_cast<T*>(&raw[c]);
#pragma unroll
                        for (uint32_t i = 0; i < 8u; ++i) e[i] = src[8u * c + i];
                    }
                }
                float big = 0.0f;
#pragma unroll
                for (uint32_t c = 0; c < HD / 8u; ++c)
#pragma unroll
                    for (uint32_t i = 0; i < 8u; ++i) big = fmaxf(big, fabsf(op_widen(reinterpret_cast<const T*>(&raw[c])[i])));
                // 2^e above the largest |q|; the scale's sign goes with q
                const int e = big > 0.0f && big < INFINITY ? min(max(ilogbf(big) + 1, -110), 128) : 15;
                const float up = copysignf(power_of_two(15 - e), p.a.scale);
                factor = factor_of(p.a.scale, e - 15, 80);      // products are below 2^38
#pragma unroll
                for (uint32_t c = 0; c < HD / 8u; ++c) {
                    float v[8];
#pragma unroll
                    for (uint32_t i = 0; i < 8u; ++i) v[i] = op_widen(reinterpret_cast<const T*>(&raw[c])[i]) * up;
                    uint4 w;      // in the order that widened keys come in
                    w.x = bits_of(__floats2half2_rn(v[0], v[4]));
                    w.y = bits_of(__floats2half2_rn(v[1], v[5]));
                    w.z = bits_of(__floats2half2_rn(v[2], v[6]));
                    w.w = bits_of(__floats2half2_rn(v[3], v[7]));
                    *reinterpret_cast<uint4*>(smem + L::kQ + c / 8u * kRows * 128u + piece_at(tid, c & 7u)) = w;
                }
                publish(bar(ctl.q_full), lane);
            }
            for (uint32_t i = 0; i < n && live; ++i) {
                const uint32_t k = k0 + i, b = k & 1u;
                const int32_t tok0 = static_cast<int32_t>(un.b0 * kBlockKeys + i * kKeys);
                // (kv_full: what its writers say of pages and NaN)
                live = mbar_wait(bar(ctl.kv_full[b]), (k >> 1) & 1u, p.spin) && mbar_wait(bar(ctl.s_full[b]), (k >> 1) & 1u, p.spin);
                if (!live) break;
                after_sync();
                uint32_t s[kKeys];
                tmem_ld32(lane_at + b * kKeys, s);
                tmem_ld32(lane_at + b * kKeys + 32u, s + 32);
                tmem_loaded();
                const uint32_t present = *reinterpret_cast<const volatile uint32_t*>(ctl.there[b]);
                uint32_t see[2] = {0xFFFFFFFFu, 0xFFFFFFFFu};
                if (tok0 + static_cast<int32_t>(kKeys) > least || present != 0x01010101u) {
                    // keys that a row does not see weigh nothing, whatever lies there
#pragma unroll
                    for (uint32_t h = 0; h < 2u; ++h) {
                        const int32_t left = limit - tok0 - static_cast<int32_t>(32u * h);
                        see[h] = left >= 32 ? 0xFFFFFFFFu : left > 0 ? (1u << left) - 1u : 0u;
                        if (!(present >> (16u * h) & 1u)) see[h] &= 0xFFFF0000u;
                        if (!(present >> (16u * h + 8u) & 1u)) see[h] &= 0x0000FFFFu;
                    }
#pragma unroll
                    for (uint32_t j = 0; j < kKeys; ++j)
                        if (!(see[j / 32u] >> (j & 31u) & 1u)) s[j] = 0xFF800000u;
                }
#pragma unroll
                for (uint32_t u = 0; u < G; ++u) {
                    const uint2 o = make_uint2(*reinterpret_cast<const volatile uint32_t*>(&ctl.odd[b][u][0]), *reinterpret_cast<const volatile uint32_t*>(&ctl.odd[b][u][2]));
                    if ((o.x & see[0]) | (o.y & see[1])) bad |= 1u << u;
                }
                float tops[4];
#pragma unroll
                for (uint32_t j = 0; j < 4u; ++j) tops[j] = __uint_as_float(s[j]);
#pragma unroll
                for (uint32_t j = 4; j < kKeys; ++j) tops[j & 3u] = fmaxf(tops[j & 3u], __uint_as_float(s[j]));
                const float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3])) * factor;
                // the maximum follows in steps: weights may reach 2^kSlack before outputs are scaled anew
                const bool grows = __any_sync(0xFFFFFFFFu, top > m + kSlack);
                float f = 1.0f;
                if (grows) {
                    const float next = fmaxf(m, top);
                    f = ex2(m - next);
                    m = next;
                    l *= f;
                }
                const f32x2 fac = pack2(factor, factor), less = pack2(-m, -m);
                f32x2 sum = pack2(0.0f, 0.0f);
                uint32_t w[kKeys / 2u];
#pragma unroll
                for (uint32_t j = 0; j < kKeys / 2u; ++j) {
                    const float2 d = unpack2(fma2(pack2(__uint_as_float(s[2 * j]), __uint_as_float(s[2 * j + 1])), fac, less));
                    const float a = ex2(d.x), c = ex2(d.y);
                    sum = add2(sum, pack2(a, c));
                    w[j] = bits_of(__floats2half2_rn(a, c));
                }
                const float2 both = unpack2(sum);
                l += both.x + both.y;
                if (i) {      // the products of the weights before
                    live = mbar_wait(bar(ctl.pv_done[b ^ 1u]), ((k - 1u) >> 1) & 1u, p.spin);
                    if (!live) break;
                    after_sync();
                    if (grows) {
#pragma unroll
                        for (uint32_t c = 0; c < HD; c += 16u) {
                            uint32_t o[16];
                            tmem_ld16(lane_at + kTmemOut + c, o);
                            tmem_loaded();
#pragma unroll
                            for (uint32_t j = 0; j < 16u; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * f);
                            tmem_st16(lane_at + kTmemOut + c, o);
                        }
                        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                    }
                }
#pragma unroll
                for (uint32_t c = 0; c < kKeys / 8u; ++c)
                    *reinterpret_cast<uint4*>(smem + L::kP + piece_at(tid, c)) = make_uint4(w[4 * c], w[4 * c + 1], w[4 * c + 2], w[4 * c + 3]);
                publish(bar(ctl.p_full), lane);
            }
            if (n && live) {
                const uint32_t k = k0 + n - 1u;
                live = mbar_wait(bar(ctl.pv_done[k & 1u]), (k >> 1) & 1u, p.spin);
                after_sync();
            }
            // ---- out, or a piece of it: [four values of all rows], the last four maximum and sum ----
            constexpr uint32_t kPlanes = HD / 4u + 1u;
            const bool has = n && live;
            T* dst = static_cast<T*>(p.a.out) + static_cast<size_t>(sq.row0 + (there ? tok : 0u)) * p.a.out_stride + static_cast<size_t>(head) * HD;
            float4* slot = reinterpret_cast<float4*>(p.part) + (static_cast<size_t>(blockIdx.x) * 2u + (un.start >= sch.x0 ? 1u : 0u)) * kPlanes * kRows + tid;
            const float by = l != 0.0f ? 1.0f / l : 0.0f;      // rows that saw nothing: zeros
#pragma unroll
            for (uint32_t c = 0; c < HD; c += 16u) {
                uint32_t o[16];
                if (has) {
                    tmem_ld16(lane_at + kTmemOut + c, o);
                    tmem_loaded();
                }
                float v[2][8];
#pragma unroll
                for (uint32_t j = 0; j < 16u; ++j) v[j / 8u][j % 8u] = !has ? 0.0f : bad >> (c / 64u) & 1u ? __uint_as_float(0x7FC00000u) : __uint_as_float(o[j]);
#pragma unroll
                for (uint32_t h = 0; h < 2u; ++h) {
                    if (whole) {
                        if (there) store_row(dst + c + 8u * h, v[h], by, p.vec_out);
                    } else {
                        slot[(c / 4u + 2u * h) * kRows] = make_float4(v[h][0], v[h][1], v[h][2], v[h][3]);
                        slot[(c / 4u + 2u * h + 1u) * kRows] = make_float4(v[h][4], v[h][5], v[h][6], v[h][7]);
                    }
                }
            }
            if (!whole) {
                slot[HD / 4u * kRows] = make_float4(m, l, 0.0f, 0.0f);
                const uint32_t c0 = sch.holder(un.start), c1 = sch.holder(un.start + un.n_blocks - 1u);
                __threadfence();
                asm volatile("bar.sync 1, 128;" ::: "memory");
                if (tid == 0) {
                    const bool last = atomicAdd(p.counters + c0, 1u) == c1 - c0;
                    if (last) p.counters[c0] = 0u;       // as the next launch finds it
                    __threadfence();
                    *reinterpret_cast<volatile uint32_t*>(&ctl.flag) = last;
                }
                asm volatile("bar.sync 1, 128;" ::: "memory");
                if (*reinterpret_cast<volatile uint32_t*>(&ctl.flag)) {
                    // past L1: other CTAs wrote these
                    const float4* first = reinterpret_cast<const float4*>(p.part) + (static_cast<size_t>(c0) * 2u + 1u) * kPlanes * kRows + tid;
                    const uint32_t n_pieces = c1 - c0 + 1u;      // the first at `first`, then a CTA's two slots on
                    auto piece = [&](uint32_t i, uint32_t plane) { return __ldcg(first + (i ? static_cast<size_t>(i) * 2u - 1u : 0u) * kPlanes * kRows + plane * kRows); };
                    float jm = -FLT_MAX, jl = 0.0f;
                    for (uint32_t i = 0; i < n_pieces; ++i) jm = fmaxf(jm, piece(i, HD / 4u).x);
                    for (uint32_t i = 0; i < n_pieces; ++i) {
                        const float4 st = piece(i, HD / 4u);
                        jl = fmaf(ex2(st.x - jm), st.y, jl);
                    }
                    const float over = jl != 0.0f ? 1.0f / jl : 0.0f;
#pragma unroll 1
                    for (uint32_t c = 0; c < HD; c += 32u) {
                        f32x2 o[16];
#pragma unroll
                        for (uint32_t j = 0; j < 16u; ++j) o[j] = pack2(0.0f, 0.0f);
#pragma unroll 1
                        for (uint32_t i = 0; i < n_pieces; ++i) {
                            float4 part[8];
#pragma unroll
                            for (uint32_t j = 0; j < 8u; ++j) part[j] = piece(i, c / 4u + j);
                            const float f = ex2(piece(i, HD / 4u).x - jm);
#pragma unroll
                            for (uint32_t j = 0; j < 8u; ++j) {
                                o[2 * j] = fma2(pack2(part[j].x, part[j].y), pack2(f, f), o[2 * j]);
                                o[2 * j + 1] = fma2(pack2(part[j].z, part[j].w), pack2(f, f), o[2 * j + 1]);
                            }
                        }
#pragma unroll
                        for (uint32_t h = 0; h < 4u; ++h) {
                            float v[8];
#pragma unroll
                            for (uint32_t j = 0; j < 4u; ++j) {
                                const float2 e = unpack2(o[4u * h + j]);
                                v[2 * j] = e.x;
                                v[2 * j + 1] = e.y;
                            }
                            if (there) store_row(dst + c + 8u * h, v, over, p.vec_out);
                        }
                    }
                }
                asm volatile("bar.sync 1, 128;" ::: "memory");
            }
        });
    } else {
        // ---- keys and values: a warp has a block of sixteen of the 64 ----
        const uint32_t mine = warp - 4u, in_page = (1u << (p.kv.page_shift - 4u)) - 1u;
        const size_t page_bytes = p.kv.block_at(1u, 0u, 0u);
        // ---- products, by warp 7 ----
        const uint32_t leader = lane == 0u ? 1u : 0u;
        uint32_t units = 0;
        auto scores = [&](uint32_t k) {
            const uint32_t b = k & 1u;
            live = live && mbar_wait(bar(ctl.kv_full[b]), (k >> 1) & 1u, p.spin);
            if (!live) return;
            after_sync();
            const uint32_t a0 = desc_lo(smem0 + L::kQ, 16u), b0 = desc_lo(smem0 + L::keys(b), 16u);
#pragma unroll
            for (uint32_t q = 0; q < HD / 16u; ++q)
                mma(tmem + b * kKeys, a0 + (q / 4u * kRows * 128u + q % 4u * 32u >> 4), b0 + (q / 4u * kKeys * 128u + q % 4u * 32u >> 4), idesc(kKeys, false), q != 0u, leader);
            commit(bar(ctl.s_full[b]), leader);
        };
        auto outputs = [&](uint32_t k, bool first) {
            const uint32_t b = k & 1u;
            live = live && mbar_wait(bar(ctl.p_full), k & 1u, p.spin);
            if (!live) return;
            after_sync();
            const uint32_t a0 = desc_lo(smem0 + L::kP, 16u), b0 = desc_lo(smem0 + L::values(b), kKeys * 128u);
#pragma unroll
            for (uint32_t q = 0; q < kKeys / 16u; ++q)
                mma(tmem + kTmemOut, a0 + (q * 32u >> 4), b0 + (q * 2048u >> 4), idesc(HD, true), !first || q != 0u, leader);
            commit(bar(ctl.pv_done[b]), leader);
        };
        for_units([&](const Unit& un, uint32_t n) {
            if (!live || !n) return;
            const uint8_t* head_base = p.kv.base + p.kv.block_at(0u, un.kvh, 0u);
            const int32_t* table = p.b.pages + static_cast<size_t>(sch.s) * p.b.pages_per_seq;
            const uint32_t subs = static_cast<uint32_t>(un.keys + 15) / 16u, sub0 = un.b0 * (kBlockKeys / 16u) + mine;
            auto page_of = [&](uint32_t i) {
                const uint32_t sub = sub0 + 4u * i;
                if (i >= n || sub >= subs) return -1;
                const int32_t pg = table[sub >> (p.kv.page_shift - 4u)];
                return static_cast<uint32_t>(pg) < p.kv.n_pages ? pg : -1;
            };
            auto block_of = [&](uint32_t i, int32_t pg) { return head_base + static_cast<uint32_t>(max(pg, 0)) * page_bytes + ((sub0 + 4u * i) & in_page) * SB; };
            Raw<HD> ahead;
            int32_t pg = page_of(0), pg_next = page_of(1);
            ahead.load(block_of(0, pg), pg >= 0, lane);
            for (uint32_t i = 0; i < n; ++i) {
                const uint32_t k = k0 + i, b = k & 1u;
                const Raw<HD> r = ahead;
                const uint8_t* block = block_of(i, pg);
                const bool there = pg >= 0;
                pg = pg_next;
                pg_next = page_of(i + 2u);
                if (i + 1u < n) ahead.load(block_of(i + 1u, pg), pg >= 0, lane);
                if (k >= 2u) {
                    live = mbar_wait(bar(ctl.pv_done[b]), ((k - 2u) >> 1) & 1u, p.spin);
                    if (!live) return;
                }
                const int32_t left = un.keys - static_cast<int32_t>((sub0 + 4u * i) * 16u);      // tokens of the block that the tile sees
                uint8_t* ks = smem + L::keys(b) + mine * 16u * 128u;
                uint8_t* vs = smem + L::values(b) + mine * 16u * 128u;
                bool odd = false;
#pragma unroll
                for (uint32_t j = 0; j < Raw<HD>::N; ++j) {
                    const uint32_t at = lane + 32u * j, key = Raw<HD>::key_of(at), pair = Raw<HD>::pair_of(at);
#pragma unroll
                    for (uint32_t c = 0; c < 4u; ++c) {
                        // word t (HD / 32) + w of a key: values 64 (w / 2) + 16 t + 8 (w % 2)
                        const uint32_t word = at % (HD / 32u) * 4u + c, t = word / (HD / 32u), w = word % (HD / 32u);
                        const uint32_t meta = r.km[j][G == 1u ? 0u : c / 2u];
                        uint32_t v[4];
                        values_of(c == 0u ? r.k[j].x : c == 1u ? r.k[j].y : c == 2u ? r.k[j].z : r.k[j].w, __byte_perm(meta, 0u, 0x3232), __byte_perm(meta, 0u, 0x1010), v);
                        *reinterpret_cast<uint4*>(ks + w / 2u * kKeys * 128u + piece_at(key, 2u * t + (w & 1u))) = make_uint4(v[0], v[1], v[2], v[3]);
                    }
#pragma unroll
                    for (uint32_t c = 0; c < 2u; ++c) {
                        // words (g, u, 0), (g, u, 1) of a pair of tokens: values 64 u + 8 g of both
                        const uint32_t words = at % (HD / 16u) * 2u + c, g = words / G, u = words % G;
                        uint2 meta = r.vm[j][G == 1u ? 0u : c];
                        // what no row sees, or is NaN (and told apart), is zero: weights of nothing are multiplied by it too
                        const bool odd0 = half_is_nan(meta.x), odd1 = half_is_nan(meta.y);
                        odd = odd || odd0 || odd1;
                        if (odd0 || static_cast<int32_t>(2u * pair) >= left) meta.x = 0u;
                        if (odd1 || static_cast<int32_t>(2u * pair + 1u) >= left) meta.y = 0u;
                        const uint32_t steps = __byte_perm(meta.x, meta.y, 0x7632), minima = __byte_perm(meta.x, meta.y, 0x5410);
                        uint32_t lo[4], hi[4];
                        values_of(c ? r.v[j].z : r.v[j].x, steps, minima, lo);
                        values_of(c ? r.v[j].w : r.v[j].y, steps, minima, hi);
                        uint8_t* to = vs + u * kKeys * 128u;
                        *reinterpret_cast<uint4*>(to + piece_at(2u * pair, g)) = make_uint4(__byte_perm(lo[0], lo[1], 0x5410), __byte_perm(lo[2], lo[3], 0x5410),
                                                                                           __byte_perm(hi[0], hi[1], 0x5410), __byte_perm(hi[2], hi[3], 0x5410));
                        *reinterpret_cast<uint4*>(to + piece_at(2u * pair + 1u, g)) = make_uint4(__byte_perm(lo[0], lo[1], 0x7632), __byte_perm(lo[2], lo[3], 0x7632),
                                                                                                __byte_perm(hi[0], hi[1], 0x7632), __byte_perm(hi[2], hi[3], 0x7632));
                    }
                }
                odd = __any_sync(0xFFFFFFFFu, odd);
#pragma unroll
                for (uint32_t u = 0; u < G; ++u) {
                    uint32_t which = 0;
                    if (odd) {
                        const uint32_t meta = reinterpret_cast<const uint32_t*>(block + 17u * HD)[u * 16u + (lane & 15u)];
                        which = __ballot_sync(0xFFFFFFFFu, half_is_nan(meta)) & 0xFFFFu;
                    }
                    if (lane == 0u) ctl.odd[b][u][mine] = static_cast<uint16_t>(which);
                }
                if (lane == 0u) ctl.there[b][mine] = there ? 1u : 0u;
                publish(bar(ctl.kv_full[b]), lane);
                if (warp == 7u) {
                    if (i == 0u) live = mbar_wait_first(bar(ctl.q_full), units++ & 1u, p.spin);      // the others wait for what comes of it
                    scores(k);
                    if (i) outputs(k - 1u, i == 1u);
                    if (!live) return;
                }
            }
            if (warp == 7u) outputs(k0 + n - 1u, n == 1u);
        });
        if (warp == 7u) {      // products under way read shared memory and write columns that are given back below
            commit(bar(ctl.drained), leader);
            mbar_wait(bar(ctl.drained), 0u, kDrainRounds);
        }
    }
    if (!live && lane == 0u) ctl.failed = 1u;
    before_sync();
    __syncthreads();
    if (tid == 0 && ctl.failed) atomicExch(p.status, 1);      // results are wrong, and said to be
    if (warp == 7u) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(kTmemColumns) : "memory");
}

template <int HD>
void launch(csdr_context* ctx, AttnParams& p) {
    constexpr size_t smem = Layout<HD>::kBytes;
    auto kern = kv_attention_tc_kernel<HD>;
    ctx->opt_in_smem(reinterpret_cast<const void*>(kern), smem);
    launch_op(ctx, kern, dim3(static_cast<unsigned>(ctx->sm_count) * 2u), kThreads, smem, 1, p);
}

}  // namespace

void launch_kv_attention_tc(csdr_context* ctx, uint32_t head_dim, AttnParams& p) {
    if (head_dim == 64) launch<64>(ctx, p);
    else launch<128>(ctx, p);
}

}  // namespace csdr
