// Attention over the quantised cache for many query rows (a batch over its
// shared prefix, wide verify passes): the same scores, weights and running
// maximum as cdq_kv_attn.cu, with both products on tcgen05.mma (kind::f16,
// M = 128 rows, fp32 accumulators in tensor memory). e4m3 caches: a code is a
// half exactly, and its one scale a position multiplies scores and weights.
//
// One CTA a multiprocessor walks its units (128 positions) in two streams,
// even and odd units, each with its own scores, accumulator and running
// maxima, joined at the end of a segment:
//   warps 0..3, 4..7  softmax of stream 0 and 1, one thread a row: two sweeps
//                     over its 128 scores (tcgen05.ld), the maxima, then the
//                     weights, which go back over the scores as halves
//                     (tcgen05.st) and are the A operand of the second product;
//   warps 8..11       the unit's codes from global memory (the next unit's
//                     already in registers), as halves into shared memory: keys
//                     as they are, values transposed (position pairs of one
//                     element side by side), K-major 8 x 16-byte core matrices;
//                     value groups are 144 bytes apart, which takes the stores
//                     of a warp off each other's banks;
//   warp 12           lane 0 issues S_i = Q K_i^T, then O += P_(i-1) V_(i-1).
// Softmax and conversion issue about 4400 instructions a unit against 1024
// cycles of tensor core: the issue slots bound it, not the memory, and two
// streams keep all pipes busy.
//
// Every wait is bounded; one that gives up sets the abort flag and the error
// code 5, every role leaves its loop, and tensor memory is released.
#include <algorithm>
#include <atomic>

#include "cdq_kv_attn.cuh"

using cdq::launch_pdl;
using cdq::pdl_release;
using cdq::pdl_wait;
using namespace cdq::kv;

namespace {

constexpr int kSoftWarps = 8, kLoadWarps = 4;
constexpr int kMmaWarp = kSoftWarps + kLoadWarps;
constexpr int kThreads = 32 * (kMmaWarp + 1);
constexpr uint32_t kSpinLimit = 1u << 22;
constexpr int kScaleSlots = 4;  // units whose scales are in shared memory

__device__ int g_kv_error;

template <int HD>
struct Cfg {
    static constexpr int kQ = kMmaRows * HD * 2;
    static constexpr int kK = kUnit * HD * 2;
    static constexpr int kVBlock = HD / 8 * 144;          // eight positions of every element
    static constexpr int kV = kUnit / 8 * kVBlock;
    static constexpr int kQAt = 0, kKAt = kQ, kVAt = kKAt + 2 * kK;
    static constexpr int kScAt = kVAt + 2 * kV;           // [kScaleSlots][3][kUnit] floats
    static constexpr int kMetaAt = kScAt + kScaleSlots * 3 * kUnit * 4;  // [2][kMmaRows][4] floats
    static constexpr int kBarAt = kMetaAt + 2 * kMmaRows * 16;
    static constexpr int kSmem = kBarAt + 256;
    static constexpr int kOs = HD + 4;                    // padded row of the joined accumulators, over keys and values
    static_assert(kMmaRows * kOs * 4 <= 2 * (kK + kV), "joined accumulators");
};

// mbarriers, by index: [2] each
enum { kKFull = 0, kKEmpty = 2, kVFull = 4, kVEmpty = 6, kSFull = 8, kPFull = 10, kBars = 12 };

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
// Waits for the phase of the given parity; false once it, or another role's
// wait, has given up.
__device__ __forceinline__ bool wait(uint32_t bar, uint32_t parity, volatile uint32_t* abort) {
    for (uint32_t spin = 0; spin < kSpinLimit; ++spin) {
        uint32_t ok;
        asm volatile(
            "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}"
            : "=r"(ok)
            : "r"(bar), "r"(parity)
            : "memory");
        if (ok) return true;
        if ((spin & 63) == 63 && *abort) return false;
    }
    *abort = 1;
    atomicExch(&g_kv_error, 5);
    return false;
}

// K-major, no swizzle: core matrices of 8 rows x 16 bytes, `lead` bytes apart
// along K, `group` bytes apart between groups of 8 rows.
__device__ __forceinline__ uint64_t operand(uint32_t addr, int lead, int group) {
    return (uint64_t)((addr >> 4) & 0x3FFFu) | ((uint64_t)(lead >> 4) << 16) | ((uint64_t)(group >> 4) << 32) | (1ull << 46);
}
// instruction descriptor: f32 accumulators, f16 A and B, both K-major, M = 128
constexpr uint32_t idesc(int n) { return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((128u >> 4) << 24); }

__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t id, uint32_t accumulate) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d),
        "l"(a), "l"(b), "r"(id), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t id, uint32_t accumulate) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(d),
        "r"(a), "l"(b), "r"(id), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void load32(uint32_t at, uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
          "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]),
          "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]),
          "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
        : "r"(at)
        : "memory");
}
__device__ __forceinline__ void load16(uint32_t at, uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, "
        "[%16];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
          "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
        : "r"(at)
        : "memory");
}
__device__ __forceinline__ void wait_loads() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void store16(uint32_t at, const uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16};" ::"r"(at),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
        "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
        : "memory");
}
__device__ __forceinline__ void wait_stores() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Pairs of float32 in one 64-bit register: one instruction does both.
__device__ __forceinline__ uint64_t pair(float lo, float hi) {
    uint64_t p;
    asm("mov.b64 %0, {%1, %2};" : "=l"(p) : "f"(lo), "f"(hi));
    return p;
}
__device__ __forceinline__ uint64_t pair(uint32_t lo, uint32_t hi) { return pair(__uint_as_float(lo), __uint_as_float(hi)); }
__device__ __forceinline__ float2 unpair(uint64_t p) {
    float2 f;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(p));
    return f;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}

// One softmax thread's state of a row.
struct Row {
    float M, l;  // the running maximum (lags by up to kLazy) and the denominator
};

// The weights of one unit for one row: scores at S, scales of the unit at sc
// ([3][kUnit]: keys, values, log2 of values); positions at or beyond lim are
// hidden (MASK). The accumulator O of HD columns is rescaled where M rises
// (`filled`: it holds anything).
template <int HD, bool MASK>
__device__ __forceinline__ void weigh(Row& R, float f, uint32_t S, uint32_t O, const float* sc, int lim, bool filled) {
    float top = -INFINITY;
    const uint64_t f2 = pair(f, f);
    uint32_t v[2][32];
    load32(S, v[0]);
#pragma unroll
    for (int c = 0; c < kUnit; c += 32) {
        wait_loads();
        if (c + 32 < kUnit) load32(S + c + 32, v[(c / 32 + 1) & 1]);
        else load32(S, v[(c / 32 + 1) & 1]);  // (the second sweep's first)
        const uint32_t(&x)[32] = v[(c / 32) & 1];
#pragma unroll
        for (int j = 0; j < 32; j += 4) {
            const float4 ks = *reinterpret_cast<const float4*>(sc + c + j);
            const float4 lv = *reinterpret_cast<const float4*>(sc + 2 * kUnit + c + j);
            float2 s = unpair(fma2(mul2(pair(x[j], x[j + 1]), pair(ks.x, ks.y)), f2, pair(lv.x, lv.y)));
            float2 t = unpair(fma2(mul2(pair(x[j + 2], x[j + 3]), pair(ks.z, ks.w)), f2, pair(lv.z, lv.w)));
            if (MASK) {
                if (c + j >= lim) s.x = -INFINITY;
                if (c + j + 1 >= lim) s.y = -INFINITY;
                if (c + j + 2 >= lim) t.x = -INFINITY;
                if (c + j + 3 >= lim) t.y = -INFINITY;
            }
            top = fmaxf(top, fmaxf(s.x, s.y));
            top = fmaxf(top, fmaxf(t.x, t.y));
        }
    }
    float raise = 1.f;
    if (top > R.M + kLazy) {
        raise = ex2(R.M - top);
        R.M = top;
        R.l *= raise;
    }
    if (__any_sync(0xFFFFFFFFu, raise != 1.f) && filled) {
#pragma unroll 1
        for (int c = 0; c < HD; c += 16) {
            uint32_t w[16];
            load16(O + c, w);
            wait_loads();
#pragma unroll
            for (int j = 0; j < 16; ++j) w[j] = __float_as_uint(__uint_as_float(w[j]) * raise);
            store16(O + c, w);
        }
    }
    const float ref = R.M == -INFINITY ? 0.f : R.M;  // (nothing seen yet: every weight is 0)
    const uint64_t ref2 = pair(-ref, -ref);
    uint64_t l2 = pair(0.f, 0.f);
#pragma unroll
    for (int c = 0; c < kUnit; c += 32) {
        wait_loads();
        if (c + 32 < kUnit) load32(S + c + 32, v[(c / 32 + 1) & 1]);
        const uint32_t(&x)[32] = v[(c / 32) & 1];
        uint32_t w[16];
#pragma unroll
        for (int j = 0; j < 32; j += 4) {
            const float4 ks = *reinterpret_cast<const float4*>(sc + c + j);
            const float4 vs = *reinterpret_cast<const float4*>(sc + kUnit + c + j);
            const uint64_t kk[2] = {pair(ks.x, ks.y), pair(ks.z, ks.w)}, vv[2] = {pair(vs.x, vs.y), pair(vs.z, vs.w)};
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int at = c + j + 2 * h;
                const float2 e = unpair(fma2(mul2(pair(x[j + 2 * h], x[j + 2 * h + 1]), kk[h]), f2, ref2));
                float2 p = make_float2(ex2(e.x), ex2(e.y));
                if (MASK) {
                    if (at >= lim) p.x = 0.f;
                    if (at + 1 >= lim) p.y = 0.f;
                }
                const uint64_t p2 = pair(p.x, p.y);
                l2 = add2(l2, p2);
                float2 y = unpair(mul2(p2, vv[h]));
                if (MASK) {  // a hidden position's scale may be NaN
                    if (at >= lim) y.x = 0.f;
                    if (at + 1 >= lim) y.y = 0.f;
                }
                w[j / 2 + h] = pack_half(y.x, y.y);
            }
        }
        store16(S + c / 2, w);  // over scores that both sweeps have in registers, or behind them
    }
    const float2 l = unpair(l2);
    R.l += l.x + l.y;
    wait_stores();
}

template <int HD>
__global__ void __launch_bounds__(kThreads, 1) attn_mma_kernel(const AttnArgs A) {
    using F = Cfg<HD>;
    extern __shared__ __align__(128) uint8_t sm[];
    __shared__ uint32_t s_scan[kThreads / 32 + 2], s_tmem;
    __shared__ volatile uint32_t s_abort;
    const uint32_t base = smem_addr(sm), bars = base + F::kBarAt;
    const auto bar = [&](int kind, int s) { return bars + 8 * (kind + s); };
    float* const s_sc = reinterpret_cast<float*>(sm + F::kScAt);
    float4* const s_meta = reinterpret_cast<float4*>(sm + F::kMetaAt);
    float* const s_o = reinterpret_cast<float*>(sm + F::kKAt);
    pdl_wait();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const bool shared_rows = A.p.prefix_len != nullptr;
    const int per_b = A.p.c.kv_heads * A.p.tiles;
    const int per_seq = A.n_q * A.group;
    const int n_rows = shared_rows ? A.batch * per_seq : per_seq;
    const int prefix_len = shared_rows ? max(0, min(*A.p.prefix_len, A.p.c.max_len)) : 0;
    const auto len_of = [&](int b) { return shared_rows ? prefix_len : seen_len(A.pos[b], A.n_q, A.max_len); };
    uint32_t u, u_end, b_first;
    int b;
    if (!my_units<kThreads>(A.p, shared_rows ? 1 : A.batch, len_of, s_scan, u, u_end, b_first, b)) return;
    const uint32_t u_begin = u;

    if (tid == 0) {
        for (int s = 0; s < 2; ++s) {
            const int counts[kBars / 2] = {32 * kLoadWarps, 1, 32 * kLoadWarps, 1, 1, 16 * kSoftWarps};
            for (int k = 0; k < kBars / 2; ++k)
                asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar(2 * k, s)), "r"(counts[k]) : "memory");
        }
        s_abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_addr(&s_tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = s_tmem;
    const uint32_t kS[2] = {tmem, tmem + kUnit}, kO[2] = {tmem + 2 * kUnit, tmem + 2 * kUnit + HD};
    pdl_release();  // (tensor memory is taken: a successor's CTA cannot take it first)

    uint32_t it = 0;  // units done: unit `it` is use it / 2 of stage it % 2
    while (u < u_end) {
        const int len = len_of(b);
        const uint32_t nu = units_of(len);
        if (u >= b_first + nu * per_b) {
            b_first += nu * per_b;
            ++b;
            continue;
        }
        const uint32_t in_b = (u - b_first) / nu;
        const int kvh = in_b / A.p.tiles, tile = in_b % A.p.tiles;
        const uint32_t seg = b_first + in_b * nu;
        const int ua = u - seg, ub = min(nu, u_end - seg), n = ub - ua;
        const int r0 = tile * kMmaRows;
        const int p0 = shared_rows ? 0 : A.pos[b];
        const int first = shared_rows ? len : p0 < len ? p0 + 1 : len;  // positions that every row sees
        const int64_t head = (int64_t)b * A.p.c.kv_heads + kvh;
        const auto row_of = [&](int r, int* rb, int* ri, int* rh) -> int64_t {  // tile row -> output row
            const int x = r0 + r, w = shared_rows ? x % per_seq : x;
            *rb = shared_rows ? x / per_seq : b;
            *ri = w / A.group;
            *rh = kvh * A.group + w % A.group;
            return ((int64_t)*rb * A.n_q + *ri) * A.n_heads + *rh;
        };

        // ---- rotated queries as the first product's A operand ----
        if (warp < kSoftWarps) {
            constexpr int kLanes = HD / 8, kAtOnce = 32 * kSoftWarps / kLanes;
#pragma unroll
            for (int i = 0; i < kMmaRows / kAtOnce; ++i) {
                const int r = i * kAtOnce + tid / kLanes, sub = tid % kLanes;
                const bool in = r0 + r < n_rows;
                int rb = 0, ri = 0, rh = 0;
                if (in) row_of(r, &rb, &ri, &rh);
                const Query x = rotated_query<HD>(A, in, rb, ri, rh, sub);
                *reinterpret_cast<uint4*>(sm + F::kQAt + (r / 8) * (HD / 8 * 128) + sub * 128 + r % 8 * 16) = x.h;
                if (sub == 0) s_meta[r].x = x.f;
            }
            fence_async();
        }
        __syncthreads();

        if (warp < kSoftWarps) {
            // ---- softmax of one stream, one thread a row ----
            const int s = warp / 4, r = tid % kMmaRows;
            const uint32_t rows_at = (uint32_t)(warp % 4) << 21;  // the warp's 32 lanes of tensor memory
            const float f = s_meta[r].x;
            const int lim = shared_rows ? len : min(first + (r0 + r) / A.group, len);
            Row R{-INFINITY, 0.f};
            bool filled = false;
            int i = (it + s) & 1;  // this stream's first unit of the segment
            uint32_t g = it + i;
            for (; i < n; i += 2, g += 2) {
                const uint32_t par = (g >> 1) & 1;
                if (!wait(bar(kSFull, s), par, &s_abort)) break;
                fence_after();
                const int at = (ua + i) * kUnit;
                const float* sc = s_sc + g % kScaleSlots * (3 * kUnit);
                if (at + kUnit > first) weigh<HD, true>(R, f, kS[s] + rows_at, kO[s] + rows_at, sc, lim - at, filled);
                else weigh<HD, false>(R, f, kS[s] + rows_at, kO[s] + rows_at, sc, lim - at, filled);
                filled = true;
                fence_before();
                arrive(bar(kPFull, s));
            }
            // its last product has to be through before the accumulator is read
            if (filled && !s_abort) wait(bar(kVEmpty, s), ((g - 2) >> 1) & 1, &s_abort);
            fence_after();
            __syncwarp();
            // ---- join the streams: meta, then the accumulators over keys and values ----
            const auto soft_sync = [] { asm volatile("bar.sync 1, %0;" ::"n"(32 * kSoftWarps) : "memory"); };
            soft_sync();  // (every thread has read its factor)
            s_meta[s * kMmaRows + r] = make_float4(R.M, R.l, 0.f, 0.f);
            soft_sync();
            const float4 o = s_meta[(s ^ 1) * kMmaRows + r];
            const float top = fmaxf(R.M, o.x), ref = top == -INFINITY ? 0.f : top, e = ex2(R.M - ref);
            const float sum = R.l * e + o.y * ex2(o.x - ref);
            const bool whole = ua == 0 && ub == (int)nu;
            for (int turn = 1; turn >= 0; --turn) {
                if (s == turn && !s_abort) {
#pragma unroll 1
                    for (int c = 0; c < HD; c += 32) {
                        uint32_t v[32];
                        float* dst = s_o + r * F::kOs + c;
                        if (filled) {
                            load32(kO[s] + rows_at + c, v);
                            wait_loads();
                        } else {
#pragma unroll
                            for (int j = 0; j < 32; ++j) v[j] = 0;
                        }
#pragma unroll
                        for (int j = 0; j < 32; j += 4) {
                            float4 y = make_float4(__uint_as_float(v[j]) * e, __uint_as_float(v[j + 1]) * e,
                                                   __uint_as_float(v[j + 2]) * e, __uint_as_float(v[j + 3]) * e);
                            if (turn == 0) {
                                const float4 z = *reinterpret_cast<const float4*>(dst + j);
                                y = make_float4(y.x + z.x, y.y + z.y, y.z + z.z, y.w + z.w);
                            }
                            *reinterpret_cast<float4*>(dst + j) = y;
                        }
                    }
                }
                fence_before();
                soft_sync();
            }
            if (s == 0) s_meta[r] = make_float4(top, sum, 0.f, 0.f);
            soft_sync();
            // ---- rows out: final, a record, or this CTA's slot ----
            const int rows = s_abort ? 0 : min(kMmaRows, n_rows - r0);
            float* cut = A.p.slots + ((int64_t)blockIdx.x * 2 + (seg + ua == u_begin ? 0 : 1)) * kMmaRows * (kMeta + HD);
            for (int x = warp; x < rows; x += kSoftWarps) {
                int rb, ri, rh;
                const int64_t row = row_of(x, &rb, &ri, &rh);
                const float4 mt = s_meta[x];
                const float* src = s_o + x * F::kOs;
                if (whole && !A.p.recs) {
                    const int p = A.pos[rb];
                    const float k = (int64_t)p + ri >= A.max_len ? nan_f() : 1.f / mt.y;
#pragma unroll
                    for (int j = 0; j < HD / 32; ++j)
                        A.out[row * HD + lane + 32 * j] =
                            __bfloat16_as_ushort(__float2bfloat16_rn(p < 0 ? 0.f : src[lane + 32 * j] * k));
                } else {
                    float* dst = whole ? A.p.recs + row * (kMeta + HD) : cut + x * (kMeta + HD);
                    if (lane == 0) *reinterpret_cast<float4*>(dst) = mt;
#pragma unroll
                    for (int j = 0; j < HD / 32; ++j) dst[kMeta + lane + 32 * j] = src[lane + 32 * j];
                }
            }
        } else if (warp < kMmaWarp) {
            // ---- codes -> halves in shared memory ----
            const int w = warp - kSoftWarps;
            const uint8_t* kc = static_cast<const uint8_t*>(A.p.c.k) + head * A.p.c.max_len * HD;
            const uint8_t* vc = static_cast<const uint8_t*>(A.p.c.v) + head * A.p.c.max_len * HD;
            const uint16_t* ks = A.p.c.k_scale + head * A.p.c.max_len;
            const uint16_t* vs = A.p.c.v_scale + head * A.p.c.max_len;
            constexpr int kKs = HD / 16;            // 16-byte pieces of a lane's keys: (eight positions, four pieces) a warp
            constexpr int kVs = HD / 32;            // groups of eight positions x four elements of a lane's values
            constexpr int kDLanes = HD / 4;         // lanes across a value row
            uint4 kr[kKs];
            uint32_t vr[kVs][8], sk, sv;
            const int k_tok = lane % 8, k_piece = lane / 8;
            const int v_piece = lane % kDLanes, v_sub = lane / kDLanes;
            const auto k_at = [&](int j, int* tok, int* piece) {  // piece of a row, by 16 bytes
                const int x = w * kKs + j;
                *tok = x / (HD / 64) * 8 + k_tok;
                *piece = x % (HD / 64) * 4 + k_piece;
            };
            const auto v_at = [&](int j) { return ((w * kVs + j) * (32 / kDLanes) + v_sub) * 8; };  // first position
            const auto fetch = [&](int un) {
                const int p = un * kUnit, left = len - p;
#pragma unroll
                for (int j = 0; j < kKs; ++j) {
                    int tok, piece;
                    k_at(j, &tok, &piece);
                    kr[j] = make_uint4(0, 0, 0, 0);
                    if (tok < left) kr[j] = __ldg(reinterpret_cast<const uint4*>(kc + (int64_t)(p + tok) * HD) + piece);
                }
#pragma unroll
                for (int j = 0; j < kVs; ++j)
#pragma unroll
                    for (int t = 0; t < 8; ++t) {
                        const int tok = v_at(j) + t;
                        vr[j][t] = 0;
                        if (tok < left) vr[j][t] = __ldg(reinterpret_cast<const uint32_t*>(vc + (int64_t)(p + tok) * HD) + v_piece);
                    }
                const int tok = tid - 32 * kSoftWarps;
                sk = tok < left ? __ldg(ks + p + tok) : 0;
                sv = tok < left ? __ldg(vs + p + tok) : 0;
            };
            fetch(ua);
            for (int i = 0; i < n; ++i) {
                const uint32_t g = it + i, s = g & 1, use = g >> 1;
                if (use && !wait(bar(kKEmpty, s), (use - 1) & 1, &s_abort)) break;
                uint8_t* kd = sm + F::kKAt + s * F::kK;
#pragma unroll
                for (int j = 0; j < kKs; ++j) {
                    int tok, piece;
                    k_at(j, &tok, &piece);
                    uint32_t h[8];
                    e4m3x4_to_half(kr[j].x, h[0], h[1]);
                    e4m3x4_to_half(kr[j].y, h[2], h[3]);
                    e4m3x4_to_half(kr[j].z, h[4], h[5]);
                    e4m3x4_to_half(kr[j].w, h[6], h[7]);
                    uint8_t* d = kd + tok / 8 * (HD / 8 * 128) + piece * 256 + tok % 8 * 16;
                    *reinterpret_cast<uint4*>(d) = make_uint4(h[0], h[1], h[2], h[3]);
                    *reinterpret_cast<uint4*>(d + 128) = make_uint4(h[4], h[5], h[6], h[7]);
                }
                // (the slot's last unit is four back; the product of its weights was through before this stage's last scores)
                float* sc = s_sc + g % kScaleSlots * (3 * kUnit) + tid - 32 * kSoftWarps;
                sc[0] = bf_lo(sk), sc[kUnit] = bf_lo(sv), sc[2 * kUnit] = fmaxf(lg2(bf_lo(sv)), kLeast);
                fence_async();
                arrive(bar(kKFull, s));
                if (use && !wait(bar(kVEmpty, s), (use - 1) & 1, &s_abort)) break;
                uint8_t* vd = sm + F::kVAt + s * F::kV;
#pragma unroll
                for (int j = 0; j < kVs; ++j) {
                    uint32_t h[4][4];  // [element][pair of positions]
#pragma unroll
                    for (int t = 0; t < 4; ++t) {
                        const uint32_t lo = __byte_perm(vr[j][2 * t], vr[j][2 * t + 1], 0x5140),
                                       hi = __byte_perm(vr[j][2 * t], vr[j][2 * t + 1], 0x7362);
                        e4m3x4_to_half(lo, h[0][t], h[1][t]);
                        e4m3x4_to_half(hi, h[2][t], h[3][t]);
                    }
                    uint8_t* d = vd + v_at(j) / 8 * F::kVBlock + v_piece / 2 * 144 + v_piece % 2 * 64;
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        *reinterpret_cast<uint4*>(d + 16 * e) = make_uint4(h[e][0], h[e][1], h[e][2], h[e][3]);
                }
                fence_async();
                arrive(bar(kVFull, s));
                if (i + 1 < n) fetch(ua + i + 1);
            }
        } else if (lane == 0) {
            // ---- the products ----
            constexpr int kKGroup = HD / 8 * 128;
            for (int i = 0; i <= n; ++i) {
                if (i < n) {
                    const uint32_t g = it + i, s = g & 1, par = (g >> 1) & 1;
                    // the scores go over the weights of the stream's last unit: its product is through
                    if (g > 1 && !wait(bar(kVEmpty, s), par ^ 1, &s_abort)) break;
                    if (!wait(bar(kKFull, s), par, &s_abort)) break;
                    fence_after();
#pragma unroll
                    for (int k = 0; k < HD / 16; ++k)
                        mma_ss(kS[s], operand(base + F::kQAt + 256 * k, 128, kKGroup),
                               operand(base + F::kKAt + s * F::kK + 256 * k, 128, kKGroup), idesc(kUnit), k != 0);
                    commit(bar(kKEmpty, s));
                    commit(bar(kSFull, s));
                }
                if (i > 0) {
                    const uint32_t g = it + i - 1, s = g & 1, par = (g >> 1) & 1;
                    if (!wait(bar(kVFull, s), par, &s_abort) || !wait(bar(kPFull, s), par, &s_abort)) break;
                    fence_after();
#pragma unroll
                    for (int k = 0; k < kUnit / 16; ++k)
                        mma_ts(kO[s], kS[s] + 8 * k,
                               operand(base + F::kVAt + s * F::kV + 2 * k * F::kVBlock, F::kVBlock, 144), idesc(HD),
                               i > 2 || k != 0);
                    commit(bar(kVEmpty, s));
                }
            }
        }
        __syncwarp();
        fence_before();
        __syncthreads();
        fence_after();
        if (s_abort) break;
        it += n;
        u = seg + ub;
    }
    if (s_abort) {
        // what the tensor core still runs ends by itself; nothing waits on it but the release below
        __syncthreads();
        if (warp == kMmaWarp && lane == 0) {
            commit(bar(kSFull, 0));
            for (uint32_t spin = 0; spin < kSpinLimit / 64; ++spin) __nanosleep(20);
        }
        __syncthreads();
    }
    if (warp == kMmaWarp) {
        __syncwarp();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
}

template <int HD>
cudaError_t launch(const AttnArgs& A, cudaStream_t s) {
    static std::atomic<uint64_t> ready[2];  // devices that the attribute is set on
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev >= 128 || !(ready[dev / 64].load() >> (dev % 64) & 1)) {
        e = cudaFuncSetAttribute(attn_mma_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<HD>::kSmem);
        if (e != cudaSuccess) return e;
        if (dev < 128) ready[dev / 64].fetch_or(1ull << (dev % 64));
    }
    return launch_pdl(attn_mma_kernel<HD>, dim3(A.p.ctas), dim3(kThreads), Cfg<HD>::kSmem, s, A);
}

}  // namespace

namespace cdq {
namespace kv {

cudaError_t mma_attn_launch(const AttnArgs& A, cudaStream_t s) {
    return A.p.c.head_dim == 64 ? launch<64>(A, s) : launch<128>(A, s);
}

cudaError_t mma_read_error(int* out) {
    int v = 0;
    const cudaError_t e = cudaMemcpyFromSymbol(&v, g_kv_error, sizeof v);
    if (e == cudaSuccess) *out = v;
    return e;
}

}  // namespace kv
}  // namespace cdq
