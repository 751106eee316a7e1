// Attention over the quantised cache for many query rows (a batch over its
// shared prefix, wide verify passes): the same scores, weights and running
// maximum as cdq_kv_attn.cu, with both products on tcgen05.mma (M = 128 rows,
// fp32 accumulators in tensor memory).
//   S = Q K^T  (kind::f8f6f4): the keys' codes enter as they lie in the cache.
//              A query row, its largest element in [128, 256), is the sum of
//              two e4m3 terms and an e5m2 one: each takes what the ones before
//              left, so that 2^-11 of an element is left out, as by a rounding
//              to half, or 2^-20 of the largest. (A third e4m3 term would leave
//              out 2^-12 of an element but 2^-17 of the largest, for its
//              smallest step is 2^-9: elements beside one 2^9 times as large
//              would have fewer bits than bf16 gave them.) Three products at
//              twice the rate of halves, and nothing of the keys to convert.
//   O = P V    (kind::f16): weights as halves, the values' codes as halves.
//
// One CTA a multiprocessor walks its units (128 positions) in two streams,
// even and odd units, each with its own scores, accumulator and running
// maximum, joined at the end of a segment:
//   warps 0..7, 8..15 softmax of stream 0 and 1, two threads a row (64
//                     positions each): the weights under the running maximum
//                     as it is (tcgen05.ld), which go back over the scores as
//                     halves (tcgen05.st) and are the A operand of the second
//                     product. Only where one is too large for a half is the
//                     maximum found exactly, position by position, and the
//                     unit done again;
//   warps 16..21      the unit's values from global memory (the next unit's
//                     already in registers) into shared memory as halves,
//                     transposed (position pairs of one element side by side);
//                     a lane takes its four elements in an order of its own,
//                     which takes a warp's stores off each other's banks;
//   warp 22           its keys by asynchronous copies, straight into K-major
//                     8 x 16-byte core matrices, and its scales;
//   warp 23           lane 0 issues S_i, then O += P_(i-1) V_(i-1).
//
// 96 rows of 28 heads over 4 of 128 (672 a kv head) over 16,384 positions take
// 70 us, 330 TFLOP/s of the two products as they are defined. A unit takes
// about 4,600 cycles (108,000 that an SM is active in a capture, less 12,000
// before the first unit for tensor memory, lengths and queries, over 20.8
// units), of which 1,280 are the tensor pipe's (three terms of a query, one of
// the weights) and about 1,000 the exponentials'. Neither bounds it: the chain of
// a stream does, S, weights over S, O, and then the next S, for there is tensor
// memory for two streams only.
//
// Every wait is bounded; one that gives up sets the abort flag and the error
// code 5, every role leaves its loop, and tensor memory is released.
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "cdq_kv_attn.cuh"

using cdq::launch_pdl;
using cdq::pdl_release;
using cdq::pdl_wait;
using namespace cdq::kv;

namespace {

constexpr int kSoftWarps = 16, kValueWarps = 6;
constexpr int kHalf = kUnit / 2;  // positions of a softmax thread
constexpr int kKeyWarp = kSoftWarps + kValueWarps, kMmaWarp = kKeyWarp + 1;
constexpr int kKeyStages = 4;   // units of keys in shared memory, two of them ahead
constexpr int kValueStages = 3;  // units of values
constexpr int kTerms = 3;       // of a query: e4m3, e4m3, e5m2
constexpr int kThreads = 32 * (kMmaWarp + 1);
constexpr uint32_t kSpinLimit = 1u << 22;
constexpr int kScaleSlots = 4;  // units whose scales are in shared memory
// The largest weight under an M that lags; a half's largest is 65504. (M is found kBelow under the maximum; three powers
// of two lower, as many less of lag: 672 rows over 16,384 positions 3 us more, for it rises more often.)
constexpr float kRoom = 32768.f;
constexpr float kMost = 0x1p100f;  // the largest sum of a half unit's 2^(s - M): 64 of 2^90 where M is found anew

__device__ int g_kv_error;

constexpr int kScale = 2 * kUnit;  // scales of a unit: of its keys, of its values

template <int HD>
struct Cfg {
    static constexpr int kQ = kMmaRows * HD;              // one term
    static constexpr int kK = kUnit * HD;
    static constexpr int kGroup = HD / 16 * 128;          // eight rows of codes
    static constexpr int kVBlock = HD * 16;               // eight positions of every element
    static constexpr int kV = kUnit / 8 * kVBlock;
    static constexpr int kQAt = 0, kKAt = kTerms * kQ, kVAt = kKAt + kKeyStages * kK;
    static constexpr int kScAt = kVAt + kValueStages * kV;           // [kScaleSlots][kScale] floats
    static constexpr int kMetaAt = kScAt + kScaleSlots * kScale * 4;  // [4][kMmaRows][2] floats
    static constexpr int kBarAt = kMetaAt + 4 * kMmaRows * 8;
    static constexpr int kSmem = kBarAt + 256;
    static constexpr int kOs = HD + 4;                    // padded row of the joined accumulators, over keys and values
    static_assert(kMmaRows * kOs * 4 <= kKeyStages * kK + kValueStages * kV, "joined accumulators");
};

// mbarriers, by index: of the key and value stages, and of the two streams
// (scores there, weights there, accumulated)
enum { kKFull = 0, kKEmpty = kKFull + kKeyStages, kVFull = kKEmpty + kKeyStages, kVEmpty = kVFull + kValueStages,
       kSFull = kVEmpty + kValueStages, kPFull = kSFull + 2, kODone = kPFull + 2, kBars = kODone + 2 };
static_assert(kBars <= 32, "barrier block");

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

// The same for a whole warp, which goes on or gives up together.
__device__ __forceinline__ bool wait_warp(uint32_t bar, uint32_t parity, volatile uint32_t* abort) {
    return __all_sync(0xFFFFFFFFu, wait(bar, parity, abort));
}

// K-major, no swizzle: core matrices of 8 rows x 16 bytes, `lead` bytes apart
// along K, `group` bytes apart between groups of 8 rows.
__device__ __forceinline__ uint64_t operand(uint32_t addr, int lead, int group) {
    return (uint64_t)((addr >> 4) & 0x3FFFu) | ((uint64_t)(lead >> 4) << 16) | ((uint64_t)(group >> 4) << 32) | (1ull << 46);
}
// instruction descriptor: f32 accumulators, A and B of the kind's first type
// (f16; e4m3), both K-major, M = 128; kE5M2A: A in e5m2
constexpr uint32_t kE5M2A = 1u << 7;
constexpr uint32_t idesc(int n) { return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((128u >> 4) << 24); }

__device__ __forceinline__ void mma_fp8(uint32_t d, uint64_t a, uint64_t b, uint32_t id, uint32_t accumulate) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n}" ::"r"(d),
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

// One softmax thread's state of a row.
struct Row {
    float M, l;  // the running maximum (it may lag by kRoom) and the denominator
};

// The two warps that share 32 rows of a stream.
__device__ __forceinline__ void pair_sync(int pair) { asm volatile("bar.sync %0, 64;" ::"r"(2 + pair) : "memory"); }
__device__ __forceinline__ bool pair_any(int pair, bool on) {  // whether any of their threads says so
    uint32_t r;
    asm volatile(
        "{\n .reg .pred p, q;\n setp.ne.u32 p, %1, 0;\n bar.red.or.pred q, %2, 64, p;\n selp.u32 %0, 1, 0, q;\n}"
        : "=r"(r)
        : "r"((uint32_t)on), "r"(2 + pair)
        : "memory");
    return r != 0;
}

// The running maximum for a unit, found exactly: max over positions of
// s_j + log2 scale_v[j], less kBelow (both of a row's threads find it); this
// thread's half of the accumulator's columns is rescaled where it rises from M.
template <int HD, bool MASK>
__device__ __noinline__ float raised_maximum(float M, float f, uint32_t S, uint32_t O, const float* sc, int lim, bool filled,
                                             int pair) {
    float top = -INFINITY;
#pragma unroll 1
    for (int c = 0; c < kUnit; c += 16) {
        uint32_t v[16];
        load16(S + c, v);
        wait_loads();
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            const float t = fmaf(__uint_as_float(v[j]) * sc[c + j], f, fmaxf(lg2(sc[kUnit + c + j]), kLeast));
            if (!MASK || c + j < lim) top = fmaxf(top, t);
        }
    }
    top -= kBelow;
    const float raise = top > M ? ex2(M - top) : 1.f;
    if (filled) {
#pragma unroll 1
        for (int c = 0; c < HD / 2; c += 16) {
            uint32_t w[16];
            load16(O + c, w);
            wait_loads();
#pragma unroll
            for (int j = 0; j < 16; ++j) w[j] = __float_as_uint(__uint_as_float(w[j]) * raise);
            store16(O + c, w);
        }
        wait_stores();
    }
    pair_sync(pair);  // (the scores are read: weights may go over them)
    return fmaxf(M, top);
}

// The weights of kHalf positions of one unit for one row, under the running
// maximum M: scores at S, scales of the unit at sc, positions at or beyond lim
// hidden (MASK). l: the sum of their 2^(s - M). Returns whether M is too low for
// them: a weight above kRoom, or terms of l that may leave float32's range.
template <bool MASK>
__device__ __forceinline__ bool sweep(float M, float f, uint32_t S, const float* sc, int lim, uint32_t (&w)[kHalf / 2], float& l) {
    const float ref = M == -INFINITY ? 0.f : M;  // (nothing seen yet: every weight is 0)
    float sum[2] = {0.f, 0.f};
    __half2 top = __float2half2_rn(0.f);
#pragma unroll
    for (int c = 0; c < kHalf; c += 16) {
        uint32_t x[16];
        load16(S + c, x);
        wait_loads();
#pragma unroll
        for (int j = 0; j < 16; j += 4) {
            const float4 ks = *reinterpret_cast<const float4*>(sc + c + j);
            const float4 vs = *reinterpret_cast<const float4*>(sc + kUnit + c + j);
            float p[4] = {ex2(fmaf(__uint_as_float(x[j]) * ks.x, f, -ref)), ex2(fmaf(__uint_as_float(x[j + 1]) * ks.y, f, -ref)),
                          ex2(fmaf(__uint_as_float(x[j + 2]) * ks.z, f, -ref)),
                          ex2(fmaf(__uint_as_float(x[j + 3]) * ks.w, f, -ref))};
            float y[4] = {p[0] * vs.x, p[1] * vs.y, p[2] * vs.z, p[3] * vs.w};
            if (MASK) {  // a hidden position's scale may be NaN
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (c + j + e >= lim) p[e] = y[e] = 0.f;
            }
            sum[0] += p[0], sum[1] += p[1];
            sum[0] += p[2], sum[1] += p[3];
            const __half2 lo = __floats2half2_rn(y[0], y[1]), hi = __floats2half2_rn(y[2], y[3]);
            top = __hmax2(top, __hmax2(lo, hi));
            w[(c + j) / 2] = *reinterpret_cast<const uint32_t*>(&lo);
            w[(c + j) / 2 + 1] = *reinterpret_cast<const uint32_t*>(&hi);
        }
    }
    l = sum[0] + sum[1];
    return fmaxf(__low2float(top), __high2float(top)) > kRoom || l > kMost;
}

// A row's half of a unit: its weights under the running maximum as it is,
// which seldom rises; where either thread of any of the warps' rows finds it
// too low, it is found exactly and the weights again. Scores lie at S + from on,
// O: this thread's half of the accumulator, `filled`: it holds anything.
template <int HD, bool MASK>
__device__ __forceinline__ void weigh(Row& R, float f, uint32_t S, uint32_t O, const float* sc, int lim, bool filled, int half,
                                      int pair) {
    const int from = half * kHalf;
    uint32_t w[kHalf / 2];
    float l;
    bool raise = !filled;
#pragma unroll 1
    for (;;) {
        if (raise) {
            const float M = raised_maximum<HD, MASK>(R.M, f, S, O, sc, lim, filled, pair);
            if (M > R.M) R.l *= ex2(R.M - M);
            R.M = M;
        }
        const bool low = sweep<MASK>(R.M, f, S + from, sc + from, lim - from, w, l);
        if (raise || !pair_any(pair, low || (R.M == -INFINITY && f == f))) break;
        raise = true;
    }
    R.l += l;
    // over scores of this half (every thread that reads them is past them)
    store16(S + from, *reinterpret_cast<const uint32_t(*)[16]>(w));
    store16(S + from + 16, *reinterpret_cast<const uint32_t(*)[16]>(w + 16));
    wait_stores();
}

template <int HD>
__global__ void __launch_bounds__(kThreads, 1) attn_mma_kernel(const AttnArgs A) {
    using F = Cfg<HD>;
    using Vec = typename std::conditional<HD == 128, float4, float2>::type;  // a lane's share of a row
    extern __shared__ __align__(128) uint8_t sm[];
    __shared__ uint32_t s_scan[kThreads / 32 + 2], s_tmem;
    __shared__ volatile uint32_t s_abort;
    const uint32_t base = smem_addr(sm), bars = base + F::kBarAt;
    const auto bar = [&](int kind, int s) { return bars + 8 * (kind + s); };
    float* const s_sc = reinterpret_cast<float*>(sm + F::kScAt);
    float2* const s_meta = reinterpret_cast<float2*>(sm + F::kMetaAt);
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
    if (!my_units<kThreads>(A.p, blockIdx.x, shared_rows ? 1 : A.batch, len_of, s_scan, u, u_end, b_first, b)) return;
    const uint32_t u_begin = u;

    if (tid == 0) {
        const auto init = [&](int first, int n, int count) {
            for (int i = first; i < first + n; ++i)
                asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bars + 8 * i), "r"(count) : "memory");
        };
        init(kKFull, kKeyStages, 32);
        init(kKEmpty, kKeyStages, 1);
        init(kVFull, kValueStages, 32 * kValueWarps);
        init(kVEmpty, kValueStages, 1);
        init(kODone, 2, 1);
        init(kSFull, 2, 1);
        init(kPFull, 2, 16 * kSoftWarps);
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

    uint32_t it = 0;  // units done: unit `it` is use it / 2 of stream it % 2, and likewise of the key and value stages
    while (u < u_end) {
        const int len = len_of(b);
        const uint32_t nu = units_of(len), nv = nu + A.p.lead;
        if (u >= b_first + nv * per_b) {
            b_first += nv * per_b;
            ++b;
            continue;
        }
        const uint32_t in_b = (u - b_first) / nv;
        const int kvh = in_b / A.p.tiles, tile = in_b % A.p.tiles;
        const uint32_t seg = b_first + in_b * nv;
        const Part part(u, u_end, seg, nu, A.p.lead);
        if (part.ua >= part.ub) break;
        const int ua = part.ua, ub = part.ub, n = ub - ua;
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
            constexpr int kLanes = HD / 8, kAtOnce = 32 * kSoftWarps / kLanes, kTurns = kMmaRows / kAtOnce;
            const int sub = tid % kLanes;
            QueryLoad q[kTurns];
#pragma unroll
            for (int i = 0; i < kTurns; ++i) {
                const int r = i * kAtOnce + tid / kLanes;
                const bool in = r0 + r < n_rows;
                int rb = 0, ri = 0, rh = 0;
                if (in) row_of(r, &rb, &ri, &rh);
                q[i] = load_query<HD>(A, in, rb, ri, rh, sub);
            }
#pragma unroll
            for (int i = 0; i < kTurns; ++i) {
                const int r = i * kAtOnce + tid / kLanes;
                const Query x = rotated_query<HD>(A, r0 + r < n_rows, q[i], sub);
                float y[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) y[j] = x.x[j] * 128.f;
                uint8_t* d = sm + F::kQAt + r / 8 * F::kGroup + sub / 2 * 128 + r % 8 * 16 + sub % 2 * 8;
#pragma unroll
                for (int term = 0; term < kTerms; ++term) {
                    uint32_t o[2] = {0, 0};
#pragma unroll
                    for (int j = 0; j < 8; j += 2) {
                        const float2 z = make_float2(y[j], y[j + 1]);
                        const uint32_t c = __nv_cvt_float2_to_fp8x2(z, __NV_SATFINITE, term < kTerms - 1 ? __NV_E4M3 : __NV_E5M2);
                        const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)c, __NV_E4M3);
                        const float2 back = __half22float2(*reinterpret_cast<const __half2*>(&h));
                        y[j] -= back.x, y[j + 1] -= back.y;
                        o[j / 4] |= c << (16 * (j / 2 & 1));
                    }
                    *reinterpret_cast<uint2*>(d + term * F::kQ) = make_uint2(o[0], o[1]);
                }
                if (sub == 0) s_meta[r].x = x.f * 0x1p-7f;
            }
            fence_async();
        }
        // (keys and values set out meanwhile)
        if (warp < kSoftWarps || warp == kMmaWarp)
            asm volatile("bar.sync 10, %0;" ::"n"(32 * (kSoftWarps + 1)) : "memory");

        if (warp < kSoftWarps) {
            // ---- softmax of one stream, one thread a row ----
            const int s = warp / 8, half = warp / 4 % 2, r = tid % kMmaRows, pair = s * 4 + warp % 4;
            const uint32_t rows_at = (uint32_t)(warp % 4) << 21;  // the warp's 32 lanes of tensor memory
            const float f = s_meta[r].x;
            const int lim = shared_rows ? len : min(first + (r0 + r) / A.group, len);
            Row R{-INFINITY, 0.f};
            bool filled = false;
            int i = (it + s) & 1;  // this stream's first unit of the segment
            uint32_t g = it + i;
            for (; i < n; i += 2, g += 2) {
                const uint32_t par = (g >> 1) & 1;
                if (pair_any(pair, !wait(bar(kSFull, s), par, &s_abort))) break;
                fence_after();
                const int at = (ua + i) * kUnit;
                const float* sc = s_sc + g % kScaleSlots * kScale;
                const uint32_t o_at = kO[s] + rows_at + half * (HD / 2);
                if (at + kUnit > first) weigh<HD, true>(R, f, kS[s] + rows_at, o_at, sc, lim - at, filled, half, pair);
                else weigh<HD, false>(R, f, kS[s] + rows_at, o_at, sc, lim - at, filled, half, pair);
                filled = true;
                fence_before();
                arrive(bar(kPFull, s));
            }
            // its last product has to be through before the accumulator is read
            if (filled) wait_warp(bar(kODone, s), ((g - 2) >> 1) & 1, &s_abort);
            fence_after();
            __syncwarp();
            // ---- join the streams: meta, then the accumulators over keys and values ----
            const auto soft_sync = [] { asm volatile("bar.sync 1, %0;" ::"n"(32 * kSoftWarps) : "memory"); };
            soft_sync();  // (every thread has read its factor)
            s_meta[(2 * s + half) * kMmaRows + r] = make_float2(R.M, R.l);
            soft_sync();
            // (both halves of a stream have its M)
            const float2 m0 = s_meta[r], m1 = s_meta[kMmaRows + r], m2 = s_meta[2 * kMmaRows + r], m3 = s_meta[3 * kMmaRows + r];
            const float top = fmaxf(m0.x, m2.x), ref = top == -INFINITY ? 0.f : top, e = ex2(R.M - ref);
            const float sum = (m0.y + m1.y) * ex2(m0.x - ref) + (m2.y + m3.y) * ex2(m2.x - ref);
            const bool whole = ua == 0 && ub == (int)nu;
            for (int turn = 1; turn >= 0; --turn) {
                if (s == turn && !__any_sync(0xFFFFFFFFu, s_abort)) {
#pragma unroll 1
                    for (int c = half * (HD / 2); c < (half + 1) * (HD / 2); c += 32) {
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
            if (warp < 4) s_meta[r] = make_float2(top, sum);
            soft_sync();
            // ---- rows out: final, a record, or this CTA's slot ----
            const int rows = s_abort ? 0 : min(kMmaRows, n_rows - r0);
            float* cut = A.p.slots + ((int64_t)blockIdx.x * 2 + (u_begin >= seg ? 0 : 1)) * kMmaRows * (kMeta + HD);
            for (int x = warp; x < rows; x += kSoftWarps) {
                const float2 mt = s_meta[x];
                const float* src = s_o + x * F::kOs;
                float* dst = cut + x * (kMeta + HD);
                if (whole) {
                    int rb, ri, rh;
                    const int64_t row = row_of(x, &rb, &ri, &rh);
                    if (!A.p.recs) {
                        const int p = A.pos[rb];
                        const float k = (int64_t)p + ri >= A.max_len ? nan_f() : 1.f / mt.y;
#pragma unroll
                        for (int j = 0; j < HD / 32; ++j)
                            A.out[row * HD + lane + 32 * j] =
                                __bfloat16_as_ushort(__float2bfloat16_rn(p < 0 ? 0.f : src[lane + 32 * j] * k));
                        continue;
                    }
                    dst = A.p.recs + row * (kMeta + HD);
                }
                if (lane == 0) *reinterpret_cast<float2*>(dst) = mt;
                *reinterpret_cast<Vec*>(dst + kMeta + HD / 32 * lane) = *reinterpret_cast<const Vec*>(src + HD / 32 * lane);
            }
        } else if (warp < kKeyWarp) {
            // ---- values: codes as halves, transposed ----
            const int w = warp - kSoftWarps;
            const uint8_t* vc = static_cast<const uint8_t*>(A.p.c.v) + head * A.p.c.max_len * HD;
            // tasks of a warp: eight positions x four elements a lane
            constexpr int kDLanes = HD / 4;         // lanes across a value row
            constexpr int kTasks = kUnit / 8 * kDLanes / 32, kVs = (kTasks + kValueWarps - 1) / kValueWarps;
            uint32_t vr[kVs][8];
            const int v_piece = lane % kDLanes, v_sub = lane / kDLanes;
            // elements (e + turn) mod 4 of the lane's four, paired over two positions: byte selectors
            const uint32_t turn = lane / 2 % 4;
            const auto bytes = [&](uint32_t e) {
                const uint32_t x = (e + turn) % 4, y = (e + 1 + turn) % 4;
                return x | (4 + x) << 4 | y << 8 | (4 + y) << 12;
            };
            const uint32_t lo_bytes = bytes(0), hi_bytes = bytes(2);
            const auto v_at = [&](int j) { return ((w + j * kValueWarps) * (32 / kDLanes) + v_sub) * 8; };  // first position
            const auto fetch = [&](int un) {
                const int p = un * kUnit, left = len - p;
                const uint32_t* src = reinterpret_cast<const uint32_t*>(vc + (int64_t)p * HD) + v_piece;
#pragma unroll
                for (int j = 0; j < kVs; ++j) {
                    if (w + j * kValueWarps >= kTasks) break;
                    if (left >= kUnit) {
#pragma unroll
                        for (int t = 0; t < 8; ++t) vr[j][t] = __ldg(src + (v_at(j) + t) * (HD / 4));
                    } else {
#pragma unroll
                        for (int t = 0; t < 8; ++t) vr[j][t] = v_at(j) + t < left ? __ldg(src + (v_at(j) + t) * (HD / 4)) : 0;
                    }
                }
            };
            fetch(ua);
            for (int i = 0; i < n; ++i) {
                const uint32_t g = it + i, st = g % kValueStages, use = g / kValueStages;
                if (use && !wait_warp(bar(kVEmpty, st), (use - 1) & 1, &s_abort)) break;
                uint8_t* vd = sm + F::kVAt + st * F::kV;
#pragma unroll
                for (int j = 0; j < kVs; ++j) {
                    if (w + j * kValueWarps >= kTasks) break;
                    uint32_t h[4][4];  // [element][pair of positions]
#pragma unroll
                    for (int t = 0; t < 4; ++t) {
                        const uint32_t lo = __byte_perm(vr[j][2 * t], vr[j][2 * t + 1], lo_bytes),
                                       hi = __byte_perm(vr[j][2 * t], vr[j][2 * t + 1], hi_bytes);
                        e4m3x4_to_half(lo, h[0][t], h[1][t]);
                        e4m3x4_to_half(hi, h[2][t], h[3][t]);
                    }
                    uint8_t* d = vd + v_at(j) / 8 * F::kVBlock + v_piece * 64;
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        *reinterpret_cast<uint4*>(d + (e + turn) % 4 * 16) = make_uint4(h[e][0], h[e][1], h[e][2], h[e][3]);
                }
                fence_async();
                arrive(bar(kVFull, st));
                if (i + 1 < n) fetch(ua + i + 1);
            }
        } else if (warp == kKeyWarp) {
            // ---- keys, as they are, and scales ----
            const uint8_t* kc = static_cast<const uint8_t*>(A.p.c.k) + head * A.p.c.max_len * HD;
            const uint16_t* ks = A.p.c.k_scale + head * A.p.c.max_len;
            const uint16_t* vs = A.p.c.v_scale + head * A.p.c.max_len;
            // a copy of a warp: eight positions x four 16-byte pieces of their rows
            constexpr int kCopies = kUnit / 8 * (HD / 64);
            const uint32_t kd = base + F::kKAt + lane / 8 * 128 + lane % 8 * 16;
            const uint8_t* src = kc + (int64_t)(lane % 8) * HD + lane / 8 * 16;
            bool ok = true;
            const auto issue = [&](int i) {
                if (i < n && ok) {
                    const uint32_t g = it + i, st = g % kKeyStages, use = g / kKeyStages;
                    if (use) ok = wait_warp(bar(kKEmpty, st), (use - 1) & 1, &s_abort);
                    const int p = (ua + i) * kUnit, left = len - p - lane % 8;
                    const uint8_t* from = src + (int64_t)p * HD;
#pragma unroll
                    for (int x = 0; x < kCopies; ++x) {
                        const int tok = x / (HD / 64) * 8, at = x % (HD / 64);  // (of the copy's first position and piece)
                        const bool in = tok < left;
                        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(
                                         kd + st * F::kK + tok / 8 * F::kGroup + at * 512),
                                     "l"(in ? from + tok * HD + at * 64 : kc), "r"(in ? 16 : 0)
                                     : "memory");
                    }
                }
                asm volatile("cp.async.commit_group;" ::: "memory");
            };
            uint32_t kn[kUnit / 32], vn[kUnit / 32];
            const auto fetch = [&](int i) {
                const int p = (ua + i) * kUnit + lane;
#pragma unroll
                for (int j = 0; j < kUnit / 32; ++j) {
                    const bool in = i < n && p + 32 * j < len;
                    kn[j] = in ? __ldg(ks + p + 32 * j) : 0;
                    vn[j] = in ? __ldg(vs + p + 32 * j) : 0;
                }
            };
            issue(0);
            issue(1);
            fetch(0);
            for (int i = 0; i < n && ok; ++i) {
                const uint32_t g = it + i;
                // the slot's last unit is four back: the scores two back waited for the product of its weights
                if (i >= kScaleSlots) ok = wait_warp(bar(kKEmpty, (g - 2) % kKeyStages), (g - 2) / kKeyStages & 1, &s_abort);
                float* sc = s_sc + g % kScaleSlots * kScale;
#pragma unroll
                for (int j = 0; j < kUnit / 32; ++j) {
                    sc[lane + 32 * j] = bf_lo(kn[j]);
                    sc[kUnit + lane + 32 * j] = bf_lo(vn[j]);
                }
                asm volatile("cp.async.wait_group 1;" ::: "memory");
                fence_async();
                arrive(bar(kKFull, g % kKeyStages));
                fetch(i + 1);
                issue(i + 2);
            }
            asm volatile("cp.async.wait_group 0;" ::: "memory");
        } else if (lane == 0) {
            // ---- the products ----
            for (int i = 0; i <= n; ++i) {
                if (i < n) {
                    const uint32_t g = it + i, s = g & 1, st = g % kKeyStages;
                    // the scores go over the weights of the stream's last unit: its product is through
                    if (g > 1 && !wait(bar(kODone, s), ((g >> 1) - 1) & 1, &s_abort)) break;
                    if (!wait(bar(kKFull, st), g / kKeyStages & 1, &s_abort)) break;
                    fence_after();
#pragma unroll
                    for (int k = 0; k < kTerms * HD / 32; ++k)
                        mma_fp8(kS[s], operand(base + F::kQAt + k / (HD / 32) * F::kQ + k % (HD / 32) * 256, 128, F::kGroup),
                                 operand(base + F::kKAt + st * F::kK + k % (HD / 32) * 256, 128, F::kGroup),
                                 idesc(kUnit) | (k / (HD / 32) == kTerms - 1 ? kE5M2A : 0), k != 0);
                    commit(bar(kKEmpty, st));
                    commit(bar(kSFull, s));
                }
                if (i > 0) {
                    const uint32_t g = it + i - 1, s = g & 1, st = g % kValueStages;
                    if (!wait(bar(kVFull, st), g / kValueStages & 1, &s_abort) || !wait(bar(kPFull, s), g >> 1 & 1, &s_abort)) break;
                    fence_after();
#pragma unroll
                    for (int k = 0; k < kUnit / 16; ++k)
                        mma_ts(kO[s], kS[s] + 8 * k + (k >= kHalf / 16 ? kHalf / 2 : 0),
                               operand(base + F::kVAt + st * F::kV + 2 * k * F::kVBlock, F::kVBlock, 128), idesc(HD),
                               i > 2 || k != 0);
                    commit(bar(kVEmpty, st));
                    commit(bar(kODone, s));
                }
            }
        }
        __syncwarp();
        fence_before();
        __syncthreads();
        fence_after();
        if (s_abort) break;
        it += n;
        u = part.next;
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
