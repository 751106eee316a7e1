// Verification of drafted tokens and sampling, from given random numbers.
//
// One launch over all rows leaves the (max, sum of 2^(x - max)) of each row's
// parts; in a second one a cluster of CTAs serves each sequence, every CTA a
// contiguous part of the vocabulary, exchanging through distributed shared
// memory:
//   1. the rows' sums decide which drafts are kept (sampling alone has one
//      row, and the cluster finds its maximum itself: one launch);
//   2. the weights e^(x - max)/Z, or max(p - q, 0), summed in 64 bits over
//      segments of 128 tokens, give the total; the segment that u * total
//      falls into is scanned.
// A drawn token is the one side of a border that a number falls on, and with
// a flat distribution over 10^5 tokens sums that err by 1e-7 put it on the
// wrong side of one in every few hundred draws: hence 64 bits in 2. A kept
// draft is a single comparison; where its sides are nearer than the first
// launch's float32 terms may err (one in 50,000) 64-bit sums of its rows
// decide. max(p - q, 0) has to be formed before Z_p and Z_q are known to 64
// bits: step 2 begins with the first launch's, picks by them the tokens where p
// is the larger, and sums both rows' shares of these and, in the same pass, Z_p
// and Z_q, which then correct the two. The choice of tokens may be off where
// p / q is within d of 1, d the relative error of Z_p / Z_q (about 1e-7), each
// such token by d p at most: the pass sums the p of those within 2^-20 too, and
// where d times it exceeds 1e-11 of the total, or d 2^-20, it is made again with
// the corrected sums.
//
// Measured, 151,936 tokens, replayed graphs: a token of bf16 logits 9.9 us (a
// launch, two passes over 9,500 logits a CTA, three cluster barriers); four
// drafts of one sequence 20.0 us; 32 sequences of up to six drafts in float32
// 82 us, of which 38 are the first launch (reading the logits, 4.8 TB/s) and 44
// the second. That one issues 0.54 of a scheduler's slots (sixty instructions a
// warp's exponential, eight of them 64-bit; the 64-bit pipe is 23% busy) while
// its SMs are active, 75% of the time (256 CTAs for 296 places, and clusters
// that end apart), and waits for fixed latencies, loads (a segment ahead) and
// barriers besides. The sum that guards the choice of tokens is 2.4 us of it;
// with the rows' sums in a pass of their own it took 12 more. In bf16 the batch
// takes 91: half the bytes, but as many loads.
#include <cooperative_groups.h>
#include <cuda_bf16.h>

#include <algorithm>
#include <atomic>

#include "cdq_internal.cuh"

namespace cg = cooperative_groups;
using cdq::pdl_release;
using cdq::pdl_wait;

namespace {

constexpr int kVec = 4;                   // neighbouring tokens of a lane
constexpr int kSeg = 32 * kVec;           // tokens of a segment: one warp pass
constexpr int kMaxDrafts = CDQ_VERIFY_MAX_DRAFTS;
constexpr int kMaxRows = 2 * kMaxDrafts + 1;
constexpr int kMaxCluster = 16;
constexpr int kAhead = 4;                 // vectors of a lane in flight in the first launch
constexpr int kMaxParts = 32;             // parts of a row there
constexpr int kStatThreads = 256;
constexpr int kMaxWarps = 32;
// More than two rows' sums of the first launch are off by, relative. A term 2^-X of a row of 2^22 errs by 30 * 3 * 2^-24 ln 2
// at most in its exponent (differences, their product with 1 / (T ln 2), that factor; X up to 22 counts, and kLag twice)
// and 2^-22 in each of up to six exponentials (a rising reference passes log2 of the row / kLag times), 16 terms are
// added in float32 (6 * 2^-24) and these sums in 64 bits: 5.6e-6 a row.
constexpr double kNear = 2e-5;
constexpr float kLag = 4.f;    // log2 that a thread's reference may lie below its largest logit
constexpr double kChoice = 1e-11;  // of the total: what a wrong choice of tokens may cost
constexpr double kApart = 0x1p-20;  // of Z_p / Z_q: more makes the choice anew
constexpr int kAlike = 3;  // steps of the high words (2^-21 to 2^-20 of a number) between numbers kApart from each other
constexpr int kMaxSegs = (CDQ_VERIFY_MAX_VOCAB + kVec) / 8 / kSeg + 2;  // of a CTA, with 8 a sequence

struct RowPart {
    double sum;
    float max, pad;
};
static_assert(kAhead == 4, "sums of a turn");
static_assert(kMaxParts * sizeof(RowPart) == CDQ_VERIFY_ROW_BYTES, "workspace of a row");

struct VerifyArgs {
    const void *target, *draft;
    int64_t t_seq, t_row, d_seq, d_row;
    const int64_t* drafts;
    const float *u_accept, *u_sample;
    int64_t* tokens;
    int32_t* n_accepted;
    RowPart* stats;  // [batch][2 k + 1][parts]: target rows, then draft rows
    int32_t k, vocab, vecs;  // vecs: vectors that cover any row
    int32_t chunk, parts;  // tokens of a CTA, a multiple of kSeg; parts of a row
    double temperature;
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ float value(const uint16_t* p) { return __uint_as_float((uint32_t)__ldg(p) << 16); }
__device__ __forceinline__ float value(const float* p) { return __ldg(p); }

// A row of n logits as vectors of four that start at multiples of their size:
// vector i holds elements 4 i - shift .. 4 i - shift + 3, -inf outside the row.
template <typename T>
struct Row {
    const T* row;
    int shift, n, whole;  // vectors [shift > 0, whole) lie inside the row
    __device__ __forceinline__ Row(const T* r, int count, int s) : row(r), shift(s), n(count), whole((count + s) / kVec) {}
    __device__ __forceinline__ Row(const T* r, int count) : Row(r, count, (int)((uintptr_t)r / sizeof(T) % kVec)) {}
    __device__ __forceinline__ void load(int i, float (&x)[kVec]) const {
        const int j = i * kVec - shift;
        if (i < whole && j >= 0) {
            vector(row + j, x);
        } else {
#pragma unroll 1
            for (int e = 0; e < kVec; ++e) {  // (rolled: an edge of the row, shifted into place)
#pragma unroll
                for (int k = 0; k + 1 < kVec; ++k) x[k] = x[k + 1];
                x[kVec - 1] = j + e >= 0 && j + e < n ? value(row + j + e) : -INFINITY;
            }
        }
    }
    // as load, for a row of another alignment: element by element
    __device__ __forceinline__ void gather(int i, float (&x)[kVec]) const {
        const int j = i * kVec - shift;
#pragma unroll
        for (int e = 0; e < kVec; ++e) x[e] = j + e >= 0 && j + e < n ? value(row + j + e) : -INFINITY;
    }
    static __device__ __forceinline__ void vector(const uint16_t* p, float (&x)[kVec]) {
        const uint2 u = __ldg(reinterpret_cast<const uint2*>(p));
        x[0] = __uint_as_float(u.x << 16), x[1] = __uint_as_float(u.x & 0xFFFF0000u);
        x[2] = __uint_as_float(u.y << 16), x[3] = __uint_as_float(u.y & 0xFFFF0000u);
    }
    static __device__ __forceinline__ void vector(const float* p, float (&x)[kVec]) {
        const float4 a = __ldg(reinterpret_cast<const float4*>(p));
        x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w;
    }
};

__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
    return v;
}

// 2^(j / 32)
__device__ const double kRoots[32] = {
    0x1.0000000000000p+0, 0x1.059b0d3158574p+0, 0x1.0b5586cf9890fp+0, 0x1.11301d0125b51p+0,
    0x1.172b83c7d517bp+0, 0x1.1d4873168b9aap+0, 0x1.2387a6e756238p+0, 0x1.29e9df51fdee1p+0,
    0x1.306fe0a31b715p+0, 0x1.371a7373aa9cbp+0, 0x1.3dea64c123422p+0, 0x1.44e086061892dp+0,
    0x1.4bfdad5362a27p+0, 0x1.5342b569d4f82p+0, 0x1.5ab07dd485429p+0, 0x1.6247eb03a5585p+0,
    0x1.6a09e667f3bcdp+0, 0x1.71f75e8ec5f74p+0, 0x1.7a11473eb0187p+0, 0x1.82589994cce13p+0,
    0x1.8ace5422aa0dbp+0, 0x1.93737b0cdc5e5p+0, 0x1.9c49182a3f090p+0, 0x1.a5503b23e255dp+0,
    0x1.ae89f995ad3adp+0, 0x1.b7f76f2fb5e47p+0, 0x1.c199bdd85529cp+0, 0x1.cb720dcef9069p+0,
    0x1.d5818dcfba487p+0, 0x1.dfc97337b9b5fp+0, 0x1.ea4afa2a490dap+0, 0x1.f50765b6e4540p+0};

// 2^(d c) for d <= 0 in 64 bits, 0 below 2^-1000 (and of a NaN): d c = n / 32 + f with
// |f| <= 1/64, 2^f by its Taylor series to the fourth power (0.0109^5 / 120 =
// 1.3e-12 of the value), 2^((n mod 32) / 32) from lane n mod 32, which holds it
// in `table`, and n div 32 added to the exponent. Eight 64-bit operations,
// where the library's function takes two to three times as many (they run at a
// ninth of the 32-bit rate here); the sums that decide a token need 1e-11.
// The whole warp calls it.
__device__ __forceinline__ double exp2_64(double d, double c, double table) {
    constexpr double kLn2 = 0.69314718055994530942;
    constexpr double c1 = kLn2, c2 = c1 * kLn2 / 2, c3 = c2 * kLn2 / 3, c4 = c3 * kLn2 / 4;
    constexpr double kMagic = 211106232532992.0;  // 1.5 * 2^47: adding it rounds to a multiple of 1/32, n in the low bits
    const double t = fma(d, c, kMagic);
    const double f = fma(d, c, kMagic - t);
    // -n, as the two numbers' exponents are the same (huge for any other t: far below, -inf, NaN)
    const unsigned long long back = __double_as_longlong(kMagic) - __double_as_longlong(t);
    const int n = -(int)(unsigned)back;
    double y = fma(c4, f, c3);
    y = fma(y, f, c2);
    y = fma(y, f, c1);
    y = fma(y, f, 1.0);
    y *= __shfl_sync(0xFFFFFFFFu, table, n & 31);
    const bool in = back < 32000;
    return in ? __hiloint2double(__double2hiint(y) + (n >> 5) * (1 << 20), __double2loint(y)) : 0.0;
}

// Running sums of a warp's values, its own included.
__device__ __forceinline__ double warp_scan(double v, int lane) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const double y = __shfl_up_sync(0xFFFFFFFFu, v, o);
        if (lane >= o) v += y;
    }
    return v;
}
// The lane whose weight t > 0 takes the running sum past aim, before being
// the sum in front of each lane; the last lane with weight if none does; -1 if
// no lane has any. over: whether one does.
__device__ __forceinline__ int pick(double t, double before, double aim, bool* over) {
    const unsigned any = __ballot_sync(0xFFFFFFFFu, t > 0.0);
    const unsigned past = __ballot_sync(0xFFFFFFFFu, t > 0.0 && before + t > aim);
    *over = past != 0;
    return past ? __ffs(past) - 1 : 31 - __clz(any);
}

// Drafts of a sequence before the first negative one (the whole warp calls it).
__device__ __forceinline__ int drafts_given(const int64_t* x, int k, int lane) {
    int given = k;
    for (int i = lane; i < k; i += 32)
        if (x[i] < 0) given = min(given, i);
    return __reduce_min_sync(0xFFFFFFFFu, given);
}

// (part, row, sequence): the (max, sum) of a part of one row, kAhead vectors a
// thread a turn. A thread adds its turns' sums in 64 bits (in 32, thousands of
// equal terms all round the same way), under a reference that it raises by
// kLag or more at a time (a factor for each small rise would add up its
// rounding). Reading the logits once bounds it for large batches.
template <typename T>
__global__ void __launch_bounds__(kStatThreads) row_stats_kernel(const VerifyArgs A) {
    __shared__ float s_max[kStatThreads / 32];
    __shared__ double s_sum[kStatThreads / 32];
    pdl_wait();
    pdl_release();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, r = blockIdx.y;
    const int64_t b = blockIdx.z;
    const int given = drafts_given(A.drafts + b * A.k, A.k, lane);
    const bool drafted = r > A.k;
    if (drafted ? r - A.k - 1 >= given : r > given) return;  // a row that nothing asks for
    const Row<T> row(drafted ? static_cast<const T*>(A.draft) + b * A.d_seq + (r - A.k - 1) * A.d_row
                             : static_cast<const T*>(A.target) + b * A.t_seq + r * A.t_row, A.vocab);
    const float c = (float)(1.4426950408889634 / A.temperature);
    const int per = (A.vecs + A.parts - 1) / A.parts;
    const int lo = blockIdx.x * per, hi = min(lo + per, A.vecs);
    float top = -INFINITY, m = -INFINITY;  // the largest logit, the reference of s
    double s = 0.0;
    for (int i0 = lo + warp * 32; i0 < hi; i0 += kAhead * kStatThreads) {
        float v[kAhead][kVec];
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            const int i = i0 + lane + k * kStatThreads;
            if (i < hi) {
                row.load(i, v[k]);
            } else {
#pragma unroll
                for (int e = 0; e < kVec; ++e) v[k][e] = -INFINITY;
            }
        }
#pragma unroll
        for (int k = 0; k < kAhead; ++k)
#pragma unroll
            for (int e = 0; e < kVec; ++e) top = fmaxf(top, v[k][e]);
        // (differences first: the type's lowest value times c is no finite number)
        const float old = m;
        if ((top - m) * c > kLag) m = top;
        const float ref = m == -INFINITY ? 0.f : m;
        s *= ex2((old - ref) * c);  // (1 where the reference stays; under a branch a batch's first launch takes 13 us more)
        float y[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            y[k] = 0.f;
#pragma unroll
            for (int e = 0; e < kVec; ++e) y[k] += ex2((v[k][e] - ref) * c);
        }
        s += (y[0] + y[1]) + (y[2] + y[3]);
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
    if (lane == 0) s_max[warp] = top;
    __syncthreads();
    top = s_max[0];
#pragma unroll
    for (int w = 1; w < kStatThreads / 32; ++w) top = fmaxf(top, s_max[w]);
    s = warp_sum(s * (double)ex2((m - (top == -INFINITY ? 0.f : top)) * c));
    if (lane == 0) s_sum[warp] = s;
    __syncthreads();
    if (warp == 0) {
        s = warp_sum(lane < kStatThreads / 32 ? s_sum[lane] : 0.0);
        if (lane == 0) A.stats[(b * gridDim.y + r) * A.parts + blockIdx.x] = RowPart{s, top, 0.f};
    }
}

// A thread's share of a row's sum in 64 bits, vectors [lo, hi).
template <typename T, int THREADS>
__device__ __noinline__ double row_share(const T* p, int n, double top, double c64, double table, int lo, int hi) {
    const Row<T> row(p, n);
    double s = 0.0;
    for (int i0 = lo + (int)threadIdx.x / 32 * 32; i0 < hi; i0 += THREADS) {
        float v[kVec];
        row.load(i0 + (int)threadIdx.x % 32, v);
#pragma unroll
        for (int e = 0; e < kVec; ++e) s += exp2_64((double)v[e] - top, c64, table);
    }
    return s;
}

struct Shared {
    float2 top[kMaxCluster];             // sampling alone: every CTA's (max, 0 or NaN)
    double z[3][kMaxCluster], total[3][kMaxCluster], total_q[kMaxCluster];
    double warp_z[3][kMaxWarps];
    float2 warp_top[kMaxWarps];
    double row_sum[kMaxRows];
    float row_max[kMaxRows];
    int kept, ok, open;
};

// One cluster a sequence (blockIdx.y). CTAs exchange by writing into every
// other's shared memory before a cluster barrier, so that all reads are local.
// DRAFTS: k > 0 (a variant of its own, for what the first launch's 32-bit sums
// ask for takes registers: a sampled token is 9.9 us without it, 11.9 with it).
template <typename T, int THREADS, bool DRAFTS>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS) verify_kernel(const VerifyArgs A) {
    constexpr int kWarps = THREADS / 32;
    extern __shared__ double seg[];  // sums of this CTA's segments (two each)
    __shared__ Shared S;
    cg::cluster_group cluster = cg::this_cluster();
    const int rank = (int)cluster.block_rank(), ranks = (int)cluster.num_blocks();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int64_t b = blockIdx.y;
    cluster.barrier_arrive();  // (every CTA runs before any writes into another's shared memory)
    const double table = kRoots[lane];
    pdl_wait();
    pdl_release();
    const int n = A.vocab;
    const T* target = static_cast<const T*>(A.target) + b * A.t_seq;
    const T* draft = A.draft ? static_cast<const T*>(A.draft) + b * A.d_seq : nullptr;
    const int64_t* x = A.drafts + b * A.k;
    const int given = DRAFTS ? drafts_given(x, A.k, lane) : 0;
    const int rows = given + 1 + (draft ? given : 0);  // target rows 0 .. given, then draft rows
    const auto row_of = [&](int r) { return r <= given ? target + r * A.t_row : draft + (r - given - 1) * A.d_row; };
    const double c64 = 1.4426950408889634074 / A.temperature;
    const int vecs = A.chunk / kVec, v_lo = rank * vecs, v_hi = min(v_lo + vecs, A.vecs);

    // 1. every row's maximum and sum; what the drafts are decided by
    constexpr int kDraftLanes = (kMaxDrafts + 31) / 32;
    float tv[kDraftLanes], dv[kDraftLanes], ua[kDraftLanes];
    if (DRAFTS) {
        if (warp == 0) {
#pragma unroll
            for (int k = 0; k < kDraftLanes; ++k) {
                const int i = lane + 32 * k;
                const int64_t t = i < given ? x[i] : n;
                tv[k] = t < n ? value(row_of(i) + t) : -INFINITY;
                dv[k] = t < n && draft ? value(row_of(given + 1 + i) + t) : -INFINITY;
                ua[k] = i < given ? A.u_accept[b * A.k + i] : 0.f;
            }
        }
        const int all_rows = A.k + 1 + (draft ? A.k : 0);
        for (int r = warp; r < rows; r += kWarps) {
            const RowPart* part = A.stats + (b * all_rows + (r <= given ? r : r - given + A.k)) * A.parts;
            const RowPart one = lane < A.parts ? part[lane] : RowPart{0.0, -INFINITY, 0.f};
            float top = one.max;
#pragma unroll
            for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
            const float ref = top == -INFINITY ? 0.f : top;
            const double sum = warp_sum(one.sum * exp2_64((double)one.max - ref, c64, table));
            if (lane == 0) S.row_max[r] = top, S.row_sum[r] = sum;
        }
        cluster.barrier_wait();
    } else {
        const Row<T> row(target, n);
        float top = -INFINITY, bad = 0.f;
        for (int i0 = v_lo + warp * 32; i0 < v_hi; i0 += kAhead * THREADS) {
            float v[kAhead][kVec];
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                if (i0 + k * THREADS < v_hi) {
                    row.load(i0 + k * THREADS + lane, v[k]);
                } else {
#pragma unroll
                    for (int e = 0; e < kVec; ++e) v[k][e] = -INFINITY;
                }
            }
#pragma unroll
            for (int k = 0; k < kAhead; ++k)
#pragma unroll
                for (int e = 0; e < kVec; ++e) top = fmaxf(top, v[k][e]), bad += v[k][e] != v[k][e];
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) {
            top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
            bad += __shfl_xor_sync(0xFFFFFFFFu, bad, o);
        }
        if (lane == 0) S.warp_top[warp] = make_float2(top, bad);
        __syncthreads();
        cluster.barrier_wait();
        if (warp == 0) {
            float2 w = lane < kWarps ? S.warp_top[lane] : make_float2(-INFINITY, 0.f);
#pragma unroll
            for (int o = 16; o; o >>= 1) {
                w.x = fmaxf(w.x, __shfl_xor_sync(0xFFFFFFFFu, w.x, o));
                w.y += __shfl_xor_sync(0xFFFFFFFFu, w.y, o);
            }
            if (lane < ranks) *cluster.map_shared_rank(&S.top[rank], lane) = w;
        }
        cluster.sync();
        if (warp == 0) {
            float2 w = lane < ranks ? S.top[lane] : make_float2(-INFINITY, 0.f);
#pragma unroll
            for (int o = 16; o; o >>= 1) {
                w.x = fmaxf(w.x, __shfl_xor_sync(0xFFFFFFFFu, w.x, o));
                w.y += __shfl_xor_sync(0xFFFFFFFFu, w.y, o);
            }
            if (lane == 0) S.row_max[0] = w.x, S.row_sum[0] = w.y == 0.f && w.x > -INFINITY ? 1.0 : 0.0;
        }
    }
    __syncthreads();
    // a lane a draft: the first that is not kept, or has no distribution
    const auto has = [&](int r) {
        return S.row_sum[r] > 0.0 && S.row_sum[r] < (double)INFINITY && S.row_max[r] < INFINITY;
    };
    unsigned long long sure = 0;  // drafts whose rows have 64-bit sums
    for (;;) {
        if (warp == 0) {
            int a = given, bad = kMaxDrafts + 1, open = kMaxDrafts + 1;
#pragma unroll
            for (int k = 0; k < kDraftLanes; ++k) {
                const int i = lane + 32 * k, ti = min(i, given), di = draft ? given + 1 + min(i, given - 1) : ti;
                // u q < p, times both sums
                const double p = exp2_64((double)tv[k] - S.row_max[ti], c64, table) * (draft ? S.row_sum[di] : 1.0);
                const double q = draft ? exp2_64((double)dv[k] - S.row_max[di], c64, table) * S.row_sum[ti] : S.row_sum[ti];
                const double uq = (double)ua[k] * q;
                if (i < given) {
                    if (!has(i) || (draft && !has(di))) bad = min(bad, i);
                    else if (!(uq < p)) a = min(a, i);
                    if (DRAFTS && !(sure >> i & 1) && fabs(uq - p) < kNear * fmax(uq, p)) open = min(open, i);
                }
            }
            a = __reduce_min_sync(0xFFFFFFFFu, a);
            bad = __reduce_min_sync(0xFFFFFFFFu, bad);
            if (DRAFTS) open = __reduce_min_sync(0xFFFFFFFFu, open);
            if (lane == 0) {
                S.kept = min(a, bad);
                S.ok = bad > a && has(a);
                if (DRAFTS) S.open = open <= min(a, bad) ? open : -1;
            }
        }
        __syncthreads();
        if (!DRAFTS) break;
        const int i = S.open;
        if (i < 0) break;
        // too near for 32-bit sums: those of the draft's rows in 64 bits
        for (int r = 0; r < (draft ? 2 : 1); ++r) {
            const int x = r ? given + 1 + i : i;
            const double s = warp_sum(row_share<T, THREADS>(row_of(x), n, S.row_max[x], c64, table, v_lo, v_hi));
            if (lane == 0) S.warp_z[r][warp] = s;
        }
        __syncthreads();
        if (warp < (draft ? 2 : 1)) {
            const double s = warp_sum(lane < kWarps ? S.warp_z[warp][lane] : 0.0);
            if (lane < ranks) *cluster.map_shared_rank(&S.z[warp][rank], lane) = s;
        }
        cluster.sync();
        if (warp < (draft ? 2 : 1)) {
            const double s = warp_sum(lane < ranks ? S.z[warp][lane] : 0.0);
            if (lane == 0) S.row_sum[warp ? given + 1 + i : i] = s;
        }
        sure |= 1ull << i;
        cluster.sync();  // (and before any writes into S.z again)
    }
    const int a = S.kept;
    int64_t token = -1;
    bool mine = rank == 0;
    if (S.ok) {
        const bool refused = a < given;
        const T* prow = row_of(a);
        const T* qrow = refused && draft ? row_of(given + 1 + a) : nullptr;
        const int64_t gone = refused && !draft ? x[a] : -1;  // a greedily chosen draft that was refused
        const double pm = S.row_max[a], qm = qrow ? S.row_max[given + 1 + a] : 0.f;
        const Row<T> P(prow, n), Q(qrow ? qrow : prow, n, P.shift);
        const bool alike = ((uintptr_t)prow - (uintptr_t)Q.row) % (kVec * sizeof(T)) == 0;
        double izp = 1.0, izq = 1.0;
        if (qrow) izp = 1.0 / S.row_sum[a], izq = 1.0 / S.row_sum[given + 1 + a];
        // 2. the weights of a lane's four tokens; their sums by segment
        bool rest = qrow != nullptr || gone >= 0;
        const auto fetch = [&](int i0, float (&v)[kVec], float (&u)[kVec]) {
            P.load(i0, v);
            if (rest && qrow) {
                if (alike) Q.load(i0, u);
                else Q.gather(i0, u);
            }
        };
        const auto weights = [&](int i0, const float (&v)[kVec], const float (&u)[kVec], double (&w)[kVec]) {
            const bool two = rest && qrow;
#pragma unroll
            for (int i = 0; i < kVec; ++i) {
                w[i] = exp2_64((double)v[i] - pm, c64, table);
                // (two rounded products: of equal distributions nothing may remain)
                if (two)
                    w[i] = fmax(__dmul_rn(w[i], izp) - __dmul_rn(exp2_64((double)u[i] - qm, c64, table), izq), 0.0);
                else if (rest && i0 * kVec - P.shift + i == gone) w[i] = 0.0;
            }
        };
        const int segs = A.chunk / kSeg;
        double* const seg_q = seg + segs;
        // with 32-bit sums: both rows' shares of the tokens where p is the larger, and the rows' sums
        bool split = DRAFTS && qrow;
        double fp = 1.0, fq = 0.0;  // a segment's weight is fp seg - fq seg_q
        const auto weight = [&](double x, double y) { return DRAFTS && split ? fmax(__dmul_rn(x, fp) - __dmul_rn(y, fq), 0.0) : x; };
        double total = 0.0, mine_before = 0.0;
        int round = 0, owner;
        for (;; ++round) {
            float v[kVec], u[kVec], nv[kVec], nu[kVec];
            double sp = 0.0, sq = 0.0, alike_p = 0.0;
            if (warp < segs) fetch(v_lo + warp * 32 + lane, nv, nu);
            for (int s = warp; s < segs; s += kWarps) {
#pragma unroll
                for (int i = 0; i < kVec; ++i) v[i] = nv[i], u[i] = nu[i];
                if (s + kWarps < segs) fetch(v_lo + (s + kWarps) * 32 + lane, nv, nu);
                if (DRAFTS && split) {
                    double x = 0.0, y = 0.0;
#pragma unroll
                    for (int i = 0; i < kVec; ++i) {
                        const double p = exp2_64((double)v[i] - pm, c64, table), q = exp2_64((double)u[i] - qm, c64, table);
                        sp += p, sq += q;
                        const double wp = __dmul_rn(p, izp), wq = __dmul_rn(q, izq);
                        if (wp > wq) x += wp, y += wq;
                        if (abs(__double2hiint(wp) - __double2hiint(wq)) <= kAlike) alike_p += wp;
                    }
                    x = warp_sum(x), y = warp_sum(y);
                    if (lane == 0) seg[s] = x, seg_q[s] = y;
                } else {
                    double w[kVec];
                    weights(v_lo + s * 32 + lane, v, u, w);
                    const double t = warp_sum((w[0] + w[1]) + (w[2] + w[3]));
                    if (lane == 0) seg[s] = t;
                }
            }
            if (DRAFTS && split) {
                sp = warp_sum(sp), sq = warp_sum(sq), alike_p = warp_sum(alike_p);
                if (lane == 0) S.warp_z[0][warp] = sp, S.warp_z[1][warp] = sq, S.warp_z[2][warp] = alike_p;
            }
            __syncthreads();
            if (warp == 0 || (DRAFTS && split && warp == 1)) {
                const double* of = DRAFTS && warp ? seg_q : seg;
                double t = 0.0;
                for (int s = lane; s < segs; s += 32) t += of[s];
                t = warp_sum(t);
                if (lane < ranks) *cluster.map_shared_rank(DRAFTS && warp ? &S.total_q[rank] : &S.total[round][rank], lane) = t;
            } else if (DRAFTS && split && warp < 5) {
                const double t = warp_sum(lane < kWarps ? S.warp_z[warp - 2][lane] : 0.0);
                if (lane < ranks) *cluster.map_shared_rank(&S.z[warp - 2][rank], lane) = t;
            }
            cluster.sync();
            double t = lane < ranks ? S.total[round][lane] : 0.0, off = 0.0;
            if (DRAFTS && split) {
                const double zp = warp_sum(lane < ranks ? S.z[0][lane] : 0.0), zq = warp_sum(lane < ranks ? S.z[1][lane] : 0.0);
                fp = 1.0 / (zp * izp), fq = 1.0 / (zq * izq);
                off = fabs(fp - fq) > kApart ? 1.0 : fabs(fp - fq) * warp_sum(lane < ranks ? S.z[2][lane] : 0.0);
                izp = 1.0 / zp, izq = 1.0 / zq;
                t = weight(t, lane < ranks ? S.total_q[lane] : 0.0);
            }
            // the CTA that u * total falls into
            const double inc = warp_scan(t, lane);
            total = __shfl_sync(0xFFFFFFFFu, inc, 31);
            if (DRAFTS && split && off > kChoice * total) {
                split = false;  // too near to each other for 32-bit sums: once more with these
                continue;
            }
            if (total > 0.0 || !rest) {
                bool over;
                owner = pick(t, inc - t, (double)A.u_sample[b] * total, &over);
                mine_before = __shfl_sync(0xFFFFFFFFu, inc - t, max(owner, 0));
                break;
            }
            rest = split = false;  // the two distributions are the same to the last bit: draw from p
        }
        mine = rank == max(owner, 0);
        if (rank == owner && warp == 0) {
            const double aim = (double)A.u_sample[b] * total;
            // the segment: 32 sums at a time, a lane each
            double at = mine_before, seg_before = mine_before;
            int hit = 0;
            for (int s0 = 0; s0 < segs; s0 += 32) {
                const double t = s0 + lane < segs ? weight(seg[s0 + lane], DRAFTS && split ? seg_q[s0 + lane] : 0.0) : 0.0;
                const double inc = warp_scan(t, lane), before = at + (inc - t);
                bool over;
                const int who = pick(t, before, aim, &over);
                if (who >= 0) {
                    hit = s0 + who;
                    seg_before = __shfl_sync(0xFFFFFFFFu, before, who);
                }
                if (over) break;
                at += __shfl_sync(0xFFFFFFFFu, inc, 31);
            }
            // the lane, then the token
            float v[kVec], u[kVec];
            double w[kVec];
            const int i0 = v_lo + hit * 32 + lane;
            fetch(i0, v, u);
            weights(i0, v, u, w);
            const double t = (w[0] + w[1]) + (w[2] + w[3]);
            const double before = seg_before + (warp_scan(t, lane) - t);
            bool over;
            const int who = max(pick(t, before, aim, &over), 0);
            double r = before;
            int64_t found = (int64_t)i0 * kVec - P.shift;
            bool done = false;
#pragma unroll
            for (int i = 0; i < kVec; ++i) {
                if (!done && w[i] > 0.0) {
                    found = (int64_t)i0 * kVec - P.shift + i;
                    done = r + w[i] > aim;
                }
                r += w[i];
            }
            token = __shfl_sync(0xFFFFFFFFu, found, who);
        }
    }
    if (mine && warp == 0) {
        int64_t* out = A.tokens + b * (A.k + 1);
        for (int i = lane; i <= A.k; i += 32) out[i] = i < a ? x[i] : i == a ? token : -1;
        if (lane == 0 && A.n_accepted) A.n_accepted[b] = a;
    }
}

// The launch of a cluster of `ranks` CTAs for each of `batch` sequences.
struct Launch {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    Launch(int threads, int batch, int ranks, int chunk, cudaStream_t s) {
        cfg.gridDim = dim3(ranks, batch);
        cfg.blockDim = dim3(threads);
        cfg.dynamicSmemBytes = (size_t)(chunk / kSeg) * 2 * sizeof(double);
        cfg.stream = s;
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = ranks;
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[1].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 2;
    }
};

// Allows the kernel its clusters and shared memory on the current device, once.
template <typename T, int THREADS, bool DRAFTS>
cudaError_t prepare(int dev) {
    static std::atomic<uint64_t> ready[2];
    if (dev < 128 && ready[dev / 64].load() >> (dev % 64) & 1) return cudaSuccess;
    const auto kernel = verify_kernel<T, THREADS, DRAFTS>;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e == cudaSuccess)
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 2 * kMaxSegs * (int)sizeof(double));
    if (e == cudaSuccess && dev < 128) ready[dev / 64].fetch_or(1ull << (dev % 64));
    return e;
}

// Clusters of 16 CTAs of 1024 threads that the device runs at once.
template <typename T>
cudaError_t wide_clusters(int dev, int chunk, int* n) {
    static std::atomic<int> known[128];
    *n = dev < 128 ? known[dev].load() : 0;
    if (*n) return cudaSuccess;
    Launch L(1024, 1, kMaxCluster, chunk, nullptr);
    L.cfg.numAttrs = 1;
    const cudaError_t e = cudaOccupancyMaxActiveClusters(n, verify_kernel<T, 1024, false>, &L.cfg);
    if (e == cudaSuccess && dev < 128) known[dev].store(*n);
    return e;
}

template <typename T>
cudaError_t launch(VerifyArgs& A, int batch, cudaStream_t s) {
    int dev = 0, wide = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess) e = prepare<T, 1024, false>(dev);
    if (e == cudaSuccess) e = prepare<T, 512, false>(dev);
    if (e == cudaSuccess) e = prepare<T, 1024, true>(dev);
    if (e == cudaSuccess) e = prepare<T, 512, true>(dev);
    const auto chunk_of = [&](int ranks) {  // (a row may start inside its first vector)
        const int per = (A.vocab + kVec - 1 + ranks - 1) / ranks;
        return (per + kSeg - 1) / kSeg * kSeg;
    };
    A.chunk = chunk_of(kMaxCluster);
    if (e == cudaSuccess) e = wide_clusters<T>(dev, A.chunk, &wide);
    if (e != cudaSuccess) return e;
    // 16 CTAs of 1024 threads a sequence while all of them run at once, else 8
    // of 512, two a multiprocessor (151,936 tokens of bf16, four drafts, each
    // side as it was when they were compared: one sequence 19.3 us with 16,
    // 29.1 with 8; six 26.8 and 33.6; sampling from 8, more than run at once,
    // 18.4 and 17.0, from 32 44.4 and 21.1).
    const int ranks = batch <= wide ? kMaxCluster : 8;
    A.chunk = chunk_of(ranks);
    if (A.k) {
        const dim3 grid(A.parts, A.k + 1 + (A.draft ? A.k : 0), batch);
        e = cdq::launch_pdl(row_stats_kernel<T>, grid, dim3(kStatThreads), 0, s, A);
        if (e != cudaSuccess) return e;
    }
    Launch L(ranks == kMaxCluster ? 1024 : 512, batch, ranks, A.chunk, s);
    const auto wide_one = A.k ? verify_kernel<T, 1024, true> : verify_kernel<T, 1024, false>;
    const auto one = A.k ? verify_kernel<T, 512, true> : verify_kernel<T, 512, false>;
    return cudaLaunchKernelEx(&L.cfg, ranks == kMaxCluster ? wide_one : one, A);
}

// Parts of a row in the first launch: four CTAs a multiprocessor in all (of
// the 148 of a B200), none of less than two turns. Sums of another number of
// parts differ within kNear, which decides nothing by itself.
int parts_of(int64_t rows, int vecs) {
    const int64_t want = (4 * 148 + rows - 1) / rows, most = (vecs + 2 * kAhead * kStatThreads - 1) / (2 * kAhead * kStatThreads);
    return (int)std::max<int64_t>(1, std::min<int64_t>({want, most, kMaxParts}));
}

}  // namespace

extern "C" {

cdq_status cdq_verify_drafts(const void* target, int64_t t_seq, int64_t t_row, const void* draft, int64_t d_seq,
                             int64_t d_row, int32_t dtype, const int64_t* drafts, const float* u_accept,
                             const float* u_sample, int32_t batch, int32_t k, int32_t vocab, double temperature,
                             int64_t* tokens, int32_t* n_accepted, void* workspace, int64_t workspace_bytes,
                             void* stream) {
    if (dtype != 0 && dtype != 1) return CDQ_ERR_UNSUPPORTED;
    if (!target || !u_sample || !tokens || batch < 1 || batch > 65535 || k < 0 || k > kMaxDrafts || vocab < 1 ||
        vocab > CDQ_VERIFY_MAX_VOCAB)
        return CDQ_ERR_ARG;
    if (k && (!drafts || !u_accept)) return CDQ_ERR_ARG;
    if (!(temperature >= 1e-30) || !(temperature <= 1e30)) return CDQ_ERR_ARG;  // (float32 factors stay finite, above 0)
    const size_t el = dtype ? 4 : 2;
    if ((uintptr_t)drafts % 8 || (uintptr_t)tokens % 8 || (uintptr_t)u_accept % 4 || (uintptr_t)u_sample % 4 ||
        (uintptr_t)n_accepted % 4)
        return CDQ_ERR_ARG;
    if ((uintptr_t)target % el || (uintptr_t)draft % el || t_seq < 0 || t_row < 0 || d_seq < 0 || d_row < 0)
        return CDQ_ERR_ARG;
    if (!k) draft = nullptr;
    const int64_t rows = batch * (k + 1LL + (draft ? k : 0));
    if (k && (!workspace || (uintptr_t)workspace % 16 || workspace_bytes < rows * CDQ_VERIFY_ROW_BYTES))
        return CDQ_ERR_WORKSPACE;
    // one CTA writes a sequence's tokens while others still read its drafts
    if (k && tokens < drafts + (int64_t)batch * k && drafts < tokens + (int64_t)batch * (k + 1)) return CDQ_ERR_ARG;
    VerifyArgs A{target, draft, t_seq, t_row, d_seq, d_row, drafts, u_accept, u_sample, tokens, n_accepted,
                 static_cast<RowPart*>(workspace), k, vocab, (vocab + 2 * kVec - 2) / kVec, 0, 0, temperature};
    A.parts = parts_of(rows, A.vecs);
    const auto s = (cudaStream_t)stream;
    const cudaError_t e = dtype ? launch<float>(A, batch, s) : launch<uint16_t>(A, batch, s);
    return e == cudaSuccess ? CDQ_OK : CDQ_ERR_CUDA;
}

}  // extern "C"
