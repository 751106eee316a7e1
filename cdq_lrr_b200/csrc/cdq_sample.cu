// Verification of drafted tokens and sampling, from given random numbers.
//
// A cluster of CTAs serves one sequence, each CTA a contiguous part of the
// vocabulary, so that everything a sequence needs is exchanged through
// distributed shared memory in one launch without a workspace:
//   1. the (max, sum of 2^(x - max)) of every target and draft row, in
//      float32 with the CTAs' sums joined, decide which drafts are kept;
//   2. for the row that the drawn token comes from, Z_p (and Z_q) in 64 bits;
//   3. the weights e^(x - max)/Z, or max(p - q, 0), summed in 64 bits over
//      segments of 256 tokens, give the total; the segment that u * total
//      falls into is scanned.
// A drawn token is the one side of a border that a number falls on, and with
// a flat distribution over 10^5 tokens sums that err by 1e-7 put it on the
// wrong side of one in every few hundred draws: hence 64 bits in 2 and 3,
// for the one row (two with a draft's) that is drawn from. A kept draft is a
// single comparison, which float32 sums decide wrongly once in about 10^6.
#include <cooperative_groups.h>
#include <cuda_bf16.h>

#include <algorithm>

#include "cdq_internal.cuh"

namespace cg = cooperative_groups;
using cdq::pdl_release;
using cdq::pdl_wait;

namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kVec = 8;                   // neighbouring tokens of a lane
constexpr int kSeg = 32 * kVec;           // tokens of a segment: one warp pass
constexpr int kTile = kWarps * kSeg;      // tokens of a CTA pass
constexpr int kMaxDrafts = CDQ_VERIFY_MAX_DRAFTS;
constexpr int kMaxRows = 2 * kMaxDrafts + 1;
constexpr int kMaxCluster = 16;
constexpr int kMaxTasks = 256;            // (row, part) tasks of a CTA's first step: at least kMaxRows
constexpr int kAhead = 4;                 // vectors of a lane in flight there

struct VerifyArgs {
    const void *target, *draft;
    int64_t t_seq, t_row, d_seq, d_row;
    const int64_t* drafts;
    const float *u_accept, *u_sample;
    int64_t* tokens;
    int32_t* n_accepted;
    int32_t k, vocab, chunk;  // chunk: tokens of a CTA, a multiple of kSeg
    double temperature;
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ float value(const uint16_t* p) { return __uint_as_float((uint32_t)__ldg(p) << 16); }
__device__ __forceinline__ float value(const float* p) { return __ldg(p); }

// elements that a row's start lies behind a 16-byte boundary
template <typename T>
__device__ __forceinline__ int row_shift(const T* row) {
    return (int)(((uintptr_t)row % 16) / sizeof(T));
}

// x[j0 .. j0 + 7], -inf outside [0, n); 16-byte loads where the eight are whole and aligned
__device__ __forceinline__ void load8(const uint16_t* row, int64_t j0, int n, float (&x)[kVec]) {
    if (j0 >= 0 && j0 + kVec <= n && (uintptr_t)(row + j0) % 16 == 0) {
        const uint4 u = __ldg(reinterpret_cast<const uint4*>(row + j0));
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[2 * i] = __uint_as_float(w[i] << 16);
            x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
        }
    } else {
#pragma unroll
        for (int i = 0; i < kVec; ++i) x[i] = j0 + i >= 0 && j0 + i < n ? value(row + j0 + i) : -INFINITY;
    }
}
__device__ __forceinline__ void load8(const float* row, int64_t j0, int n, float (&x)[kVec]) {
    if (j0 >= 0 && j0 + kVec <= n && (uintptr_t)(row + j0) % 16 == 0) {
        const float4 a = __ldg(reinterpret_cast<const float4*>(row + j0));
        const float4 b = __ldg(reinterpret_cast<const float4*>(row + j0) + 1);
        x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
    } else {
#pragma unroll
        for (int i = 0; i < kVec; ++i) x[i] = j0 + i >= 0 && j0 + i < n ? value(row + j0 + i) : -INFINITY;
    }
}

__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
    return v;
}

// 2^z for z <= 0 in 64 bits: z = i + f with |f| <= 1/2, the Taylor series of
// e^(f ln 2) to the tenth power (0.3466^11 / 11! = 2e-13 of the value), and i
// added to the exponent; 0 below 2^-1000. Fourteen 64-bit operations, all
// multiply-adds, where the library's function takes about twice as many; the
// sums that decide a token need 1e-11.
__device__ __forceinline__ double exp2_64(double z) {
    constexpr double kLn2 = 0.69314718055994530942;
    constexpr double c1 = kLn2, c2 = c1 * kLn2 / 2, c3 = c2 * kLn2 / 3, c4 = c3 * kLn2 / 4, c5 = c4 * kLn2 / 5,
                     c6 = c5 * kLn2 / 6, c7 = c6 * kLn2 / 7, c8 = c7 * kLn2 / 8, c9 = c8 * kLn2 / 9, c10 = c9 * kLn2 / 10;
    constexpr double kMagic = 6755399441055744.0;  // 1.5 * 2^52: adding it rounds to a whole number in the low bits
    const double t = z + kMagic;
    const double f = z - (t - kMagic);
    double y = fma(c10, f, c9);
    y = fma(y, f, c8);
    y = fma(y, f, c7);
    y = fma(y, f, c6);
    y = fma(y, f, c5);
    y = fma(y, f, c4);
    y = fma(y, f, c3);
    y = fma(y, f, c2);
    y = fma(y, f, c1);
    y = fma(y, f, 1.0);
    const int i = __double2loint(t);
    return z > -1000.0 ? __hiloint2double(__double2hiint(y) + i * (1 << 20), __double2loint(y)) : 0.0;
}

struct Shared {
    float2 part[kMaxCluster][kMaxRows];  // every CTA's (max, sum) of each row, written by that CTA
    double z[kMaxCluster][2], total[2][kMaxCluster];
    double warp_z[kWarps][2];
    float row_max[kMaxRows], row_sum[kMaxRows];
    float2 task[kMaxTasks];              // (max, sum) of each task of the first step
    int kept, ok;
};

// One cluster a sequence (blockIdx.y). CTAs exchange by writing into every
// other's shared memory before a cluster barrier, so that all reads are local.
template <typename T>
__global__ void __launch_bounds__(kThreads, 2) verify_kernel(const VerifyArgs A) {
    extern __shared__ double seg[];  // sums of this CTA's segments
    __shared__ Shared S;
    cg::cluster_group cluster = cg::this_cluster();
    const int rank = (int)cluster.block_rank(), ranks = (int)cluster.num_blocks();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int64_t b = blockIdx.y;
    cluster.barrier_arrive();  // (every CTA runs before any writes into another's shared memory)
    pdl_wait();
    pdl_release();
    const int n = A.vocab;
    const T* target = static_cast<const T*>(A.target) + b * A.t_seq;
    const T* draft = A.draft ? static_cast<const T*>(A.draft) + b * A.d_seq : nullptr;
    const int64_t* x = A.k ? A.drafts + b * A.k : nullptr;
    int given = A.k;  // drafts before the first negative one
    if (A.k) {
        for (int i = lane; i < A.k; i += 32)
            if (x[i] < 0) given = min(given, i);
        given = __reduce_min_sync(0xFFFFFFFFu, given);
    }
    const int rows = given + 1 + (draft ? given : 0);  // target rows 0 .. given, then draft rows
    const auto row_of = [&](int r) { return r <= given ? target + r * A.t_row : draft + (r - given - 1) * A.d_row; };
    const float c = (float)(1.4426950408889634 / A.temperature);

    // 1. (max, sum) of every row: its part of this CTA in `parts` tasks of a
    // warp, four vectors of a lane in flight
    const int parts = max(1, min(kMaxTasks / rows, (4 * kWarps + rows - 1) / rows));
    const int per_task = (A.chunk / kVec + parts - 1) / parts;  // vectors
    for (int task = warp; task < rows * parts; task += kWarps) {
        const int r = task / parts, q = task % parts;
        const T* row = row_of(r);
        const int64_t j_lo = (int64_t)rank * A.chunk - row_shift(row);
        const int v_hi = min((q + 1) * per_task, A.chunk / kVec);
        float m = -INFINITY, s = 0.f;
        for (int i0 = q * per_task + lane; i0 < v_hi; i0 += 32 * kAhead) {
            float v[kAhead][kVec];
            float top = m;
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                const int i = i0 + 32 * k;
                load8(row, i < v_hi ? j_lo + (int64_t)i * kVec : (int64_t)n, n, v[k]);
            }
#pragma unroll
            for (int k = 0; k < kAhead; ++k)
#pragma unroll
                for (int e = 0; e < kVec; ++e) top = fmaxf(top, v[k][e]);
            // (differences first: the type's lowest value times c is no finite number)
            const float ref = top == -INFINITY ? 0.f : top;
            s *= ex2((m - ref) * c);
            m = top;
#pragma unroll
            for (int k = 0; k < kAhead; ++k)
#pragma unroll
                for (int e = 0; e < kVec; ++e) s += ex2((v[k][e] - ref) * c);
        }
        float top = m;
#pragma unroll
        for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
        s *= top == -INFINITY ? 1.f : ex2((m - top) * c);
#pragma unroll
        for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
        if (lane == 0) S.task[task] = make_float2(top, s);
    }
    __syncthreads();
    cluster.barrier_wait();
    for (int i = tid; i < rows * ranks; i += kThreads) {  // one row to one CTA
        const int r = i / ranks, q = i % ranks;
        float top = -INFINITY, s = 0.f;
        for (int t = 0; t < parts; ++t) top = fmaxf(top, S.task[r * parts + t].x);
        for (int t = 0; t < parts; ++t)
            s += S.task[r * parts + t].y * (top == -INFINITY ? 1.f : ex2((S.task[r * parts + t].x - top) * c));
        *cluster.map_shared_rank(&S.part[rank][r], q) = make_float2(top, s);
    }
    cluster.sync();
    for (int r = tid; r < rows; r += kThreads) {
        float top = -INFINITY, s = 0.f;
        for (int q = 0; q < ranks; ++q) top = fmaxf(top, S.part[q][r].x);
        for (int q = 0; q < ranks; ++q)
            s += S.part[q][r].y * (top == -INFINITY ? 1.f : ex2((S.part[q][r].x - top) * c));
        S.row_max[r] = top;
        S.row_sum[r] = s;
    }
    __syncthreads();
    // a lane a draft: the first that is not kept, or has no distribution
    const auto has = [&](int r) { return S.row_sum[r] > 0.f && S.row_sum[r] < INFINITY && S.row_max[r] < INFINITY; };
    if (warp == 0) {
        int a = given, bad = kMaxDrafts + 1;
        for (int i = lane; i < given; i += 32) {
            if (!has(i) || (draft && !has(given + 1 + i))) {
                bad = min(bad, i);
                continue;
            }
            const int64_t t = x[i];
            double p = 0.0, q = draft ? 0.0 : 1.0;
            if (t < n) {
                p = exp(((double)value(row_of(i) + t) - S.row_max[i]) / A.temperature) / S.row_sum[i];
                if (draft)
                    q = exp(((double)value(row_of(given + 1 + i) + t) - S.row_max[given + 1 + i]) / A.temperature) /
                        S.row_sum[given + 1 + i];
            }
            if (!((double)A.u_accept[b * A.k + i] * q < p)) a = min(a, i);
        }
        a = __reduce_min_sync(0xFFFFFFFFu, a);
        bad = __reduce_min_sync(0xFFFFFFFFu, bad);
        if (lane == 0) {
            S.kept = min(a, bad);
            S.ok = bad > a && has(a);
        }
    }
    __syncthreads();
    const int a = S.kept;
    int64_t token = -1;
    bool mine = rank == 0;
    if (S.ok) {
        const bool refused = a < given;
        const T* prow = row_of(a);
        const T* qrow = refused && draft ? row_of(given + 1 + a) : nullptr;
        const int64_t gone = refused && !draft ? x[a] : -1;  // a greedily chosen draft that was refused
        const double c64 = 1.4426950408889634074 / A.temperature;
        const double pm = S.row_max[a], qm = qrow ? S.row_max[given + 1 + a] : 0.f;
        const int64_t j_lo = (int64_t)rank * A.chunk - row_shift(prow), j_hi = min(j_lo + A.chunk, (int64_t)n);
        double izp = 1.0, izq = 1.0;
        if (qrow) {
            // 2. the normalising sums, needed where two distributions are subtracted
            double sp = 0.0, sq = 0.0;
            for (int64_t j = j_lo + warp * kSeg + lane * kVec; j < j_hi; j += kTile) {
                float v[kVec], w[kVec];
                load8(prow, j, n, v);
                load8(qrow, j, n, w);
#pragma unroll
                for (int i = 0; i < kVec; ++i) {
                    sp += exp2_64(((double)v[i] - pm) * c64);
                    sq += exp2_64(((double)w[i] - qm) * c64);
                }
            }
            sp = warp_sum(sp);
            sq = warp_sum(sq);
            if (lane == 0) S.warp_z[warp][0] = sp, S.warp_z[warp][1] = sq;
            __syncthreads();
            if (tid < 2 * ranks) {
                double t = 0.0;
                for (int w = 0; w < kWarps; ++w) t += S.warp_z[w][tid & 1];
                *cluster.map_shared_rank(&S.z[rank][tid & 1], tid >> 1) = t;
            }
            cluster.sync();
            double zp = 0.0, zq = 0.0;
            for (int q = 0; q < ranks; ++q) zp += S.z[q][0], zq += S.z[q][1];
            izp = 1.0 / zp;
            izq = 1.0 / zq;
        }
        // 3. the weights of eight tokens; their sums by segment
        bool rest = qrow != nullptr || gone >= 0;
        const auto weights = [&](int64_t j, double (&w)[kVec]) {
            float v[kVec], u[kVec];
            load8(prow, j, n, v);
            if (rest && qrow) load8(qrow, j, n, u);
#pragma unroll
            for (int i = 0; i < kVec; ++i) {
                w[i] = exp2_64(((double)v[i] - pm) * c64);
                if (rest) {
                    // (two rounded products: of equal distributions nothing may remain)
                    if (qrow)
                        w[i] = fmax(__dmul_rn(w[i], izp) - __dmul_rn(exp2_64(((double)u[i] - qm) * c64), izq), 0.0);
                    else if (j + i == gone) w[i] = 0.0;
                }
            }
        };
        const int segs = A.chunk / kSeg;
        double total = 0.0;
        int round = 0;
        for (;; ++round) {
            for (int s = warp; s < segs; s += kWarps) {
                double w[kVec], t = 0.0;
                const int64_t j = j_lo + s * kSeg + lane * kVec;
                if (j < j_hi) {
                    weights(j, w);
#pragma unroll
                    for (int i = 0; i < kVec; ++i) t += w[i];
                }
                t = warp_sum(t);
                if (lane == 0) seg[s] = t;
            }
            __syncthreads();
            if (warp == 0) {
                double t = 0.0;
                for (int s = lane; s < segs; s += 32) t += seg[s];
                t = warp_sum(t);
                if (lane < ranks) *cluster.map_shared_rank(&S.total[round][rank], lane) = t;
            }
            cluster.sync();
            total = 0.0;
            for (int q = 0; q < ranks; ++q) total += S.total[round][q];
            if (total > 0.0 || !rest) break;
            rest = false;  // the two distributions are the same to the last bit: draw from p
        }
        // the CTA that u * total falls into (the last with weight where rounding passes them all)
        const double aim = (double)A.u_sample[b] * total;
        double run = 0.0, before = 0.0;
        int owner = -1;
        for (int q = 0; q < ranks; ++q) {
            const double t = S.total[round][q];
            if (t > 0.0 && (owner < 0 || before + S.total[round][owner] <= aim)) owner = q, before = run;
            run += t;
        }
        mine = rank == owner;
        if (mine && warp == 0) {
            // the segment: 32 sums at a time, a lane each
            double at = before, seg_before = before;
            int hit = -1;
            for (int s0 = 0; s0 < segs; s0 += 32) {
                const double t = s0 + lane < segs ? seg[s0 + lane] : 0.0;
                double inc = t;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const double y = __shfl_up_sync(0xFFFFFFFFu, inc, o);
                    if (lane >= o) inc += y;
                }
                const double mine_before = at + (inc - t);
                const unsigned any = __ballot_sync(0xFFFFFFFFu, t > 0.0);
                const unsigned over = __ballot_sync(0xFFFFFFFFu, t > 0.0 && mine_before + t > aim);
                if (any) {
                    const int who = over ? __ffs(over) - 1 : 31 - __clz(any);
                    hit = s0 + who;
                    seg_before = __shfl_sync(0xFFFFFFFFu, mine_before, who);
                }
                if (over) break;
                at += __shfl_sync(0xFFFFFFFFu, inc, 31);
            }
            double w[kVec], t = 0.0;
            const int64_t j = j_lo + (int64_t)hit * kSeg + lane * kVec;
            if (j < j_hi) weights(j, w);
            else
                for (int i = 0; i < kVec; ++i) w[i] = 0.0;
#pragma unroll
            for (int i = 0; i < kVec; ++i) t += w[i];
            double inc = t;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const double y = __shfl_up_sync(0xFFFFFFFFu, inc, o);
                if (lane >= o) inc += y;
            }
            const double lane_before = seg_before + (inc - t);
            const unsigned any = __ballot_sync(0xFFFFFFFFu, t > 0.0);
            const unsigned over = __ballot_sync(0xFFFFFFFFu, t > 0.0 && lane_before + t > aim);
            const int who = over ? __ffs(over) - 1 : any ? 31 - __clz(any) : 0;
            double r = lane_before;
            int64_t found = j;
            bool done = false;
#pragma unroll
            for (int i = 0; i < kVec; ++i) {
                if (!done && w[i] > 0.0) {
                    found = j + i;
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

template <typename T>
cudaError_t launch(const VerifyArgs& A, int batch, int ranks, size_t smem, cudaStream_t s) {
    static bool wide[128] = {};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= 128 || !wide[dev]) {
        e = cudaFuncSetAttribute(verify_kernel<T>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (e != cudaSuccess) return e;
        if (dev >= 0 && dev < 128) wide[dev] = true;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ranks, batch);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = ranks;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, verify_kernel<T>, A);
}

}  // namespace

extern "C" cdq_status cdq_verify_drafts(const void* target, int64_t t_seq, int64_t t_row, const void* draft,
                                        int64_t d_seq, int64_t d_row, int32_t dtype, const int64_t* drafts,
                                        const float* u_accept, const float* u_sample, int32_t batch, int32_t k,
                                        int32_t vocab, double temperature, int64_t* tokens, int32_t* n_accepted,
                                        void* stream) {
    if (dtype != 0 && dtype != 1) return CDQ_ERR_UNSUPPORTED;
    if (!target || !u_sample || !tokens || batch < 1 || batch > 65535 || k < 0 || k > kMaxDrafts || vocab < 1 ||
        vocab > CDQ_VERIFY_MAX_VOCAB)
        return CDQ_ERR_ARG;
    if (k && (!drafts || !u_accept)) return CDQ_ERR_ARG;
    if (!(temperature > 0.0) || !(temperature < INFINITY)) return CDQ_ERR_ARG;
    const size_t el = dtype ? 4 : 2;
    if ((uintptr_t)target % el || (uintptr_t)draft % el || t_seq < 0 || t_row < 0 || d_seq < 0 || d_row < 0)
        return CDQ_ERR_ARG;
    // 16 CTAs a sequence while the batch leaves multiprocessors idle, else 8
    const int ranks = batch <= 8 ? 16 : 8;
    VerifyArgs A{target, draft, t_seq, t_row, d_seq, d_row, drafts, u_accept, u_sample, tokens, n_accepted,
                 k, vocab, 0, temperature};
    const int per = (vocab + 7 + ranks - 1) / ranks;  // a row may start up to 7 elements into its first vector
    A.chunk = (per + kSeg - 1) / kSeg * kSeg;
    const size_t smem = (size_t)(A.chunk / kSeg) * sizeof(double);
    const auto s = (cudaStream_t)stream;
    const cudaError_t e = dtype ? launch<float>(A, batch, ranks, smem, s) : launch<uint16_t>(A, batch, ranks, smem, s);
    return e == cudaSuccess ? CDQ_OK : CDQ_ERR_CUDA;
}
