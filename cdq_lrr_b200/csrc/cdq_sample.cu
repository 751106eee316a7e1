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

struct Shared {
    float2 part[kMaxRows];          // this CTA's (max, sum) of each row, read by the cluster
    double z[2], total;             // this CTA's part of Z_p, Z_q and of the weights
    float2 warp_part[kWarps][kMaxRows];
    double warp_z[kWarps][2];
    float row_max[kMaxRows], row_sum[kMaxRows];
    int kept, ok;
};

// One cluster a sequence (blockIdx.y).
template <typename T>
__global__ void __launch_bounds__(kThreads) verify_kernel(const VerifyArgs A) {
    extern __shared__ double seg[];  // sums of this CTA's segments
    __shared__ Shared S;
    cg::cluster_group cluster = cg::this_cluster();
    const int rank = (int)cluster.block_rank(), ranks = (int)cluster.num_blocks();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int64_t b = blockIdx.y;
    pdl_wait();
    pdl_release();
    const int n = A.vocab;
    const T* target = static_cast<const T*>(A.target) + b * A.t_seq;
    const T* draft = A.draft ? static_cast<const T*>(A.draft) + b * A.d_seq : nullptr;
    const int64_t* x = A.k ? A.drafts + b * A.k : nullptr;
    int given = 0;  // drafts before the first negative one
    while (given < A.k && x[given] >= 0) ++given;
    const int rows = given + 1 + (draft ? given : 0);  // target rows 0 .. given, then draft rows
    const auto row_of = [&](int r) { return r <= given ? target + r * A.t_row : draft + (r - given - 1) * A.d_row; };
    const float c = (float)(1.4426950408889634 / A.temperature);

    // 1. (max, sum) of every row
    for (int r = 0; r < rows; ++r) {
        const T* row = row_of(r);
        const int64_t j_lo = (int64_t)rank * A.chunk - row_shift(row), j_hi = min(j_lo + A.chunk, (int64_t)n);
        float m = -INFINITY, s = 0.f;
        for (int64_t j = j_lo + warp * kSeg + lane * kVec; j < j_hi; j += kTile) {
            float v[kVec];
            load8(row, j, n, v);
            float top = m;
#pragma unroll
            for (int i = 0; i < kVec; ++i) top = fmaxf(top, v[i]);
            // (differences first: the type's lowest value times c is no finite number)
            const float ref = top == -INFINITY ? 0.f : top;
            s *= ex2((m - ref) * c);
            m = top;
#pragma unroll
            for (int i = 0; i < kVec; ++i) s += ex2((v[i] - ref) * c);
        }
        float top = m;
#pragma unroll
        for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
        s *= top == -INFINITY ? 1.f : ex2((m - top) * c);
#pragma unroll
        for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
        if (lane == 0) S.warp_part[warp][r] = make_float2(top, s);
    }
    __syncthreads();
    for (int r = tid; r < rows; r += kThreads) {
        float top = -INFINITY, s = 0.f;
        for (int w = 0; w < kWarps; ++w) top = fmaxf(top, S.warp_part[w][r].x);
        for (int w = 0; w < kWarps; ++w)
            s += S.warp_part[w][r].y * (top == -INFINITY ? 1.f : ex2((S.warp_part[w][r].x - top) * c));
        S.part[r] = make_float2(top, s);
    }
    cluster.sync();
    for (int r = tid; r < rows; r += kThreads) {
        float2 p[kMaxCluster];
        float top = -INFINITY, s = 0.f;
        for (int q = 0; q < ranks; ++q) {
            p[q] = *cluster.map_shared_rank(&S.part[r], q);
            top = fmaxf(top, p[q].x);
        }
        for (int q = 0; q < ranks; ++q) s += p[q].y * (top == -INFINITY ? 1.f : ex2((p[q].x - top) * c));
        S.row_max[r] = top;
        S.row_sum[r] = s;
    }
    __syncthreads();
    const auto has = [&](int r) { return S.row_sum[r] > 0.f && S.row_sum[r] < INFINITY && S.row_max[r] < INFINITY; };
    if (tid == 0) {
        int a = 0, ok = 1;
        for (; a < given; ++a) {
            if (!has(a) || (draft && !has(given + 1 + a))) {
                ok = 0;
                break;
            }
            const int64_t t = x[a];
            double p = 0.0, q = draft ? 0.0 : 1.0;
            if (t < n) {
                p = exp(((double)value(row_of(a) + t) - S.row_max[a]) / A.temperature) / S.row_sum[a];
                if (draft)
                    q = exp(((double)value(row_of(given + 1 + a) + t) - S.row_max[given + 1 + a]) / A.temperature) /
                        S.row_sum[given + 1 + a];
            }
            if (!((double)A.u_accept[b * A.k + a] * q < p)) break;
        }
        S.kept = a;
        S.ok = ok && has(a);
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
        const double pm = S.row_max[a], qm = qrow ? S.row_max[given + 1 + a] : 0.f;
        const double inv_t = 1.0 / A.temperature;
        const int64_t j_lo = (int64_t)rank * A.chunk - row_shift(prow), j_hi = min(j_lo + A.chunk, (int64_t)n);
        double zp = 1.0, zq = 1.0;
        if (qrow) {
            // 2. the normalising sums, needed where two distributions are subtracted
            double sp = 0.0, sq = 0.0;
            for (int64_t j = j_lo + warp * kSeg + lane * kVec; j < j_hi; j += kTile) {
                float v[kVec], w[kVec];
                load8(prow, j, n, v);
                load8(qrow, j, n, w);
#pragma unroll
                for (int i = 0; i < kVec; ++i) {
                    sp += exp(((double)v[i] - pm) * inv_t);
                    sq += exp(((double)w[i] - qm) * inv_t);
                }
            }
            sp = warp_sum(sp);
            sq = warp_sum(sq);
            if (lane == 0) S.warp_z[warp][0] = sp, S.warp_z[warp][1] = sq;
            __syncthreads();
            if (tid < 2) {
                double t = 0.0;
                for (int w = 0; w < kWarps; ++w) t += S.warp_z[w][tid];
                S.z[tid] = t;
            }
            cluster.sync();
            zp = zq = 0.0;
            for (int q = 0; q < ranks; ++q) {
                zp += *cluster.map_shared_rank(&S.z[0], q);
                zq += *cluster.map_shared_rank(&S.z[1], q);
            }
        }
        // 3. the weights of eight tokens; their sums by segment
        bool rest = qrow != nullptr || gone >= 0;
        const auto weights = [&](int64_t j, double (&w)[kVec]) {
            float v[kVec], u[kVec];
            load8(prow, j, n, v);
            if (rest && qrow) load8(qrow, j, n, u);
#pragma unroll
            for (int i = 0; i < kVec; ++i) {
                w[i] = exp(((double)v[i] - pm) * inv_t);
                if (rest) {
                    if (qrow) w[i] = fmax(w[i] / zp - exp(((double)u[i] - qm) * inv_t) / zq, 0.0);
                    else if (j + i == gone) w[i] = 0.0;
                }
            }
        };
        const int segs = A.chunk / kSeg;
        double total = 0.0, before = 0.0;
        int last = -1, owner = -1;
        for (;;) {
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
                if (lane == 0) S.total = t;
            }
            cluster.sync();
            total = 0.0;
            for (int q = 0; q < ranks; ++q) total += *cluster.map_shared_rank(&S.total, q);
            if (total > 0.0 || !rest) break;
            cluster.sync();  // every CTA has read the totals
            rest = false;    // the two distributions are the same to the last bit: draw from p
        }
        // the CTA that u * total falls into, and the last one that holds any weight
        const double aim = (double)A.u_sample[b] * total;
        double run = 0.0;
        for (int q = 0; q < ranks; ++q) {
            const double t = *cluster.map_shared_rank(&S.total, q);
            if (owner < 0 && t > 0.0) {
                last = q;
                before = run;
                if (run + t > aim) owner = q;
            }
            run += t;
        }
        if (owner < 0) owner = last;
        mine = rank == owner;
        if (mine && warp == 0) {
            // the segment, then the token; the last one with weight where rounding passes them all
            double at = before, seg_before = before;
            int hit = -1, last_seg = 0;
            for (int s = 0; s < segs; ++s) {
                if (seg[s] > 0.0) {
                    last_seg = s;
                    seg_before = at;
                    if (at + seg[s] > aim) {
                        hit = s;
                        break;
                    }
                }
                at += seg[s];
            }
            if (hit < 0) hit = last_seg;
            double w[kVec], t = 0.0;
            const int64_t j = j_lo + hit * kSeg + lane * kVec;
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
    cluster.sync();  // no CTA leaves while another may read its shared memory
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
