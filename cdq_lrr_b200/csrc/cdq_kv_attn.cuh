// What the two attention kernels over the quantised cache share: how the
// positions of a batch are shared out over CTAs, and where partial results go.
#pragma once

#include "cdq_internal.cuh"
#include "cdq_kv.cuh"

namespace cdq {
namespace kv {

constexpr int kUnit = 128;             // positions of the unit of work
constexpr float kBelow = 7.f;          // M is set this far (log2) below the largest s_j + log2 scale_v[j],
constexpr float kLazy = 15.f;          // and raised only when it lags by more than this
constexpr float kLeast = -83.f;        // log2 of a value scale, at least (see cdq_kv_attn.cu)
constexpr int kMeta = 4;               // floats in front of a partial's accumulators: (M, l, -, -)

// One pass over a cache: every (sequence, kv head, row tile) is a segment of
// ceil(len / kUnit) units (one where len is 0) behind `lead` blank ones, which
// stand for what it costs a CTA to begin and to finish with one; in that order,
// CTA i takes the i-th ceil(U / ctas) of all U units, so that ragged batches
// load every multiprocessor alike. A segment that one CTA has whole goes to the output
// (or to its rows' records, where another pass adds to them); of one that is
// cut, each CTA leaves its part in one of its two slots: 0 if the segment
// holds the CTA's first unit, else 1. The first CTA leaves the units a CTA
// takes, and each sequence's first unit, for the launch that joins the parts.
struct Pass {
    cdq_kv_cache c;
    const int32_t* prefix_len;  // set: c is the prefix, one "sequence" whose rows span the batch
    float* slots;               // [ctas][2][tile rows][kMeta + HD]
    float* recs;                // [row][kMeta + HD]; null: whole segments are final
    uint32_t* share;            // [1 + sequences]: units a CTA, first unit of each sequence (null: nothing to join)
    int32_t ctas, tiles, tile_rows, lead;
};

struct AttnArgs {
    Pass p;
    Pass also;  // of the CTAs behind p.ctas, where the launch has any
    const uint16_t* q;
    int64_t q_seq, q_tok;
    const int32_t* pos;
    Rope rope;
    uint16_t* out;
    float scale_log2;
    int32_t batch, n_q, n_heads, group, max_len;
    int32_t cluster;  // CTAs of a cluster that has a segment to itself and joins it (0: none)
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float lg2(float x) {
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float nan_f() { return __int_as_float(0x7FC00000); }

// Positions that the newest rows of a sequence see.
__device__ __forceinline__ int seen_len(int p, int n_q, int max_len) {
    return p < 0 ? 0 : (int)min((int64_t)p + n_q, (int64_t)max_len);
}
__device__ __forceinline__ int units_of(int len) { return len > kUnit ? (len + kUnit - 1) / kUnit : 1; }

// Finds the units [u, u_end) of a pass's CTA and the sequence b, with first unit
// b_first, that the first one belongs to; the first CTA leaves the shares for
// the join. Every thread of the CTA calls it (THREADS of them); false: no
// units. scratch: THREADS / 32 + 2 words of shared memory.
template <int THREADS, class LenOf>
__device__ __forceinline__ bool my_units(const Pass& P, uint32_t cta, int seqs, const LenOf& len_of, uint32_t* scratch,
                                         uint32_t& u, uint32_t& u_end, uint32_t& b_first, int& b) {
    constexpr int kW = THREADS / 32;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int per_b = P.c.kv_heads * P.tiles;  // segments of a sequence
    const int each = (seqs + THREADS - 1) / THREADS;
    const int lo = min(tid * each, seqs), hi = min(lo + each, seqs);
    uint32_t mine = 0;
    for (int j = lo; j < hi; ++j) mine += (units_of(len_of(j)) + P.lead) * per_b;
    uint32_t inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(0xFFFFFFFFu, inc, o);
        if (lane >= o) inc += y;
    }
    if (lane == 31) scratch[warp] = inc;
    __syncthreads();
    uint32_t at = inc - mine, U = 0;
#pragma unroll
    for (int w = 0; w < kW; ++w) {
        if (w < warp) at += scratch[w];
        U += scratch[w];
    }
    const uint32_t share = (U + P.ctas - 1) / P.ctas;
    u = min(cta * share, U);
    u_end = min(u + share, U);
    const bool tell = cta == 0 && P.share;
    if (tell && tid == 0) P.share[0] = share;
    for (int j = lo; j < hi; ++j) {
        const uint32_t w = (units_of(len_of(j)) + P.lead) * per_b;
        if (tell) P.share[1 + j] = at;
        if (u >= at && u < at + w) scratch[kW] = j, scratch[kW + 1] = at;
        at += w;
    }
    __syncthreads();
    b = scratch[kW];
    b_first = scratch[kW + 1];
    return u < u_end;
}

// The part [ua, ub) of a segment's nu units that a CTA's units [u, u_end) are,
// u in the segment that begins at seg; empty where they are blank ones.
struct Part {
    int ua, ub;
    uint32_t next;  // the CTA's first unit behind it
    __device__ __forceinline__ Part(uint32_t u, uint32_t u_end, uint32_t seg, uint32_t nu, uint32_t lead) {
        const uint32_t from = seg + lead;
        ua = u > from ? u - from : 0;
        ub = u_end > from ? min(nu, u_end - from) : 0;
        next = ub == (int)nu ? from + nu : u_end;
    }
};

// Eight elements of a query row as they are loaded, with the rotary rows.
struct QueryLoad {
    uint4 x, c, s;
};
// in: the row exists; its HD / 8 lanes (sub: the lane's place) call together.
template <int HD>
__device__ __forceinline__ QueryLoad load_query(const AttnArgs& A, bool in, int rb, int ri, int rh, int sub) {
    QueryLoad q;
    q.x = make_uint4(0, 0, 0, 0);
    q.c = q.s = make_uint4(0x7FC07FC0u, 0x7FC07FC0u, 0x7FC07FC0u, 0x7FC07FC0u);
    if (in) q.x = __ldg(reinterpret_cast<const uint4*>(A.q + rb * A.q_seq + ri * A.q_tok + rh * HD) + sub);
    if (A.rope.cos_t) {
        const int64_t t = in ? (int64_t)(A.rope.pos ? A.rope.pos[rb] : A.pos[rb]) + ri : 0;
        if (in && t >= 0 && t < A.rope.rows) {
            q.c = __ldg(reinterpret_cast<const uint4*>(A.rope.cos_t + t * HD) + sub);
            q.s = __ldg(reinterpret_cast<const uint4*>(A.rope.sin_t + t * HD) + sub);
        }
    }
    return q;
}
// The row rotated and divided by its power of two, elements in [-2, 2) with
// the scale's sign, and the factor f >= 0 of its scores in log2 units (NaN
// for a row that is not finite, whose elements are zeros).
struct Query {
    float x[8];
    float f;
};
template <int HD>
__device__ __forceinline__ Query rotated_query(const AttnArgs& A, bool in, const QueryLoad& q, int sub) {
    constexpr int kLanes = HD / 8;
    const uint32_t xw[4] = {q.x.x, q.x.y, q.x.z, q.x.w};
    float x[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) x[2 * j] = bf_lo(xw[j]), x[2 * j + 1] = bf_hi(xw[j]);
    if (A.rope.cos_t) {
        const uint32_t cw[4] = {q.c.x, q.c.y, q.c.z, q.c.w}, sw[4] = {q.s.x, q.s.y, q.s.z, q.s.w};
        const float sgn = sub < kLanes / 2 ? -1.f : 1.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float o = sgn * __shfl_xor_sync(0xFFFFFFFFu, x[j], kLanes / 2);
            x[j] = fmaf(o, j & 1 ? bf_hi(sw[j / 2]) : bf_lo(sw[j / 2]), x[j] * (j & 1 ? bf_hi(cw[j / 2]) : bf_lo(cw[j / 2])));
        }
    }
    float amax = 0.f;
    bool nan = false;
#pragma unroll
    for (int j = 0; j < 8; ++j) amax = fmaxf(amax, fabsf(x[j])), nan |= x[j] != x[j];
    if (nan) amax = INFINITY;
#pragma unroll
    for (int o = 1; o < kLanes; o <<= 1) amax = fmaxf(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, o));
    // 2^-e and 2^e, e the exponent of the largest element, within +-126
    const bool fine = amax <= 3.402823466e38f;
    const uint32_t ex = min(max(__float_as_uint(amax) >> 23, 1u), 253u);
    const float down = copysignf(__uint_as_float((254 - ex) << 23), A.scale_log2), up = __uint_as_float(ex << 23);
    Query r;
#pragma unroll
    for (int j = 0; j < 8; ++j) r.x[j] = in && fine ? x[j] * down : 0.f;
    r.f = fine ? fabsf(A.scale_log2) * up : nan_f();
    return r;
}

// The tcgen05 kernel (cdq_kv_mma.cu): row tiles of kMmaRows, e4m3.
constexpr int kMmaRows = 128;
cudaError_t mma_attn_launch(const AttnArgs& A, cudaStream_t s);
cudaError_t mma_read_error(int* out);

}  // namespace kv
}  // namespace cdq
