// Writing the quantised key/value cache and reading it back.
#include <algorithm>

#include "cdq_internal.cuh"
#include "cdq_kv.cuh"

using cdq::launch_pdl;
using cdq::pdl_release;
using cdq::pdl_wait;
using namespace cdq::kv;

namespace {

constexpr int kThreads = 256;
constexpr int kAhead = 4;  // rows of a lane in flight

struct AppendArgs {
    cdq_kv_cache c;
    const uint16_t *k, *v;
    int64_t k_seq, k_tok, v_seq, v_tok;
    const int32_t* pos;
    Rope rope;
    int32_t n;
};

// Pairs of float32 in one 64-bit register: one instruction does both.
__device__ __forceinline__ uint64_t pair(float lo, float hi) {
    uint64_t p;
    asm("mov.b64 %0, {%1, %2};" : "=l"(p) : "f"(lo), "f"(hi));
    return p;
}
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
__device__ __forceinline__ uint64_t pair_bf(uint32_t w) { return pair(bf_lo(w), bf_hi(w)); }

// A row of head_dim elements is HD / 8 neighbouring lanes of 8 elements (one
// 16-byte load each); a lane takes one position of a sequence (blockIdx.z),
// its heads kAhead at a time, their loads first, so that the rotary rows are
// read and unpacked once a position. blockIdx.y picks keys or values. The
// rotation's partner element (HD / 2 away) is the same slot of the lane
// HD / 16 away, the largest magnitude a shuffle reduction over the row's
// (e2m1: the group's four) lanes. Inputs are read and codes written once: 16 x
// 4,096 positions, 4 heads of 128, to e2m1 take 44 us for 172 MB, 3.9 TB/s, to
// e4m3 44 us for 202 MB, 4.6 TB/s. Of the 44, 28 are issue slots (126
// instructions for two rows of 128, a warp), the rest are loads and the chain
// of shuffles behind them. A step's one position is 1.9 us, a launch.
template <int FMT, int HD, bool KEYS>
__device__ __forceinline__ void append_rows(const AppendArgs& A) {
    constexpr int kLanes = HD / 8, kRows = kThreads / kLanes;
    const int sub = threadIdx.x % kLanes;
    const int64_t b = blockIdx.z;
    const int p0 = A.pos[b];
    if (p0 < 0) return;
    const int i = blockIdx.x * kRows + threadIdx.x / kLanes;
    const int64_t p = (int64_t)p0 + i;
    const bool live = i < A.n && p < A.c.max_len;
    const uint4* src = reinterpret_cast<const uint4*>(KEYS ? A.k + b * A.k_seq + (live ? i * A.k_tok : 0)
                                                           : A.v + b * A.v_seq + (live ? i * A.v_tok : 0)) + sub;
    const int64_t row0 = b * A.c.kv_heads * A.c.max_len + p;
    uint64_t cs[4], sn[4];
    const bool turned = KEYS && A.rope.cos_t;
    if (turned) {
        const int64_t t = (int64_t)(A.rope.pos ? A.rope.pos[b] : p0) + i;
        uint4 cu = make_uint4(0x7FC07FC0u, 0x7FC07FC0u, 0x7FC07FC0u, 0x7FC07FC0u), su = cu;
        if (live && t >= 0 && t < A.rope.rows) {
            cu = __ldg(reinterpret_cast<const uint4*>(A.rope.cos_t + t * HD) + sub);
            su = __ldg(reinterpret_cast<const uint4*>(A.rope.sin_t + t * HD) + sub);
        }
        const uint32_t flip = sub < kLanes / 2 ? 0x80008000u : 0u;  // the first half takes -sin
        cs[0] = pair_bf(cu.x), cs[1] = pair_bf(cu.y), cs[2] = pair_bf(cu.z), cs[3] = pair_bf(cu.w);
        sn[0] = pair_bf(su.x ^ flip), sn[1] = pair_bf(su.y ^ flip), sn[2] = pair_bf(su.z ^ flip), sn[3] = pair_bf(su.w ^ flip);
    }
    for (int h0 = 0; h0 < A.c.kv_heads; h0 += kAhead) {
        uint4 xu[kAhead];
#pragma unroll
        for (int a = 0; a < kAhead; ++a) {
            xu[a] = make_uint4(0, 0, 0, 0);
            if (live && h0 + a < A.c.kv_heads) xu[a] = __ldg(src + (int64_t)(h0 + a) * kLanes);
        }
#pragma unroll
        for (int a = 0; a < kAhead; ++a) {
            if (h0 + a >= A.c.kv_heads) break;
            uint64_t x[4] = {pair_bf(xu[a].x), pair_bf(xu[a].y), pair_bf(xu[a].z), pair_bf(xu[a].w)};
            if (turned) {
                // products of two bf16 are exact in float32: one rounding
                const uint32_t ow[4] = {__shfl_xor_sync(0xFFFFFFFFu, xu[a].x, kLanes / 2),
                                        __shfl_xor_sync(0xFFFFFFFFu, xu[a].y, kLanes / 2),
                                        __shfl_xor_sync(0xFFFFFFFFu, xu[a].z, kLanes / 2),
                                        __shfl_xor_sync(0xFFFFFFFFu, xu[a].w, kLanes / 2)};
#pragma unroll
                for (int j = 0; j < 4; ++j) x[j] = fma2(pair_bf(ow[j]), sn[j], mul2(x[j], cs[j]));
            }
            // the largest magnitude; a sum of x * 0 is NaN where an element is no number
            float amax = 0.f;
            uint64_t none = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float2 f = unpair(x[j]);
                amax = fmaxf(fmaxf(amax, fabsf(f.x)), fabsf(f.y));
                none = fma2(x[j], 0, none);
            }
            const float2 f = unpair(none);
            if (f.x + f.y != 0.f) amax = INFINITY;
#pragma unroll
            for (int o = 1; o < (FMT == kE4M3 ? kLanes : kGroup / 8); o <<= 1)
                amax = fmaxf(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, o));
            const uint16_t sb = group_scale<FMT>(amax);
            const float s = bf(sb);
            // x / s (Markstein's correction of x * (1 / s) by its exact remainder: a
            // quotient on the border of two codes comes out exactly)
            float inv;
            asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(s));
            inv = fmaf(fmaf(-s, inv, 1.f), inv, inv);
            const uint64_t inv2 = pair(inv, inv), neg2 = pair(-s, -s);
            uint32_t o[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint64_t q = mul2(x[j], inv2);
                const float2 y = unpair(fma2(fma2(q, neg2, x[j]), inv2, q));
                if (FMT == kE4M3) o[j] = __nv_cvt_float2_to_fp8x2(y, __NV_SATFINITE, __NV_E4M3);
                else o[j] = __nv_cvt_float2_to_fp4x2(y, __NV_E2M1, cudaRoundNearest) & 0xFFu;
            }
            if (!live) continue;
            const bool ok = s == s;
            const int64_t row = row0 + (int64_t)(h0 + a) * A.c.max_len;
            uint8_t* codes = static_cast<uint8_t*>(KEYS ? A.c.k : A.c.v) + row * row_bytes<FMT>(HD);
            uint16_t* scales = (KEYS ? A.c.k_scale : A.c.v_scale) + row * row_scales<FMT>(HD);
            if (FMT == kE4M3) {
                reinterpret_cast<uint2*>(codes)[sub] =
                    ok ? make_uint2(o[0] | o[1] << 16, o[2] | o[3] << 16) : make_uint2(0, 0);
                if (sub == 0) scales[0] = sb;
            } else {
                reinterpret_cast<uint32_t*>(codes)[sub] = ok ? o[0] | o[1] << 8 | o[2] << 16 | o[3] << 24 : 0;
                if (sub % (kGroup / 8) == 0) scales[sub / (kGroup / 8)] = sb;
            }
        }
    }
}

template <int FMT, int HD>
__global__ void __launch_bounds__(kThreads) append_kernel(const AppendArgs A) {
    pdl_wait();
    pdl_release();
    if (blockIdx.y == 0) append_rows<FMT, HD, true>(A);
    else append_rows<FMT, HD, false>(A);
}

struct ReadArgs {
    cdq_kv_cache c;
    const int32_t* pos;
    uint16_t *k, *v;
    int32_t rows;  // n * kv_heads of a sequence
};

// Lanes of a row as in append_kernel, kAhead rows a lane; reading the codes
// and writing bf16 bounds it: the same positions take 30 us, 5.7 TB/s.
template <int FMT, int HD>
__global__ void __launch_bounds__(kThreads) read_kernel(const ReadArgs A) {
    constexpr int kLanes = HD / 8, kRows = kThreads / kLanes;
    pdl_wait();
    pdl_release();
    const bool key = blockIdx.y == 0;
    const int sub = threadIdx.x % kLanes;
    const int64_t b = blockIdx.z;
    const int p0 = A.pos ? A.pos[b] : 0;
    const uint8_t* codes = static_cast<const uint8_t*>(key ? A.c.k : A.c.v);
    const uint16_t* scales = key ? A.c.k_scale : A.c.v_scale;
    uint16_t* out = (key ? A.k : A.v) + b * A.rows * HD;
    const uint32_t r0 = blockIdx.x * (kAhead * kRows) + threadIdx.x / kLanes;
    uint32_t c[kAhead][FMT == kE4M3 ? 2 : 1];
    uint16_t s[kAhead];
#pragma unroll
    for (int a = 0; a < kAhead; ++a) {
        const uint32_t r = r0 + a * kRows, i = r / A.c.kv_heads, h = r % A.c.kv_heads;
        const int64_t p = (int64_t)p0 + i, src = (b * A.c.kv_heads + h) * A.c.max_len + p;
        c[a][0] = 0, s[a] = 0;
        if (FMT == kE4M3) c[a][FMT == kE4M3 ? 1 : 0] = 0;
        if (r < (uint32_t)A.rows && p0 >= 0 && p < A.c.max_len) {
            if (FMT == kE4M3) {
                const uint2 u = __ldg(reinterpret_cast<const uint2*>(codes + src * row_bytes<FMT>(HD)) + sub);
                c[a][0] = u.x, c[a][FMT == kE4M3 ? 1 : 0] = u.y;
                s[a] = __ldg(scales + src);
            } else {
                c[a][0] = __ldg(reinterpret_cast<const uint32_t*>(codes + src * row_bytes<FMT>(HD)) + sub);
                s[a] = __ldg(scales + src * row_scales<FMT>(HD) + sub / (kGroup / 8));
            }
        }
    }
#pragma unroll
    for (int a = 0; a < kAhead; ++a) {
        const uint32_t r = r0 + a * kRows;
        if (r >= (uint32_t)A.rows) break;
        uint32_t hh[4];
        if (FMT == kE4M3) {
            e4m3x4_to_half(c[a][0], hh[0], hh[1]);
            e4m3x4_to_half(c[a][FMT == kE4M3 ? 1 : 0], hh[2], hh[3]);
        } else {
            e2m1x8_to_half(c[a][0], hh);
        }
        uint32_t o[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&hh[j]));
            o[j] = pack_bf(f.x * bf(s[a]), f.y * bf(s[a]));
        }
        reinterpret_cast<uint4*>(out + (int64_t)r * HD)[sub] = make_uint4(o[0], o[1], o[2], o[3]);
    }
}

// The reading grid: rows of one sequence in x, keys and values in y. False
// where a dimension does not fit.
bool grid_of(const cdq_kv_cache* c, int32_t n, int32_t* rows, dim3* grid) {
    const int64_t r = (int64_t)n * c->kv_heads;
    if (r > 0x3FFFFFFF) return false;
    const int per = kAhead * kThreads / (c->head_dim / 8);
    *rows = (int32_t)r;
    *grid = dim3((unsigned)((r + per - 1) / per), 2, c->batch);
    return true;
}

}  // namespace

namespace cdq {
namespace kv {

cdq_status check_cache(const cdq_kv_cache* c) {
    if (!c) return CDQ_ERR_ARG;
    if (c->format != kE4M3 && c->format != kE2M1) return CDQ_ERR_UNSUPPORTED;
    if (c->head_dim != 64 && c->head_dim != 128) return CDQ_ERR_UNSUPPORTED;
    if (c->batch < 1 || c->batch > 65535 || c->kv_heads < 1 || c->kv_heads > 1024 || c->max_len < 1 ||
        c->max_len > (1 << 30))
        return CDQ_ERR_SHAPE;
    if (!at(c->k, 16) || !at(c->v, 16) || !at(c->k_scale, 8) || !at(c->v_scale, 8)) return CDQ_ERR_ARG;
    return CDQ_OK;
}

cdq_status check_rope(const uint16_t* cos_t, const uint16_t* sin_t, int32_t rows, const int32_t* pos, Rope* out) {
    *out = Rope{};
    if (!cos_t) return CDQ_OK;
    if (!at(cos_t, 16) || !at(sin_t, 16) || rows < 1 || (pos && !at(pos, 4))) return CDQ_ERR_ARG;
    *out = Rope{cos_t, sin_t, pos, rows};
    return CDQ_OK;
}

bool strided(const void* p, int64_t seq, int64_t tok) {
    return at(p, 16) && seq >= 0 && tok >= 0 && seq % 8 == 0 && tok % 8 == 0;
}

}  // namespace kv
}  // namespace cdq

extern "C" {

cdq_status cdq_kv_append(const cdq_kv_cache* cache, const uint16_t* k, int64_t k_seq, int64_t k_tok,
                         const uint16_t* v, int64_t v_seq, int64_t v_tok, const int32_t* pos, int32_t n,
                         const uint16_t* cos_t, const uint16_t* sin_t, int32_t table_rows, const int32_t* table_pos,
                         void* stream) {
    cdq_status st = check_cache(cache);
    if (st) return st;
    AppendArgs A{};
    if ((st = check_rope(cos_t, sin_t, table_rows, table_pos, &A.rope))) return st;
    if (!strided(k, k_seq, k_tok) || !strided(v, v_seq, v_tok) || !at(pos, 4) || n < 1) return CDQ_ERR_ARG;
    A.c = *cache;
    A.k = k, A.v = v, A.k_seq = k_seq, A.k_tok = k_tok, A.v_seq = v_seq, A.v_tok = v_tok;
    A.pos = pos, A.n = n;
    if (n > 0x3FFFFFFF) return CDQ_ERR_SHAPE;
    const int per = kThreads / (cache->head_dim / 8);
    const dim3 grid((n + per - 1) / per, 2, cache->batch);
    auto s = (cudaStream_t)stream;
    cudaError_t e;
    if (cache->format == kE4M3)
        e = cache->head_dim == 64 ? launch_pdl(append_kernel<kE4M3, 64>, grid, dim3(kThreads), 0, s, A)
                                  : launch_pdl(append_kernel<kE4M3, 128>, grid, dim3(kThreads), 0, s, A);
    else
        e = cache->head_dim == 64 ? launch_pdl(append_kernel<kE2M1, 64>, grid, dim3(kThreads), 0, s, A)
                                  : launch_pdl(append_kernel<kE2M1, 128>, grid, dim3(kThreads), 0, s, A);
    return e == cudaSuccess ? CDQ_OK : CDQ_ERR_CUDA;
}

cdq_status cdq_kv_read(const cdq_kv_cache* cache, const int32_t* pos, int32_t n, uint16_t* k, uint16_t* v,
                       void* stream) {
    cdq_status st = check_cache(cache);
    if (st) return st;
    if (!at(k, 16) || !at(v, 16) || (pos && !at(pos, 4)) || n < 1) return CDQ_ERR_ARG;
    ReadArgs A{};
    A.c = *cache, A.pos = pos, A.k = k, A.v = v;
    dim3 grid;
    if (!grid_of(cache, n, &A.rows, &grid)) return CDQ_ERR_SHAPE;
    auto s = (cudaStream_t)stream;
    cudaError_t e;
    if (cache->format == kE4M3)
        e = cache->head_dim == 64 ? launch_pdl(read_kernel<kE4M3, 64>, grid, dim3(kThreads), 0, s, A)
                                  : launch_pdl(read_kernel<kE4M3, 128>, grid, dim3(kThreads), 0, s, A);
    else
        e = cache->head_dim == 64 ? launch_pdl(read_kernel<kE2M1, 64>, grid, dim3(kThreads), 0, s, A)
                                  : launch_pdl(read_kernel<kE2M1, 128>, grid, dim3(kThreads), 0, s, A);
    return e == cudaSuccess ? CDQ_OK : CDQ_ERR_CUDA;
}

}  // extern "C"
