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

struct AppendArgs {
    cdq_kv_cache c;
    const uint16_t *k, *v;
    int64_t k_seq, k_tok, v_seq, v_tok;
    const int32_t* pos;
    Rope rope;
    int32_t n;
    int64_t rows;  // batch * n * kv_heads
};

// A row of head_dim elements is HD / 8 neighbouring lanes of 8 elements (one
// 16-byte load each); blockIdx.y picks keys or values. The rotation's partner
// element (HD / 2 away) is the same slot of the lane HD / 16 away, the
// largest magnitude a shuffle reduction over the row's (e2m1: the group's
// four) lanes.
template <int FMT, int HD>
__global__ void __launch_bounds__(kThreads) append_kernel(const AppendArgs A) {
    constexpr int kLanes = HD / 8;
    pdl_wait();
    pdl_release();
    const bool key = blockIdx.y == 0;
    const int sub = threadIdx.x % kLanes;
    const int64_t row = (int64_t)blockIdx.x * (kThreads / kLanes) + threadIdx.x / kLanes;
    const bool in = row < A.rows;
    const int64_t r = in ? row : 0;
    const int h = (int)(r % A.c.kv_heads);
    const int64_t tok = r / A.c.kv_heads;
    const int i = (int)(tok % A.n);
    const int64_t b = tok / A.n;
    const int p0 = A.pos[b];
    const int64_t p = (int64_t)p0 + i;
    const bool live = in && p0 >= 0 && p < A.c.max_len;
    const uint16_t* src = key ? A.k + b * A.k_seq + i * A.k_tok : A.v + b * A.v_seq + i * A.v_tok;
    uint4 u = make_uint4(0, 0, 0, 0);
    if (live) u = __ldg(reinterpret_cast<const uint4*>(src + h * HD) + sub);
    float x[8];
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        x[2 * j] = bf_lo(w[j]);
        x[2 * j + 1] = bf_hi(w[j]);
    }
    if (key && A.rope.cos_t) {
        const int64_t t = (int64_t)(A.rope.pos ? A.rope.pos[b] : p0) + i;
        const bool ok = t >= 0 && t < A.rope.rows;
        uint4 cu = make_uint4(0x7FC07FC0u, 0x7FC07FC0u, 0x7FC07FC0u, 0x7FC07FC0u), su = cu;
        if (live && ok) {
            cu = __ldg(reinterpret_cast<const uint4*>(A.rope.cos_t + t * HD) + sub);
            su = __ldg(reinterpret_cast<const uint4*>(A.rope.sin_t + t * HD) + sub);
        }
        const uint32_t cw[4] = {cu.x, cu.y, cu.z, cu.w}, sw[4] = {su.x, su.y, su.z, su.w};
        const float sgn = sub < kLanes / 2 ? -1.f : 1.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float o = sgn * __shfl_xor_sync(0xFFFFFFFFu, x[j], kLanes / 2);
            const float cs = j & 1 ? bf_hi(cw[j / 2]) : bf_lo(cw[j / 2]);
            const float sn = j & 1 ? bf_hi(sw[j / 2]) : bf_lo(sw[j / 2]);
            x[j] = fmaf(o, sn, x[j] * cs);  // products of two bf16 are exact in float32: one rounding
        }
    }
    // the largest magnitude of the scale's elements, NaN if any is NaN
    float amax = 0.f;
    bool nan = false;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        amax = fmaxf(amax, fabsf(x[j]));
        nan |= x[j] != x[j];
    }
    if (nan) amax = INFINITY;
#pragma unroll
    for (int o = 1; o < (FMT == kE4M3 ? kLanes : kGroup / 8); o <<= 1)
        amax = fmaxf(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, o));
    if (!live) return;
    const uint16_t sb = group_scale<FMT>(amax);
    const float s = bf(sb);
    const bool ok = s == s;
    float y[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) y[j] = ok ? x[j] / s : 0.f;
    const int64_t dst = (b * A.c.kv_heads + h) * A.c.max_len + p;
    uint8_t* codes = static_cast<uint8_t*>(key ? A.c.k : A.c.v) + dst * row_bytes<FMT>(HD);
    uint16_t* scales = (key ? A.c.k_scale : A.c.v_scale) + dst * row_scales<FMT>(HD);
    if (FMT == kE4M3) {
        uint32_t o[2] = {0, 0};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t c = __nv_cvt_float2_to_fp8x2(make_float2(y[2 * j], y[2 * j + 1]), __NV_SATFINITE, __NV_E4M3);
            o[j / 2] |= c << (16 * (j & 1));
        }
        reinterpret_cast<uint2*>(codes)[sub] = make_uint2(o[0], o[1]);
        if (sub == 0) scales[0] = sb;
    } else {
        uint32_t o = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t c = __nv_cvt_float2_to_fp4x2(make_float2(y[2 * j], y[2 * j + 1]), __NV_E2M1, cudaRoundNearest);
            o |= (c & 0xFFu) << (8 * j);
        }
        reinterpret_cast<uint32_t*>(codes)[sub] = o;
        if (sub % (kGroup / 8) == 0) scales[sub / (kGroup / 8)] = sb;
    }
}

struct ReadArgs {
    cdq_kv_cache c;
    const int32_t* pos;
    uint16_t *k, *v;
    int32_t n;
    int64_t rows;
};

template <int FMT, int HD>
__global__ void __launch_bounds__(kThreads) read_kernel(const ReadArgs A) {
    constexpr int kLanes = HD / 8;
    pdl_wait();
    pdl_release();
    const bool key = blockIdx.y == 0;
    const int sub = threadIdx.x % kLanes;
    const int64_t row = (int64_t)blockIdx.x * (kThreads / kLanes) + threadIdx.x / kLanes;
    if (row >= A.rows) return;
    const int h = (int)(row % A.c.kv_heads);
    const int64_t tok = row / A.c.kv_heads;
    const int i = (int)(tok % A.n);
    const int64_t b = tok / A.n;
    const int p0 = A.pos ? A.pos[b] : 0;
    const int64_t p = (int64_t)p0 + i;
    uint4 out = make_uint4(0, 0, 0, 0);
    if (p0 >= 0 && p < A.c.max_len) {
        const int64_t src = (b * A.c.kv_heads + h) * A.c.max_len + p;
        const uint8_t* codes = static_cast<const uint8_t*>(key ? A.c.k : A.c.v) + src * row_bytes<FMT>(HD);
        const uint16_t* scales = (key ? A.c.k_scale : A.c.v_scale) + src * row_scales<FMT>(HD);
        uint32_t hh[4];
        float s;
        if (FMT == kE4M3) {
            const uint2 c = __ldg(reinterpret_cast<const uint2*>(codes) + sub);
            s = bf(__ldg(scales));
            e4m3x4_to_half(c.x, hh[0], hh[1]);
            e4m3x4_to_half(c.y, hh[2], hh[3]);
        } else {
            const uint32_t c = __ldg(reinterpret_cast<const uint32_t*>(codes) + sub);
            s = bf(__ldg(scales + sub / (kGroup / 8)));
            e2m1x8_to_half(c, hh);
        }
        uint32_t o[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&hh[j]));
            o[j] = pack_bf(f.x * s, f.y * s);
        }
        out = make_uint4(o[0], o[1], o[2], o[3]);
    }
    reinterpret_cast<uint4*>((key ? A.k : A.v) + row * HD)[sub] = out;
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
    if (!at(cos_t, 16) || !at(sin_t, 16) || rows < 1) return CDQ_ERR_ARG;
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
    if (!strided(k, k_seq, k_tok) || !strided(v, v_seq, v_tok) || !pos || n < 1) return CDQ_ERR_ARG;
    A.c = *cache;
    A.k = k, A.v = v, A.k_seq = k_seq, A.k_tok = k_tok, A.v_seq = v_seq, A.v_tok = v_tok;
    A.pos = pos, A.n = n;
    A.rows = (int64_t)cache->batch * n * cache->kv_heads;
    const int per = kThreads / (cache->head_dim / 8);
    const int64_t blocks = (A.rows + per - 1) / per;
    if (blocks > 0x7FFFFFFF) return CDQ_ERR_SHAPE;
    const dim3 grid((unsigned)blocks, 2);
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
    if (!at(k, 16) || !at(v, 16) || n < 1) return CDQ_ERR_ARG;
    ReadArgs A{};
    A.c = *cache, A.pos = pos, A.k = k, A.v = v, A.n = n;
    A.rows = (int64_t)cache->batch * n * cache->kv_heads;
    const int per = kThreads / (cache->head_dim / 8);
    const int64_t blocks = (A.rows + per - 1) / per;
    if (blocks > 0x7FFFFFFF) return CDQ_ERR_SHAPE;
    const dim3 grid((unsigned)blocks, 2);
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
