// The quantised key/value cache: formats, conversions and what its kernels
// share. Buffers are [batch][kv head][position] rows of head_dim codes, and
// scales beside them:
//   e4m3  one code a byte, one bf16 scale a row,
//         s = bf16(max(amax, 2^-100) / 448), code = e4m3(x / s);
//   e2m1  two codes a byte (the even element in the low nibble), one bf16
//         scale per 32 elements, s = bf16(max(amax, 2^-100) / 6),
//         code = e2m1(x / s).
// Codes round to nearest even and saturate. The floor under amax keeps s
// normal and positive, so an all-zero row needs no case of its own. The scale
// has 8 significant bits on purpose: a bf16 element divided by it either is a
// border between two codes exactly or lies further from one than a float32
// division errs, so no element is decided by a rounding of the quotient. A
// row (group) that holds a NaN or an infinity gets scale NaN and codes 0.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp4.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "cdq.h"

namespace cdq {
namespace kv {

constexpr int kE4M3 = CDQ_KV_E4M3, kE2M1 = CDQ_KV_E2M1;
constexpr int kGroup = 32;  // e2m1 elements per scale

template <int FMT>
__host__ __device__ constexpr int row_bytes(int hd) {
    return FMT == kE4M3 ? hd : hd / 2;
}
template <int FMT>
__host__ __device__ constexpr int row_scales(int hd) {
    return FMT == kE4M3 ? 1 : hd / kGroup;
}
template <int FMT>
__host__ __device__ constexpr float code_max() {
    return FMT == kE4M3 ? 448.f : 6.f;
}

__device__ __forceinline__ float bf(uint16_t v) { return __uint_as_float((uint32_t)v << 16); }
__device__ __forceinline__ float bf_lo(uint32_t v) { return __uint_as_float(v << 16); }
__device__ __forceinline__ float bf_hi(uint32_t v) { return __uint_as_float(v & 0xFFFF0000u); }
__device__ __forceinline__ uint32_t pack_bf(float lo, float hi) {
    const __nv_bfloat162 p = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&p);
}

// Four e4m3 codes -> four halves, exactly (lo: codes 0 and 1).
__device__ __forceinline__ void e4m3x4_to_half(uint32_t c, uint32_t& lo, uint32_t& hi) {
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\t"
        "cvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
        : "=r"(lo), "=r"(hi)
        : "r"(c));
}
// Eight e2m1 codes -> eight halves, exactly (h[0]: codes 0 and 1).
__device__ __forceinline__ void e2m1x8_to_half(uint32_t c, uint32_t (&h)[4]) {
    asm("{\n\t.reg .b8 a, b, d, e;\n\tmov.b32 {a, b, d, e}, %4;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, a;\n\tcvt.rn.f16x2.e2m1x2 %1, b;\n\t"
        "cvt.rn.f16x2.e2m1x2 %2, d;\n\tcvt.rn.f16x2.e2m1x2 %3, e;\n\t}"
        : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
        : "r"(c));
}

// Scale of a group from its largest magnitude (bf16 bits; NaN when that is
// not finite).
template <int FMT>
__device__ __forceinline__ uint16_t group_scale(float amax) {
    if (!(amax <= 3.402823466e38f)) return 0x7FC0;
    // amax / code_max, corrected by its exact remainder to the rounded quotient
    constexpr float top = code_max<FMT>(), inv = 1.f / top;
    const float a = fmaxf(amax, 0x1p-100f), q = a * inv;
    return __bfloat16_as_ushort(__float2bfloat16_rn(fmaf(fmaf(-q, top, a), inv, q)));
}

// Rotary tables [rows][head_dim] and the row of a sequence's first new
// position (null: its cache position).
struct Rope {
    const uint16_t *cos_t, *sin_t;
    const int32_t* pos;
    int32_t rows;
};

// Argument checks shared by the cache's entry points.
cdq_status check_cache(const cdq_kv_cache* c);
bool strided(const void* p, int64_t seq, int64_t tok);
cdq_status check_rope(const uint16_t* cos_t, const uint16_t* sin_t, int32_t rows, const int32_t* pos, Rope* out);
inline bool at(const void* p, size_t a) { return p && (uintptr_t)p % a == 0; }

}  // namespace kv
}  // namespace cdq
