// Attention over the quantised cache (cdq_kv.cuh): grouped-query attention of
// a few new positions of every sequence, and of a whole batch over a prefix
// that all its sequences share.
//
// The rows of one kv head, (new position i, head of the group g), r = i * G +
// g, go through mma.m16n8k16 as its N side, eight a tile; sixteen keys, then
// sixteen elements of their values, are the M side, so that a tile of eight
// rows leaves no half of an instruction empty:
//   S[j][r] = sum_d code_k[j][d] q[r][d]      the codes as halves, exact;
//   s_j     = S * scale_k[j] * f_r            log2 units;
//   l += 2^(s_j - M),   O[d][r] += code_v[j][d] 2^(s_j - M) scale_v[j],   out = O / l
// with M a running maximum not of the scores but of s_j + log2 scale_v[j], less
// kBelow: the weights 2^(s_j - M) scale_v[j] that enter the second product are
// at most 2^kLazy whatever the scales are, and the largest at least 2^kBelow.
// Rounding them to half then costs at most 2^-11 of a weight or 2^-32 of the
// largest (a half's smallest step is 2^-24), whichever is more. The second
// counts where one position outweighs very many others: 2^20 of them in one
// warp, whose M is its own, can lose 2^-12 of the largest contribution. (With M
// at the maximum itself all weights below 2^-25 of it are lost: 2^20 positions
// at 2^-25.2 have a share of 0.026.) l is a float32 sum too: equal terms round
// alike, which costs 2^-11 at most where a warp has 2^18 of them (a cache of 45
// GB, a segment a CTA), added by eight lanes. The logarithm is
// held at kLeast = -83 and above, so that the terms of l, at most 2^(kLazy + 83),
// have room to be summed in float32; values all smaller than that (by their
// scales) have as many fewer bits. q is rotated in float32, divided by its
// row's power of two and rounded to half (2^-11). Neither operand is ever
// dequantised: scales multiply scores and weights.
//
// Both products contract over an order of elements that is free: a lane takes
// neighbouring bytes of a key row as its k slices (q is laid out to match) and
// four neighbouring positions of the values. Scores come out with a position a
// lane row, weights go in with a position a lane column: 8x8 transposes
// between lanes (movmatrix) turn them.
//
// What bounds it: for long sequences the reading of the cache and the
// conversions (64 ragged sequences of up to 32,768 positions, 14 heads over 2
// of 64, e4m3: 62.7 us for 319 MB, 5.1 TB/s; 131,072 positions, 28 heads over
// 4 of 128, e2m1: 29.9 us for 75.5 MB; with the rows as the M side, half of it
// empty at 7 rows, 68.3 and 38.2); for few units the chain of a launch, the
// lengths, the rotated queries, one unit and the join: 5.5 us for 640
// positions.
//
// Positions are split over CTAs (and over a CTA's warps); partial (M, l, O) of
// a row are joined by a second launch when there is more than one part, or by
// the cluster of CTAs that has a short cache's segment to itself.
#include <cooperative_groups.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "cdq_kv_attn.cuh"

namespace cg = cooperative_groups;
using cdq::launch_pdl;
using cdq::pdl_release;
using cdq::pdl_wait;
using namespace cdq::kv;

namespace {

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr int kStep = 32;              // positions of a warp step
constexpr int kMaxCluster = 8;
static_assert(kStep * kWarps == kUnit, "a CTA step is the unit of work");

__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// 16 bytes into shared memory, asynchronously; zeros behind the first n
__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, int n) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
// B = 4 or 8 bytes, or zeros
template <int B>
__device__ __forceinline__ void copy_small(uint32_t dst, const void* src, bool in) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(B), "r"(in ? B : 0) : "memory");
}
__device__ __forceinline__ uint32_t load_u16(const uint16_t* p) {
    uint16_t v;
    asm volatile("ld.global.nc.u16 %0, [%1];" : "=h"(v) : "l"(p));
    return v;
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// The t-th of lane row g's HD / 8 elements of a value row.
template <int FMT, int HD>
__device__ __forceinline__ int value_dim(int g, int t) {
    return FMT == kE4M3 ? (HD / 8) * g + t : kGroup * (t / 4) + 4 * g + t % 4;
}

template <int FMT, int HD, int NT>
struct Cfg {
    static constexpr int kRows = 8 * NT;
    static constexpr int kRowsB = 2 * kStep * row_bytes<FMT>(HD);
    static constexpr int kScaleB = FMT == kE4M3 ? 0 : kStep * row_scales<FMT>(HD) * 2;
    static constexpr int kStage = kRowsB + 2 * kScaleB;  // a warp step's keys, values (e2m1: and the scales of each)
    // (a stage less is a CTA more on a multiprocessor: 131,072 positions of e2m1, 28 heads of 128, take 30.3 us with two
    // stages and four CTAs, 31.9 with three and three; e4m3 rows of 64 take the same either way)
    static constexpr int kStages = kStage >= 4096 ? 2 : 3;
    static constexpr int kKinds = FMT == kE4M3 ? 3 : 2 * (HD / kGroup) + 1;  // scale arrays of a step
    static constexpr int kOs = HD + 4;                   // padded row of the joined accumulators
    static constexpr int kRing = kWarps * kStages * kStage;
    static constexpr int kJoin = kWarps * kRows * kOs * 4;
    static constexpr int kBig = kRing > kJoin ? kRing : kJoin;  // the ring is drained when warps join
    static constexpr int kScales = kWarps * kKinds * kStep * 4;
    static constexpr int kMetaB = kWarps * kRows * 2 * 4;
    static constexpr int kQ = kRows * (HD + 8) * 2;
    static constexpr int kSmem = kBig + kScales + kMetaB + kRows * 8 + kQ;
    // registers for this many CTAs a multiprocessor without spilling more than a few words (64 rows of one sequence:
    // five of heads of 64 take 61.7 us where four take 62.4, but 6.2 where four take 6.0 for a short one)
    static constexpr int kMinCtas = HD == 64 || (NT == 1 && FMT == kE2M1) ? 4 : NT == 1 || (NT == 2 && FMT == kE2M1) ? 3 : 2;
};

// The element of a key row at which lane c's four of slice s start.
template <int FMT>
__device__ __forceinline__ int key_dim(int s, int c) {
    return FMT == kE4M3 ? 64 * (s / 4) + 16 * c + 4 * (s % 4) : kGroup * (s / 2) + 8 * c + 4 * (s % 2);
}
// Lane row g's elements of the values of the four positions at v0, as they
// lie: four elements value_dim(g, 4w ..) a word w (e2m1: in its low half).
template <int FMT, int HD>
__device__ __forceinline__ void value_words(const uint8_t* v0, int g, uint32_t (&v)[4][HD / 32]) {
    constexpr int RB = row_bytes<FMT>(HD);
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        if (FMT == kE2M1) {
#pragma unroll
            for (int w = 0; w < HD / 32; ++w) v[t][w] = *reinterpret_cast<const uint16_t*>(v0 + t * RB + 16 * w + 2 * g);
        } else if (HD == 64) {
            const uint2 x = *reinterpret_cast<const uint2*>(v0 + t * RB + 8 * g);
            v[t][0] = x.x, v[t][1] = x.y;
        } else {
            const uint4 x = *reinterpret_cast<const uint4*>(v0 + t * RB + 16 * g);
            v[t][0] = x.x, v[t][1] = x.y, v[t][HD / 32 - 2] = x.z, v[t][HD / 32 - 1] = x.w;
        }
    }
}
// Those of one word as halves: pairs of the first two positions, of the last two.
template <int FMT>
__device__ __forceinline__ void value_pairs(uint32_t v0, uint32_t v1, uint32_t v2, uint32_t v3, uint32_t (&lo)[4],
                                            uint32_t (&hi)[4]) {
    if (FMT == kE4M3) {
        e4m3x4_to_half(__byte_perm(v0, v1, 0x5140), lo[0], lo[1]);
        e4m3x4_to_half(__byte_perm(v0, v1, 0x7362), lo[2], lo[3]);
        e4m3x4_to_half(__byte_perm(v2, v3, 0x5140), hi[0], hi[1]);
        e4m3x4_to_half(__byte_perm(v2, v3, 0x7362), hi[2], hi[3]);
    } else {
        // nibbles of four elements: position pairs side by side in a byte
        // (one word a pair of positions: elements 0, 2 of the four in its low half, 1, 3 in its high)
        const uint32_t v01 = v0 | (v0 << 12), v23 = v2 | (v2 << 12);
        const uint32_t w01 = (v1 << 4) | (v1 << 16), w23 = (v3 << 4) | (v3 << 16);
        uint32_t x[4], z[4];
        e2m1x8_to_half((v01 & 0x0F0F0F0Fu) | (w01 & 0xF0F0F0F0u), x);
        e2m1x8_to_half((v23 & 0x0F0F0F0Fu) | (w23 & 0xF0F0F0F0u), z);
        lo[0] = x[0], lo[1] = x[2], lo[2] = x[1], lo[3] = x[3];
        hi[0] = z[0], hi[1] = z[2], hi[2] = z[1], hi[3] = z[3];
    }
}
__device__ __forceinline__ uint32_t transposed(uint32_t a) {  // an 8x8 matrix of halves over the warp
    uint32_t d;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}

// What a warp holds of the 8 NT rows of its tile, and its two products over
// kStep positions of its own. A lane has the scores of rows 8n + 2c and
// 8n + 2c + 1 for the positions 16 (t / 2) + 2 (t % 2) + `at`, t < 4.
template <int FMT, int HD, int NT>
struct Rows {
    static constexpr int kKs = HD / 16;               // k slices of the first product
    static constexpr int kNt = HD / 16;               // accumulator tiles of the second
    static constexpr int kGs = row_scales<FMT>(HD);
    static constexpr int RB = row_bytes<FMT>(HD);
    static constexpr int kBlocks = NT == 1 ? 2 : 1;   // (registers) blocks of 16 positions between looks at the maximum
    // values into registers before the look at the maximum (35 rows over 16 x 16,000 positions of e4m3, heads of 128:
    // 120 us instead of 140; e2m1 and 8 rows have no registers for it: 145 instead of 138)
    static constexpr bool kEarly = FMT == kE4M3 && NT > 1;
    static constexpr bool kQRegs = NT * HD <= 128;    // q operands stay in registers
    int g, c, at;
    const __half* s_q;
    const int* s_lim;                                 // positions that each row sees
    float l[NT][2], M[NT][2], f[NT][2];               // l: this lane's positions
    float o[NT][kNt][4];                              // two elements of a tile by the two rows
    uint32_t q[kQRegs ? NT : 1][kQRegs ? kKs : 1][2];

    __device__ __forceinline__ uint2 load_q(int n, int s) const {
        return *reinterpret_cast<const uint2*>(s_q + (8 * n + g) * (HD + 8) + key_dim<FMT>(s, c));
    }
    __device__ __forceinline__ Rows(int lane, const __half* sq, const float* s_f, const int* lim)
        : g(lane >> 2), c(lane & 3), at(4 * (g >> 1) + (g & 1)), s_q(sq), s_lim(lim) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int e = 0; e < 2; ++e) M[n][e] = -INFINITY, l[n][e] = 0.f, f[n][e] = s_f[8 * n + 2 * c + e];
#pragma unroll
            for (int t = 0; t < kNt; ++t) o[n][t][0] = o[n][t][1] = o[n][t][2] = o[n][t][3] = 0.f;
            if (kQRegs)
#pragma unroll
                for (int s = 0; s < kKs; ++s) {
                    const uint2 x = load_q(n, s);
                    q[kQRegs ? n : 0][kQRegs ? s : 0][0] = x.x, q[kQRegs ? n : 0][kQRegs ? s : 0][1] = x.y;
                }
        }
    }
    // d += sixteen keys' slice by the rows of tile n
    __device__ __forceinline__ void key_product(float (&d)[4], const uint32_t (&a)[4], int n, int s) const {
        if (kQRegs) {
            mma16816(d, a, q[kQRegs ? n : 0][kQRegs ? s : 0][0], q[kQRegs ? n : 0][kQRegs ? s : 0][1]);
        } else {
            const uint2 x = load_q(n, s);
            mma16816(d, a, x.x, x.y);
        }
    }
    // positions base .. base + kStep - 1, whose keys and then values are at kr
    template <bool kMask>
    __device__ __forceinline__ void step(const uint8_t* kr, const float* my_sc, int base) {
#pragma unroll
        for (int h0 = 0; h0 < 2; h0 += kBlocks) block<kMask>(kr, my_sc, base, h0);
    }
    template <bool kMask>
    __device__ __forceinline__ void block(const uint8_t* kr, const float* my_sc, int base, int h0) {
        float s[kBlocks][2][NT][2], lv[kBlocks][2];
        int lim[NT][2];
        if (kMask)
#pragma unroll
            for (int n = 0; n < NT; ++n) lim[n][0] = s_lim[8 * n + 2 * c] - base, lim[n][1] = s_lim[8 * n + 2 * c + 1] - base;
        bool up = false;
#pragma unroll
        for (int h = 0; h < kBlocks; ++h) {
            uint32_t kw[2][FMT == kE4M3 ? HD / 16 : HD / 32];
            float sc[2][kGs];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int p = 16 * (h0 + h) + 2 * j + at;
                const uint8_t* row = kr + p * RB;
                if (FMT == kE4M3) {
#pragma unroll
                    for (int i = 0; i < HD / 64; ++i) {
                        const uint4 x = *reinterpret_cast<const uint4*>(row + 64 * i + 16 * c);
                        kw[j][4 * i] = x.x, kw[j][4 * i + 1] = x.y, kw[j][4 * i + 2] = x.z, kw[j][4 * i + 3] = x.w;
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < HD / kGroup; ++i)
                        kw[j][i] = *reinterpret_cast<const uint32_t*>(row + 16 * i + 4 * c);
                }
                lv[h][j] = my_sc[2 * kGs * kStep + p];
#pragma unroll
                for (int i = 0; i < kGs; ++i) sc[j][i] = my_sc[i * kStep + p];
            }
            constexpr int kPer = kKs / kGs;  // slices under one scale
#pragma unroll
            for (int i = 0; i < kGs; ++i) {
                float d[NT][4];
#pragma unroll
                for (int n = 0; n < NT; ++n) d[n][0] = d[n][1] = d[n][2] = d[n][3] = 0.f;
                uint32_t x[4], y[4];
                if (FMT == kE2M1) e2m1x8_to_half(kw[0][i], x), e2m1x8_to_half(kw[1][i], y);
#pragma unroll
                for (int sl = 0; sl < kPer; ++sl) {
                    uint32_t a[4];
                    if (FMT == kE4M3) {
                        e4m3x4_to_half(kw[0][sl], a[0], a[2]);
                        e4m3x4_to_half(kw[1][sl], a[1], a[3]);
                    } else {
                        a[0] = x[2 * sl], a[1] = y[2 * sl], a[2] = x[2 * sl + 1], a[3] = y[2 * sl + 1];
                    }
#pragma unroll
                    for (int n = 0; n < NT; ++n) key_product(d[n], a, n, kPer * i + sl);
                }
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int j = 0; j < 2; ++j)
#pragma unroll
                        for (int e = 0; e < 2; ++e)
                            s[h][j][n][e] = i ? fmaf(d[n][2 * j + e], sc[j][i], s[h][j][n][e]) : d[n][2 * j + e] * sc[j][0];
            }
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float& v = s[h][j][n][e];
                        v *= f[n][e];
                        if (kMask && 16 * (h0 + h) + 2 * j + at >= lim[n][e]) v = -INFINITY;
                        up |= v + lv[h][j] > M[n][e] + kLazy;
                    }
        }
        uint32_t v[4][HD / 32];  // a block's values
        if (kEarly) value_words<FMT, HD>(kr + (kStep + 16 * h0 + 4 * c) * RB, g, v);
        if (__any_sync(0xFFFFFFFFu, up)) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float t = -INFINITY;
#pragma unroll
                    for (int h = 0; h < kBlocks; ++h) t = fmaxf(t, fmaxf(s[h][0][n][e] + lv[h][0], s[h][1][n][e] + lv[h][1]));
#pragma unroll
                    for (int x = 4; x < 32; x <<= 1) t = fmaxf(t, __shfl_xor_sync(0xFFFFFFFFu, t, x));
                    if (t > M[n][e] + kLazy) {
                        t -= kBelow;
                        const float raise = ex2(M[n][e] - t);
                        M[n][e] = t;
                        l[n][e] *= raise;
#pragma unroll
                        for (int i = 0; i < kNt; ++i) o[n][i][e] *= raise, o[n][i][2 + e] *= raise;
                    }
                }
        }
#pragma unroll
        for (int h = 0; h < kBlocks; ++h) {
            float vsc[2][kGs];
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int i = 0; i < kGs; ++i) vsc[j][i] = my_sc[(kGs + i) * kStep + 16 * (h0 + h) + 2 * j + at];
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float ref = M[n][e] == -INFINITY ? 0.f : M[n][e];  // (nothing seen yet: every weight is 0)
#pragma unroll
                    for (int j = 0; j < 2; ++j) l[n][e] += s[h][j][n][e] = ex2(s[h][j][n][e] - ref);
                }
            // the operand of the positions' weights under value scale i, for tile n
            const auto weights = [&](int n, int i, uint32_t (&b)[2]) {
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    float y[2] = {s[h][j][n][0] * vsc[j][i], s[h][j][n][1] * vsc[j][i]};
                    if (kMask) {  // a hidden position's scale may be NaN
#pragma unroll
                        for (int e = 0; e < 2; ++e)
                            if (16 * (h0 + h) + 2 * j + at >= lim[n][e]) y[e] = 0.f;
                    }
                    b[j] = transposed(pack_half(y[0], y[1]));
                }
            };
            uint32_t b[NT][2];
            if (!kEarly) value_words<FMT, HD>(kr + (kStep + 16 * (h0 + h) + 4 * c) * RB, g, v);
            // O += V P: pairs of positions of two elements, sixteen elements a tile
#pragma unroll
            for (int w = 0; w < HD / 32; ++w) {
                if (FMT == kE2M1 || w == 0)
#pragma unroll
                    for (int n = 0; n < NT; ++n) weights(n, FMT == kE2M1 ? w : 0, b[n]);
                uint32_t lo[4], hi[4];
                value_pairs<FMT>(v[0][w], v[1][w], v[2][w], v[3][w], lo, hi);
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const uint32_t a[4] = {lo[2 * i], lo[2 * i + 1], hi[2 * i], hi[2 * i + 1]};
#pragma unroll
                    for (int n = 0; n < NT; ++n) mma16816(o[n][2 * w + i], a, b[n][0], b[n][1]);
                }
            }
        }
    }
    // a row's denominator over its eight lanes
    __device__ __forceinline__ void close() {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e)
#pragma unroll
                for (int x = 4; x < 32; x <<= 1) l[n][e] += __shfl_xor_sync(0xFFFFFFFFu, l[n][e], x);
    }
    // (M, l) of the rows and their accumulators [row][padded row of `os` floats]
    __device__ __forceinline__ void store(float* meta, float* acc, int os) const {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int r = 8 * n + 2 * c + e;
                if (g == 0) meta[2 * r] = M[n][e], meta[2 * r + 1] = l[n][e];
#pragma unroll
                for (int i = 0; i < kNt; ++i)
                    *reinterpret_cast<float2*>(acc + r * os + value_dim<FMT, HD>(g, 2 * i)) =
                        make_float2(o[n][i][e], o[n][i][2 + e]);
            }
    }
};

template <int FMT, int HD, int NT>
__global__ void __launch_bounds__(kThreads, Cfg<FMT, HD, NT>::kMinCtas) attn_kernel(const __grid_constant__ AttnArgs A) {
    using F = Cfg<FMT, HD, NT>;
    constexpr int kRows = F::kRows;
    constexpr int kGs = row_scales<FMT>(HD);
    constexpr int RB = row_bytes<FMT>(HD);
    extern __shared__ __align__(16) uint8_t sm[];
    float* s_o = reinterpret_cast<float*>(sm);                      // [kWarps][kRows][kOs], over the ring
    float* s_sc = reinterpret_cast<float*>(sm + F::kBig);           // [kWarps][kKinds][kStep]
    float* s_meta = s_sc + kWarps * F::kKinds * kStep;              // [kWarps][kRows][2]
    float* s_f = s_meta + kWarps * kRows * 2;                       // [kRows] score factors
    int* s_lim = reinterpret_cast<int*>(s_f + kRows);               // [kRows] positions that a row sees
    __half* s_q = reinterpret_cast<__half*>(s_lim + kRows);         // [kRows][HD + 8]
    __shared__ uint32_t s_scan[kWarps + 2];
    pdl_wait();
    pdl_release();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const bool second = blockIdx.x >= A.p.ctas;
    const Pass& P = second ? A.also : A.p;
    const uint32_t cta = blockIdx.x - (second ? A.p.ctas : 0);
    const bool shared_rows = P.prefix_len != nullptr;
    const int per_b = P.c.kv_heads * P.tiles;  // segments of a sequence
    const int per_seq = A.n_q * A.group;
    const int n_rows = shared_rows ? A.batch * per_seq : per_seq;
    const int prefix_len = shared_rows ? max(0, min(*P.prefix_len, P.c.max_len)) : 0;
    const auto len_of = [&](int b) { return shared_rows ? prefix_len : seen_len(A.pos[b], A.n_q, A.max_len); };

    uint32_t u, u_end, b_first;
    int b;
    if (A.cluster) {  // a segment's units, alike over the cluster's CTAs
        const uint32_t seg = blockIdx.x / A.cluster, rank = blockIdx.x % A.cluster;
        b = seg / per_b, b_first = 0;
        const uint32_t nu = units_of(len_of(b)), per = (nu + A.cluster - 1) / A.cluster;
        u = seg % per_b * nu + min(rank * per, nu);
        u_end = seg % per_b * nu + min(rank * per + per, nu);
    } else if (!my_units<kThreads>(P, cta, shared_rows ? 1 : A.batch, len_of, s_scan, u, u_end, b_first, b)) {
        return;
    }
    const uint32_t u_begin = u;

    uint8_t* ring = sm + warp * F::kStages * F::kStage;
    const uint32_t ring_a = (uint32_t)__cvta_generic_to_shared(ring);
    float* my_sc = s_sc + warp * F::kKinds * kStep;

    while (u < u_end) {
        // ---- the segment that unit u belongs to ----
        const int len = len_of(b);
        const uint32_t nu = units_of(len), nv = nu + P.lead;
        if (u >= b_first + nv * per_b) {
            b_first += nv * per_b;
            ++b;
            continue;
        }
        const uint32_t in_b = (u - b_first) / nv;
        const int kvh = in_b / P.tiles, tile = in_b % P.tiles;
        const uint32_t seg = b_first + in_b * nv;
        const Part part(u, u_end, seg, nu, P.lead);
        if (part.ua >= part.ub) break;
        const int ua = part.ua, ub = part.ub;
        const int r0 = tile * kRows;
        const int p0 = shared_rows ? 0 : A.pos[b];
        const int first = shared_rows ? len : p0 < len ? p0 + 1 : len;  // positions that every row sees
        const int64_t head = (int64_t)b * P.c.kv_heads + kvh;
        const uint8_t* kc = static_cast<const uint8_t*>(P.c.k) + head * P.c.max_len * RB;
        const uint8_t* vc = static_cast<const uint8_t*>(P.c.v) + head * P.c.max_len * RB;
        const uint16_t* ks = P.c.k_scale + head * P.c.max_len * kGs;
        const uint16_t* vs = P.c.v_scale + head * P.c.max_len * kGs;
        const auto row_of = [&](int r, int* rb, int* ri, int* rh) -> int64_t {  // tile row -> output row
            const int x = r0 + r, w = shared_rows ? x % per_seq : x;
            *rb = shared_rows ? x / per_seq : b;
            *ri = w / A.group;
            *rh = kvh * A.group + w % A.group;
            return ((int64_t)*rb * A.n_q + *ri) * A.n_heads + *rh;
        };

        // a step's rows are contiguous: 16 bytes a lane at a time
        const auto issue = [&](int un, int slot) {
            const int base = un * kUnit + warp * kStep;
            if (un < ub && base < len) {
                const uint8_t* sk = kc + (int64_t)base * RB + lane * 16;
                const uint8_t* sv = vc + (int64_t)base * RB + lane * 16;
                const uint32_t d = ring_a + slot * F::kStage + lane * 16;
                if (base + kStep <= len) {
#pragma unroll
                    for (int i = 0; i < kStep * RB / 512; ++i) {
                        copy16(d + i * 512, sk + i * 512);
                        copy16(d + kStep * RB + i * 512, sv + i * 512);
                    }
                } else {  // zeros behind the last position
                    const int left = (len - base) * RB - lane * 16;
#pragma unroll
                    for (int i = 0; i < kStep * RB / 512; ++i) {
                        const bool in = i * 512 < left;
                        copy16(d + i * 512, in ? sk + i * 512 : kc, in ? 16 : 0);
                        copy16(d + kStep * RB + i * 512, in ? sv + i * 512 : vc, in ? 16 : 0);
                    }
                }
                if constexpr (FMT == kE2M1) {
                    const bool in = base + lane < len;
                    const int64_t at = in ? (int64_t)(base + lane) * kGs : 0;
                    const uint32_t ds = ring_a + slot * F::kStage + F::kRowsB + lane * kGs * 2;
                    copy_small<kGs * 2>(ds, ks + at, in);
                    copy_small<kGs * 2>(ds + F::kScaleB, vs + at, in);
                }
            }
            copy_commit();
        };
        uint32_t nks = 0, nvs = 0;  // e4m3: the next step's scales of position `lane`
        const auto fetch_scales = [&](int un) {
            const int j = un * kUnit + warp * kStep + lane;
            const bool in = un < ub && j < len;
            nks = in ? load_u16(ks + j) : 0;
            nvs = in ? load_u16(vs + j) : 0;
        };
#pragma unroll
        for (int s = 0; s < F::kStages - 1; ++s) issue(ua + s, s);
        if (FMT == kE4M3) fetch_scales(ua);

        // ---- rotated queries, divided by a power of two per row, as halves ----
        {
            constexpr int kLanes = HD / 8;  // lanes of a row, eight elements each
            constexpr int kAtOnce = kThreads / kLanes;
#pragma unroll
            for (int it = 0; it < (kRows + kAtOnce - 1) / kAtOnce; ++it) {
                const int r = it * kAtOnce + tid / kLanes, sub = tid % kLanes;
                const bool in = r < kRows && r0 + r < n_rows;
                int rb = 0, ri = 0, rh = 0;
                if (in) row_of(r, &rb, &ri, &rh);
                const Query x = rotated_query<HD>(A, in, load_query<HD>(A, in, rb, ri, rh, sub), sub);
                if (r < kRows) {
                    *reinterpret_cast<uint4*>(s_q + r * (HD + 8) + sub * 8) =
                        make_uint4(pack_half(x.x[0], x.x[1]), pack_half(x.x[2], x.x[3]), pack_half(x.x[4], x.x[5]),
                                   pack_half(x.x[6], x.x[7]));
                    if (sub == 0) {
                        s_f[r] = x.f;
                        s_lim[r] = shared_rows ? len : min(first + (r0 + r) / A.group, len);
                    }
                }
            }
        }
        __syncthreads();

        Rows<FMT, HD, NT> tile_of(lane, s_q, s_f, s_lim);
        int slot = 0;
        for (int un = ua; un < ub; ++un) {
            const int base = un * kUnit + warp * kStep;
            if (base >= len) break;  // (only the last unit ends early)
            issue(un + F::kStages - 1, slot == 0 ? F::kStages - 1 : slot - 1);
            if (FMT == kE2M1) copy_wait<F::kStages - 1>();
            __syncwarp();  // (the step before has read its scales)
            const uint8_t* kr = ring + slot * F::kStage;
            // the step's scales as floats: keys, values, log2 of the largest value scale
            if (FMT == kE4M3) {
                const float x = bf_lo(nvs);
                my_sc[lane] = bf_lo(nks);
                my_sc[kStep + lane] = x;
                my_sc[2 * kStep + lane] = fmaxf(lg2(x), kLeast);
                fetch_scales(un + 1);
                copy_wait<F::kStages - 1>();
            } else {
                const uint32_t* sc = reinterpret_cast<const uint32_t*>(kr + F::kRowsB) + lane * (kGs / 2);
                float top = 0.f;
#pragma unroll
                for (int i = 0; i < kGs / 2; ++i) {
                    const uint32_t a = sc[i], x = sc[F::kScaleB / 4 + i];
                    my_sc[2 * i * kStep + lane] = bf_lo(a), my_sc[(2 * i + 1) * kStep + lane] = bf_hi(a);
                    my_sc[(kGs + 2 * i) * kStep + lane] = bf_lo(x), my_sc[(kGs + 2 * i + 1) * kStep + lane] = bf_hi(x);
                    top = fmaxf(fmaxf(top, bf_lo(x)), bf_hi(x));
                }
                my_sc[2 * kGs * kStep + lane] = fmaxf(lg2(top), kLeast);
            }
            __syncwarp();
            if (base + kStep > first) tile_of.template step<true>(kr, my_sc, base);
            else tile_of.template step<false>(kr, my_sc, base);
            slot = slot + 1 == F::kStages ? 0 : slot + 1;
            __syncwarp();  // the slot is read: the next issue may fill it
        }
        copy_wait<0>();
        tile_of.close();
        __syncthreads();  // every warp's ring is drained: the accumulators go over it
        tile_of.store(s_meta + warp * kRows * 2, s_o + warp * kRows * F::kOs, F::kOs);
        __syncthreads();
        // ---- join the warps; whole segments are final (or records), cut ones go to a slot ----
        const bool whole = ua == 0 && ub == (int)nu;
        float* cut = P.slots + ((int64_t)cta * 2 + (u_begin >= seg ? 0 : 1)) * kRows * (kMeta + HD);
        const int rows = min(kRows, n_rows - r0);
        for (int r = warp; r < rows; r += kWarps) {
            float lw[kWarps], Mw[kWarps], top = -INFINITY, sum = 0.f;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                const float* x = s_meta + (w * kRows + r) * 2;
                Mw[w] = x[0], lw[w] = x[1];
                top = fmaxf(top, Mw[w]);
            }
            const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                Mw[w] = ex2(Mw[w] - ref);
                sum = fmaf(lw[w], Mw[w], sum);
            }
            float v[HD / 32];
#pragma unroll
            for (int j = 0; j < HD / 32; ++j) {
                v[j] = 0.f;
#pragma unroll
                for (int w = 0; w < kWarps; ++w) v[j] = fmaf(Mw[w], s_o[(w * kRows + r) * F::kOs + lane + 32 * j], v[j]);
            }
            int rb, ri, rh;
            const int64_t row = row_of(r, &rb, &ri, &rh);
            if (whole && !P.recs) {
                const int p = A.pos[rb];
                const bool over = (int64_t)p + ri >= A.max_len;
                const float k = over ? nan_f() : 1.f / sum;
#pragma unroll
                for (int j = 0; j < HD / 32; ++j)
                    A.out[row * HD + lane + 32 * j] = __bfloat16_as_ushort(__float2bfloat16_rn(p < 0 ? 0.f : v[j] * k));
            } else if (A.cluster) {  // (over the first warp's part: this warp alone reads the row)
                __syncwarp();
                if (lane == 0) *reinterpret_cast<float2*>(s_meta + r * 2) = make_float2(top, sum);
#pragma unroll
                for (int j = 0; j < HD / 32; ++j) s_o[r * F::kOs + lane + 32 * j] = v[j];
            } else {
                float* dst = whole ? P.recs + row * (kMeta + HD) : cut + r * (kMeta + HD);
                if (lane == 0) *reinterpret_cast<float4*>(dst) = make_float4(top, sum, 0.f, 0.f);
#pragma unroll
                for (int j = 0; j < HD / 32; ++j) dst[kMeta + lane + 32 * j] = v[j];
            }
        }
        u = part.next;
        __syncthreads();  // shared memory may be filled again
    }
    if (A.cluster) {
        // ---- join the cluster's CTAs, a warp a row ----
        cg::cluster_group cluster = cg::this_cluster();
        cluster.sync();
        const uint32_t seg = blockIdx.x / A.cluster, rank = blockIdx.x % A.cluster;
        const int nu = units_of(len_of(b)), per = (nu + A.cluster - 1) / A.cluster, parts = (nu + per - 1) / per;
        const int kvh = seg % per_b / A.p.tiles, r0 = seg % A.p.tiles * kRows;
        if (parts > 1)
            for (int r = rank * kWarps + warp; r < min(kRows, n_rows - r0); r += A.cluster * kWarps) {
                float2 m[kMaxCluster];
                float a[kMaxCluster][HD / 32];
#pragma unroll
                for (int k = 0; k < kMaxCluster; ++k) {
                    m[k] = make_float2(-INFINITY, 0.f);
                    if (k < parts) m[k] = *reinterpret_cast<const float2*>(cluster.map_shared_rank(s_meta, k) + r * 2);
#pragma unroll
                    for (int j = 0; j < HD / 32; ++j)
                        a[k][j] = k < parts ? cluster.map_shared_rank(s_o, k)[r * F::kOs + lane + 32 * j] : 0.f;
                }
                float top = -INFINITY, sum = 0.f, v[HD / 32];
#pragma unroll
                for (int k = 0; k < kMaxCluster; ++k) top = fmaxf(top, m[k].x);
                const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll
                for (int j = 0; j < HD / 32; ++j) v[j] = 0.f;
#pragma unroll
                for (int k = 0; k < kMaxCluster; ++k) {
                    const float e = ex2(m[k].x - ref);
                    sum = fmaf(m[k].y, e, sum);
#pragma unroll
                    for (int j = 0; j < HD / 32; ++j) v[j] = fmaf(a[k][j], e, v[j]);
                }
                const int i = (r0 + r) / A.group;
                const float k = (int64_t)A.pos[b] + i >= A.max_len ? nan_f() : 1.f / sum;
                const int64_t row = ((int64_t)b * A.n_q + i) * A.n_heads + kvh * A.group + (r0 + r) % A.group;
#pragma unroll
                for (int j = 0; j < HD / 32; ++j) A.out[row * HD + lane + 32 * j] = __bfloat16_as_ushort(__float2bfloat16_rn(v[j] * k));
            }
        cluster.sync();  // (the others' reads of this CTA's part)
    }
}

struct JoinArgs {
    Pass own, prefix;  // prefix.prefix_len null: own alone
    const int32_t* pos;
    uint16_t* out;
    int32_t batch, n_q, n_heads, group, max_len;
};

// kW warps a row, four warps a CTA or one row: the parts that the passes left
// of it, spread over its warps (kDeep loads in flight each), their weighted
// sums added in warp order. A row whose only segment one CTA had whole is
// final already. A chain of three loads from L2 (shares, parts, and before
// them the predecessor's end) bounds it: about 2 us behind the pass in a graph.
template <int HD, int kW>
__global__ void __launch_bounds__(kW == 1 ? 128 : 32 * kW) join_kernel(const JoinArgs A) {
    using Vec = typename std::conditional<HD == 128, float4, float2>::type;  // a lane's share of a row
    constexpr int kF = kMeta + HD, kL = HD / 32;
    constexpr int kDeep = 6;
    __shared__ float s_m[kW][2];
    __shared__ Vec s_v[kW][32];
    pdl_wait();
    pdl_release();
    const int lane = threadIdx.x & 31, warp = kW == 1 ? 0 : threadIdx.x >> 5;
    const uint32_t row = kW == 1 ? blockIdx.x * 4 + (threadIdx.x >> 5) : blockIdx.x;
    if (row >= (uint32_t)A.batch * A.n_q * A.n_heads) return;
    const uint32_t head = row % A.n_heads, bi = row / A.n_heads, i = bi % A.n_q, b = bi / A.n_q;
    const uint32_t kvh = head / A.group, r = i * A.group + head % A.group;
    const int p = A.pos[b];

    // the parts of this row: a record of its own, or slots of CTAs i0 .. i0 + n - 1
    struct Parts {
        const float* base;
        int n;
        int64_t stride, skip;  // skip: the first CTA's slot
    };
    const auto parts_of = [&](const Pass& P, uint32_t first, uint32_t nu, uint32_t share, uint32_t x) {
        const uint32_t seg = first + (kvh * P.tiles + x / P.tile_rows) * (nu + P.lead), from = seg + P.lead;
        const uint32_t i0 = from / share, i1 = (from + nu - 1) / share;
        Parts q;
        q.n = i1 - i0 + 1;
        q.stride = (int64_t)2 * P.tile_rows * kF;
        q.skip = i0 * share >= seg ? 0 : P.tile_rows * kF;
        q.base = P.slots + i0 * q.stride + x % P.tile_rows * kF;
        if (q.n == 1) q.base = P.recs ? P.recs + (int64_t)row * kF : nullptr, q.skip = 0;
        return q;
    };
    const Parts own = parts_of(A.own, A.own.share[1 + b], units_of(seen_len(p, A.n_q, A.max_len)), A.own.share[0], r);
    Parts pre{};
    bool bad = (int64_t)p + i >= A.max_len;
    if (A.prefix.prefix_len) {
        const int pl = *A.prefix.prefix_len;
        bad |= pl > A.prefix.c.max_len;
        pre = parts_of(A.prefix, 0, units_of(max(0, min(pl, A.prefix.c.max_len))), A.prefix.share[0],
                       b * A.n_q * A.group + r);
    } else if (own.n == 1) {
        return;  // final already
    }
    const auto at = [&](const Parts& q, int s) { return q.base + (s ? s * q.stride : q.skip); };
    const int n = own.n + pre.n;
    float top = -INFINITY, sum = 0.f, v[kL];
#pragma unroll
    for (int j = 0; j < kL; ++j) v[j] = 0.f;
    // a warp's parts, with a running maximum
    for (int s0 = warp; s0 < n; s0 += kDeep * kW) {
        float2 x[kDeep];
        Vec a[kDeep];
#pragma unroll
        for (int k = 0; k < kDeep; ++k) {
            const int s = s0 + k * kW;
            x[k] = make_float2(-INFINITY, 0.f), a[k] = Vec{};
            if (s < n) {
                const float* src = s < own.n ? at(own, s) : at(pre, s - own.n);
                x[k] = *reinterpret_cast<const float2*>(src);
                a[k] = reinterpret_cast<const Vec*>(src + kMeta)[lane];
            }
        }
#pragma unroll
        for (int k = 0; k < kDeep; ++k) {
            const float t = fmaxf(top, x[k].x), ref = t == -INFINITY ? 0.f : t;
            const float w0 = ex2(top - ref), w1 = ex2(x[k].x - ref);
            sum = sum * w0 + x[k].y * w1;
#pragma unroll
            for (int j = 0; j < kL; ++j) v[j] = fmaf(v[j], w0, reinterpret_cast<const float*>(&a[k])[j] * w1);
            top = t;
        }
    }
    if (kW > 1) {
        if (lane == 0) s_m[warp][0] = top, s_m[warp][1] = sum;
#pragma unroll
        for (int j = 0; j < kL; ++j) reinterpret_cast<float*>(&s_v[warp][lane])[j] = v[j];
        __syncthreads();
        if (warp) return;
        top = -INFINITY, sum = 0.f;
#pragma unroll
        for (int w = 0; w < kW; ++w) top = fmaxf(top, s_m[w][0]);
        const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll
        for (int j = 0; j < kL; ++j) v[j] = 0.f;
#pragma unroll
        for (int w = 0; w < kW; ++w) {
            const float e = ex2(s_m[w][0] - ref);
            sum = fmaf(s_m[w][1], e, sum);
            const Vec y = s_v[w][lane];
#pragma unroll
            for (int j = 0; j < kL; ++j) v[j] = fmaf(reinterpret_cast<const float*>(&y)[j], e, v[j]);
        }
    }
    uint32_t o[kL / 2];
#pragma unroll
    for (int j = 0; j < kL; ++j) v[j] = p < 0 ? 0.f : bad ? nan_f() : v[j] / sum;
#pragma unroll
    for (int j = 0; j < kL / 2; ++j) o[j] = pack_bf(v[2 * j], v[2 * j + 1]);
    uint32_t* out = reinterpret_cast<uint32_t*>(A.out + (int64_t)row * HD) + lane * (kL / 2);
#pragma unroll
    for (int j = 0; j < kL / 2; ++j) out[j] = o[j];
}

// The kernel of a pass's row tiles (of 8 NT rows), its resident CTAs on one
// multiprocessor of device `dev` (its shared-memory limit is set at the first
// call; 0 on an error) or its launch.
template <int FMT, int HD, int NT>
struct Variant {
    static cudaError_t launch(const AttnArgs& A, cudaStream_t s) {
        const auto k = attn_kernel<FMT, HD, NT>;
        constexpr int sm = Cfg<FMT, HD, NT>::kSmem;
        if (!A.cluster) return launch_pdl(k, dim3(A.p.ctas + A.also.ctas), dim3(kThreads), sm, s, A);
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(A.p.ctas), cfg.blockDim = dim3(kThreads), cfg.dynamicSmemBytes = sm, cfg.stream = s;
        cudaLaunchAttribute attr[2];
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        attr[1].id = cudaLaunchAttributeClusterDimension;
        attr[1].val.clusterDim.x = A.cluster, attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
        cfg.attrs = attr, cfg.numAttrs = 2;
        return cudaLaunchKernelEx(&cfg, k, A);
    }
    static int resident(int dev) {
        static std::atomic<int> known[128];
        if (dev < 0 || dev >= 128) return 0;
        int n = known[dev].load(std::memory_order_relaxed);
        if (n) return n;
        const auto k = attn_kernel<FMT, HD, NT>;
        constexpr int sm = Cfg<FMT, HD, NT>::kSmem;
        if (cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, sm) != cudaSuccess ||
            cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, k, kThreads, sm) != cudaSuccess)
            return 0;
        known[dev].store(n, std::memory_order_relaxed);
        return n;
    }
};
struct Kernel {
    cudaError_t (*launch)(const AttnArgs&, cudaStream_t);
    int (*resident)(int);
};
template <int FMT, int HD, int NT>
constexpr Kernel kernel() {
    return {Variant<FMT, HD, NT>::launch, Variant<FMT, HD, NT>::resident};
}
// nt: 1, 2, for heads of 128 also 3
template <int FMT>
Kernel kernel_of(int hd, int nt) {
    if (hd == 64)
        return nt == 1 ? kernel<FMT, 64, 1>() : kernel<FMT, 64, 2>();
    return nt == 1 ? kernel<FMT, 128, 1>() : nt == 2 ? kernel<FMT, 128, 2>() : kernel<FMT, 128, 3>();
}
Kernel kernel_of(const Pass& p) {
    return p.c.format == kE4M3 ? kernel_of<kE4M3>(p.c.head_dim, p.tile_rows / 8)
                               : kernel_of<kE2M1>(p.c.head_dim, p.tile_rows / 8);
}

cudaError_t launch_attn(const AttnArgs& A, cudaStream_t s) {
    return A.p.tile_rows == kMmaRows ? mma_attn_launch(A, s) : kernel_of(A.p).launch(A, s);
}

// A pass's kernel, tiles and CTAs: as many as are resident at once, or one a
// unit. (Both sides below are e4m3 times in us; the lengths that count are the
// cache's, for the host does not know those of its sequences.)
bool plan_pass(const cdq_kv_cache* c, int64_t seqs, int64_t rows, int dev, int sms, Pass* P) {
    P->c = *c;
    const int64_t len_units = (c->max_len + kUnit - 1) / kUnit, heads = seqs * c->kv_heads;
    int res = 1;
    if (heads * len_units >= (1ll << 31)) return false;
    // The tcgen05 kernel pads its rows to 128 and starts slowly: it is for many rows over many units a multiprocessor.
    // 16 x 16,000 positions, heads of 128: 63 rows 145 (169 the other kernel), 77 rows 145 (217); 32 x 8,000 of 64:
    // 63 rows 66 (57), 77 rows 68 (69), 91 rows 66 (79). Over a prefix: 126 rows of 60,000 positions, heads of 128 (13
    // units a multiprocessor), 72 (101), heads of 64 (6) 37 (38), of 8,000 (1) 25 (19); 336 rows of 8,000, heads of 128
    // (5) 63 (51).
    const int64_t wide = (rows + kMmaRows - 1) / kMmaRows;
    if (c->format == kE4M3 && rows > (c->head_dim == 64 ? 72 : 48) && heads * wide * len_units >= 8ll * sms) {
        P->tile_rows = kMmaRows;
        P->tiles = (int)wide;
    } else {
        // As few tiles as the widest allows (heads of 64: 16 rows, of 128: 24), of the narrowest that holds them; but
        // tiles of 8 where full caches are no more than a unit a CTA, where latency is what counts. 35 rows over 8 x
        // 5,000 positions, heads of 64: 15.7 in tiles of 16, 18.7 of 8, 21 of 24; over 700: 6.5 of 8, 7.3 of 16; over
        // 16 x 16,000, heads of 128: 152 of 24, 179 of 16, 204 of 8.
        P->tile_rows = 8;
        P->tiles = (int)((rows + 7) / 8);
        res = kernel_of(*P).resident(dev);
        if (P->tiles > 1 && heads * P->tiles * len_units > (int64_t)res * sms) {
            const int most = c->head_dim == 64 ? 16 : 24;
            P->tiles = (int)((rows + most - 1) / most);
            const int64_t per = (rows + P->tiles - 1) / P->tiles;
            P->tile_rows = per <= 8 ? 8 : per <= 16 ? 16 : 24;
            res = kernel_of(*P).resident(dev);
        }
    }
    // What beginning and finishing a segment costs, in units (none where every CTA has one unit at most, for it would
    // leave CTAs idle: 640 positions 6.1 us, with it 6.8). 96 rows of 28 heads over a prefix of 16,384 positions: 87 us
    // in all with 4 for the tcgen05 kernel, 89 with 6, 98 with 2, 100 with none; 35 rows over 8 ragged sequences of up
    // to 5,000: 15.7 with 2, 18.2 with none.
    P->lead = heads * P->tiles * len_units <= (int64_t)res * sms ? 0 : P->tile_rows == kMmaRows ? 4 : 2;
    const int64_t units = heads * P->tiles * (len_units + P->lead);
    P->ctas = (int)std::min<int64_t>(heads * P->tiles * len_units, (int64_t)res * sms);
    return res > 0 && units < (1ll << 31);
}

struct Plan {
    Pass own, prefix;
    bool one;  // one launch for both
    int cluster;
    bool many;  // the join takes sixteen warps a row
    int64_t rows, bytes, own_slots, pre_slots, recs, share;  // bytes of each part of the workspace
    bool join;
};

cdq_status plan(const cdq_kv_cache* c, int n_heads, int n_q, const cdq_kv_cache* prefix, Plan* P) {
    cdq_status st = check_cache(c);
    if (st) return st;
    if (n_q < 1 || n_q > CDQ_KV_MAX_NEW || n_heads < c->kv_heads || n_heads % c->kv_heads || n_heads > 65535)
        return CDQ_ERR_ARG;
    int dev = 0, sms = 0;
    if (prefix) {
        if ((st = check_cache(prefix))) return st;
        if (prefix->batch != 1 || prefix->kv_heads != c->kv_heads || prefix->head_dim != c->head_dim ||
            prefix->format != c->format)
            return CDQ_ERR_SHAPE;
    }
    if (cudaGetDevice(&dev) != cudaSuccess ||
        cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
        return CDQ_ERR_CUDA;
    const int64_t per_seq = (int64_t)n_q * (n_heads / c->kv_heads);
    P->rows = (int64_t)c->batch * n_q * n_heads;
    if (P->rows > 0x7FFFFFFF) return CDQ_ERR_SHAPE;
    P->own = P->prefix = Pass{};
    if (!plan_pass(c, c->batch, per_seq, dev, sms, &P->own)) return CDQ_ERR_CUDA;
    const int64_t rec = (kMeta + c->head_dim) * 4;
    const auto slots = [&](const Pass& p) { return (int64_t)p.ctas * 2 * p.tile_rows * rec; };
    // A cluster a segment, which joins its parts itself, where a cache has few units and all clusters are resident:
    // one sequence of 640 positions 5.5 us, with a
    // join in a launch of its own 6.2; 2,000 6.3 and 7.9; 4,000 7.8 and 6.8. (Three quarters of the places: clusters do
    // not pack.)
    const int64_t len_units = (c->max_len + kUnit - 1) / kUnit, segs = (int64_t)c->batch * c->kv_heads * P->own.tiles;
    P->cluster = (int)std::min<int64_t>(len_units, kMaxCluster);
    if (prefix || len_units < 2 || len_units > 2 * kMaxCluster || P->own.tile_rows == kMmaRows ||
        segs * P->cluster > (int64_t)kernel_of(P->own).resident(dev) * sms * 3 / 4)
        P->cluster = 0;
    else
        P->own.ctas = (int)segs * P->cluster, P->own.lead = 0;
    // a segment of one unit is never cut
    P->join = prefix || (c->max_len > kUnit && !P->cluster);
    P->own_slots = P->join ? slots(P->own) : 0;
    P->pre_slots = P->recs = 0;
    P->one = false;
    if (prefix) {
        if (!plan_pass(prefix, 1, per_seq * c->batch, dev, sms, &P->prefix)) return CDQ_ERR_CUDA;
        P->pre_slots = slots(P->prefix);
        // alike, and all of both resident at once: one launch (four samples of a 1,500-token prompt: 8.1 us,
        // with two 11.9)
        P->one = P->prefix.tile_rows == P->own.tile_rows && P->own.tile_rows != kMmaRows &&
                 P->own.ctas + P->prefix.ctas <= kernel_of(P->own).resident(dev) * sms;
        P->recs = P->rows * rec;
    }
    // Sixteen warps a row where a row has many parts: 131,072 positions over 592 CTAs 30.0 us in all, with a warp a row
    // 47.5; 8,000 positions 6.8 and 13.7. With fewer parts only while there is a multiprocessor a row: four samples of a
    // 1,500-token prompt (56 rows) 7.6 and 8.1, 35 rows over 8 x 2,500 positions (560 rows) 14.8 and 13.0.
    const int64_t parts = std::max<int64_t>(
        P->own.ctas / segs, prefix ? P->prefix.ctas / (prefix->kv_heads * P->prefix.tiles) : 0);
    P->many = parts > 16 || (parts > 8 && P->rows <= sms);
    P->share = P->join ? (4 * (c->batch + 3LL) + 15) / 16 * 16 : 0;  // of both passes
    P->bytes = P->own_slots + P->pre_slots + 2 * P->recs + P->share;
    return CDQ_OK;
}

}  // namespace

extern "C" {

cdq_status cdq_kv_attend_workspace(const cdq_kv_cache* cache, int32_t n_heads, int32_t n_q, const cdq_kv_cache* prefix,
                                   int64_t* bytes) {
    if (!bytes) return CDQ_ERR_ARG;
    Plan P;
    const cdq_status st = plan(cache, n_heads, n_q, prefix, &P);
    if (st == CDQ_OK) *bytes = P.bytes;
    return st;
}

cdq_status cdq_kv_attend(const cdq_kv_cache* cache, const uint16_t* q, int64_t q_seq, int64_t q_tok, int32_t n_heads,
                         int32_t n_q, const int32_t* pos, const uint16_t* cos_t, const uint16_t* sin_t,
                         int32_t table_rows, const int32_t* table_pos, float scale, const cdq_kv_cache* prefix,
                         const int32_t* prefix_len, uint16_t* out, void* workspace, int64_t workspace_bytes,
                         void* stream) {
    cdq_status st = check_cache(cache);
    if (st) return st;
    if (!strided(q, q_seq, q_tok) || !at(pos, 4) || !at(out, 16) || (prefix && !at(prefix_len, 4))) return CDQ_ERR_ARG;
    // one CTA writes its rows while another still reads its queries
    const int64_t row = (int64_t)n_heads * cache->head_dim;
    const uint16_t* q_end = q + (cache->batch - 1) * q_seq + (n_q - 1) * q_tok + row;
    if (out < q_end && q < out + (int64_t)cache->batch * n_q * row) return CDQ_ERR_ARG;
    Plan P;
    if ((st = plan(cache, n_heads, n_q, prefix, &P))) return st;
    AttnArgs A{};
    if ((st = check_rope(cos_t, sin_t, table_rows, table_pos, &A.rope))) return st;
    if (P.bytes && (!workspace || (uintptr_t)workspace % 16 || workspace_bytes < P.bytes)) return CDQ_ERR_WORKSPACE;
    const auto s = (cudaStream_t)stream;
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    P.own.slots = reinterpret_cast<float*>(ws);
    if (P.join) P.own.share = reinterpret_cast<uint32_t*>(ws + P.bytes - P.share);
    if (prefix) {
        P.prefix.share = P.own.share + 1 + cache->batch;
        P.prefix.slots = reinterpret_cast<float*>(ws + P.own_slots);
        P.own.recs = reinterpret_cast<float*>(ws + P.own_slots + P.pre_slots);
        P.prefix.recs = reinterpret_cast<float*>(ws + P.own_slots + P.pre_slots + P.recs);
        P.prefix.prefix_len = prefix_len;
    }
    A.q = q, A.q_seq = q_seq, A.q_tok = q_tok, A.pos = pos, A.out = out;
    A.scale_log2 = scale * 1.4426950408889634f;
    A.batch = cache->batch, A.n_q = n_q, A.n_heads = n_heads, A.group = n_heads / cache->kv_heads;
    A.max_len = cache->max_len;
    A.p = P.own;
    if (P.one) A.also = P.prefix;
    A.cluster = P.cluster;
    if (launch_attn(A, s) != cudaSuccess) return CDQ_ERR_CUDA;
    if (prefix && !P.one) {
        A.p = P.prefix;
        if (launch_attn(A, s) != cudaSuccess) return CDQ_ERR_CUDA;
    }
    if (P.join) {
        const JoinArgs J{P.own, P.prefix, pos, out, A.batch, n_q, n_heads, A.group, A.max_len};
        cudaError_t e;
        const dim3 few((unsigned)((P.rows + 3) / 4)), grid((unsigned)P.rows);
        if (cache->head_dim == 64)
            e = P.many ? launch_pdl(join_kernel<64, 16>, grid, dim3(512), 0, s, J)
                     : launch_pdl(join_kernel<64, 1>, few, dim3(128), 0, s, J);
        else
            e = P.many ? launch_pdl(join_kernel<128, 16>, grid, dim3(512), 0, s, J)
                     : launch_pdl(join_kernel<128, 1>, few, dim3(128), 0, s, J);
        if (e != cudaSuccess) return CDQ_ERR_CUDA;
    }
    return CDQ_OK;
}

}  // extern "C"
