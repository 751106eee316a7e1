// Attention over the quantised cache (cdq_kv.cuh): grouped-query attention of
// a few new positions of every sequence, and of a whole batch over a prefix
// that all its sequences share.
//
// The rows of one kv head, (new position i, head of the group g), r = i * G +
// g, form the M = 16 side of mma.m16n8k16; a warp walks the positions sixteen
// at a time:
//   S[r][j] = sum_d q[r][d] code_k[j][d]      the codes as halves, exact;
//   s_j     = S * scale_k[j] * f_r            log2 units;
//   l      += 2^(s_j - m),  O[r][d] += 2^(s_j + log2(scale_v[j]) - M) code_v[j][d]
// with a running maximum m of s_j for the denominator and another, M, of
// s_j + log2(scale_v[j]) for the numerator: the weights that enter the second
// product are at most 2^8 whatever the scales are, so rounding them to half
// costs 2^-12 of the largest contribution and no range. q is rotated in
// float32, divided by its row's power of two and rounded to half (2^-12).
// Neither operand is ever dequantised: scales multiply scores and weights.
//
// Both products contract over an order of elements that is free: a lane takes
// neighbouring bytes of a key row as its k slices (q is laid out to match),
// and a lane's four positions of a value slice are the four whose weights it
// already holds, so weights go from accumulator to operand without a shuffle.
//
// Positions are split over CTAs (and over a CTA's warps); partial (m, l, M, O)
// of a row are joined by a second launch when there is more than one part.
#include <algorithm>

#include "cdq_internal.cuh"
#include "cdq_kv.cuh"

using cdq::launch_pdl;
using cdq::pdl_release;
using cdq::pdl_wait;
using namespace cdq::kv;

namespace {

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr int kStep = 16;              // positions of a warp step
constexpr float kLazy = 8.f;           // M is raised only when it lags by more than this (log2)
constexpr int kMetaF = 4;              // floats of a partial's (m, l, M, -)
constexpr int kMaxParts = 256;         // parts of one row

struct AttnArgs {
    cdq_kv_cache c;          // the cache that this launch reads
    const uint16_t* q;
    int64_t q_seq, q_tok;
    const int32_t* pos;
    cdq_kv_rope rope;
    const int32_t* prefix_len;  // set: c is the prefix (one sequence's cache, rows of the whole batch)
    uint16_t* out;              // set: one part, the final result
    float* meta;                // partials: [row][parts][kMetaF]
    float* acc;                 // [row][parts][HD]
    float scale_log2;
    int32_t batch, n_q, n_heads, group, row_tiles, max_len;
    int32_t splits, part0, parts;  // this launch's splits, its first part, parts of a row in all
};

__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float lg2(float x) {
    float y;
    asm("lg2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// A warp step's data as one lane holds it: its slices of two key rows, of
// four value rows, and those four positions' scales.
template <int FMT, int HD>
struct Chunk {
    static constexpr int kK = FMT == kE4M3 ? HD / 16 : HD / 32;  // 32-bit words of a key row
    static constexpr int kV = FMT == kE4M3 ? HD / 32 : HD / 32;  // words (e2m1: half words) of a value row
    static constexpr int kS = FMT == kE4M3 ? 1 : HD / 64;        // words of a position's scales
    uint32_t k[2][kK], v[4][kV], ks[4][kS], vs[4][kS];
};

// positions base .. base + 15, those beyond `last` replaced by it
template <int FMT, int HD>
__device__ __forceinline__ void load_chunk(Chunk<FMT, HD>& x, const uint8_t* kc, const uint8_t* vc, const uint16_t* ks,
                                           const uint16_t* vs, int base, int last, int g, int c) {
    constexpr int RB = row_bytes<FMT>(HD);
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        const int j = min(base + 4 * (g >> 1) + 2 * t + (g & 1), last);
        const uint8_t* row = kc + (int64_t)j * RB;
        if (FMT == kE4M3) {
#pragma unroll
            for (int i = 0; i < HD / 64; ++i) {
                const uint4 u = __ldg(reinterpret_cast<const uint4*>(row + 64 * i) + c);
                x.k[t][4 * i] = u.x, x.k[t][4 * i + 1] = u.y, x.k[t][4 * i + 2] = u.z, x.k[t][4 * i + 3] = u.w;
            }
        } else {
#pragma unroll
            for (int i = 0; i < HD / kGroup; ++i) x.k[t][i] = __ldg(reinterpret_cast<const uint32_t*>(row + 16 * i) + c);
        }
    }
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        const int j = min(base + 4 * c + t, last);
        const uint8_t* row = vc + (int64_t)j * RB;
        if (FMT == kE4M3) {
            if (HD == 64) {
                const uint2 u = __ldg(reinterpret_cast<const uint2*>(row) + g);
                x.v[t][0] = u.x, x.v[t][1] = u.y;
            } else {
                const uint4 u = __ldg(reinterpret_cast<const uint4*>(row) + g);
                x.v[t][0] = u.x, x.v[t][1] = u.y, x.v[t][HD / 32 - 2] = u.z, x.v[t][HD / 32 - 1] = u.w;
            }
            x.ks[t][0] = __ldg(ks + j);
            x.vs[t][0] = __ldg(vs + j);
        } else {
#pragma unroll
            for (int i = 0; i < HD / kGroup; ++i) x.v[t][i] = __ldg(reinterpret_cast<const uint16_t*>(row + 16 * i) + g);
#pragma unroll
            for (int i = 0; i < HD / 64; ++i) {
                x.ks[t][i] = __ldg(reinterpret_cast<const uint32_t*>(ks + (int64_t)j * (HD / kGroup)) + i);
                x.vs[t][i] = __ldg(reinterpret_cast<const uint32_t*>(vs + (int64_t)j * (HD / kGroup)) + i);
            }
        }
    }
}

// scale `i` of a position
template <int FMT, int KS>
__device__ __forceinline__ float scale_of(const uint32_t (&s)[KS], int i) {
    if (FMT == kE4M3) return bf_lo(s[0]);
    return i & 1 ? bf_hi(s[i / 2]) : bf_lo(s[i / 2]);
}

// The element of a value row that column n of accumulator tile t stands for.
template <int FMT, int HD>
__device__ __forceinline__ int value_dim(int n, int t) {
    return FMT == kE4M3 ? (HD / 8) * n + t : kGroup * (t / 4) + 4 * n + t % 4;
}

// One CTA: (row tile, split) x kv head x sequence. MT tiles of 16 rows; HALF:
// at most 8 rows, the upper half of the only tile is padding.
template <int FMT, int HD, int MT, bool HALF>
__global__ void __launch_bounds__(kThreads) attn_kernel(const AttnArgs A) {
    constexpr int kRows = 16 * MT;
    constexpr int kH = HALF ? 1 : 2;      // halves of a tile that hold rows
    constexpr int kKs = HD / 16;          // k slices of the first product
    constexpr int kNt = HD / 8;           // accumulator tiles of the second
    constexpr int kOs = HD + 4;           // padded row of the joined accumulators
    extern __shared__ float sm[];
    float* s_o = sm;                                            // [kWarps][kRows][kOs]
    float* s_meta = s_o + kWarps * kRows * kOs;                 // [kWarps][kRows][3]
    float* s_f = s_meta + kWarps * kRows * 3;                   // [kRows] score factors
    __half* s_q = reinterpret_cast<__half*>(s_f + kRows);       // [kRows][HD + 8]
    pdl_wait();
    pdl_release();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, c = lane & 3;
    const int tile = blockIdx.x % A.row_tiles, split = blockIdx.x / A.row_tiles;
    const int kvh = blockIdx.y;
    const bool shared_rows = A.prefix_len != nullptr;
    const int b0 = blockIdx.z;  // the sequence (0 when the launch's rows span the batch)
    const int per_seq = A.n_q * A.group;
    const int n_rows = shared_rows ? A.batch * per_seq : per_seq;
    const int r0 = tile * kRows;
    int len, first;  // positions that any row sees, and that every row sees
    if (shared_rows) {
        len = max(0, min(*A.prefix_len, A.c.max_len));
        first = len;
    } else {
        const int p = A.pos[b0];
        len = p < 0 ? 0 : (int)min((int64_t)p + A.n_q, (int64_t)A.max_len);
        first = p < len ? p + 1 : len;
    }
    // this split's positions: whole steps of the CTA
    const int blocks = (len + kStep * kWarps - 1) / (kStep * kWarps);
    const int per = (blocks + A.splits - 1) / A.splits;
    const int t0 = min(split * per * kStep * kWarps, len), t1 = min(t0 + per * kStep * kWarps, len);

    const auto row_id = [&](int r, int* b, int* i, int* head) -> int64_t {  // row r of the tile -> output row
        const int x = r0 + r;
        *b = shared_rows ? x / per_seq : b0;
        const int w = shared_rows ? x % per_seq : x;
        *i = w / A.group;
        *head = kvh * A.group + w % A.group;
        return ((int64_t)*b * A.n_q + *i) * A.n_heads + *head;
    };

    if (t0 < t1) {
        // rotated queries, divided by a power of two per row, as halves
        for (int r = warp; r < kRows; r += kWarps) {
            float x[HD / 32];
            float amax = 0.f;
            bool nan = false;
            const bool in = r0 + r < n_rows;
            if (in) {
                int b, i, head;
                row_id(r, &b, &i, &head);
                const uint16_t* src = A.q + b * A.q_seq + i * A.q_tok + head * HD;
                const int64_t t = A.rope.cos_t ? (int64_t)(A.rope.rope_pos ? A.rope.rope_pos[b] : A.pos[b]) + i : 0;
                const bool ok = t >= 0 && t < A.rope.rows;
#pragma unroll
                for (int j = 0; j < HD / 32; ++j) {
                    const int d = lane + 32 * j;
                    x[j] = bf(src[d]);
                    if (A.rope.cos_t) {
                        const float o = bf(src[d ^ (HD / 2)]), sgn = d < HD / 2 ? -1.f : 1.f;
                        x[j] = ok ? fmaf(sgn * o, bf(A.rope.sin_t[t * HD + d]), x[j] * bf(A.rope.cos_t[t * HD + d]))
                                  : __int_as_float(0x7FC00000);
                    }
                    amax = fmaxf(amax, fabsf(x[j]));
                    nan |= x[j] != x[j];
                }
            } else {
#pragma unroll
                for (int j = 0; j < HD / 32; ++j) x[j] = 0.f;
            }
            if (nan) amax = INFINITY;
#pragma unroll
            for (int o = 16; o; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, o));
            const bool fine = amax <= 3.402823466e38f;
            const int e = fine && amax > 0.f ? ilogbf(amax) : 0;
#pragma unroll
            for (int j = 0; j < HD / 32; ++j) {
                const int d = lane + 32 * j;
                s_q[r * (HD + 8) + d] = __float2half_rn(fine ? scalbnf(x[j], -e) : 0.f);
            }
            if (lane == 0) s_f[r] = fine ? scalbnf(A.scale_log2, e) : __int_as_float(0x7FC00000);
        }
    }
    __syncthreads();

    float m[MT][kH], l[MT][kH], M[MT][kH];
    float o[MT][kNt][4];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
#pragma unroll
        for (int h = 0; h < kH; ++h) m[t][h] = M[t][h] = -INFINITY, l[t][h] = 0.f;
#pragma unroll
        for (int n = 0; n < kNt; ++n) o[t][n][0] = o[t][n][1] = o[t][n][2] = o[t][n][3] = 0.f;
    }
    if (t0 + warp * kStep < t1) {
        // q operands: slice s of lane c covers the elements that it reads of a key row
        uint32_t qa[MT][kKs][4];
        float f[MT][kH];
        int lim[MT][kH];
#pragma unroll
        for (int t = 0; t < MT; ++t) {
#pragma unroll
            for (int s = 0; s < kKs; ++s) {
                const int d = FMT == kE4M3 ? 64 * (s / 4) + 16 * c + 4 * (s % 4) : kGroup * (s / 2) + 8 * c + 4 * (s % 2);
                const uint2 lo = *reinterpret_cast<const uint2*>(s_q + (16 * t + g) * (HD + 8) + d);
                const uint2 hi = HALF ? make_uint2(0, 0)
                                      : *reinterpret_cast<const uint2*>(s_q + (16 * t + g + 8) * (HD + 8) + d);
                qa[t][s][0] = lo.x, qa[t][s][1] = hi.x, qa[t][s][2] = lo.y, qa[t][s][3] = hi.y;
            }
#pragma unroll
            for (int h = 0; h < kH; ++h) {
                const int r = 16 * t + g + 8 * h;
                f[t][h] = s_f[r];
                lim[t][h] = shared_rows ? len : min(first + (r0 + r) / A.group, len);
            }
        }
        const int64_t head = (int64_t)b0 * A.c.kv_heads + kvh;
        const uint8_t* kc = static_cast<const uint8_t*>(A.c.k) + head * A.c.max_len * row_bytes<FMT>(HD);
        const uint8_t* vc = static_cast<const uint8_t*>(A.c.v) + head * A.c.max_len * row_bytes<FMT>(HD);
        const uint16_t* ks = A.c.k_scale + head * A.c.max_len * row_scales<FMT>(HD);
        const uint16_t* vs = A.c.v_scale + head * A.c.max_len * row_scales<FMT>(HD);
        constexpr int kGs = row_scales<FMT>(HD);

        Chunk<FMT, HD> nx;
        load_chunk<FMT, HD>(nx, kc, vc, ks, vs, t0 + warp * kStep, t1 - 1, g, c);
        for (int base = t0 + warp * kStep; base < t1; base += kStep * kWarps) {
            Chunk<FMT, HD> x = nx;
            if (base + kStep * kWarps < t1)
                load_chunk<FMT, HD>(nx, kc, vc, ks, vs, base + kStep * kWarps, t1 - 1, g, c);
            const bool mask = base + kStep > min(first, t1);
            // scores: s[tile of 8 positions][half][column]
            float s[MT][2][kH][2];
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                float d[MT][kGs][4];
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int i = 0; i < kGs; ++i) d[mt][i][0] = d[mt][i][1] = d[mt][i][2] = d[mt][i][3] = 0.f;
#pragma unroll
                for (int sl = 0; sl < kKs; ++sl) {
                    uint32_t kb0, kb1;
                    if (FMT == kE4M3) {
                        kb0 = e4m3x2_to_half2(x.k[t][sl] & 0xFFFFu);
                        kb1 = e4m3x2_to_half2(x.k[t][sl] >> 16);
                    } else {
                        kb0 = e2m1x2_to_half2(x.k[t][sl / 2] >> (16 * (sl % 2)));
                        kb1 = e2m1x2_to_half2(x.k[t][sl / 2] >> (16 * (sl % 2) + 8));
                    }
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt) mma16816(d[mt][FMT == kE4M3 ? 0 : sl / 2], qa[mt][sl], kb0, kb1);
                }
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int h = 0; h < kH; ++h)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            float a = 0.f;
#pragma unroll
                            for (int i = 0; i < kGs; ++i) {
                                const float sc = scale_of<FMT>(x.ks[2 * t + e], i);
                                a = i ? fmaf(d[mt][i][2 * h + e], sc, a) : d[mt][i][2 * h + e] * sc;
                            }
                            a *= f[mt][h];
                            if (mask && base + 4 * c + 2 * t + e >= min(lim[mt][h], t1)) a = -INFINITY;
                            s[mt][t][h][e] = a;
                        }
            }
            // value scales and their logarithms
            float vsc[4][kGs], lv[4];
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                float top = 0.f;
#pragma unroll
                for (int i = 0; i < kGs; ++i) {
                    vsc[t][i] = scale_of<FMT>(x.vs[t], i);
                    top = fmaxf(top, vsc[t][i]);
                }
                lv[t] = lg2(top);
            }
            uint32_t pa[MT][kGs][4];
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
                float raise[kH];
                bool any = false;
#pragma unroll
                for (int h = 0; h < kH; ++h) {
                    float top = -INFINITY;
#pragma unroll
                    for (int t = 0; t < 4; ++t) top = fmaxf(top, s[mt][t / 2][h][t % 2] + lv[t]);
                    top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
                    top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
                    raise[h] = 1.f;
                    if (top > M[mt][h] + kLazy) {
                        raise[h] = ex2(M[mt][h] - top);
                        M[mt][h] = top;
                        any = true;
                    }
                }
                if (__any_sync(0xFFFFFFFFu, any)) {
#pragma unroll
                    for (int n = 0; n < kNt; ++n) {
                        o[mt][n][0] *= raise[0], o[mt][n][1] *= raise[0];
                        if (!HALF) o[mt][n][2] *= raise[kH - 1], o[mt][n][3] *= raise[kH - 1];
                    }
                }
#pragma unroll
                for (int h = 0; h < kH; ++h) {
                    float top = m[mt][h];
#pragma unroll
                    for (int t = 0; t < 4; ++t) top = fmaxf(top, s[mt][t / 2][h][t % 2]);
                    const float ref = top == -INFINITY ? 0.f : top;
                    l[mt][h] *= ex2(m[mt][h] - ref);
                    m[mt][h] = top;
                    const float up = top == -INFINITY || M[mt][h] == -INFINITY ? 0.f : ex2(ref - M[mt][h]);
                    float w[4];
#pragma unroll
                    for (int t = 0; t < 4; ++t) {
                        const float p = ex2(s[mt][t / 2][h][t % 2] - ref);
                        l[mt][h] += p;
                        w[t] = p * up;
                    }
#pragma unroll
                    for (int i = 0; i < kGs; ++i) {
                        float y[4];
#pragma unroll
                        for (int t = 0; t < 4; ++t) {
                            y[t] = w[t] * vsc[t][i];
                            // a hidden position's scale may be NaN
                            if (mask && s[mt][t / 2][h][t % 2] == -INFINITY) y[t] = 0.f;
                        }
                        pa[mt][i][h] = pack_half(y[0], y[1]);
                        pa[mt][i][2 + h] = pack_half(y[2], y[3]);
                    }
                }
                if (HALF)
#pragma unroll
                    for (int i = 0; i < kGs; ++i) pa[mt][i][1] = pa[mt][i][3] = 0;
            }
            // O += P V: pairs of positions of one element, eight elements a tile
            if (FMT == kE4M3) {
#pragma unroll
                for (int w = 0; w < HD / 32; ++w) {
                    const uint32_t a0 = __byte_perm(x.v[0][w], x.v[1][w], 0x5140), a1 = __byte_perm(x.v[0][w], x.v[1][w], 0x7362);
                    const uint32_t b0v = __byte_perm(x.v[2][w], x.v[3][w], 0x5140), b1v = __byte_perm(x.v[2][w], x.v[3][w], 0x7362);
                    const uint32_t lo[4] = {e4m3x2_to_half2(a0 & 0xFFFFu), e4m3x2_to_half2(a0 >> 16),
                                            e4m3x2_to_half2(a1 & 0xFFFFu), e4m3x2_to_half2(a1 >> 16)};
                    const uint32_t hi[4] = {e4m3x2_to_half2(b0v & 0xFFFFu), e4m3x2_to_half2(b0v >> 16),
                                            e4m3x2_to_half2(b1v & 0xFFFFu), e4m3x2_to_half2(b1v >> 16)};
#pragma unroll
                    for (int e = 0; e < 4; ++e)
#pragma unroll
                        for (int mt = 0; mt < MT; ++mt) mma16816(o[mt][4 * w + e], pa[mt][0], lo[e], hi[e]);
                }
            } else {
#pragma unroll
                for (int w = 0; w < HD / kGroup; ++w) {
                    // nibbles of four elements: position pairs side by side in a byte
                    const uint32_t ae = (x.v[0][w] & 0x0F0Fu) | ((x.v[1][w] & 0x0F0Fu) << 4);
                    const uint32_t ao = ((x.v[0][w] >> 4) & 0x0F0Fu) | (x.v[1][w] & 0xF0F0u);
                    const uint32_t be = (x.v[2][w] & 0x0F0Fu) | ((x.v[3][w] & 0x0F0Fu) << 4);
                    const uint32_t bo = ((x.v[2][w] >> 4) & 0x0F0Fu) | (x.v[3][w] & 0xF0F0u);
                    const uint32_t lo[4] = {e2m1x2_to_half2(ae), e2m1x2_to_half2(ao), e2m1x2_to_half2(ae >> 8),
                                            e2m1x2_to_half2(ao >> 8)};
                    const uint32_t hi[4] = {e2m1x2_to_half2(be), e2m1x2_to_half2(bo), e2m1x2_to_half2(be >> 8),
                                            e2m1x2_to_half2(bo >> 8)};
#pragma unroll
                    for (int e = 0; e < 4; ++e)
#pragma unroll
                        for (int mt = 0; mt < MT; ++mt) mma16816(o[mt][4 * w + e], pa[mt][w], lo[e], hi[e]);
                }
            }
        }
        // a row's denominator over its four lanes
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int h = 0; h < kH; ++h) {
                float top = m[mt][h];
                top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
                const float ref = top == -INFINITY ? 0.f : top;
                float t = l[mt][h] * ex2(m[mt][h] - ref);
                t += __shfl_xor_sync(0xFFFFFFFFu, t, 1);
                t += __shfl_xor_sync(0xFFFFFFFFu, t, 2);
                m[mt][h] = top;
                l[mt][h] = t;
            }
    }
    // join the warps
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int h = 0; h < kH; ++h) {
            const int r = 16 * mt + g + 8 * h;
            if (c == 0) {
                float* w = s_meta + (warp * kRows + r) * 3;
                w[0] = m[mt][h], w[1] = l[mt][h], w[2] = M[mt][h];
            }
            float* w = s_o + (warp * kRows + r) * kOs;
#pragma unroll
            for (int n = 0; n < kNt; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) w[value_dim<FMT, HD>(2 * c + e, n)] = o[mt][n][2 * h + e];
        }
    __syncthreads();
    const int rows = min(HALF ? 8 : kRows, n_rows - r0);
    for (int r = warp; r < rows; r += kWarps) {
        float mw[kWarps], lw[kWarps], Mw[kWarps], top = -INFINITY, Top = -INFINITY, sum = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float* x = s_meta + (w * kRows + r) * 3;
            mw[w] = x[0], lw[w] = x[1], Mw[w] = x[2];
            top = fmaxf(top, mw[w]);
            Top = fmaxf(Top, Mw[w]);
        }
        const float ref = top == -INFINITY ? 0.f : top, Ref = Top == -INFINITY ? 0.f : Top;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            sum += lw[w] * ex2(mw[w] - ref);
            Mw[w] = ex2(Mw[w] - Ref);
        }
        int b, i, head;
        const int64_t row = row_id(r, &b, &i, &head);
        if (A.out) {
            const int p = A.pos[b];
            const bool over = (int64_t)p + i >= A.max_len;
            const float k = p < 0 ? 0.f : over ? __int_as_float(0x7FC00000) : ex2(Ref - ref) / sum;
#pragma unroll
            for (int j = 0; j < HD / 32; ++j) {
                const int d = lane + 32 * j;
                float v = 0.f;
#pragma unroll
                for (int w = 0; w < kWarps; ++w) v = fmaf(Mw[w], s_o[(w * kRows + r) * kOs + d], v);
                A.out[row * HD + d] = __bfloat16_as_ushort(__float2bfloat16_rn(p < 0 ? 0.f : v * k));
            }
        } else {
            const int64_t at = row * A.parts + A.part0 + split;
            if (lane == 0) reinterpret_cast<float4*>(A.meta)[at] = make_float4(top, sum, Top, 0.f);
            if (top == -INFINITY && sum == 0.f) continue;  // nothing seen: the accumulators are not read
#pragma unroll
            for (int j = 0; j < HD / 32; ++j) {
                const int d = lane + 32 * j;
                float v = 0.f;
#pragma unroll
                for (int w = 0; w < kWarps; ++w) v = fmaf(Mw[w], s_o[(w * kRows + r) * kOs + d], v);
                A.acc[at * HD + d] = v;
            }
        }
    }
}

struct JoinArgs {
    const float* meta;
    const float* acc;
    const int32_t* pos;
    const int32_t* prefix_len;
    uint16_t* out;
    int32_t parts, n_q, n_heads, max_len, prefix_max;
};

// One CTA a row: its parts' weights, then the weighted accumulators, the
// parts spread over the warps and their sums added in warp order.
template <int HD>
__global__ void __launch_bounds__(kThreads) join_kernel(const JoinArgs A) {
    __shared__ float s_w[kMaxParts];
    __shared__ float s_v[kWarps][HD];
    pdl_wait();
    pdl_release();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int64_t row = blockIdx.x;
    const int i = (int)(row / A.n_heads % A.n_q);
    const int b = (int)(row / A.n_heads / A.n_q);
    const float4* meta = reinterpret_cast<const float4*>(A.meta) + row * A.parts;
    // every warp reduces the parts' (m, l, M) itself
    float top = -INFINITY, Top = -INFINITY, sum = 0.f;
    for (int s = lane; s < A.parts; s += 32) {
        const float4 x = meta[s];
        top = fmaxf(top, x.x), Top = fmaxf(Top, x.z);
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
        Top = fmaxf(Top, __shfl_xor_sync(0xFFFFFFFFu, Top, o));
    }
    const float ref = top == -INFINITY ? 0.f : top, Ref = Top == -INFINITY ? 0.f : Top;
    for (int s = lane; s < A.parts; s += 32) {
        const float4 x = meta[s];
        const bool seen = !(x.x == -INFINITY && x.y == 0.f);
        sum += x.y * ex2(x.x - ref);
        if (warp == 0) s_w[s] = seen ? ex2(x.z - Ref) : -1.f;
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
    __syncthreads();
    float v[HD / 32];
#pragma unroll
    for (int j = 0; j < HD / 32; ++j) v[j] = 0.f;
    for (int s = warp; s < A.parts; s += kWarps) {
        const float w = s_w[s];
        if (w < 0.f) continue;
        const float* x = A.acc + (row * A.parts + s) * HD;
#pragma unroll
        for (int j = 0; j < HD / 32; ++j) v[j] = fmaf(w, x[lane + 32 * j], v[j]);
    }
#pragma unroll
    for (int j = 0; j < HD / 32; ++j) s_v[warp][lane + 32 * j] = v[j];
    __syncthreads();
    if (tid < HD) {
        float a = s_v[0][tid];
#pragma unroll
        for (int w = 1; w < kWarps; ++w) a += s_v[w][tid];
        const int p = A.pos[b];
        const bool bad = (int64_t)p + i >= A.max_len || (A.prefix_len && *A.prefix_len > A.prefix_max);
        a = p < 0 ? 0.f : bad ? __int_as_float(0x7FC00000) : a * (ex2(Ref - ref) / sum);
        A.out[row * HD + tid] = __bfloat16_as_ushort(__float2bfloat16_rn(a));
    }
}

template <int HD, int MT>
constexpr size_t smem_bytes() {
    return (size_t)kWarps * 16 * MT * (HD + 4) * 4 + kWarps * 16 * MT * 3 * 4 + 16 * MT * 4 + 16 * MT * (HD + 8) * 2;
}

template <int FMT, int HD, int MT, bool HALF>
cudaError_t launch(const AttnArgs& A, dim3 grid, cudaStream_t s) {
    constexpr size_t sm = smem_bytes<HD, MT>();
    if (sm > 48 * 1024) {
        const cudaError_t e =
            cudaFuncSetAttribute(attn_kernel<FMT, HD, MT, HALF>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sm);
        if (e != cudaSuccess) return e;
    }
    return launch_pdl(attn_kernel<FMT, HD, MT, HALF>, grid, dim3(kThreads), sm, s, A);
}

template <int FMT, int HD>
cudaError_t launch_rows(const AttnArgs& A, int rows, dim3 grid, cudaStream_t s) {
    if (rows <= 8) return launch<FMT, HD, 1, true>(A, grid, s);
    if (rows <= 16) return launch<FMT, HD, 1, false>(A, grid, s);
    return launch<FMT, HD, 2, false>(A, grid, s);
}

cudaError_t launch_attn(const AttnArgs& A, int rows, dim3 grid, cudaStream_t s) {
    if (A.c.format == kE4M3)
        return A.c.head_dim == 64 ? launch_rows<kE4M3, 64>(A, rows, grid, s) : launch_rows<kE4M3, 128>(A, rows, grid, s);
    return A.c.head_dim == 64 ? launch_rows<kE2M1, 64>(A, rows, grid, s) : launch_rows<kE2M1, 128>(A, rows, grid, s);
}

int tiles_of(int64_t rows) { return (int)(rows <= 16 ? 1 : (rows + 31) / 32); }

// Parts that the positions of a cache are split into: enough CTAs for three a
// multiprocessor, no part shorter than two CTA steps.
int splits_for(int64_t items, int max_len, int sms) {
    const int64_t want = (3LL * sms + items - 1) / items;
    const int64_t most = (max_len + 2 * kStep * kWarps - 1) / (2 * kStep * kWarps);
    return (int)std::max<int64_t>(1, std::min<int64_t>({want, most, kMaxParts / 2}));
}

struct Plan {
    int row_tiles, splits, p_tiles, p_splits;
    int64_t rows, bytes;
};

cdq_status plan(const cdq_kv_cache* c, int n_heads, int n_q, const cdq_kv_cache* prefix, Plan* P) {
    cdq_status st = check_cache(c);
    if (st) return st;
    if (n_q < 1 || n_q > CDQ_KV_MAX_NEW || n_heads < c->kv_heads || n_heads % c->kv_heads || n_heads > 65535)
        return CDQ_ERR_ARG;
    int dev = 0, sms = 0;
    if (cudaGetDevice(&dev) != cudaSuccess ||
        cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
        return CDQ_ERR_CUDA;
    const int64_t per_seq = (int64_t)n_q * (n_heads / c->kv_heads);
    P->rows = (int64_t)c->batch * n_q * n_heads;
    P->row_tiles = tiles_of(per_seq);
    P->splits = splits_for((int64_t)P->row_tiles * c->kv_heads * c->batch, c->max_len, sms);
    P->p_tiles = P->p_splits = 0;
    if (prefix) {
        if ((st = check_cache(prefix))) return st;
        if (prefix->batch != 1 || prefix->kv_heads != c->kv_heads || prefix->head_dim != c->head_dim ||
            prefix->format != c->format)
            return CDQ_ERR_SHAPE;
        P->p_tiles = tiles_of(per_seq * c->batch);
        P->p_splits = splits_for((int64_t)P->p_tiles * c->kv_heads, prefix->max_len, sms);
    }
    const int64_t parts = P->splits + P->p_splits;
    if (P->rows > 0x7FFFFFFF || (int64_t)P->row_tiles * P->splits > 0x7FFFFFFF) return CDQ_ERR_SHAPE;
    P->bytes = parts == 1 ? 0 : P->rows * parts * (kMetaF + c->head_dim) * 4;
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
                         int32_t n_q, const int32_t* pos, const cdq_kv_rope* rope, float scale,
                         const cdq_kv_cache* prefix, const int32_t* prefix_len, uint16_t* out, void* workspace,
                         int64_t workspace_bytes, void* stream) {
    Plan P;
    cdq_status st = plan(cache, n_heads, n_q, prefix, &P);
    if (st) return st;
    AttnArgs A{};
    if ((st = check_rope(rope, &A.rope))) return st;
    if (!strided(q, q_seq, q_tok) || !pos || !out || (prefix && !prefix_len)) return CDQ_ERR_ARG;
    if (P.bytes && (!workspace || (uintptr_t)workspace % 16 || workspace_bytes < P.bytes)) return CDQ_ERR_WORKSPACE;
    auto s = (cudaStream_t)stream;
    A.q = q, A.q_seq = q_seq, A.q_tok = q_tok, A.pos = pos;
    A.scale_log2 = scale * 1.4426950408889634f;
    A.batch = cache->batch, A.n_q = n_q, A.n_heads = n_heads, A.group = n_heads / cache->kv_heads;
    A.max_len = cache->max_len;
    A.parts = P.splits + P.p_splits;
    const bool single = A.parts == 1;
    A.meta = single ? nullptr : static_cast<float*>(workspace);
    A.acc = single ? nullptr : A.meta + P.rows * A.parts * kMetaF;
    A.out = single ? out : nullptr;
    A.c = *cache;
    A.row_tiles = P.row_tiles, A.splits = P.splits, A.part0 = 0;
    const int64_t per_seq = (int64_t)n_q * A.group;
    if (launch_attn(A, (int)per_seq, dim3(P.row_tiles * P.splits, cache->kv_heads, cache->batch), s) != cudaSuccess)
        return CDQ_ERR_CUDA;
    if (prefix) {
        A.c = *prefix;
        A.prefix_len = prefix_len;
        A.row_tiles = P.p_tiles, A.splits = P.p_splits, A.part0 = P.splits;
        if (launch_attn(A, (int)std::min<int64_t>(per_seq * cache->batch, 1 << 20),
                        dim3(P.p_tiles * P.p_splits, cache->kv_heads, 1), s) != cudaSuccess)
            return CDQ_ERR_CUDA;
    }
    if (!single) {
        JoinArgs J{A.meta, A.acc, pos, prefix ? prefix_len : nullptr, out, A.parts, n_q, n_heads, cache->max_len,
                   prefix ? prefix->max_len : 0};
        const cudaError_t e = cache->head_dim == 64
                                  ? launch_pdl(join_kernel<64>, dim3((unsigned)P.rows), dim3(kThreads), 0, s, J)
                                  : launch_pdl(join_kernel<128>, dim3((unsigned)P.rows), dim3(kThreads), 0, s, J);
        if (e != cudaSuccess) return CDQ_ERR_CUDA;
    }
    return CDQ_OK;
}

}  // extern "C"
