// prefix_paths.cuh -- the arithmetic of one warp over the rows of one key
// head, for bf16, INT8 and fp32 caches (prefix_decode.cu runs them).
//
// A path holds up to ROWS query rows and their running (m, l, o), and takes
// KEYS cache rows a step: issue() starts a step's copies of K and V into a
// stage of shared memory, compute() folds them in, finish() writes the state.
// Row i of a block is query head hk * ratio + (row0 + i) % ratio of request
// first_req + (row0 + i) / ratio.
//
// A lane copies exactly the bytes that it will use, into words that only it
// reads (chunk i of lane n at 32 i + n, so neither side has bank conflicts):
// a stage is an extension of the lane's registers, and waiting for the lane's
// own copies is all the synchronisation there is.
#pragma once
#include <cuda_fp16.h>

#include "prefix.cuh"
#include "sm100.cuh"

namespace attn {
namespace prefix {

using sm100::ex2;
using sm100::f2;
using sm100::f2_split;
using sm100::fma2;
using sm100::pack_bf16;

__device__ __forceinline__ void mma_bf16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel) { return __byte_perm(a, b, sel); }

__device__ __forceinline__ float quad_max(float v) {
    v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
    return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
}
__device__ __forceinline__ float quad_sum(float v) {
    v += __shfl_xor_sync(0xffffffffu, v, 1);
    return v + __shfl_xor_sync(0xffffffffu, v, 2);
}
// a and b as bf16, and what that leaves of them
__device__ __forceinline__ void bf16_parts(float a, float b, uint32_t &hi, uint32_t &lo) {
    hi = pack_bf16(a, b);
    lo = pack_bf16(a - __uint_as_float(hi << 16), b - __uint_as_float(hi & 0xffff0000u));
}

// Copies to a stage and reads from it.  The data are read once (16 bytes past
// L1) or by lanes that share sectors (smaller pieces, through L1).
__device__ __forceinline__ void copy16(uint32_t dst, const void *src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
template <int N>
__device__ __forceinline__ void copy_small(uint32_t dst, const void *src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(N) : "memory");
}
__device__ __forceinline__ uint4 lds16(uint32_t a) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ uint2 lds8(uint32_t a) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ uint32_t lds4(uint32_t a) {
    uint32_t v;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
    return v;
}

// Address of query row `row` of a block (clamped to the block's rows).
template <typename T>
__device__ __forceinline__ const T *query(const Params &p, int first_req, int row, int hk, int d) {
    const int s = first_req + row / p.ratio, h = hk * p.ratio + row % p.ratio;
    return static_cast<const T *>(p.q) + s * p.q_stride + (long long)h * d;
}

// ---------------------------------------------------------------------------
// bf16: both products on mma.sync m16n8k16, 8 or 16 query rows.
//
// A dot product may take its k positions in any order, and an output its n
// positions, so each lane's share of a cache row is 16 contiguous bytes and
// serves as it was loaded:
//   scores: lane (g, c) = (lane / 4, lane % 4) holds dims (4 j + c) 8 .. + 7 of
//     key g, whose four words are the B fragments of k-steps 2j and 2j + 1;
//   values: lane (g, c) holds dims 8 g .. 8 g + 7 (of each 64) of keys 2c,
//     2c + 1, 2c + 8, 2c + 9; one byte permutation pairs two keys' values of a
//     dim into a B fragment, and dim 8 g + i is column g of n-tile i.
// Probabilities are rounded to bf16 for the second product (their sum is not);
// with 8 rows, the rounding's rest goes through the 8 MMA rows that are free.
// ---------------------------------------------------------------------------
template <int D, bool HI>                 // HI: rows 8 .. 15 are used
struct Bf16Path {
    static constexpr int ROWS = HI ? 16 : 8, KEYS = D <= 64 ? 32 : 16;
    static constexpr int KT = KEYS / 8, KH = KEYS / 16, KC = D / 32, B64 = D / 64, REM = D % 64 != 0;
    static constexpr int NT = D / 8, NR = HI ? 2 : 1;         // n-tiles of the output; rows of a lane
    static constexpr int OFF_V = KT * KC * 512, OFF_W = OFF_V + KH * 4 * B64 * 512, STAGE = OFF_W + REM * KH * 4 * 256;
    uint32_t q[2 * KC][2 * NR];
    float o[NT][4], m[NR], l[NR];
    const char *kb, *vb;

    __device__ __forceinline__ void begin(const Params &p, int first_req, int row0, int rows, int hk) {
        const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
#pragma unroll
        for (int r = 0; r < NR; r++) {
            const __nv_bfloat16 *a = query<__nv_bfloat16>(p, first_req, row0 + min(g + 8 * r, rows - 1), hk, D);
#pragma unroll
            for (int j = 0; j < KC; j++) {
                const uint4 x = __ldg(reinterpret_cast<const uint4 *>(a) + 4 * j + c);
                q[2 * j][r] = x.x; q[2 * j][NR + r] = x.y;
                q[2 * j + 1][r] = x.z; q[2 * j + 1][NR + r] = x.w;
            }
            m[r] = -INFINITY;
            l[r] = 0.f;
        }
#pragma unroll
        for (int i = 0; i < NT; i++)
#pragma unroll
            for (int e = 0; e < 4; e++) o[i][e] = 0.f;
        kb = static_cast<const char *>(p.k) + (long long)hk * D * 2 + c * 16;
        vb = static_cast<const char *>(p.v) + (long long)hk * D * 2;
    }
    __device__ __forceinline__ void issue(const Params &p, uint32_t st, int row) const {
        const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
        const long long stride = p.row_stride * 2;
#pragma unroll
        for (int t = 0; t < KT; t++) {
            const char *at = kb + __shfl_sync(0xffffffffu, row, t * 8 + g) * stride;
#pragma unroll
            for (int j = 0; j < KC; j++) copy16(st + (t * KC + j) * 512 + lane * 16, at + 64 * j);
        }
#pragma unroll
        for (int n = 0; n < 4 * KH; n++) {
            const char *at = vb + __shfl_sync(0xffffffffu, row, (n >> 1) * 8 + 2 * c + (n & 1)) * stride;
#pragma unroll
            for (int x = 0; x < B64; x++) copy16(st + OFF_V + (n * B64 + x) * 512 + lane * 16, at + 128 * x + 16 * g);
            if constexpr (REM) copy_small<8>(st + OFF_W + n * 256 + lane * 8, at + 128 * B64 + 8 * g);
        }
    }
    template <bool EDGE>                  // EDGE: some keys of the step have no row
    __device__ __forceinline__ void compute(const Params &p, uint32_t st, unsigned mask) {
        const int lane = threadIdx.x & 31, c = lane & 3;
        st += lane * 16;
        float s[KT][4];
#pragma unroll
        for (int t = 0; t < KT; t++) {
            s[t][0] = s[t][1] = s[t][2] = s[t][3] = 0.f;
#pragma unroll
            for (int j = 0; j < KC; j++) {
                const uint4 k = lds16(st + (t * KC + j) * 512);
                mma(s[t], q[2 * j], k.x, k.y);
                mma(s[t], q[2 * j + 1], k.z, k.w);
            }
        }
        if (EDGE) {
#pragma unroll
            for (int t = 0; t < KT; t++)
#pragma unroll
                for (int e = 0; e < 4; e++)
                    if (!(mask >> (t * 8 + 2 * c + (e & 1)) & 1)) s[t][e] = -INFINITY;
        }
        float neg[NR];
#pragma unroll
        for (int r = 0; r < NR; r++) {
            float mx = s[0][2 * r];
#pragma unroll
            for (int t = 0; t < KT; t++) mx = fmaxf(mx, fmaxf(s[t][2 * r], s[t][2 * r + 1]));
            mx = fmaxf(m[r], quad_max(mx) * p.scale_log2);
            neg[r] = mx == -INFINITY ? 0.f : -mx;
            if (__any_sync(0xffffffffu, mx != m[r])) {
                const float a = ex2(m[r] + neg[r]);
                l[r] *= a;
#pragma unroll
                for (int i = 0; i < NT; i++)
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        if (!HI || e >> 1 == r) o[i][e] *= a;
            }
            m[r] = mx;
        }
#pragma unroll
        for (int t = 0; t < KT; t++)
#pragma unroll
            for (int e = 0; e < 2 * NR; e++) {
                s[t][e] = ex2(fmaf(s[t][e], p.scale_log2, neg[e >> 1]));
                l[e >> 1] += s[t][e];
            }
#pragma unroll
        for (int h = 0; h < KH; h++) {
            uint32_t a[4];
            if constexpr (HI) {
                a[0] = pack_bf16(s[2 * h][0], s[2 * h][1]);
                a[1] = pack_bf16(s[2 * h][2], s[2 * h][3]);
                a[2] = pack_bf16(s[2 * h + 1][0], s[2 * h + 1][1]);
                a[3] = pack_bf16(s[2 * h + 1][2], s[2 * h + 1][3]);
            } else {
                bf16_parts(s[2 * h][0], s[2 * h][1], a[0], a[1]);
                bf16_parts(s[2 * h + 1][0], s[2 * h + 1][1], a[2], a[3]);
            }
            // a key with no row has probability 0, and values that may be NaN
            auto there = [&](int i) { return !EDGE || (mask >> (h * 16 + (i >> 1) * 8 + 2 * c + (i & 1)) & 1); };
#pragma unroll
            for (int x = 0; x < B64; x++) {
                uint32_t v[4][4];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    uint4 y = lds16(st + OFF_V + ((h * 4 + i) * B64 + x) * 512);
                    if (!there(i)) y = make_uint4(0, 0, 0, 0);
                    v[i][0] = y.x; v[i][1] = y.y; v[i][2] = y.z; v[i][3] = y.w;
                }
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const uint32_t sel = i & 1 ? 0x7632 : 0x5410;
                    mma_bf16(o[8 * x + i], a, prmt(v[0][i / 2], v[1][i / 2], sel), prmt(v[2][i / 2], v[3][i / 2], sel));
                }
            }
            if constexpr (REM) {
                uint32_t v[4][2];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    uint2 y = lds8(st - lane * 8 + OFF_W + (h * 4 + i) * 256);
                    if (!there(i)) y = make_uint2(0, 0);
                    v[i][0] = y.x; v[i][1] = y.y;
                }
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const uint32_t sel = i & 1 ? 0x7632 : 0x5410;
                    mma_bf16(o[8 * B64 + i], a, prmt(v[0][i / 2], v[1][i / 2], sel), prmt(v[2][i / 2], v[3][i / 2], sel));
                }
            }
        }
    }
    __device__ __forceinline__ static void mma(float (&d)[4], const uint32_t (&a)[2 * NR], uint32_t b0, uint32_t b1) {
        const uint32_t x[4] = {a[0], HI ? a[NR - 1] : 0u, a[NR], HI ? a[2 * NR - 1] : 0u};
        mma_bf16(d, x, b0, b1);
    }
    __device__ __forceinline__ void finish(float *out, float2 *ml, int rows) {
        const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
        if constexpr (!HI) {
#pragma unroll
            for (int i = 0; i < NT; i++) { o[i][0] += o[i][2]; o[i][1] += o[i][3]; }
        }
#pragma unroll
        for (int r = 0; r < NR; r++) {
            const float sum = quad_sum(l[r]);
            const int row = g + 8 * r;
            if (row >= rows) continue;
            if (c == 0) ml[row] = make_float2(m[r], sum);
#pragma unroll
            for (int n = 0; n < 2; n++) {        // columns 2c, 2c + 1 of every n-tile
                float *at = out + row * D;
#pragma unroll
                for (int x = 0; x < B64; x++) {
#pragma unroll
                    for (int i = 0; i < 8; i += 4)
                        *reinterpret_cast<float4 *>(at + 64 * x + 8 * (2 * c + n) + i) =
                            make_float4(o[8 * x + i][2 * r + n], o[8 * x + i + 1][2 * r + n], o[8 * x + i + 2][2 * r + n],
                                        o[8 * x + i + 3][2 * r + n]);
                }
                if constexpr (REM)
                    *reinterpret_cast<float4 *>(at + 64 * B64 + 4 * (2 * c + n)) =
                        make_float4(o[8 * B64][2 * r + n], o[8 * B64 + 1][2 * r + n], o[8 * B64 + 2][2 * r + n],
                                    o[8 * B64 + 3][2 * r + n]);
            }
        }
    }
};

// ---------------------------------------------------------------------------
// INT8 codes: the same products in f16, in which a code is exact; 8 query rows.
//
// A query and a weight go in as two f16 parts, high in MMA row g and the rest
// in row g + 8, whose sums are added: 22 bits of each.  The query row is
// first scaled by a power of two that puts its largest element in [2^7, 2^8),
// the weights p * vscale by one, kept for the piece, that keeps them under 2,
// so the second parts stay above f16's smallest numbers.  A code c becomes f16
// as the low byte of 1024 + (c + 128) minus 1152, all exact.  The tensor core
// rounds its sums towards zero, which drifts over a long piece, so every
// FOLD steps the output sums move to fp32 registers.
// ---------------------------------------------------------------------------
__device__ __forceinline__ uint32_t codes_f16(uint32_t biased, uint32_t sel) {   // two bytes of code + 128
    const uint32_t x = prmt(biased, 0x64646464u, sel);
    const __half2 r = __hsub2(*reinterpret_cast<const __half2 *>(&x), __floats2half2_rn(1152.f, 1152.f));
    return *reinterpret_cast<const uint32_t *>(&r);
}
// high and low f16 parts of two floats
__device__ __forceinline__ void f16_parts(float a, float b, uint32_t &hi, uint32_t &lo) {
    const __half2 h = __floats2half2_rn(a, b);
    const float2 f = __half22float2(h);
    const __half2 r = __floats2half2_rn(a - f.x, b - f.y);
    hi = *reinterpret_cast<const uint32_t *>(&h);
    lo = *reinterpret_cast<const uint32_t *>(&r);
}
// 2^e as a float, e in [-126, 127]
__device__ __forceinline__ float pow2i(int e) { return __int_as_float((e + 127) << 23); }
// exponent of x > 0, within [-100, 100]
__device__ __forceinline__ int exponent(float x) { return min(100, max(-100, (__float_as_int(x) >> 23 & 255) - 127)); }

template <int D>
struct I8Path {
    static constexpr int ROWS = 8, KEYS = 32, FOLD = 8;
    static constexpr int KT = KEYS / 8, KH = KEYS / 16, B64 = D / 64, REM = D % 64 != 0;
    static constexpr int KW = D / 16;                         // words of a K row per lane = k-steps
    static constexpr int NT = D / 8;
    static constexpr int OFF_KR = KT * B64 * 512, OFF_V = OFF_KR + REM * KT * 256, OFF_VR = OFF_V + KH * 4 * B64 * 256;
    static constexpr int OFF_S = OFF_VR + REM * KH * 4 * 128, STAGE = OFF_S + 256;
    uint32_t q[KW][4];
    float o[NT][4], f[NT][2], m, l;
    float qscale;                                             // scale log2(e) / the query's power of two
    float wscale;                                             // the weights' power of two
    int folded, hk_;
    const char *kb, *vb;

    __device__ __forceinline__ void begin(const Params &p, int first_req, int row0, int rows, int hk) {
        const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
        const float *a = query<float>(p, first_req, row0 + min(g, rows - 1), hk, D);
        float4 x[KW];
        float amax = 0.f;
#pragma unroll
        for (int j = 0; j < KW; j++) {
            // word j of this lane: 16 codes of each 64 dims, then 8 of the last 32
            const int dim = j < 4 * B64 ? 64 * (j / 4) + 16 * c + 4 * (j % 4) : 64 * B64 + 8 * c + 4 * (j - 4 * B64);
            x[j] = __ldg(reinterpret_cast<const float4 *>(a + dim));
            amax = fmaxf(amax, fmaxf(fmaxf(fabsf(x[j].x), fabsf(x[j].y)), fmaxf(fabsf(x[j].z), fabsf(x[j].w))));
        }
        amax = quad_max(amax);
        const int e = amax > 0.f ? 7 - exponent(amax) : 0;
        const float up = pow2i(e);
        qscale = p.scale_log2 * pow2i(-e);
#pragma unroll
        for (int j = 0; j < KW; j++) {
            f16_parts(x[j].x * up, x[j].y * up, q[j][0], q[j][1]);
            f16_parts(x[j].z * up, x[j].w * up, q[j][2], q[j][3]);
        }
#pragma unroll
        for (int i = 0; i < NT; i++) {
#pragma unroll
            for (int n = 0; n < 4; n++) o[i][n] = 0.f;
            f[i][0] = f[i][1] = 0.f;
        }
        m = -INFINITY;
        l = 0.f;
        wscale = 0.f;
        folded = 0;
        hk_ = hk;
        kb = static_cast<const char *>(p.k) + (long long)hk * D;
        vb = static_cast<const char *>(p.v) + (long long)hk * D;
    }
    __device__ __forceinline__ void issue(const Params &p, uint32_t st, int row) const {
        const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
        const long long at_scale = (long long)row * p.kv_heads + hk_;
        copy_small<4>(st + OFF_S + lane * 4, p.kscale + at_scale);
        copy_small<4>(st + OFF_S + 128 + lane * 4, p.vscale + at_scale);
#pragma unroll
        for (int t = 0; t < KT; t++) {
            const char *at = kb + __shfl_sync(0xffffffffu, row, t * 8 + g) * p.row_stride;
#pragma unroll
            for (int x = 0; x < B64; x++) copy16(st + (t * B64 + x) * 512 + lane * 16, at + 64 * x + 16 * c);
            if constexpr (REM) copy_small<8>(st + OFF_KR + t * 256 + lane * 8, at + 64 * B64 + 8 * c);
        }
#pragma unroll
        for (int n = 0; n < 4 * KH; n++) {
            const char *at = vb + __shfl_sync(0xffffffffu, row, (n >> 1) * 8 + 2 * c + (n & 1)) * p.row_stride;
#pragma unroll
            for (int x = 0; x < B64; x++) copy_small<8>(st + OFF_V + (n * B64 + x) * 256 + lane * 8, at + 64 * x + 8 * g);
            if constexpr (REM) copy_small<4>(st + OFF_VR + n * 128 + lane * 4, at + 64 * B64 + 4 * g);
        }
    }
    __device__ __forceinline__ void fold() {
#pragma unroll
        for (int i = 0; i < NT; i++)
#pragma unroll
            for (int n = 0; n < 2; n++) {
                f[i][n] += o[i][n] + o[i][n + 2];
                o[i][n] = o[i][n + 2] = 0.f;
            }
        folded = 0;
    }
    __device__ __forceinline__ void scale_output(float a) {
#pragma unroll
        for (int i = 0; i < NT; i++) {
#pragma unroll
            for (int n = 0; n < 4; n++) o[i][n] *= a;
            f[i][0] *= a;
            f[i][1] *= a;
        }
    }
    template <bool EDGE>
    __device__ __forceinline__ void compute(const Params &, uint32_t st, unsigned mask) {
        const int lane = threadIdx.x & 31, c = lane & 3;
        const float my_ks = __uint_as_float(lds4(st + OFF_S + lane * 4)), my_vs = __uint_as_float(lds4(st + OFF_S + 128 + lane * 4));
        float s[KT][4];
#pragma unroll
        for (int t = 0; t < KT; t++) {
            s[t][0] = s[t][1] = s[t][2] = s[t][3] = 0.f;
            uint32_t w[KW];
#pragma unroll
            for (int x = 0; x < B64; x++) {
                const uint4 k = lds16(st + (t * B64 + x) * 512 + lane * 16);
                w[4 * x] = k.x; w[4 * x + 1] = k.y; w[4 * x + 2] = k.z; w[4 * x + 3] = k.w;
            }
            if constexpr (REM) {
                const uint2 k = lds8(st + OFF_KR + t * 256 + lane * 8);
                w[4 * B64] = k.x; w[4 * B64 + 1] = k.y;
            }
#pragma unroll
            for (int j = 0; j < KW; j++) {
                w[j] ^= 0x80808080u;
                mma_f16(s[t], q[j], codes_f16(w[j], 0x4140), codes_f16(w[j], 0x4342));
            }
        }
        // weights' scale: the power of two over the largest vscale so far
        const bool valid = !EDGE || (mask >> lane & 1);
        const unsigned big = __reduce_max_sync(0xffffffffu, valid ? __float_as_uint(my_vs) & 0x7fffffffu : 0u);
        if (big && (wscale == 0.f || __uint_as_float(big) * wscale >= 2.f)) {
            const float now = pow2i(-exponent(__uint_as_float(big)));
            if (wscale != 0.f) scale_output(now / wscale);
            wscale = now;
        }
        float mx = -INFINITY;
#pragma unroll
        for (int t = 0; t < KT; t++)
#pragma unroll
            for (int n = 0; n < 2; n++) {
                const int key = t * 8 + 2 * c + n;
                const float ks = __shfl_sync(0xffffffffu, my_ks, key);
                s[t][n] = !EDGE || (mask >> key & 1) ? (s[t][n] + s[t][n + 2]) * qscale * ks : -INFINITY;
                mx = fmaxf(mx, s[t][n]);
            }
        mx = fmaxf(m, quad_max(mx));
        const float neg = mx == -INFINITY ? 0.f : -mx;
        if (__any_sync(0xffffffffu, mx != m)) {
            const float a = ex2(m + neg);
            l *= a;
            scale_output(a);
        }
        m = mx;
        uint32_t hi[KT], lo[KT];
#pragma unroll
        for (int t = 0; t < KT; t++) {
            float w[2];
#pragma unroll
            for (int n = 0; n < 2; n++) {
                const int key = t * 8 + 2 * c + n;
                const float e = ex2(s[t][n] + neg);
                const float vs = __shfl_sync(0xffffffffu, my_vs, key);
                l += e;
                w[n] = !EDGE || (mask >> key & 1) ? e * vs * wscale : 0.f;
            }
            f16_parts(w[0], w[1], hi[t], lo[t]);
        }
#pragma unroll
        for (int h = 0; h < KH; h++) {
            const uint32_t a[4] = {hi[2 * h], lo[2 * h], hi[2 * h + 1], lo[2 * h + 1]};
#pragma unroll
            for (int x = 0; x < 2 * B64 + REM; x++) {         // 4 dims of each of the lane's keys
                uint32_t v[4];
#pragma unroll
                for (int i = 0; i < 4; i++) v[i] = lds4(x < 2 * B64 ? st + OFF_V + ((h * 4 + i) * B64 + x / 2) * 256 + lane * 8 + x % 2 * 4
                                                                    : st + OFF_VR + (h * 4 + i) * 128 + lane * 4);
                const uint32_t a01 = prmt(v[0], v[1], 0x5140) ^ 0x80808080u, a23 = prmt(v[0], v[1], 0x7362) ^ 0x80808080u;
                const uint32_t b01 = prmt(v[2], v[3], 0x5140) ^ 0x80808080u, b23 = prmt(v[2], v[3], 0x7362) ^ 0x80808080u;
                mma_f16(o[4 * x], a, codes_f16(a01, 0x4140), codes_f16(b01, 0x4140));
                mma_f16(o[4 * x + 1], a, codes_f16(a01, 0x4342), codes_f16(b01, 0x4342));
                mma_f16(o[4 * x + 2], a, codes_f16(a23, 0x4140), codes_f16(b23, 0x4140));
                mma_f16(o[4 * x + 3], a, codes_f16(a23, 0x4342), codes_f16(b23, 0x4342));
            }
        }
        if (++folded == FOLD) fold();
    }
    __device__ __forceinline__ void finish(float *out, float2 *ml, int rows) {
        const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
        fold();
        const float sum = quad_sum(l);
        if (g >= rows) return;
        if (c == 0) ml[g] = make_float2(m, sum);
        const float down = wscale == 0.f ? 0.f : 1.f / wscale;
#pragma unroll
        for (int n = 0; n < 2; n++) {
            float *at = out + g * D;
#pragma unroll
            for (int x = 0; x < B64; x++)
#pragma unroll
                for (int i = 0; i < 8; i += 4)
                    *reinterpret_cast<float4 *>(at + 64 * x + 8 * (2 * c + n) + i) =
                        make_float4(f[8 * x + i][n] * down, f[8 * x + i + 1][n] * down, f[8 * x + i + 2][n] * down,
                                    f[8 * x + i + 3][n] * down);
            if constexpr (REM)
                *reinterpret_cast<float4 *>(at + 64 * B64 + 4 * (2 * c + n)) =
                    make_float4(f[8 * B64][n] * down, f[8 * B64 + 1][n] * down, f[8 * B64 + 2][n] * down,
                                f[8 * B64 + 3][n] * down);
        }
    }
};

// ---------------------------------------------------------------------------
// fp32: fp32 FMAs on pairs, R query rows.
//
// LPK lanes share a key, each with E = D / LPK of its dims, so a score is a
// dot product of E terms and log2(LPK) shuffles; each group of LPK lanes keeps
// its own running softmax over its keys (every 32/LPK-th) and the groups join
// once, in finish().  At most 4 R flops stand against a byte (R/2 of them), so
// up to 8 rows the FMA pipe keeps up with the memory.
// ---------------------------------------------------------------------------
template <int D, int R>
struct F32Path {
    static constexpr int ROWS = R;
    // q and o take 2 E R registers: 64 at most, 96 for 12 dims of 4 rows
    static constexpr int LPK = R == 8 ? (D == 32 ? 8 : 16) : D <= 64 && R < 4 || D == 32 ? 4 : 8;
    static constexpr int E = D / LPK, W = E % 4 ? 2 : 4, N = E / W;   // floats per lane, per copy, copies
    static constexpr int G = 32 / LPK;                        // keys at a time
    static constexpr int U = D == 32 ? 4 : 2;                    // keys of a group per step
    static constexpr int KEYS = G * U, CHUNK = 32 * W * 4;
    static constexpr int OFF_V = U * N * CHUNK, STAGE = 2 * OFF_V;
    static_assert(KEYS <= 32 && LPK * E == D && N * W == E, "lane geometry");
    uint64_t q[R][E / 2], o[R][E / 2];
    float m[R], l[R];
    const float *kb, *vb;

    __device__ __forceinline__ static void read(uint64_t (&x)[E / 2], uint32_t at) {
#pragma unroll
        for (int i = 0; i < N; i++) {
            if constexpr (W == 4)
                asm volatile("ld.shared.v2.u64 {%0,%1}, [%2];" : "=l"(x[2 * i]), "=l"(x[2 * i + 1]) : "r"(at + i * CHUNK) : "memory");
            else
                asm volatile("ld.shared.u64 %0, [%1];" : "=l"(x[i]) : "r"(at + i * CHUNK) : "memory");
        }
    }
    __device__ __forceinline__ void begin(const Params &p, int first_req, int row0, int rows, int hk) {
        const int sub = (threadIdx.x & 31) % LPK;
        const uint64_t s2 = f2(p.scale_log2, p.scale_log2);
#pragma unroll
        for (int r = 0; r < R; r++) {
            const float *a = query<float>(p, first_req, row0 + min(r, rows - 1), hk, D) + sub * W;
#pragma unroll
            for (int i = 0; i < E / 2; i++) {
                const float2 x = __ldg(reinterpret_cast<const float2 *>(a + i / (W / 2) * (LPK * W) + i % (W / 2) * 2));
                q[r][i] = fma2(f2(x.x, x.y), s2, 0ull);
                o[r][i] = 0ull;
            }
            m[r] = -INFINITY;
            l[r] = 0.f;
        }
        kb = static_cast<const float *>(p.k) + (long long)hk * D + sub * W;
        vb = static_cast<const float *>(p.v) + (long long)hk * D + sub * W;
    }
    __device__ __forceinline__ void issue(const Params &p, uint32_t st, int row) const {
        const int lane = threadIdx.x & 31, g = lane / LPK;
        st += lane * W * 4;
#pragma unroll
        for (int u = 0; u < U; u++) {
            const long long at = __shfl_sync(0xffffffffu, row, u * G + g) * p.row_stride;
#pragma unroll
            for (int i = 0; i < N; i++) {
                const uint32_t to = st + (u * N + i) * CHUNK;
                if constexpr (W == 4) {
                    copy16(to, kb + at + i * LPK * W);
                    copy16(to + OFF_V, vb + at + i * LPK * W);
                } else {
                    copy_small<8>(to, kb + at + i * LPK * W);
                    copy_small<8>(to + OFF_V, vb + at + i * LPK * W);
                }
            }
        }
    }
    template <bool EDGE>
    __device__ __forceinline__ void compute(const Params &, uint32_t st, unsigned mask) {
        const int lane = threadIdx.x & 31, g = lane / LPK;
        st += lane * W * 4;
        float x[R][U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            uint64_t k[E / 2];
            read(k, st + u * N * CHUNK);
#pragma unroll
            for (int r = 0; r < R; r++) {
                uint64_t a = 0ull;
#pragma unroll
                for (int i = 0; i < E / 2; i++) a = fma2(q[r][i], k[i], a);
                float lo, hi;
                f2_split(a, lo, hi);
                x[r][u] = lo + hi;
            }
        }
#pragma unroll
        for (int d = LPK / 2; d > 0; d >>= 1)
#pragma unroll
            for (int r = 0; r < R; r++)
#pragma unroll
                for (int u = 0; u < U; u++) x[r][u] += __shfl_xor_sync(0xffffffffu, x[r][u], d);
#pragma unroll
        for (int r = 0; r < R; r++) {
            float mx = m[r];
#pragma unroll
            for (int u = 0; u < U; u++) {
                if (EDGE && !(mask >> (u * G + g) & 1)) x[r][u] = -INFINITY;
                mx = fmaxf(mx, x[r][u]);
            }
            const float neg = mx == -INFINITY ? 0.f : -mx;
            if (mx != m[r]) {
                const float a = ex2(m[r] + neg);
                l[r] *= a;
#pragma unroll
                for (int i = 0; i < E / 2; i++) o[r][i] = fma2(o[r][i], f2(a, a), 0ull);
                m[r] = mx;
            }
#pragma unroll
            for (int u = 0; u < U; u++) {
                x[r][u] = ex2(x[r][u] + neg);
                l[r] += x[r][u];
            }
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            uint64_t v[E / 2];
            read(v, st + OFF_V + u * N * CHUNK);
            if (EDGE && !(mask >> (u * G + g) & 1)) {       // probability 0, and values that may be NaN
#pragma unroll
                for (int i = 0; i < E / 2; i++) v[i] = 0ull;
            }
#pragma unroll
            for (int r = 0; r < R; r++)
#pragma unroll
                for (int i = 0; i < E / 2; i++) o[r][i] = fma2(f2(x[r][u], x[r][u]), v[i], o[r][i]);
        }
    }
    __device__ __forceinline__ void finish(float *out, float2 *ml, int rows) {
        const int lane = threadIdx.x & 31, sub = lane % LPK;
#pragma unroll
        for (int r = 0; r < R; r++) {
            float mx = m[r];
#pragma unroll
            for (int d = LPK; d < 32; d <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
            const float a = mx == -INFINITY ? 0.f : ex2(m[r] - mx);
            float sum = l[r] * a;
#pragma unroll
            for (int d = LPK; d < 32; d <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
#pragma unroll
            for (int i = 0; i < E / 2; i++) {
                float lo, hi;
                f2_split(o[r][i], lo, hi);
                lo *= a;
                hi *= a;
#pragma unroll
                for (int d = LPK; d < 32; d <<= 1) {
                    lo += __shfl_xor_sync(0xffffffffu, lo, d);
                    hi += __shfl_xor_sync(0xffffffffu, hi, d);
                }
                const int dim = i / (W / 2) * (LPK * W) + sub * W + i % (W / 2) * 2;
                if (lane < LPK && r < rows) *reinterpret_cast<float2 *>(out + r * D + dim) = make_float2(lo, hi);
            }
            if (lane == 0 && r < rows) ml[r] = make_float2(mx, sum);
        }
    }
};

}  // namespace prefix
}  // namespace attn
