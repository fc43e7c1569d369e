// prefix_paths.cuh -- the arithmetic of one warp over the rows of one key
// head, for bf16, INT8 and fp32 caches (prefix_decode.cu runs them).
//
// A path holds up to ROWS query rows and their running (m, l, o), and takes
// KEYS cache rows a step, K and V each in a slot of shared memory: place() finds
// the head, begin() reads the queries, copy_k() and copy_v() start the copies,
// scores() and values() fold them in, finish() writes the state.  LEAN paths hold
// few enough registers for two CTAs per SM.
// Row i of a block is query head hk * ratio + (row0 + i) % ratio of request
// first_req + (row0 + i) / ratio.
//
// bf16 and INT8 form the scores as S^T = K Q^T and the outputs as O^T = V^T P^T
// with mma.sync m16n8k16: the cache side is the 16-row operand, so a tile of 8
// columns of queries costs one instruction where a 16-row tile of queries
// would be mostly empty, and K and V fragments serve NT such tiles.  A lane
// (g, c) = (lane / 4, lane % 4) gets S of keys g, g + 8 and columns 2c, 2c + 1;
// the columns' probabilities, packed, become the second product's operand by
// one 8 x 8 transposition (movmatrix), and the columns of O^T are the lane's
// own again, so a rescaling needs no exchange.
//
// The warp copies the rows as they lie in memory, 16 bytes a lane, to rows of
// shared memory in which the 16- or 32-byte pieces change places by row number,
// so that what eight lanes read together lies in different banks.
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
using sm100::bf16_parts;

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

// Copies to a stage and reads from it.
__device__ __forceinline__ void copy16(uint32_t dst, const void *src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t dst, const void *src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
// Order of the 16-byte pieces of a row in shared memory: as they are; the
// 64-byte halves of each 128 bytes swapped in odd rows; whole 32-byte sectors
// XORed with (row / 2) % 4; or pieces XORed for 8 x 8 tiles (TILES): with row % 8
// where rows lie a multiple of 128 bytes apart, else with (row / 2) % 4.
enum Order { AS_IS, HALVES, SECTORS, TILES };
template <int PITCH, Order ORDER>
__device__ __forceinline__ constexpr uint32_t order_bits(int row) {
    return ORDER == HALVES ? (row & 1) << 6
         : ORDER == SECTORS ? (row >> 1 & 3) << 5
         : ORDER == TILES ? (PITCH % 128 == 0 ? row & 7 : row >> 1 & 3) << 4 : 0;
}
// KEYS rows of BYTES, the first at `base`, to `st` at PITCH.  RUNS: lane n's
// `row` is the cache row of key n, and every 16 keys' rows follow one another
// (pages of 16 rows or more); otherwise each key has a row of its own.
template <int KEYS, int BYTES, int PITCH, Order ORDER, bool RUNS>
__device__ __forceinline__ void copy_rows(uint32_t st, const char *base, long long stride, int row) {
    constexpr int CPR = BYTES / 16;                             // copies per row
    constexpr int P = CPR % 3 ? 1 : 3, RP = 32 * P / CPR;       // after P copies, RP rows on, lanes repeat
    const int lane = threadIdx.x & 31;
    static_assert(KEYS * CPR % 32 == 0 && (P == 1 || RP % 8 == 0 || CPR == 24), "whole warps of copies");
    constexpr int SPAN = KEYS < 16 ? KEYS : 16, PER = SPAN * CPR / 32;   // rows of a run, its copies
#pragma unroll
    for (int s = 0; s < KEYS / SPAN; s++) {
        const char *run = RUNS ? base + __shfl_sync(0xffffffffu, row, s * SPAN) * stride : nullptr;
#pragma unroll
        for (int i = 0; i < PER; i++) {
            const int n = i % P * 32 + lane, lk = n / CPR, ch = n % CPR;          // within the period
            const int first = s * SPAN + i / P * RP;
            const char *src = RUNS ? run + (i / P * RP) * stride + lk * stride + ch * 16
                                   : base + __shfl_sync(0xffffffffu, row, first + lk) * stride + ch * 16;
            copy16(st + first * PITCH + ((lk * PITCH + ch * 16) ^ order_bits<PITCH, ORDER>(first + lk)), src);
        }
    }
}
// Pitch of INT8 V rows in SECTORS order: a multiple of 64, and of 128 past it.
constexpr int v_pitch(int bytes) { return bytes <= 64 ? 64 : (bytes + 127) / 128 * 128; }
// Byte `off` of V row 2c + odd + 8 n, from the row's start; `lane_off` is off's
// part that depends on the lane (under 128), XORed with c << 5 already.
template <int PITCH>
__device__ __forceinline__ uint32_t v_at(int odd, uint32_t lane_off, int off) {
    return PITCH == 64 ? (lane_off ^ (odd ? 64u : 0u)) + off : odd * PITCH + lane_off + off;
}
// Four 8 x 8 tiles of 16-bit elements: lane n gives the address of row n % 8 of
// tile n / 8 and gets elements (g, 2c), (g, 2c + 1) of each, or (2c, g),
// (2c + 1, g) with T.
template <bool T>
__device__ __forceinline__ void tiles(uint32_t (&r)[4], uint32_t a) {
    if constexpr (T)
        asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                     : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
    else
        asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                     : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
    return r;
}
// over the 8 lanes of the same c
__device__ __forceinline__ float keys_max(float v) {
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}
__device__ __forceinline__ float keys_sum(float v) {
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
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
// bf16, 8 NT query rows: column n of tile t is row 8 t + n.
//
// The second product takes a probability as two bf16 parts, its rounding and
// the rest (2^-17 of it at most is left out), so that what rounding the output
// costs is all the error there is, over few keys as over many.  With one part the
// error is 1.4 times that, and 16 rows on an 8192-row prefix take 25.9 us and not
// 26.4 (8 x 128), 28.5 and not 30.1 (16 x 64).
// ---------------------------------------------------------------------------
template <int D, int NT>
struct Bf16Path {
    using Type = __nv_bfloat16;           // of q and out
    static constexpr int ROWS = 8 * NT, KEYS = D <= 64 ? 32 : 16, LEAN = NT == 1, SCRATCH = 0;
    static constexpr int KM = KEYS / 16, KS = D / 16;         // 16-key tiles; 16-dim tiles
    static constexpr int PITCH = 2 * D, SLOT = KEYS * PITCH;
    uint32_t q[NT][KS][2], hi[NT][KM][2], lo[NT][KM][2];          // queries; the step's probabilities
    float o[NT][KS][4], m[NT][2], l[NT][2];
    const char *kb, *vb;

    __device__ __forceinline__ void begin(const Params &p, uint32_t, int first_req, int row0, int rows, int hk) {
        const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
#pragma unroll
        for (int t = 0; t < NT; t++) {
            const __nv_bfloat16 *a = query<__nv_bfloat16>(p, first_req, row0 + min(8 * t + g, rows - 1), hk, D) + 2 * c;
#pragma unroll
            for (int j = 0; j < KS; j++) {
                q[t][j][0] = __ldg(reinterpret_cast<const uint32_t *>(a + 16 * j));
                q[t][j][1] = __ldg(reinterpret_cast<const uint32_t *>(a + 16 * j + 8));
#pragma unroll
                for (int e = 0; e < 4; e++) o[t][j][e] = 0.f;
            }
            m[t][0] = m[t][1] = -INFINITY;
            l[t][0] = l[t][1] = 0.f;
        }
    }
    __device__ __forceinline__ void place(const Params &p, int hk) {
        kb = static_cast<const char *>(p.k) + (long long)hk * D * 2;
        vb = static_cast<const char *>(p.v) + (long long)hk * D * 2;
    }
    template <bool RUNS>
    __device__ __forceinline__ void copy_k(const Params &p, uint32_t st, int row) const {
        copy_rows<KEYS, 2 * D, PITCH, TILES, RUNS>(st, kb, p.row_stride * 2, row);
    }
    template <bool RUNS>
    __device__ __forceinline__ void copy_v(const Params &p, uint32_t st, int row) const {
        copy_rows<KEYS, 2 * D, PITCH, TILES, RUNS>(st, vb, p.row_stride * 2, row);
    }
    template <bool EDGE>                  // EDGE: some keys of the step have no row
    __device__ __forceinline__ void scores(const Params &p, uint32_t st, unsigned mask) {
        const int lane = threadIdx.x & 31, g = lane >> 2;
        // the row and piece that this lane addresses: tiles (keys, dims), (+8, dims), (keys, +8), (+8, +8)
        const uint32_t kst = st + ((lane >> 3 & 1) * 8 + (lane & 7)) * PITCH;
        const uint32_t kbits = order_bits<PITCH, TILES>(lane & 7) ^ (lane >> 4) << 4;
        float s[NT][KM][4];
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
            for (int i = 0; i < KM; i++) s[t][i][0] = s[t][i][1] = s[t][i][2] = s[t][i][3] = 0.f;
#pragma unroll
        for (int i = 0; i < KM; i++)
#pragma unroll
            for (int j = 0; j < KS; j++) {
                uint32_t a[4];
                tiles<false>(a, kst + i * 16 * PITCH + (kbits ^ 32 * j));
#pragma unroll
                for (int t = 0; t < NT; t++) mma_bf16(s[t][i], a, q[t][j][0], q[t][j][1]);
            }
        // all tiles' maxima first, so that their exchanges overlap, and one vote
        float neg[NT][2], alpha[NT][2];
        bool grows = false;
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
                float mx = -INFINITY;
#pragma unroll
                for (int i = 0; i < KM; i++) {
                    if (EDGE) {
                        if (!(mask >> (16 * i + g) & 1)) s[t][i][e] = -INFINITY;
                        if (!(mask >> (16 * i + g + 8) & 1)) s[t][i][e + 2] = -INFINITY;
                    }
                    mx = fmaxf(mx, fmaxf(s[t][i][e], s[t][i][e + 2]));
                }
                neg[t][e] = mx;
            }
#pragma unroll
        for (int d = 4; d < 32; d <<= 1)
#pragma unroll
            for (int t = 0; t < NT; t++)
#pragma unroll
                for (int e = 0; e < 2; e++) neg[t][e] = fmaxf(neg[t][e], __shfl_xor_sync(0xffffffffu, neg[t][e], d));
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const float mx = fmaxf(m[t][e], neg[t][e] * p.scale_log2);
                grows |= mx != m[t][e];
                neg[t][e] = mx == -INFINITY ? 0.f : -mx;
                alpha[t][e] = ex2(m[t][e] + neg[t][e]);
                m[t][e] = mx;
            }
        if (__any_sync(0xffffffffu, grows)) {
#pragma unroll
            for (int t = 0; t < NT; t++) {
                l[t][0] *= alpha[t][0];
                l[t][1] *= alpha[t][1];
#pragma unroll
                for (int j = 0; j < KS; j++)
#pragma unroll
                    for (int e = 0; e < 4; e++) o[t][j][e] *= alpha[t][e & 1];
            }
        }
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
            for (int i = 0; i < KM; i++) {
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    s[t][i][e] = ex2(fmaf(s[t][i][e], p.scale_log2, neg[t][e & 1]));
                    l[t][e & 1] += s[t][i][e];
                }
#pragma unroll
                for (int n = 0; n < 2; n++) {
                    bf16_parts(s[t][i][2 * n], s[t][i][2 * n + 1], hi[t][i][n], lo[t][i][n]);
                    hi[t][i][n] = transposed(hi[t][i][n]);
                    lo[t][i][n] = transposed(lo[t][i][n]);
                }
            }
    }
    template <bool EDGE>
    __device__ __forceinline__ void values(const Params &, uint32_t st, unsigned mask) {
        const int lane = threadIdx.x & 31, c = lane & 3;
        // tiles (keys, dims), (keys, +8), (+8, dims), (+8, +8), read transposed
        const uint32_t vst = st + ((lane >> 4) * 8 + (lane & 7)) * PITCH;
        const uint32_t vbits = order_bits<PITCH, TILES>(lane & 7) ^ (lane >> 3 & 1) << 4;
#pragma unroll
        for (int i = 0; i < KM; i++)
#pragma unroll
            for (int j = 0; j < KS; j++) {
                uint32_t a[4];
                tiles<true>(a, vst + i * 16 * PITCH + (vbits ^ 32 * j));
                if (EDGE) {               // keys with no row have probability 0, and values that may be NaN
#pragma unroll
                    for (int n = 0; n < 4; n++) {
                        const unsigned two = mask >> (16 * i + (n >> 1) * 8 + 2 * c) & 3;
                        a[n] &= (two & 1 ? 0xffffu : 0u) | (two & 2 ? 0xffff0000u : 0u);
                    }
                }
#pragma unroll
                for (int t = 0; t < NT; t++) {
                    mma_bf16(o[t][j], a, hi[t][i][0], hi[t][i][1]);
                    mma_bf16(o[t][j], a, lo[t][i][0], lo[t][i][1]);
                }
            }
    }
    __device__ __forceinline__ void finish(float *out, float2 *ml, int rows) {
        const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const float sum = keys_sum(l[t][e]);
                const int row = 8 * t + 2 * c + e;
                if (row >= rows) continue;
                if (g == 0) ml[row] = make_float2(m[t][e], sum);
#pragma unroll
                for (int j = 0; j < KS; j++) {
                    out[row * D + 16 * j + g] = o[t][j][e];
                    out[row * D + 16 * j + g + 8] = o[t][j][e + 2];
                }
            }
    }
};

// ---------------------------------------------------------------------------
// INT8 codes, 4 NT query rows: the same products in f16, in which a code is
// exact.
//
// A query and a weight w = p * vscale go in as two f16 parts, columns 2 r and
// 2 r + 1 of the row's tile, whose results are added: 22 bits of each.  The
// query row is first scaled by a power of two that puts its largest element in
// [2^7, 2^8), a row's weights by one that puts the largest of them so far in
// [2^14, 2^15), so the second parts stay above f16's smallest numbers (a weight
// 2^-17 of the largest keeps its 22 bits, any other 2^-39 of the largest).  The
// largest weight and not the largest vscale sets that power: a row with a wide
// vscale and no probability would take the bits of all others.  It follows the
// weights down when the maximum of the scores grows.  A code c becomes f16
// as the low byte of 1024 + (c + 128) minus 1152, all exact.  The tensor core
// rounds its sums towards zero, which drifts over a long piece, so every
// FOLD steps the output sums move to fp32 registers.
//
// A dot product may take its k positions in any order, and O^T its rows: lane
// (g, c) reads 16 contiguous codes of a K row (four k-steps' fragments) and 8
// dims of a V row, whose pairs of keys one byte permutation brings together.
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
// exponent of x >= 0, within [-97, 127]
__device__ __forceinline__ int exponent(float x) { return min(127, max(-97, (__float_as_int(x) >> 23) - 127)); }
// Is a weight at or past the next power of two above the row's largest so far?
__device__ __forceinline__ bool outgrows(float weight, float top) {
    return weight > __int_as_float(__float_as_int(top) | 0x007fffff);
}
// What the sums of weights are multiplied by when the row's largest weight
// becomes `now`, and the weights before lose the factor alpha.
__device__ __forceinline__ float rescaling(float alpha, float top, float now) {
    return alpha * pow2i(min(127, max(-126, exponent(top) - exponent(now))));
}

template <int D, int NT>
struct I8Path {
    using Type = float;
    static constexpr int ROWS = 4 * NT, KEYS = 32, FOLD = 8, LEAN = NT == 1, SCRATCH = 0;
    static constexpr int KM = KEYS / 16, B64 = D / 64, REM = D % 64 != 0;
    static constexpr int KW = D / 16;                         // words of a K row per lane = k-steps = 16-dim tiles
    // a V slot holds its rows and both scales (K's are used with V's, once the code sums are there)
    static constexpr int VP = v_pitch(D), OFF_S = KEYS * VP, SLOT = OFF_S + 2 * 4 * KEYS;
    static constexpr bool SWAP = D == 128;
    uint32_t q[NT][KW][2];
    float s[NT][KM][4];                                       // the step's code sums
    float o[NT][KW][4], f[NT][KW][2], m[NT], l[NT];
    float qscale[NT];                                         // scale log2(e) / the query row's power of two
    float top[NT];                                            // the row's largest weight |p vscale|
    int folded, head;
    const char *kb, *vb;

    __device__ __forceinline__ void begin(const Params &p, uint32_t, int first_req, int row0, int rows, int hk) {
        const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
#pragma unroll
        for (int t = 0; t < NT; t++) {
            const float *a = query<float>(p, first_req, row0 + min(4 * t + (g >> 1), rows - 1), hk, D);
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
            qscale[t] = __shfl_sync(0xffffffffu, p.scale_log2 * pow2i(-e), 8 * c);   // of row c
#pragma unroll
            for (int j = 0; j < KW; j++) {
                uint32_t hi, lo;
                f16_parts(x[j].x * up, x[j].y * up, hi, lo);
                q[t][j][0] = g & 1 ? lo : hi;
                f16_parts(x[j].z * up, x[j].w * up, hi, lo);
                q[t][j][1] = g & 1 ? lo : hi;
#pragma unroll
                for (int n = 0; n < 4; n++) o[t][j][n] = 0.f;
                f[t][j][0] = f[t][j][1] = 0.f;
            }
            m[t] = -INFINITY;
            l[t] = top[t] = 0.f;
        }
        folded = 0;
    }
    __device__ __forceinline__ void place(const Params &p, int hk) {
        head = hk;
        kb = static_cast<const char *>(p.k) + (long long)hk * D;
        vb = static_cast<const char *>(p.v) + (long long)hk * D;
    }
    template <bool RUNS>
    __device__ __forceinline__ void copy_k(const Params &p, uint32_t st, int row) const {
        copy_rows<KEYS, D, D, SWAP ? HALVES : AS_IS, RUNS>(st, kb, p.row_stride, row);
    }
    template <bool RUNS>
    __device__ __forceinline__ void copy_v(const Params &p, uint32_t st, int row) const {
        const int lane = threadIdx.x & 31;
        const long long at_scale = (long long)row * p.kv_heads + head;
        copy4(st + OFF_S + lane * 4, p.kscale + at_scale);
        copy4(st + OFF_S + 128 + lane * 4, p.vscale + at_scale);
        copy_rows<KEYS, D, VP, SECTORS, RUNS>(st, vb, p.row_stride, row);
    }
    __device__ __forceinline__ void fold() {
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
            for (int j = 0; j < KW; j++)
#pragma unroll
                for (int n = 0; n < 2; n++) {
                    f[t][j][n] += o[t][j][2 * n] + o[t][j][2 * n + 1];
                    o[t][j][2 * n] = o[t][j][2 * n + 1] = 0.f;
                }
        folded = 0;
    }
    __device__ __forceinline__ void scale_output(int t, float a) {
#pragma unroll
        for (int j = 0; j < KW; j++) {
#pragma unroll
            for (int n = 0; n < 4; n++) o[t][j][n] *= a;
            f[t][j][0] *= a;
            f[t][j][1] *= a;
        }
    }
    // Two 16-dim tiles from one word (4 dims) of each of the lane's keys 2c, 2c + 1, 2c + 8, 2c + 9.
    __device__ __forceinline__ void pair(int j, const uint32_t (&w)[NT][2], uint32_t v0, uint32_t v1, uint32_t v2, uint32_t v3) {
        const uint32_t a01 = prmt(v0, v1, 0x5140) ^ 0x80808080u, a23 = prmt(v0, v1, 0x7362) ^ 0x80808080u;
        const uint32_t b01 = prmt(v2, v3, 0x5140) ^ 0x80808080u, b23 = prmt(v2, v3, 0x7362) ^ 0x80808080u;
        const uint32_t x[4] = {codes_f16(a01, 0x4140), codes_f16(a01, 0x4342), codes_f16(b01, 0x4140), codes_f16(b01, 0x4342)};
        const uint32_t y[4] = {codes_f16(a23, 0x4140), codes_f16(a23, 0x4342), codes_f16(b23, 0x4140), codes_f16(b23, 0x4342)};
#pragma unroll
        for (int t = 0; t < NT; t++) {
            mma_f16(o[t][j], x, w[t][0], w[t][1]);
            mma_f16(o[t][j + 1], y, w[t][0], w[t][1]);
        }
    }
    template <bool EDGE>
    __device__ __forceinline__ void scores(const Params &, uint32_t st, unsigned) {
        const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
        const uint32_t kst = st + g * D, swap = SWAP ? (g & 1) * 64 : 0;
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
            for (int i = 0; i < KM; i++) s[t][i][0] = s[t][i][1] = s[t][i][2] = s[t][i][3] = 0.f;
#pragma unroll
        for (int i = 0; i < KM; i++) {
            uint32_t w[2][KW];                                // codes + 128 of keys g and g + 8
#pragma unroll
            for (int n = 0; n < 2; n++) {
                const uint32_t at = kst + (16 * i + 8 * n) * D;
#pragma unroll
                for (int x = 0; x < B64; x++) {
                    const uint4 k = lds16(at + 64 * x + 16 * c + (x & 1 ? -swap : swap));
                    w[n][4 * x] = k.x; w[n][4 * x + 1] = k.y; w[n][4 * x + 2] = k.z; w[n][4 * x + 3] = k.w;
                }
                if constexpr (REM) {
                    const uint2 k = lds8(at + 64 * B64 + 8 * c);
                    w[n][4 * B64] = k.x; w[n][4 * B64 + 1] = k.y;
                }
            }
#pragma unroll
            for (int j = 0; j < KW; j++) {
                const uint32_t u = w[0][j] ^ 0x80808080u, v = w[1][j] ^ 0x80808080u;
                const uint32_t a[4] = {codes_f16(u, 0x4140), codes_f16(v, 0x4140), codes_f16(u, 0x4342), codes_f16(v, 0x4342)};
#pragma unroll
                for (int t = 0; t < NT; t++) mma_f16(s[t][i], a, q[t][j][0], q[t][j][1]);
            }
        }
    }
    template <bool EDGE>
    __device__ __forceinline__ void values(const Params &, uint32_t st, unsigned mask) {
        const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
        const uint32_t vst = st + 2 * c * VP, v8 = 8 * g ^ c << 5, v4 = 4 * g ^ c << 5;
        // scales of the lane's keys: g, g + 8 of each 16; absent keys' scales are not numbers to go by
        float ks[KM][2], vs[KM][2];
#pragma unroll
        for (int i = 0; i < KM; i++)
#pragma unroll
            for (int n = 0; n < 2; n++) {
                const int key = 16 * i + 8 * n + g;
                ks[i][n] = __uint_as_float(lds4(st + OFF_S + key * 4));
                vs[i][n] = __uint_as_float(lds4(st + OFF_S + 128 + key * 4));
                if (EDGE && !(mask >> key & 1)) vs[i][n] = 0.f;
            }
        // all tiles' maxima first, so that their exchanges overlap, and one vote
        uint32_t pw[KM][NT][2];
        float neg[NT], alpha[NT], big[NT];
        bool grows = false;
#pragma unroll
        for (int t = 0; t < NT; t++) {
            neg[t] = -INFINITY;
#pragma unroll
            for (int i = 0; i < KM; i++)
#pragma unroll
                for (int n = 0; n < 2; n++) {
                    float x = (s[t][i][2 * n] + s[t][i][2 * n + 1]) * qscale[t] * ks[i][n];
                    if (EDGE && !(mask >> (16 * i + 8 * n + g) & 1)) x = -INFINITY;
                    s[t][i][2 * n] = x;
                    neg[t] = fmaxf(neg[t], x);
                }
        }
#pragma unroll
        for (int d = 4; d < 32; d <<= 1)
#pragma unroll
            for (int t = 0; t < NT; t++) neg[t] = fmaxf(neg[t], __shfl_xor_sync(0xffffffffu, neg[t], d));
#pragma unroll
        for (int t = 0; t < NT; t++) {
            const float mx = fmaxf(m[t], neg[t]);
            grows |= mx != m[t];
            neg[t] = mx == -INFINITY ? 0.f : -mx;
            alpha[t] = ex2(m[t] + neg[t]);
            m[t] = mx;
            l[t] *= alpha[t];
            big[t] = 0.f;
#pragma unroll
            for (int i = 0; i < KM; i++)
#pragma unroll
                for (int n = 0; n < 2; n++) {
                    const float e = ex2(s[t][i][2 * n] + neg[t]);
                    l[t] += e;
                    s[t][i][2 * n] = e * vs[i][n];
                    big[t] = fmaxf(big[t], fabsf(s[t][i][2 * n]));
                }
            grows |= outgrows(big[t], top[t]);
        }
        if (__any_sync(0xffffffffu, grows)) {
#pragma unroll
            for (int d = 4; d < 32; d <<= 1)
#pragma unroll
                for (int t = 0; t < NT; t++) big[t] = fmaxf(big[t], __shfl_xor_sync(0xffffffffu, big[t], d));
#pragma unroll
            for (int t = 0; t < NT; t++) {
                const float now = fmaxf(top[t] * alpha[t], big[t]);
                scale_output(t, rescaling(alpha[t], top[t], now));
                top[t] = now;
            }
        }
#pragma unroll
        for (int t = 0; t < NT; t++) {
            const float wscale = pow2i(14 - exponent(top[t]));
#pragma unroll
            for (int i = 0; i < KM; i++)
#pragma unroll
                for (int n = 0; n < 2; n++) {
                    const float w = s[t][i][2 * n] * wscale;
                    const __half hi = __float2half_rn(w);
                    const __half2 both = __halves2half2(hi, __float2half_rn(w - __half2float(hi)));
                    pw[i][t][n] = transposed(*reinterpret_cast<const uint32_t *>(&both));
                }
        }
#pragma unroll
        for (int i = 0; i < KM; i++) {
#pragma unroll
            for (int x = 0; x < B64; x++) {
                uint2 v[4];
#pragma unroll
                for (int n = 0; n < 4; n++)
                    v[n] = lds8(vst + (i * 16 + (n >> 1) * 8) * VP + v_at<VP>(n & 1, x & 1 ? v8 ^ 64 : v8, x / 2 * 128));
                pair(4 * x, pw[i], v[0].x, v[1].x, v[2].x, v[3].x);
                pair(4 * x + 2, pw[i], v[0].y, v[1].y, v[2].y, v[3].y);
            }
            if constexpr (REM) {
                uint32_t v[4];
#pragma unroll
                for (int n = 0; n < 4; n++)
                    v[n] = lds4(vst + (i * 16 + (n >> 1) * 8) * VP + v_at<VP>(n & 1, B64 ? v4 ^ 64 : v4, 0));
                pair(4 * B64, pw[i], v[0], v[1], v[2], v[3]);
            }
        }
        if (++folded == FOLD) fold();
    }
    __device__ __forceinline__ void finish(float *out, float2 *ml, int rows) {
        const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
        fold();
#pragma unroll
        for (int t = 0; t < NT; t++) {
            const float sum = keys_sum(l[t]), down = pow2i(exponent(top[t]) - 14);
            const int row = 4 * t + c;
            if (row >= rows) continue;
            if (g == 0) ml[row] = make_float2(m[t], sum);
            // tile j's rows g and g + 8 are dims 2j and 2j + 1 (of 8, or 4) of the lane's
#pragma unroll
            for (int j = 0; j < KW; j += 2) {
                const int dim = j < 4 * B64 ? 64 * (j / 4) + 8 * g + 2 * (j % 4) : 64 * B64 + 4 * g;
                *reinterpret_cast<float4 *>(out + row * D + dim) =
                    make_float4(f[t][j][0] * down, f[t][j][1] * down, f[t][j + 1][0] * down, f[t][j + 1][1] * down);
            }
        }
    }
};

// ---------------------------------------------------------------------------
// INT8 codes, 2 query rows: both products in integers, so no code is converted.
//
// A query and a weight p * vscale become integers of 30 bits, the row's largest
// element and its largest weight so far (as above) in [2^29, 2^30), and go in as
// four signed digits of base 256, columns 4 r to 4 r + 3 of the tile from the
// highest down.  The sums are exact:
// under 2^21 of a score's digits, and 2^19 a step of an output's, for FOLD steps.
// Lane (g, c) has the pair of digits 2 (c & 1) of row c / 2, and the two lanes
// of a row exchange theirs.  Not numbers: a query's makes the score's scale one,
// a vscale's the output.
//
// The weights of keys g and g + 8 share the 16-bit elements of the transposition,
// so a lane's word of 4 keys is 2c, 2c + 8, 2c + 1, 2c + 9, and of V four words
// (4 keys, 4 dims) turn into it with 8 byte permutations.
// (64 requests with up to 8192 rows, 16 x 64: 117 us a call, 126 with two f16 parts
// and converted codes; more query rows would need a second tile of digits.)
// ---------------------------------------------------------------------------
__device__ __forceinline__ void mma_s8(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// x, |x| <= 2^30, as four signed bytes of base 256
__device__ __forceinline__ uint32_t digits(int x) { return ((uint32_t)x + 0x00808080u) ^ 0x00808080u; }

template <int D>
struct I8Digits : I8Path<D, 1> {
    using Base = I8Path<D, 1>;
    using Base::B64;
    using Base::KM;
    using Base::KW;
    using Base::OFF_S;
    using Base::REM;
    using Base::SWAP;
    using Base::VP;
    static constexpr int ROWS = 2, FOLD = 64;
    uint32_t q[KW];
    float s[KM][2];                                           // the step's code sums
    int o[KW][4];
    float f[KW][2], m, l, qscale, top, bad;
    int folded;

    __device__ __forceinline__ void begin(const Params &p, uint32_t, int first_req, int row0, int rows, int hk) {
        const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
        const float *a = query<float>(p, first_req, row0 + min(g >> 2, rows - 1), hk, D);
        float4 x[KW];
        float amax = 0.f, poison = 0.f;
#pragma unroll
        for (int j = 0; j < KW; j++) {
            // word j of this lane: 16 codes of each 64 dims, then 8 of the last 32
            const int dim = j < 4 * B64 ? 64 * (j / 4) + 16 * c + 4 * (j % 4) : 64 * B64 + 8 * c + 4 * (j - 4 * B64);
            x[j] = __ldg(reinterpret_cast<const float4 *>(a + dim));
            amax = fmaxf(amax, fmaxf(fmaxf(fabsf(x[j].x), fabsf(x[j].y)), fmaxf(fabsf(x[j].z), fabsf(x[j].w))));
            poison += x[j].x * 0.f + x[j].y * 0.f + (x[j].z * 0.f + x[j].w * 0.f);
        }
        amax = quad_max(amax);
        poison += __shfl_xor_sync(0xffffffffu, poison, 1);
        poison += __shfl_xor_sync(0xffffffffu, poison, 2);
        const int e = amax > 0.f ? 29 - max((__float_as_int(amax) >> 23) - 127, -97) : 0;      // both powers are numbers
        const float up = pow2i(e);
        qscale = __shfl_sync(0xffffffffu, p.scale_log2 * pow2i(-e) + poison, 16 * (c >> 1));   // of row c / 2
        const uint32_t digit = 3 - (g & 3);
#pragma unroll
        for (int j = 0; j < KW; j++) {
            const uint32_t d0 = digits(__float2int_rn(x[j].x * up)), d1 = digits(__float2int_rn(x[j].y * up));
            const uint32_t d2 = digits(__float2int_rn(x[j].z * up)), d3 = digits(__float2int_rn(x[j].w * up));
            const uint32_t pick = digit | (4 + digit) << 4;
            q[j] = prmt(prmt(d0, d1, pick), prmt(d2, d3, pick), 0x5410);
#pragma unroll
            for (int n = 0; n < 4; n++) o[j][n] = 0;
            f[j][0] = f[j][1] = 0.f;
        }
        m = -INFINITY;
        l = top = bad = 0.f;
        folded = 0;
    }
    __device__ __forceinline__ void fold() {
#pragma unroll
        for (int j = 0; j < KW; j++)
#pragma unroll
            for (int n = 0; n < 2; n++) {
                f[j][n] += fmaf((float)o[j][2 * n], 256.f, (float)o[j][2 * n + 1]);
                o[j][2 * n] = o[j][2 * n + 1] = 0;
            }
        folded = 0;
    }
    __device__ __forceinline__ void scale_output(float a) {
        fold();
#pragma unroll
        for (int j = 0; j < KW; j++) {
            f[j][0] *= a;
            f[j][1] *= a;
        }
    }
    template <bool EDGE>
    __device__ __forceinline__ void scores(const Params &, uint32_t st, unsigned) {
        const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
        const uint32_t kst = st + g * D, swap = SWAP ? (g & 1) * 64 : 0;
        const float mine = c & 1 ? 1.f : 65536.f, others = c & 1 ? 65536.f : 1.f;
#pragma unroll
        for (int i = 0; i < KM; i++) {
            uint32_t w[2][KW];                                // codes of keys g and g + 8
#pragma unroll
            for (int n = 0; n < 2; n++) {
                const uint32_t at = kst + (16 * i + 8 * n) * D;
#pragma unroll
                for (int x = 0; x < B64; x++) {
                    const uint4 k = lds16(at + 64 * x + 16 * c + (x & 1 ? -swap : swap));
                    w[n][4 * x] = k.x; w[n][4 * x + 1] = k.y; w[n][4 * x + 2] = k.z; w[n][4 * x + 3] = k.w;
                }
                if constexpr (REM) {
                    const uint2 k = lds8(at + 64 * B64 + 8 * c);
                    w[n][4 * B64] = k.x; w[n][4 * B64 + 1] = k.y;
                }
            }
            int sum[4] = {0, 0, 0, 0};
#pragma unroll
            for (int j = 0; j < KW; j += 2) mma_s8(sum, w[0][j], w[1][j], w[0][j + 1], w[1][j + 1], q[j], q[j + 1]);
#pragma unroll
            for (int n = 0; n < 2; n++) {
                const float x = (float)(sum[2 * n] * 256 + sum[2 * n + 1]);
                s[i][n] = fmaf(__shfl_xor_sync(0xffffffffu, x, 1), others, x * mine);
            }
        }
    }
    template <bool EDGE>
    __device__ __forceinline__ void values(const Params &, uint32_t st, unsigned mask) {
        const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
        const uint32_t vst = st + 2 * c * VP, v8 = 8 * g ^ c << 5, v4 = 4 * g ^ c << 5;
        // scales of the lane's keys: g, g + 8 of each 16; absent keys' scales are not numbers to go by
        float vs[KM][2], mx = -INFINITY;
#pragma unroll
        for (int i = 0; i < KM; i++)
#pragma unroll
            for (int n = 0; n < 2; n++) {
                const int key = 16 * i + 8 * n + g;
                const bool there = !EDGE || (mask >> key & 1);
                const float ks = __uint_as_float(lds4(st + OFF_S + key * 4));
                vs[i][n] = __uint_as_float(lds4(st + OFF_S + 128 + key * 4));
                if (!there) vs[i][n] = 0.f;
                bad = fmaf(vs[i][n], 0.f, bad);
                s[i][n] = there ? s[i][n] * qscale * ks : -INFINITY;
                mx = fmaxf(mx, s[i][n]);
            }
        mx = fmaxf(m, keys_max(mx));
        const float neg = mx == -INFINITY ? 0.f : -mx, alpha = ex2(m + neg);
        float big = 0.f;
        l *= alpha;
#pragma unroll
        for (int i = 0; i < KM; i++)
#pragma unroll
            for (int n = 0; n < 2; n++) {
                const float e = ex2(s[i][n] + neg);
                l += e;
                vs[i][n] *= e;
                big = fmaxf(big, fabsf(vs[i][n]));
            }
        if (__any_sync(0xffffffffu, mx != m || outgrows(big, top))) {
            const float now = fmaxf(top * alpha, keys_max(big));
            scale_output(rescaling(alpha, top, now));
            top = now;
        }
        m = mx;
        const float wscale = pow2i(29 - exponent(top));
        uint32_t w[KM];
#pragma unroll
        for (int i = 0; i < KM; i++) {
            uint32_t d[2];
#pragma unroll
            for (int n = 0; n < 2; n++) d[n] = digits(__float2int_rn(vs[i][n] * wscale));
            w[i] = transposed(prmt(d[0], d[1], c & 1 ? 0x4051 : 0x6273));
        }
        // 4 dims of 4 keys to 4 keys of each dim
        auto turn = [](uint32_t (&x)[4], uint32_t v0, uint32_t v1, uint32_t v2, uint32_t v3) {
            const uint32_t a = prmt(v0, v2, 0x5140), b = prmt(v1, v3, 0x5140), e = prmt(v0, v2, 0x7362), h = prmt(v1, v3, 0x7362);
            x[0] = prmt(a, b, 0x5410); x[1] = prmt(a, b, 0x7632); x[2] = prmt(e, h, 0x5410); x[3] = prmt(e, h, 0x7632);
        };
        static_assert(KM == 2, "a step is one product's depth");
#pragma unroll
        for (int x = 0; x < B64; x++) {
            uint2 v[2][4];
#pragma unroll
            for (int i = 0; i < 2; i++)
#pragma unroll
                for (int n = 0; n < 4; n++)
                    v[i][n] = lds8(vst + (i * 16 + (n >> 1) * 8) * VP + v_at<VP>(n & 1, x & 1 ? v8 ^ 64 : v8, x / 2 * 128));
#pragma unroll
            for (int h = 0; h < 2; h++) {
                uint32_t y[2][4];
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    if (h == 0) turn(y[i], v[i][0].x, v[i][1].x, v[i][2].x, v[i][3].x);
                    else turn(y[i], v[i][0].y, v[i][1].y, v[i][2].y, v[i][3].y);
                }
                mma_s8(o[4 * x + 2 * h], y[0][0], y[0][1], y[1][0], y[1][1], w[0], w[1]);
                mma_s8(o[4 * x + 2 * h + 1], y[0][2], y[0][3], y[1][2], y[1][3], w[0], w[1]);
            }
        }
        if constexpr (REM) {
            uint32_t v[4], y[2][4];
#pragma unroll
            for (int i = 0; i < 2; i++) {
#pragma unroll
                for (int n = 0; n < 4; n++)
                    v[n] = lds4(vst + (i * 16 + (n >> 1) * 8) * VP + v_at<VP>(n & 1, B64 ? v4 ^ 64 : v4, 0));
                turn(y[i], v[0], v[1], v[2], v[3]);
            }
            mma_s8(o[4 * B64], y[0][0], y[0][1], y[1][0], y[1][1], w[0], w[1]);
            mma_s8(o[4 * B64 + 1], y[0][2], y[0][3], y[1][2], y[1][3], w[0], w[1]);
        }
        if (++folded == FOLD) fold();
    }
    __device__ __forceinline__ void finish(float *out, float2 *ml, int rows) {
        const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
        fold();
        const float down = pow2i(exponent(top) - 29), sum = keys_sum(l), nan = keys_sum(bad);
        const float mine = c & 1 ? 1.f : 65536.f, others = c & 1 ? 65536.f : 1.f;
#pragma unroll
        for (int j = 0; j < KW; j++)
#pragma unroll
            for (int n = 0; n < 2; n++)
                f[j][n] = fmaf(__shfl_xor_sync(0xffffffffu, f[j][n], 1), others, f[j][n] * mine) * down + nan;
        const int row = c >> 1;
        if (row >= rows) return;
        if (g == 0 && !(c & 1)) ml[row] = make_float2(m, sum);
        // tile j's rows g and g + 8 are dims 2j and 2j + 1 (of 8, or 4) of the lane's; the two lanes take turns
#pragma unroll
        for (int j = 0; j < KW; j += 2) {
            if ((j / 2 & 1) != (c & 1)) continue;
            const int dim = j < 4 * B64 ? 64 * (j / 4) + 8 * g + 2 * (j % 4) : 64 * B64 + 4 * g;
            *reinterpret_cast<float4 *>(out + row * D + dim) = make_float4(f[j][0], f[j][1], f[j + 1][0], f[j + 1][1]);
        }
    }
};

// ---------------------------------------------------------------------------
// fp32: fp32 FMAs on pairs, R query rows.
//
// LPK lanes share a key, each with E = D / LPK of its dims, so a score is a dot
// product of E terms and a sum over LPK lanes; each group of LPK lanes keeps
// its own running softmax over its keys (every 32/LPK-th) and the groups join
// once, in finish().  At most 4 R flops stand against a byte (R/2 of them), so
// up to 8 rows the FMA pipe keeps up with the memory.
//
// SPREAD (8 rows): a step's R U scores of a group are summed by halving, a lane
// handing on half of its values at each stage and keeping the other, so the
// lanes end with R U / LPK scores each (8 / LPK of a row's lanes) instead of all
// of them in every lane; each lane does the softmax of its own, and the
// probabilities reach the group through a scratch of shared memory, as pairs.
// (All scores in all lanes took 1,010 instructions a step of 8 keys at d 128,
// 256 of them FMAs.)
// ---------------------------------------------------------------------------
template <int D, int R>
struct F32Path {
    using Type = float;
    static constexpr int ROWS = R;
    static constexpr bool SPREAD = R == 8;
    // 8 or 16 lanes read 128 bytes of a row together; q and o take 2 E R registers, 64 to 96
    static constexpr int LPK = R >= 4 && D > 32 ? 16 : 8, LEAN = R <= 4;
    static constexpr int E = D / LPK, W = E % 4 ? 2 : 4, N = E / W;   // floats per lane, per read, reads
    static constexpr int G = 32 / LPK;                        // keys at a time
    static constexpr int U = (D >= 96 ? 8 : D == 64 ? 16 : 32) / G;   // keys of a group per step
    static constexpr int KEYS = G * U, SLOT = KEYS * D * 4;
    static constexpr int L = SPREAD ? LPK / R : 1;            // lanes of a row
    static constexpr int MINE = SPREAD ? U / L : U;           // scores of a row in a lane
    static constexpr int M = SPREAD ? 1 : R;                  // rows whose m and l a lane keeps
    static constexpr int SCRATCH = SPREAD ? G * R * U * 8 : 0;
    static_assert(KEYS <= 32 && LPK * E == D && N * W == E && (!SPREAD || (LPK % R == 0 && MINE % 2 == 0)), "lane geometry");
    uint64_t q[R][E / 2], o[R][E / 2];
    float m[M], l[M], x[SPREAD ? 1 : R][U];                   // x: the step's scores, then probabilities
    uint32_t scratch;
    const char *kb, *vb;

    __device__ __forceinline__ static void read(uint64_t (&x)[E / 2], uint32_t at) {
#pragma unroll
        for (int i = 0; i < N; i++) {
            if constexpr (W == 4) {
                pair(x[2 * i], x[2 * i + 1], at + i * LPK * 16);
            } else {
                asm volatile("ld.shared.u64 %0, [%1];" : "=l"(x[i]) : "r"(at + i * LPK * 8) : "memory");
            }
        }
    }
    __device__ __forceinline__ static void pair(uint64_t &a, uint64_t &b, uint32_t at) {
        asm volatile("ld.shared.v2.u64 {%0,%1}, [%2];" : "=l"(a), "=l"(b) : "r"(at) : "memory");
    }
    __device__ __forceinline__ void begin(const Params &p, uint32_t scratch_, int first_req, int row0, int rows, int hk) {
        const int sub = (threadIdx.x & 31) % LPK;
        const uint64_t s2 = f2(p.scale_log2, p.scale_log2);
        scratch = scratch_;
#pragma unroll
        for (int r = 0; r < R; r++) {
            const float *a = query<float>(p, first_req, row0 + min(r, rows - 1), hk, D) + sub * W;
#pragma unroll
            for (int i = 0; i < E / 2; i++) {
                const float2 x = __ldg(reinterpret_cast<const float2 *>(a + i / (W / 2) * (LPK * W) + i % (W / 2) * 2));
                q[r][i] = fma2(f2(x.x, x.y), s2, 0ull);
                o[r][i] = 0ull;
            }
        }
#pragma unroll
        for (int r = 0; r < M; r++) {
            m[r] = -INFINITY;
            l[r] = 0.f;
        }
    }
    __device__ __forceinline__ void place(const Params &p, int hk) {
        kb = static_cast<const char *>(p.k) + (long long)hk * D * 4;
        vb = static_cast<const char *>(p.v) + (long long)hk * D * 4;
    }
    template <bool RUNS>
    __device__ __forceinline__ void copy_k(const Params &p, uint32_t st, int row) const {
        copy_rows<KEYS, D * 4, D * 4, AS_IS, RUNS>(st, kb, p.row_stride * 4, row);
    }
    template <bool RUNS>
    __device__ __forceinline__ void copy_v(const Params &p, uint32_t st, int row) const {
        copy_rows<KEYS, D * 4, D * 4, AS_IS, RUNS>(st, vb, p.row_stride * 4, row);
    }
    __device__ __forceinline__ void scale_output(int r, float a) {
#pragma unroll
        for (int i = 0; i < E / 2; i++) o[r][i] = fma2(o[r][i], f2(a, a), 0ull);
    }
    template <bool EDGE>
    __device__ __forceinline__ void scores(const Params &, uint32_t st, unsigned mask) {
        const int lane = threadIdx.x & 31, g = lane / LPK;
        st += g * D * 4 + lane % LPK * W * 4;
        float y[R * U];                   // score r U + u: this lane's part, then the sum
#pragma unroll
        for (int u = 0; u < U; u++) {
            uint64_t k[E / 2];
            read(k, st + u * G * D * 4);
#pragma unroll
            for (int r = 0; r < R; r++) {
                uint64_t a = 0ull;
#pragma unroll
                for (int i = 0; i < E / 2; i++) a = fma2(q[r][i], k[i], a);
                float lo, hi;
                f2_split(a, lo, hi);
                y[r * U + u] = lo + hi;
            }
        }
        if constexpr (SPREAD) {
            const int sub = lane % LPK;
#pragma unroll
            for (int d = LPK / 2, n = R * U / 2; d > 0; d >>= 1, n >>= 1) {
                const bool upper = sub & d;
#pragma unroll
                for (int i = 0; i < R * U / 2; i++) {
                    if (i >= n) break;
                    const float send = upper ? y[i] : y[i + n], keep = upper ? y[i + n] : y[i];
                    y[i] = keep + __shfl_xor_sync(0xffffffffu, send, d);
                }
            }
            // now scores sub MINE + i: row sub / L, keys (sub % L) MINE + i of the group
            float mx = m[0];
#pragma unroll
            for (int i = 0; i < MINE; i++) {
                if (EDGE && !(mask >> (((sub % L) * MINE + i) * G + g) & 1)) y[i] = -INFINITY;
                mx = fmaxf(mx, y[i]);
            }
#pragma unroll
            for (int d = 1; d < L; d <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
            const float neg = mx == -INFINITY ? 0.f : -mx;
            if (__any_sync(0xffffffffu, mx != m[0])) {
                const float a = ex2(m[0] + neg);
                l[0] *= a;
#pragma unroll
                for (int r = 0; r < R; r++) scale_output(r, __shfl_sync(0xffffffffu, a, g * LPK + r * L));
                m[0] = mx;
            }
            const uint32_t to = scratch + (g * R * U + sub * MINE) * 8;
            __syncwarp();                 // the last step's probabilities are read
#pragma unroll
            for (int i = 0; i < MINE; i += 2) {
                const float a = ex2(y[i] + neg), b = ex2(y[i + 1] + neg);
                l[0] += a + b;
                asm volatile("st.shared.v4.f32 [%0], {%1,%1,%2,%2};" ::"r"(to + i * 8), "f"(a), "f"(b) : "memory");
            }
            __syncwarp();
        } else {
#pragma unroll
            for (int d = LPK / 2; d > 0; d >>= 1)
#pragma unroll
                for (int i = 0; i < R * U; i++) y[i] += __shfl_xor_sync(0xffffffffu, y[i], d);
#pragma unroll
            for (int r = 0; r < R; r++) {
                float mx = m[r];
#pragma unroll
                for (int u = 0; u < U; u++) {
                    if (EDGE && !(mask >> (u * G + g) & 1)) y[r * U + u] = -INFINITY;
                    mx = fmaxf(mx, y[r * U + u]);
                }
                const float neg = mx == -INFINITY ? 0.f : -mx;
                if (mx != m[r]) {
                    const float a = ex2(m[r] + neg);
                    l[r] *= a;
                    scale_output(r, a);
                    m[r] = mx;
                }
#pragma unroll
                for (int u = 0; u < U; u++) {
                    x[r][u] = ex2(y[r * U + u] + neg);
                    l[r] += x[r][u];
                }
            }
        }
    }
    template <bool EDGE>
    __device__ __forceinline__ void values(const Params &, uint32_t st, unsigned mask) {
        const int lane = threadIdx.x & 31, g = lane / LPK;
        st += g * D * 4 + lane % LPK * W * 4;
        auto value = [&](uint64_t (&v)[E / 2], int u) {
            read(v, st + u * G * D * 4);
            if (EDGE && !(mask >> (u * G + g) & 1)) {       // probability 0, and values that may be NaN
#pragma unroll
                for (int i = 0; i < E / 2; i++) v[i] = 0ull;
            }
        };
        if constexpr (SPREAD) {
#pragma unroll
            for (int u = 0; u < U; u += 2) {
                uint64_t v[E / 2], w[E / 2];
                value(v, u);
                value(w, u + 1);
#pragma unroll
                for (int r = 0; r < R; r++) {
                    uint64_t a, b;
                    pair(a, b, scratch + (g * R * U + r * U + u) * 8);
#pragma unroll
                    for (int i = 0; i < E / 2; i++) o[r][i] = fma2(b, w[i], fma2(a, v[i], o[r][i]));
                }
            }
        } else {
#pragma unroll
            for (int u = 0; u < U; u++) {
                uint64_t v[E / 2];
                value(v, u);
#pragma unroll
                for (int r = 0; r < R; r++)
#pragma unroll
                    for (int i = 0; i < E / 2; i++) o[r][i] = fma2(f2(x[r][u], x[r][u]), v[i], o[r][i]);
            }
        }
    }
    __device__ __forceinline__ void finish(float *out, float2 *ml, int rows) {
        const int lane = threadIdx.x & 31, sub = lane % LPK, g = lane / LPK;
        float a[M];
#pragma unroll
        for (int r = 0; r < M; r++) {
            float mx = m[r];
#pragma unroll
            for (int d = LPK; d < 32; d <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
            a[r] = mx == -INFINITY ? 0.f : ex2(m[r] - mx);
            float sum = l[r] * a[r];
#pragma unroll
            for (int d = 1; d < L; d <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
#pragma unroll
            for (int d = LPK; d < 32; d <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
            const int row = SPREAD ? sub / L : r;
            if (g == 0 && row < rows && (SPREAD ? sub % L == 0 : sub == 0)) ml[row] = make_float2(mx, sum);
        }
#pragma unroll
        for (int r = 0; r < R; r++) {
            const float b = SPREAD ? __shfl_sync(0xffffffffu, a[0], g * LPK + r * L) : a[SPREAD ? 0 : r];
#pragma unroll
            for (int i = 0; i < E / 2; i++) {
                float lo, hi;
                f2_split(o[r][i], lo, hi);
                lo *= b;
                hi *= b;
#pragma unroll
                for (int d = LPK; d < 32; d <<= 1) {
                    lo += __shfl_xor_sync(0xffffffffu, lo, d);
                    hi += __shfl_xor_sync(0xffffffffu, hi, d);
                }
                const int dim = i / (W / 2) * (LPK * W) + sub * W + i % (W / 2) * 2;
                if (lane < LPK && r < rows) *reinterpret_cast<float2 *>(out + r * D + dim) = make_float2(lo, hi);
            }
        }
    }
};

}  // namespace prefix
}  // namespace attn
