// norm_rope.cu -- heads of Q and K divided by their root mean square, weighted
// and turned by their positions in one pass: attn_norm_rope_ex,
// attn_norm_rope_bwd_ex and attn_norm_rope_append_ex.
//
// A head x of d elements becomes R (x w r), r = (mean x^2 + eps)^-1/2, R the
// rotation of rope.cu.  With g the gradient of that, turned back (R^T), the
// gradients are
//   dw = sum over tokens and heads of g x r,
//   dx = r (g w - x r^2 mean(g w x)).
// r is formed again from x, which the backward pass reads anyway.
//
// Some 12 flops per element, 30 backward: memory bounds both.  A group of
// lanes takes a few heads of one token and keeps its place in the token's row
// over the tokens that it strides over, so the weights stay where they are, and
// a token's cosines and sines are read once for its heads.  Two kinds of kernels:
//   direct, where the turned part is a multiple of 8 elements (4 in interleaved
//   pairs) and rows are aligned to 4: a lane has both elements of its pairs, in
//   fours, so a head needs no exchange but its sum;
//   exchange, for the rest: a group is the smallest power of two of lanes that
//   covers a head with 16 bytes each, takes kHeads heads, and where the two
//   elements of a pair lie in different lanes, they meet in shared memory.
// Through the exchange kernels the direct ones' cases took 2 to 4 times as long
// (4096 tokens of 12/12 x 128 in fp32 53 us for 19.7, gradients 90 for 35; prompts 607 for 153).
#include <algorithm>

#include "common.cuh"
#include "sm100.cuh"

namespace attn {
namespace nrope {

constexpr int kThreads = 256;
constexpr int kHeads = 4, kHeadsBwd = 2;  // heads of a group
constexpr int kCtas = 2;                  // of kThreads per SM, that the registers leave
// The direct kernels' heads of a group and CTAs per SM.  Forward, 32749 tokens of 32/8 x 128 in bf16 with 4 heads and 3
// CTAs 157 us (153 with inverse_root below), 4 and 4 (spilling) 177, 8 and 2 177, 4 and 2 220; 4096 of 12/12 x 128 in fp32 with 3 and 3 19.7 us,
// 4 and 3 22.2, 2 and 3 20.3.  Backward with the next token's loads on their way while this one's are worked on, 2 CTAs
// (us; without those loads fp32 36.2 and bf16 29.8 where they take 34.1 and 23, with 3 CTAs fp32 55):
//   fp32, 4096 tokens of 12/12 x 128 with 1 head 41, 2 35, 3 42;
//   bf16 in interleaved pairs, 8192 of 16/4 x 64 with 2 heads 30.3, 3 26.9, 4 23.8; 4096 of 32/8 x 128 55, 45.7, 52.4;
//   bf16 in halves, 8192 of 16/4 x 64 24.4, 27.4, 36.7; 4096 of 32/8 x 128 48.6, 41.8, 62; 12/12 x 96 27.1, 25.9, 43.
// (In halves 4 heads spill 136 bytes and 3 16; interleaved none.  32/8 x 128 are 320 threads with 2 heads in halves and
// with 4 interleaved, two CTAs of 256, and 224 or 448 with 3.)
constexpr int direct_heads(size_t element) { return element == 2 ? 4 : 3; }
constexpr int direct_ctas(bool codes) { return codes ? 2 : 3; }
constexpr int direct_heads_bwd(size_t element, bool pairs) { return element == 4 ? 2 : pairs ? 4 : 3; }

struct Params {
    const void *q, *k, *v;                // inputs of the forward pass
    void *q_out, *k_out, *v_out;          // outputs; k_out, v_out: cache bases when slots != NULL
    const void *dq_out, *dk_out;          // backward: gradients of the outputs,
    void *dq, *dk;                        // of the inputs,
    double *partial;                      // and of the weights: [CTA][2][d] (NULL: not wanted)
    const float *q_weight, *k_weight;     // NULL: ones
    const float *table;
    const int *positions;
    const long long *slots;               // NULL: row t of k_out
    float *kscale, *vscale;               // INT8 cache
    int *err;
    long long q_stride, k_stride, v_stride, qo_stride, ko_stride;
    long long rows;                       // cache rows (slots != NULL)
    int tokens, seq_len, d, rot, max_pos, interleaved;
    int heads[3];                         // of q, k and v
    int chunks[3];                        // groups of them
    int lanes, per_token, tokens_per_block;   // lanes of a group; threads of a token
    int threads;                          // of a CTA
    int items, turned;                    // direct kernels: items of a head, those that turn
    float eps, inv_d;
};

// Where a thread works: a token of the block's, a chunk of heads of one
// tensor, a 16-byte vector of a head.
struct Place {
    int token, kind, head, n, item;       // kind: 0 q, 1 k, 2 v; n heads from `head`
    unsigned mask;                        // lanes of the group
    bool there;
};
template <int HEADS>
__device__ __forceinline__ Place place_of(const Params &p, int u) {
    Place x;
    x.token = u / p.per_token;
    const int r = u - x.token * p.per_token;
    int chunk = r / p.lanes;
    x.item = r - chunk * p.lanes;
    x.kind = 0;
    while (x.kind < 2 && chunk >= p.chunks[x.kind]) chunk -= p.chunks[x.kind++];
    x.head = chunk * HEADS;
    x.n = min(HEADS, p.heads[x.kind] - x.head);
    const int first = (threadIdx.x & 31) & ~(p.lanes - 1);
    x.mask = p.lanes == 32 ? 0xffffffffu : ((1u << p.lanes) - 1) << first;
    x.there = x.token < p.tokens_per_block;
    return x;
}

__device__ __forceinline__ bool in_cache(const Params &p, long long row) { return !p.slots || (row >= 0 && row < p.rows); }

// Row of the table of token t; as in rope.cu, a position outside it is
// reported unless the token has no place in the cache.
__device__ __forceinline__ int checked_position(const Params &p, int pos, long long row) {
    if ((unsigned)pos >= (unsigned)p.max_pos) {
        if (in_cache(p, row)) atomicExch(p.err, 0x701);
        pos = pos < 0 ? 0 : p.max_pos - 1;
    }
    return pos;
}
__device__ __forceinline__ int position_of(const Params &p, int t, long long row) {
    return checked_position(p, p.positions ? __ldg(p.positions + t) : t % p.seq_len, row);
}
// Positions of tokens first, first + stride, ...: each one asked for a token
// before its use, and looked at when it is used.
struct Positions {
    int next, step;
    __device__ __forceinline__ Positions(const Params &p, int t, int stride, bool wanted) {
        next = step = 0;
        if (!wanted) return;
        if (p.positions) {
            if (t < p.tokens) next = __ldg(p.positions + t);
        } else {
            next = t % p.seq_len;
            step = stride % p.seq_len;
        }
    }
    // this token's; asks for that of token t
    __device__ __forceinline__ int advance(const Params &p, int t, bool wanted) {
        const int pos = next;
        if (!wanted) return pos;
        if (p.positions) {
            if (t < p.tokens) next = __ldg(p.positions + t);
        } else {
            next += step;
            if (next >= p.seq_len) next -= p.seq_len;
        }
        return pos;
    }
};

// 16 bytes of elements as they lie in memory, and as floats.  WIDE: addresses
// are multiples of 16 bytes; otherwise of an element.
template <typename T, bool WIDE> struct Vec {
    static constexpr int E = 16 / (int)sizeof(T);
    uint4 raw;
    __device__ __forceinline__ void load(const T *p) {
        if constexpr (WIDE) {
            raw = *reinterpret_cast<const uint4 *>(p);
        } else if constexpr (sizeof(T) == 4) {
            const uint32_t *w = reinterpret_cast<const uint32_t *>(p);
            raw = make_uint4(w[0], w[1], w[2], w[3]);
        } else {
            const uint16_t *h = reinterpret_cast<const uint16_t *>(p);
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; i++) w[i] = h[2 * i] | (uint32_t)h[2 * i + 1] << 16;
            raw = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
    __device__ __forceinline__ void store(T *p) const {
        if constexpr (WIDE) {
            *reinterpret_cast<uint4 *>(p) = raw;
        } else {
            const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
            for (int i = 0; i < 4; i++) {
                if constexpr (sizeof(T) == 4) {
                    reinterpret_cast<uint32_t *>(p)[i] = w[i];
                } else {
                    reinterpret_cast<uint16_t *>(p)[2 * i] = (uint16_t)w[i];
                    reinterpret_cast<uint16_t *>(p)[2 * i + 1] = (uint16_t)(w[i] >> 16);
                }
            }
        }
    }
    __device__ __forceinline__ void get(float (&x)[E]) const {
        const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if constexpr (sizeof(T) == 4) {
                x[i] = __uint_as_float(w[i]);
            } else {
                x[2 * i] = __uint_as_float(w[i] << 16);
                x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
            }
        }
    }
    __device__ __forceinline__ void set(const float (&x)[E]) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if constexpr (sizeof(T) == 4) {
                w[i] = __float_as_uint(x[i]);
            } else {
                const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
                w[i] = *reinterpret_cast<const uint32_t *>(&h);
            }
        }
        raw = make_uint4(w[0], w[1], w[2], w[3]);
    }
};

// Sums, and the maximum, over the lanes of a group.
template <int N>
__device__ __forceinline__ void group_sums(float (&v)[N], const Params &p, unsigned mask) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        if (o >= p.lanes) continue;
#pragma unroll
        for (int i = 0; i < N; i++) v[i] += __shfl_xor_sync(mask, v[i], o);
    }
}
__device__ __forceinline__ float group_sum(float v, const Params &p, unsigned mask) {
    float x[1] = {v};
    group_sums(x, p, mask);
    return x[0];
}
__device__ __forceinline__ float group_max(float v, const Params &p, unsigned mask) {
    for (int o = p.lanes >> 1; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(mask, v, o));
    return v;
}
// Codes of E values under a scale (its reciprocal given), packed.
template <int E>
__device__ __forceinline__ uint32_t codes_of(const float (&y)[E], float inv) {
    static_assert(E == 4, "fp32 values");
    uint32_t codes = 0;
#pragma unroll
    for (int i = 0; i < E; i++) {
        const float q = roundf(__fmul_rn(y[i], inv));
        codes |= (uint32_t)(uint8_t)(int8_t)(int)fminf(127.f, fmaxf(-127.f, q)) << 8 * i;
    }
    return codes;
}

// Cosine and signed sine of this thread's elements e0 .. e0 + E - 1 at one
// position: an element becomes x c + s partner.  back: the transpose.
template <int E>
__device__ __forceinline__ void angles(const Params &p, int pos, int e0, bool back, float (&c)[E], float (&s)[E]) {
    const int half = p.rot / 2;
    const float2 *row = reinterpret_cast<const float2 *>(p.table) + (long long)pos * half;
#pragma unroll
    for (int i = 0; i < E; i++) {
        const int e = e0 + i;
        c[i] = s[i] = 0.f;
        if (e >= p.rot) continue;
        const bool second = p.interleaved ? e & 1 : e >= half;
        const float2 cs = __ldg(row + (p.interleaved ? e >> 1 : second ? e - half : e));
        c[i] = cs.x;
        s[i] = second != back ? cs.y : -cs.y;
    }
}
// The E elements turned.  `row`: d floats of shared memory of the group's own,
// element e at (e % E) (d / E) + e / E, so that lanes side by side write, and read
// their partners, at addresses side by side.
template <int E>
__device__ __forceinline__ void turn(const Params &p, int e0, bool there, unsigned mask, float *row, const float (&c)[E],
                                     const float (&s)[E], float (&x)[E]) {
    if (p.interleaved) {
#pragma unroll
        for (int i = 0; i < E; i += 2) {
            if (e0 + i >= p.rot) continue;
            const float a = x[i], b = x[i + 1];
            x[i] = fmaf(a, c[i], s[i] * b);
            x[i + 1] = fmaf(b, c[i + 1], s[i + 1] * a);
        }
        return;
    }
    const int half = p.rot / 2, items = p.d / E;
    __syncwarp(mask);                     // the row's last readers are done
    if (there) {
#pragma unroll
        for (int i = 0; i < E; i++) row[i * items + e0 / E] = x[i];
    }
    __syncwarp(mask);
    if (there) {
#pragma unroll
        for (int i = 0; i < E; i++) {
            const int e = e0 + i, other = e < half ? e + half : e - half;
            if (e < p.rot) x[i] = fmaf(x[i], c[i], s[i] * row[other % E * items + other / E]);
        }
    }
}
// Floats of shared memory from one group's row to the next: in other banks.
__host__ __device__ __forceinline__ int row_pitch(const Params &p) { return p.d + p.lanes; }

// CODES: k and v into an INT8 cache, quantised as quantize_int8_kernel does (kv.cu).
template <typename T, bool WIDE, bool CODES>
__global__ void __launch_bounds__(kThreads, 2)
norm_rope_kernel(const __grid_constant__ Params p)
{
    pdl_begin();                          // launched by launch_pdl
    using V = Vec<T, WIDE>;
    constexpr int E = V::E;
    extern __shared__ float exchange[];   // a row per group
    const Place x = place_of<kHeads>(p, (int)(blockIdx.y * blockDim.x + threadIdx.x));
    if (!x.there) return;
    const int e0 = x.item * E;
    const bool there = e0 < p.d;          // lanes past the head take part in the sums alone
    float *row_buf = exchange + threadIdx.x / p.lanes * row_pitch(p);
    const float *weight = x.kind == 0 ? p.q_weight : p.k_weight;
    float w[E];
#pragma unroll
    for (int i = 0; i < E; i++) w[i] = weight && x.kind < 2 && there ? __ldg(weight + e0 + i) : 1.f;

    const T *from = static_cast<const T *>(x.kind == 0 ? p.q : x.kind == 1 ? p.k : p.v) + x.head * p.d + e0;
    const long long from_stride = x.kind == 0 ? p.q_stride : x.kind == 1 ? p.k_stride : p.v_stride;
    const long long to_stride = x.kind == 0 ? p.qo_stride : p.ko_stride;
    void *to = x.kind == 0 ? p.q_out : x.kind == 1 ? p.k_out : p.v_out;

    for (int t = (int)blockIdx.x * p.tokens_per_block + x.token; t < p.tokens; t += (int)gridDim.x * p.tokens_per_block) {
        const long long slot = p.slots ? __ldg(p.slots + t) : (long long)t;
        if (x.kind > 0 && !in_cache(p, slot)) continue;       // (the whole group)
        V raw[kHeads];
#pragma unroll
        for (int h = 0; h < kHeads; h++)
            if (h < x.n && there) raw[h].load(from + t * from_stride + h * p.d);
        float c[E], s[E];
        const bool turns = x.kind < 2 && p.rot > 0;
        if (turns && there) angles<E>(p, position_of(p, t, slot), e0, false, c, s);
        const long long at = (x.kind == 0 ? (long long)t : slot) * to_stride + x.head * p.d + e0;
        float y[kHeads][E], sum[kHeads];
#pragma unroll
        for (int h = 0; h < kHeads; h++) {
            sum[h] = 0.f;
#pragma unroll
            for (int i = 0; i < E; i++) y[h][i] = 0.f;
            if (h < x.n && there) raw[h].get(y[h]);
#pragma unroll
            for (int i = 0; i < E; i++) sum[h] = fmaf(y[h][i], y[h][i], sum[h]);
        }
#pragma unroll
        for (int h = 0; h < kHeads; h++) {
            if (h >= x.n) break;
            if (x.kind < 2) {
                const float r = __frsqrt_rn(fmaf(group_sum(sum[h], p, x.mask), p.inv_d, p.eps));
#pragma unroll
                for (int i = 0; i < E; i++) y[h][i] *= r * w[i];
                if (turns) turn<E>(p, e0, there, x.mask, row_buf, c, s, y[h]);
            }
            if (CODES && x.kind > 0) {
                float amax = 1e-8f;
#pragma unroll
                for (int i = 0; i < E; i++) amax = fmaxf(amax, fabsf(y[h][i]));
                const float scale = __fdiv_rn(group_max(amax, p, x.mask), 127.0f), inv = __fdiv_rn(1.0f, scale);
                if (!there) continue;
                if constexpr (CODES) *reinterpret_cast<uint32_t *>(static_cast<int8_t *>(to) + at + h * p.d) = codes_of(y[h], inv);
                if (x.item == 0) (x.kind == 1 ? p.kscale : p.vscale)[slot * p.heads[x.kind] + x.head + h] = scale;
            } else if (there) {
                if (x.kind < 2) raw[h].set(y[h]);
                raw[h].store(static_cast<T *>(to) + at + h * p.d);
            }
        }
    }
}

// The weights' gradients are sums over all tokens and heads.  A lane adds up to
// kChain terms of a column in fp32 and then empties them into its group's sums,
// in 64 bits and in shared memory, and so do the CTAs' parts and their sum, so
// the error does not grow with the tokens.  (All but the last sum in fp32: of
// 12/12 x 128 in fp32, 4096 tokens 34.0 us and an error of 1.3e-7 against 64
// bits, 65536 tokens 404 us and 4.3e-7; so 35.2 and 414 us and 7.4e-8 both, of
// which a term's own roundings are some 6e-8.  Chains of 8 terms and parts in
// fp32 34.9 us and 8.4e-8, chains of 2 terms 35.8 us.)
constexpr int kChain = 4;
template <int HEADS> constexpr int chain_tokens() { return kChain / HEADS > 1 ? kChain / HEADS : 1; }
template <int N>
__device__ __forceinline__ void empty_into(double *sums, float (&x)[N]) {
    double2 *at = reinterpret_cast<double2 *>(sums);
#pragma unroll
    for (int i = 0; i < N / 2; i++) {
        double2 y = at[i];
        y.x += x[2 * i];
        y.y += x[2 * i + 1];
        at[i] = y;
        x[2 * i] = x[2 * i + 1] = 0.f;
    }
}

// Each CTA's part of them: the groups' sums of a column, in the order of the
// groups.  sums: d of each group, at their columns.
template <int HEADS>
__device__ __forceinline__ void write_partial(const Params &p, const double *sums) {
    for (int col = threadIdx.x; col < 2 * p.d; col += p.threads) {
        const int kind = col >= p.d, e = col - kind * p.d;
        double sum = 0.;
        for (int u = 0; u < p.threads; u += p.lanes) {
            const Place y = place_of<HEADS>(p, (int)blockIdx.y * p.threads + u);
            if (y.there && y.kind == kind) sum += sums[u / p.lanes * p.d + e];
        }
        p.partial[((long long)blockIdx.y * gridDim.x + blockIdx.x) * 2 * p.d + col] = sum;
    }
}

// Gradients of q and k, and each CTA's part of the weights'.
template <typename T, bool WIDE>
__global__ void __launch_bounds__(kThreads, 2)
norm_rope_bwd_kernel(const __grid_constant__ Params p)
{
    pdl_begin();                          // launched by launch_pdl
    using V = Vec<T, WIDE>;
    constexpr int E = V::E;
    extern __shared__ __align__(16) double sums[];            // of each group, and behind them
    float *exchange = reinterpret_cast<float *>(sums + p.threads / p.lanes * p.d);    // a row per group
    const Place x = place_of<kHeadsBwd>(p, (int)(blockIdx.y * blockDim.x + threadIdx.x));
    const int e0 = x.item * E;
    const bool there = x.there && e0 < p.d;
    float *row_buf = exchange + threadIdx.x / p.lanes * row_pitch(p);
    const float *weight = x.kind == 0 ? p.q_weight : p.k_weight;
    float w[E], dw[E];
#pragma unroll
    for (int i = 0; i < E; i++) {
        w[i] = weight && there ? __ldg(weight + e0 + i) : 1.f;
        dw[i] = 0.f;
    }
    const int in_row = x.head * p.d + e0;
    const T *from = static_cast<const T *>(x.kind == 0 ? p.q : p.k) + in_row;
    const T *grad = static_cast<const T *>(x.kind == 0 ? p.dq_out : p.dk_out) + in_row;
    T *to = static_cast<T *>(x.kind == 0 ? p.dq : p.dk) + in_row;
    const long long stride = x.kind == 0 ? p.q_stride : p.k_stride, grad_stride = x.kind == 0 ? p.qo_stride : p.ko_stride;
    const int last = x.there ? p.tokens : 0;
    double *mine = sums + threadIdx.x / p.lanes * p.d + e0;
    if (there) {
#pragma unroll
        for (int i = 0; i < E; i++) mine[i] = 0.;
    }

    int chain = 0;
    for (int t = (int)blockIdx.x * p.tokens_per_block + x.token; t < last; t += (int)gridDim.x * p.tokens_per_block) {
        V xr[kHeadsBwd], gr[kHeadsBwd];
#pragma unroll
        for (int h = 0; h < kHeadsBwd; h++)
            if (h < x.n && there) {
                xr[h].load(from + t * stride + h * p.d);
                gr[h].load(grad + t * grad_stride + h * p.d);
            }
        float c[E], s[E];
        if (p.rot > 0 && there) angles<E>(p, position_of(p, t, t), e0, true, c, s);
#pragma unroll
        for (int h = 0; h < kHeadsBwd; h++) {
            if (h >= x.n) break;
            float a[E], g[E], square = 0.f, dot = 0.f;
#pragma unroll
            for (int i = 0; i < E; i++) a[i] = g[i] = 0.f;
            if (there) {
                xr[h].get(a);
                gr[h].get(g);
            }
            if (p.rot > 0) turn<E>(p, e0, there, x.mask, row_buf, c, s, g);
#pragma unroll
            for (int i = 0; i < E; i++) {
                square = fmaf(a[i], a[i], square);
                dot = fmaf(g[i] * w[i], a[i], dot);
            }
            square = group_sum(square, p, x.mask);
            dot = group_sum(dot, p, x.mask);
            const float r = __frsqrt_rn(fmaf(square, p.inv_d, p.eps)), back = r * r * (dot * p.inv_d);
            if (there) {
#pragma unroll
                for (int i = 0; i < E; i++) {
                    dw[i] = fmaf(g[i], a[i] * r, dw[i]);
                    a[i] = r * fmaf(a[i], -back, g[i] * w[i]);
                }
                xr[h].set(a);
                xr[h].store(to + t * stride + h * p.d);
            }
        }
        if (p.partial && ++chain == chain_tokens<kHeadsBwd>()) {
            if (there) empty_into(mine, dw);
            chain = 0;
        }
    }
    if (!p.partial) return;
    if (there) empty_into(mine, dw);
    __syncthreads();
    write_partial<kHeadsBwd>(p, sums);
}

// ---------------------------------------------------------------------------
// The direct kernels: both elements of every pair in one lane, so nothing is
// exchanged but the sums.  A lane has four elements of a head (rotation
// interleaved), or four of the first half and the four rot/2 behind them, or
// four that do not turn; the arithmetic is in packed pairs of floats.
// ---------------------------------------------------------------------------
using sm100::f2;
using sm100::f2_split;
using sm100::fma2;
using sm100::mul2;

// Four elements as they lie in memory, and as two packed pairs of floats.
template <typename T> struct Four;
template <> struct Four<float> {
    float4 raw;
    __device__ __forceinline__ void zero() { raw = make_float4(0.f, 0.f, 0.f, 0.f); }
    __device__ __forceinline__ void load(const float *p) { raw = *reinterpret_cast<const float4 *>(p); }
    __device__ __forceinline__ void store(float *p) const { *reinterpret_cast<float4 *>(p) = raw; }
    __device__ __forceinline__ void get(uint64_t (&x)[2]) const { x[0] = f2(raw.x, raw.y); x[1] = f2(raw.z, raw.w); }
    __device__ __forceinline__ void set(const uint64_t (&x)[2]) { f2_split(x[0], raw.x, raw.y); f2_split(x[1], raw.z, raw.w); }
};
template <> struct Four<__nv_bfloat16> {
    uint2 raw;
    __device__ __forceinline__ void zero() { raw = make_uint2(0, 0); }
    __device__ __forceinline__ void load(const __nv_bfloat16 *p) { raw = *reinterpret_cast<const uint2 *>(p); }
    __device__ __forceinline__ void store(__nv_bfloat16 *p) const { *reinterpret_cast<uint2 *>(p) = raw; }
    __device__ __forceinline__ void get(uint64_t (&x)[2]) const {
        x[0] = f2(__uint_as_float(raw.x << 16), __uint_as_float(raw.x & 0xffff0000u));
        x[1] = f2(__uint_as_float(raw.y << 16), __uint_as_float(raw.y & 0xffff0000u));
    }
    __device__ __forceinline__ void set(const uint64_t (&x)[2]) {
        float a, b;
        f2_split(x[0], a, b);
        raw.x = sm100::pack_bf16(a, b);
        f2_split(x[1], a, b);
        raw.y = sm100::pack_bf16(a, b);
    }
};
__device__ __forceinline__ uint64_t swapped(uint64_t x) {
    float a, b;
    f2_split(x, a, b);
    return f2(b, a);
}
__device__ __forceinline__ float sum_of(uint64_t x) {
    float a, b;
    f2_split(x, a, b);
    return a + b;
}
// 1 / sqrt(x).  For fp32 results the approximation (within 2^-22.9) and one step
// of Newton's, within 2^-23 (the rounded one is some 20 instructions); what is
// rounded to bf16 takes the approximation.  Of 0 and infinity as it is.
template <typename T> __device__ __forceinline__ float inverse_root(float x) {
    const float r = rsqrtf(x);
    if constexpr (sizeof(T) == 2) return r;
    const float better = r * fmaf(-0.5f * x * r, r, 1.5f);
    return x > 0.f && x < INFINITY ? better : r;
}

// An item's place in the head, and cosines and sines of its pairs, packed:
// interleaved (c0, c0), (c1, c1) and (-s0, s0), (-s1, s1); in halves c0 c1,
// c2 c3 and s0 s1, s2 s3.
template <bool PAIRS> struct Item {
    int off;                              // of its first element in the head
    bool turns;
    __device__ __forceinline__ Item(const Params &p, int item) {
        turns = item < p.turned;
        off = PAIRS || turns ? item * 4 : p.rot + (item - p.turned) * 4;
    }
    __device__ __forceinline__ void angles(const Params &p, int pos, int item, uint64_t (&c)[2], uint64_t (&s)[2]) const {
        const float4 *row = reinterpret_cast<const float4 *>(p.table + ((long long)pos * (p.rot / 2) + item * (PAIRS ? 2 : 4)) * 2);
        const float4 x = __ldg(row);
        if constexpr (PAIRS) {
            c[0] = f2(x.x, x.x); s[0] = f2(-x.y, x.y);
            c[1] = f2(x.z, x.z); s[1] = f2(-x.w, x.w);
        } else {
            const float4 y = __ldg(row + 1);
            c[0] = f2(x.x, x.z); s[0] = f2(x.y, x.w);
            c[1] = f2(y.x, y.z); s[1] = f2(y.y, y.w);
        }
    }
};
__device__ __forceinline__ uint64_t negated(uint64_t x) { return x ^ 0x8000000080000000ull; }

// Weights of both kinds in shared memory (by all threads, before a barrier).
__device__ __forceinline__ void bring_weights(const Params &p, float (&weights)[2][128]) {
    for (int i = threadIdx.x; i < 2 * p.d; i += (int)blockDim.x) {
        const int kind = i >= p.d, e = i - kind * p.d;
        const float *from = kind ? p.k_weight : p.q_weight;
        weights[kind][e] = from ? __ldg(from + e) : 1.f;
    }
}
__device__ __forceinline__ void pairs_of(const float *p, uint64_t (&x)[2]) {
    const float4 v = *reinterpret_cast<const float4 *>(p);
    x[0] = f2(v.x, v.y);
    x[1] = f2(v.z, v.w);
}

template <typename T, int D, bool PAIRS, bool CODES>
__global__ void __launch_bounds__(kThreads, direct_ctas(CODES))
norm_rope_direct_kernel(const __grid_constant__ Params p)
{
    pdl_begin();                          // launched by launch_pdl
    constexpr int H = direct_heads(sizeof(T));
    __shared__ __align__(16) float weights[2][128];
    bring_weights(p, weights);
    __syncthreads();
    const Place x = place_of<H>(p, (int)(blockIdx.y * blockDim.x + threadIdx.x));
    if (!x.there) return;
    const Item<PAIRS> item(p, x.item);
    const bool there = x.item < p.items, turns = item.turns && x.kind < 2 && there;
    const bool second = !PAIRS && item.turns && there;       // a second vector (V's heads are cut up alike)
    const int half = p.rot / 2, n = there ? x.n : 0;

    const int stride = (int)gridDim.x * p.tokens_per_block;
    int t = (int)blockIdx.x * p.tokens_per_block + x.token;
    const int in_row = x.head * D + item.off;
    const long long from_stride = x.kind == 0 ? p.q_stride : x.kind == 1 ? p.k_stride : p.v_stride;
    const long long to_stride = x.kind == 0 ? p.qo_stride : p.ko_stride;
    const T *src = static_cast<const T *>(x.kind == 0 ? p.q : x.kind == 1 ? p.k : p.v) + in_row + t * from_stride;
    void *to = x.kind == 0 ? p.q_out : x.kind == 1 ? p.k_out : p.v_out;
    Positions positions(p, t, stride, turns);
    long long next_slot = p.slots && t < p.tokens ? __ldg(p.slots + t) : 0;
    for (; t < p.tokens; t += stride, src += stride * from_stride) {
        const long long slot = p.slots ? next_slot : t;
        const bool skip = x.kind > 0 && !in_cache(p, slot);   // (the whole group)
        Four<T> a[H], b[H];
#pragma unroll
        for (int h = 0; h < H; h++) {
            a[h].zero();
            b[h].zero();
            if (h < n && !skip) {
                a[h].load(src + h * D);
                if (second) b[h].load(src + h * D + half);
            }
        }
        if (p.slots && t + stride < p.tokens) next_slot = __ldg(p.slots + t + stride);
        const int pos = positions.advance(p, t + stride, turns);
        if (skip) continue;
        const long long at = (x.kind == 0 ? (long long)t : slot) * to_stride + in_row;
        T *dst = static_cast<T *>(to) + at;
        if (!CODES && x.kind == 2) {
#pragma unroll
            for (int h = 0; h < H; h++)
                if (h < n) {
                    a[h].store(dst + h * D);
                    if (second) b[h].store(dst + h * D + half);
                }
            continue;
        }
        float r[H];
        // The weights go into the angles, for all heads: in halves (u, v) becomes r (u wc - v vs, v vc + u ws), interleaved
        // (u, v) becomes r ((u, v) (wc, vc) + (v, u) (-vs, ws)).
        uint64_t wc[2], vs[2], vc[2], ws[2];
        if (x.kind < 2) {
#pragma unroll
            for (int h = 0; h < H; h++) {
                uint64_t u[2], sum;
                a[h].get(u);
                sum = fma2(u[1], u[1], mul2(u[0], u[0]));
                if constexpr (!PAIRS) {
                    b[h].get(u);
                    sum = fma2(u[1], u[1], fma2(u[0], u[0], sum));
                }
                r[h] = sum_of(sum);
            }
            uint64_t c[2] = {f2(1.f, 1.f), f2(1.f, 1.f)}, s[2] = {0, 0};
            if (turns) item.angles(p, checked_position(p, pos, slot), x.item, c, s);
            const float *weight = weights[x.kind] + (there ? item.off : 0);
            uint64_t w[2];
            pairs_of(weight, w);
            if constexpr (PAIRS) {
#pragma unroll
                for (int i = 0; i < 2; i++) { wc[i] = mul2(w[i], c[i]); vs[i] = mul2(swapped(w[i]), s[i]); }
            } else {
                uint64_t v[2] = {0, 0};
                if (second) pairs_of(weight + half, v);
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    wc[i] = mul2(w[i], c[i]); ws[i] = mul2(w[i], s[i]);
                    vc[i] = mul2(v[i], c[i]); vs[i] = negated(mul2(v[i], s[i]));
                }
            }
            group_sums(r, p, x.mask);
#pragma unroll
            for (int h = 0; h < H; h++) r[h] = inverse_root<T>(fmaf(r[h], p.inv_d, p.eps));
        }
#pragma unroll
        for (int h = 0; h < H; h++) {
            uint64_t u[2], v[2];
            a[h].get(u);
            b[h].get(v);
            if (x.kind < 2) {
                const uint64_t rr = f2(r[h], r[h]);
                if constexpr (PAIRS) {
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        const uint64_t y = mul2(u[i], wc[i]);
                        u[i] = mul2(turns ? fma2(swapped(u[i]), vs[i], y) : y, rr);
                    }
                } else {                  // (what does not turn has no v, and sines of 0)
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        const uint64_t y = u[i], z = v[i];
                        u[i] = mul2(fma2(z, vs[i], mul2(y, wc[i])), rr);
                        v[i] = mul2(fma2(y, ws[i], mul2(z, vc[i])), rr);
                    }
                }
            }
            if constexpr (CODES) {
                if (x.kind > 0) {
                    float y[4], z[4], amax = 1e-8f;
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        f2_split(u[i], y[2 * i], y[2 * i + 1]);
                        f2_split(v[i], z[2 * i], z[2 * i + 1]);
                    }
#pragma unroll
                    for (int i = 0; i < 4; i++) amax = fmaxf(amax, fmaxf(fabsf(y[i]), second ? fabsf(z[i]) : 0.f));
                    const float scale = __fdiv_rn(group_max(amax, p, x.mask), 127.0f), inv = __fdiv_rn(1.0f, scale);
                    if (h >= n) continue;
                    int8_t *codes = static_cast<int8_t *>(to) + at + h * D;
                    *reinterpret_cast<uint32_t *>(codes) = codes_of(y, inv);
                    if (second) *reinterpret_cast<uint32_t *>(codes + half) = codes_of(z, inv);
                    if (x.item == 0) (x.kind == 1 ? p.kscale : p.vscale)[slot * p.heads[x.kind] + x.head + h] = scale;
                    continue;
                }
            }
            if (h < n) {
                a[h].set(u);
                a[h].store(dst + h * D);
                if (second) {
                    b[h].set(v);
                    b[h].store(dst + h * D + half);
                }
            }
        }
    }
}

template <typename T, int D, bool PAIRS>
__global__ void __launch_bounds__(kThreads, kCtas)
norm_rope_bwd_direct_kernel(const __grid_constant__ Params p)
{
    pdl_begin();                          // launched by launch_pdl
    constexpr int H = direct_heads_bwd(sizeof(T), PAIRS);
    extern __shared__ __align__(16) double sums[];            // of each group
    __shared__ __align__(16) float weights[2][128];
    bring_weights(p, weights);
    __syncthreads();
    const Place x = place_of<H>(p, (int)(blockIdx.y * blockDim.x + threadIdx.x));
    const Item<PAIRS> item(p, x.item);
    const bool there = x.there && x.item < p.items, turns = item.turns && there, second = !PAIRS && turns;
    const int half = p.rot / 2, n = there ? x.n : 0;
    const int last = x.there ? p.tokens : 0, stride = (int)gridDim.x * p.tokens_per_block;
    int t = (int)blockIdx.x * p.tokens_per_block + x.token;
    const int in_row = x.head * D + item.off;
    const long long from_stride = x.kind == 0 ? p.q_stride : p.k_stride, grad_stride = x.kind == 0 ? p.qo_stride : p.ko_stride;
    const T *from = static_cast<const T *>(x.kind == 0 ? p.q : p.k) + in_row + t * from_stride;
    const T *grad = static_cast<const T *>(x.kind == 0 ? p.dq_out : p.dk_out) + in_row + t * grad_stride;
    T *to = static_cast<T *>(x.kind == 0 ? p.dq : p.dk) + in_row + t * from_stride;
    uint64_t w[2], v[2] = {0, 0};         // weights of the two vectors
    const float *weight = weights[x.kind & 1] + (there ? item.off : 0);
    pairs_of(weight, w);
    if (second) pairs_of(weight + half, v);
    uint64_t dw[2] = {0, 0}, dv[2] = {0, 0};
    double *mine = sums + threadIdx.x / p.lanes * D + item.off;
    if (there) {
#pragma unroll
        for (int i = 0; i < 4; i++) mine[i] = 0.;
        if (second) {
#pragma unroll
            for (int i = 0; i < 4; i++) mine[half + i] = 0.;
        }
    }
    auto empty = [&] {
        auto into = [&](double *sums, uint64_t (&x)[2]) {
            float y[4];
            f2_split(x[0], y[0], y[1]);
            f2_split(x[1], y[2], y[3]);
            empty_into(sums, y);
            x[0] = x[1] = 0;
        };
        if (there) into(mine, dw);
        if (second) into(mine + half, dv);
    };

    // the next token's loads are on their way while this one's are worked on
    Four<T> next_xa[H], next_xb[H], next_ga[H], next_gb[H];
    Positions positions(p, t, stride, turns && x.there);
    auto bring = [&](int t) {
#pragma unroll
        for (int h = 0; h < H; h++) {
            next_xa[h].zero(); next_xb[h].zero(); next_ga[h].zero(); next_gb[h].zero();
            if (h < n && t < last) {
                next_xa[h].load(from + h * D);
                next_ga[h].load(grad + h * D);
                if (second) {
                    next_xb[h].load(from + h * D + half);
                    next_gb[h].load(grad + h * D + half);
                }
            }
        }
    };
    bring(t);
    while (t < last) {
#pragma unroll 1
        for (int chain = 0; chain < chain_tokens<H>() && t < last; chain++, t += stride, to += stride * from_stride) {
            Four<T> xa[H], xb[H], ga[H], gb[H];
#pragma unroll
            for (int h = 0; h < H; h++) { xa[h] = next_xa[h]; xb[h] = next_xb[h]; ga[h] = next_ga[h]; gb[h] = next_gb[h]; }
            from += stride * from_stride;
            grad += stride * grad_stride;
            const int pos = positions.advance(p, t + stride, turns);
            bring(t + stride);
            uint64_t c[2] = {f2(1.f, 1.f), f2(1.f, 1.f)}, s[2] = {0, 0};
            if (turns) item.angles(p, checked_position(p, pos, t), x.item, c, s);
            // the gradient turned back: in halves (g c + f s, f c - g s), interleaved (g, f) c + (f, g) (s, -s)
            auto back = [&](int h, uint64_t (&g)[2], uint64_t (&f)[2]) {
                ga[h].get(g);
                if constexpr (PAIRS) {
                    if (turns) {
#pragma unroll
                        for (int i = 0; i < 2; i++) g[i] = fma2(swapped(g[i]), negated(s[i]), mul2(g[i], c[i]));
                    }
                } else {
                    gb[h].get(f);
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        const uint64_t y = g[i], z = f[i];
                        g[i] = fma2(z, s[i], mul2(y, c[i]));
                        f[i] = fma2(y, negated(s[i]), mul2(z, c[i]));
                    }
                }
            };
            float sq[2 * H];          // squares; products with the gradient
#pragma unroll
            for (int h = 0; h < H; h++) {
                uint64_t g[2], f[2], u[2];
                back(h, g, f);
                xa[h].get(u);
                uint64_t square = fma2(u[1], u[1], mul2(u[0], u[0]));
                uint64_t dot = fma2(mul2(g[1], w[1]), u[1], mul2(mul2(g[0], w[0]), u[0]));
                if (second) {
                    xb[h].get(u);
                    square = fma2(u[1], u[1], fma2(u[0], u[0], square));
                    dot = fma2(mul2(f[1], v[1]), u[1], fma2(mul2(f[0], v[0]), u[0], dot));
                }
                sq[2 * h] = sum_of(square);
                sq[2 * h + 1] = sum_of(dot);
            }
            group_sums(sq, p, x.mask);
#pragma unroll
            for (int h = 0; h < H; h++) {
                const float r = inverse_root<T>(fmaf(sq[2 * h], p.inv_d, p.eps)), k = -r * r * (sq[2 * h + 1] * p.inv_d);
                if (h >= n) continue;
                const uint64_t rr = f2(r, r), kk = f2(k, k);
                uint64_t g[2], f[2], u[2];
                back(h, g, f);
                xa[h].get(u);
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    dw[i] = fma2(g[i], mul2(u[i], rr), dw[i]);
                    u[i] = mul2(fma2(u[i], kk, mul2(g[i], w[i])), rr);
                }
                xa[h].set(u);
                xa[h].store(to + h * D);
                if (second) {
                    xb[h].get(u);
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        dv[i] = fma2(f[i], mul2(u[i], rr), dv[i]);
                        u[i] = mul2(fma2(u[i], kk, mul2(f[i], v[i])), rr);
                    }
                    xb[h].set(u);
                    xb[h].store(to + h * D + half);
                }
            }
        }
        if (p.partial) empty();
    }
    if (!p.partial) return;
    __syncthreads();
    write_partial<H>(p, sums);
}

// Columns of the CTAs' parts, 32 to a CTA, summed in an order that the sizes alone decide.
__global__ void __launch_bounds__(1024)
norm_weight_kernel(const double *__restrict__ partial, int parts, int d, float *__restrict__ dq_weight,
                   float *__restrict__ dk_weight, int accumulate)
{
    pdl_begin();                          // launched by launch_pdl
    __shared__ double sums[32][33];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, col = (int)blockIdx.x * 32 + lane;
    double sum = 0.0;
    for (int i = warp; i < parts; i += 32) sum += __ldcg(partial + (long long)i * 2 * d + col);
    sums[warp][lane] = sum;
    __syncthreads();
    if (warp) return;
    sum = 0.0;
    for (int i = 0; i < 32; i++) sum += sums[i][lane];
    float *to = col < d ? dq_weight : dk_weight;
    if (!to) return;
    to += col < d ? col : col - d;
    *to = (float)(accumulate ? sum + (double)*to : sum);
}

}  // namespace nrope
}  // namespace attn

namespace attn_host {

int sm_count_here();
using attn::nrope::Params;

namespace {

using attn::nrope::kThreads;

// The shape and its strides (0: dense); tensors by the callers.
Params norm_params(const attn_rope_shape *s, const attn_head_norm *n, const float *table, const int *positions, int k_heads, int v_heads,
                   int *err) {
    Params p = {};
    const long long qw = (long long)s->heads * s->head_dim, kw = (long long)s->kv_heads * s->head_dim;
    p.q_stride = s->q_row_stride ? s->q_row_stride : qw;
    p.k_stride = s->k_row_stride ? s->k_row_stride : kw;
    p.v_stride = s->v_row_stride ? s->v_row_stride : kw;
    p.qo_stride = s->q_out_row_stride ? s->q_out_row_stride : qw;
    p.ko_stride = s->k_out_row_stride ? s->k_out_row_stride : kw;
    p.q_weight = n->q_weight; p.k_weight = n->k_weight; p.eps = n->eps;
    p.inv_d = 1.f / (float)s->head_dim;
    p.table = table; p.positions = positions; p.err = err;
    p.tokens = s->tokens; p.seq_len = s->seq_len; p.d = s->head_dim; p.rot = s->rot_dim; p.max_pos = s->max_pos;
    p.interleaved = s->interleaved;
    p.heads[0] = s->heads; p.heads[1] = k_heads; p.heads[2] = v_heads;
    return p;
}

// Divides a token's row into groups of `heads` heads of `vec` elements a lane;
// CTAs of up to kThreads that are resident, which stride over the tokens
// (.y: slices of a row).
dim3 divide(Params &p, bool direct, int vec, int heads, int ctas) {
    p.turned = p.interleaved ? p.rot / vec : p.rot / 2 / vec;
    p.items = direct && !p.interleaved ? p.turned + (p.d - p.rot) / vec : p.d / vec;
    int groups = 0;
    for (int i = 0; i < 3; i++) groups += p.chunks[i] = (p.heads[i] + heads - 1) / heads;
    p.lanes = 1;
    while (p.lanes < p.items) p.lanes *= 2;
    p.per_token = groups * p.lanes;
    p.tokens_per_block = std::max(1, kThreads / p.per_token);
    p.threads = std::min((p.per_token * p.tokens_per_block + 31) / 32 * 32, kThreads);
    const int slices = (p.per_token + p.threads - 1) / p.threads;
    const int steps = (p.tokens + p.tokens_per_block - 1) / p.tokens_per_block;
    return dim3(std::max(1, std::min(steps, std::max(1, sm_count_here() * (ctas * kThreads / p.threads) / slices))), slices);
}

bool even(const void *ptr) { return ((uintptr_t)ptr & 15) == 0; }
// Addresses and strides that fours of T, and both elements of every pair in one lane, ask for?
template <typename T, size_t N>
bool direct_fits(const Params &p, const void *const (&tensors)[N], const long long (&strides)[5]) {
    for (const void *x : tensors)
        if ((uintptr_t)x % (4 * sizeof(T))) return false;
    for (long long x : strides)
        if (x % 4) return false;
    return even(p.table) && p.rot % (p.interleaved ? 4 : 8) == 0;
}

template <typename T, int D, bool CODES>
cudaError_t launch_direct(const Params &p, dim3 grid, cudaStream_t s) {
    using namespace attn::nrope;
    return launch_pdl(p.interleaved ? norm_rope_direct_kernel<T, D, true, CODES> : norm_rope_direct_kernel<T, D, false, CODES>, grid,
                      dim3(p.threads), 0, s, p);
}
template <typename T, int D>
cudaError_t launch_bwd_direct(const Params &p, dim3 grid, size_t smem, cudaStream_t s) {
    using namespace attn::nrope;
    return launch_pdl(p.interleaved ? norm_rope_bwd_direct_kernel<T, D, true> : norm_rope_bwd_direct_kernel<T, D, false>, grid,
                      dim3(p.threads), smem, s, p);
}

template <typename T, bool CODES>
int launch_forward(Params p, cudaStream_t s) {
    using namespace attn::nrope;
    constexpr int W = 16 / (int)sizeof(T);
    const void *const tensors[] = {p.q, p.k, p.v, p.q_out, p.k_out, p.v_out};
    const long long strides[] = {p.q_stride, p.k_stride, p.v_stride, p.qo_stride, p.ko_stride};
    if (direct_fits<T>(p, tensors, strides)) {
        const dim3 grid = divide(p, true, 4, direct_heads(sizeof(T)), direct_ctas(CODES));
        return check_pdl(p.d == 32   ? launch_direct<T, 32, CODES>(p, grid, s)
                         : p.d == 64 ? launch_direct<T, 64, CODES>(p, grid, s)
                         : p.d == 96 ? launch_direct<T, 96, CODES>(p, grid, s)
                                     : launch_direct<T, 128, CODES>(p, grid, s),
                         "norm_rope_direct_kernel");
    }
    bool wide = true;
    for (const void *x : tensors) wide = wide && even(x);
    for (long long x : strides) wide = wide && x % W == 0;
    const dim3 grid = divide(p, false, W, kHeads, kCtas);
    const size_t smem = (size_t)p.threads / p.lanes * row_pitch(p) * 4;
    return check_pdl(launch_pdl(wide ? norm_rope_kernel<T, true, CODES> : norm_rope_kernel<T, false, CODES>, grid, dim3(p.threads), smem, s, p),
                     "norm_rope_kernel");
}

// *parts: the CTAs' parts of the weights' gradients.
template <typename T>
int launch_backward(Params p, int *parts, cudaStream_t s) {
    using namespace attn::nrope;
    constexpr int W = 16 / (int)sizeof(T);
    const void *const tensors[] = {p.q, p.k, p.dq_out, p.dk_out, p.dq, p.dk};
    const long long strides[] = {p.q_stride, p.k_stride, 0, p.qo_stride, p.ko_stride};
    const bool direct = direct_fits<T>(p, tensors, strides);
    const dim3 grid = divide(p, direct, direct ? 4 : W, direct ? direct_heads_bwd(sizeof(T), p.interleaved) : kHeadsBwd, kCtas);
    *parts = (int)(grid.x * grid.y);
    const size_t smem = (size_t)p.threads / p.lanes * (p.d * 8 + (direct ? 0 : row_pitch(p) * 4));
    if (direct)
        return check_pdl(p.d == 32   ? launch_bwd_direct<T, 32>(p, grid, smem, s)
                         : p.d == 64 ? launch_bwd_direct<T, 64>(p, grid, smem, s)
                         : p.d == 96 ? launch_bwd_direct<T, 96>(p, grid, smem, s)
                                     : launch_bwd_direct<T, 128>(p, grid, smem, s),
                         "norm_rope_bwd_direct_kernel");
    bool wide = true;
    for (const void *x : tensors) wide = wide && even(x);
    for (long long x : strides) wide = wide && x % W == 0;
    return check_pdl(launch_pdl(wide ? norm_rope_bwd_kernel<T, true> : norm_rope_bwd_kernel<T, false>, grid, dim3(p.threads), smem, s, p),
                     "norm_rope_bwd_kernel");
}

}  // namespace

int launch_norm_rope(const attn_rope_shape *s, const attn_head_norm *n, int dtype, const float *table, const int *positions, const void *q,
                     const void *k, void *q_out, void *k_out, int *err, cudaStream_t stream) {
    Params p = norm_params(s, n, table, positions, k ? s->kv_heads : 0, 0, err);
    p.q = q; p.k = k; p.q_out = q_out; p.k_out = k_out;
    return dtype == ATTN_F32 ? launch_forward<float, false>(p, stream) : launch_forward<__nv_bfloat16, false>(p, stream);
}

int launch_norm_rope_append(const attn_rope_shape *s, const attn_head_norm *n, const attn_paged_kv *c, int dtype, const float *table,
                            const int *positions, const long long *slots, const void *q, const void *k, const void *v, void *q_out, int *err,
                            cudaStream_t stream) {
    Params p = norm_params(s, n, table, positions, s->kv_heads, s->kv_heads, err);
    p.q = q; p.k = k; p.v = v; p.q_out = q_out;
    p.k_out = c->k; p.v_out = c->v;
    p.ko_stride = c->row_stride ? c->row_stride : (long long)s->kv_heads * s->head_dim;
    p.slots = slots;
    p.rows = c->rows;
    p.kscale = c->kscale; p.vscale = c->vscale;
    if (c->kv_dtype == ATTN_I8) return launch_forward<float, true>(p, stream);
    return dtype == ATTN_F32 ? launch_forward<float, false>(p, stream) : launch_forward<__nv_bfloat16, false>(p, stream);
}

// The largest of the grids that either type and kernel may take.
size_t norm_rope_bwd_workspace(const attn_rope_shape *s) {
    size_t parts = 1;
    const attn_head_norm n = {};
    for (int i = 0; i < 8; i++) {
        using namespace attn::nrope;
        Params p = norm_params(s, &n, nullptr, nullptr, i & 1 ? s->kv_heads : 0, 0, nullptr);
        const int bytes = i & 2 ? 2 : 4;
        const dim3 grid = i < 4 ? divide(p, true, 4, direct_heads_bwd(bytes, p.interleaved), kCtas) : divide(p, false, 16 / bytes, kHeadsBwd, kCtas);
        parts = std::max(parts, (size_t)grid.x * grid.y);
    }
    return (parts * 2 * s->head_dim * 8 + 255) / 256 * 256;
}

int launch_norm_rope_bwd(const attn_rope_shape *s, const attn_head_norm *n, int dtype, const float *table, const int *positions, const void *q,
                         const void *k, const void *dq_out, const void *dk_out, void *dq, void *dk, float *dq_weight, float *dk_weight,
                         int accumulate, void *ws, int *err, cudaStream_t stream) {
    Params p = norm_params(s, n, table, positions, k ? s->kv_heads : 0, 0, err);
    p.q = q; p.k = k; p.dq_out = dq_out; p.dk_out = dk_out; p.dq = dq; p.dk = dk;
    const bool weights = dq_weight || dk_weight;
    p.partial = weights ? static_cast<double *>(ws) : nullptr;
    int parts = 0;
    if (p.tokens > 0) {
        const int st = dtype == ATTN_F32 ? launch_backward<float>(p, &parts, stream) : launch_backward<__nv_bfloat16>(p, &parts, stream);
        if (st) return st;
    }
    if (!weights) return ATTN_OK;
    return check_pdl(launch_pdl(attn::nrope::norm_weight_kernel, dim3(2 * p.d / 32), dim3(1024), 0, stream, (const double *)p.partial, parts, p.d,
                                dq_weight, dk_weight, accumulate),
                     "norm_weight_kernel");
}

}  // namespace attn_host
