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
// lanes (the smallest power of two that covers a head with 16 bytes each)
// takes kHeads heads of one token and keeps its place in the token's row over
// the tokens that it strides over, so the weights stay in registers, and a
// token's cosines and sines are read once for its heads.  Where the two
// elements of a pair lie in different lanes, they meet in shared memory.
#include <algorithm>

#include "common.cuh"

namespace attn {
namespace nrope {

constexpr int kThreads = 256;
constexpr int kHeads = 4, kHeadsBwd = 2;  // heads of a group
constexpr int kCtas = 2;                  // per SM, that the registers leave
constexpr int direct_ctas(bool pairs) { return pairs ? 3 : 2; }

struct Params {
    const void *q, *k, *v;                // inputs of the forward pass
    void *q_out, *k_out, *v_out;          // outputs; k_out, v_out: cache bases when slots != NULL
    const void *dq_out, *dk_out;          // backward: gradients of the outputs,
    void *dq, *dk;                        // of the inputs,
    float *partial;                       // and of the weights: [CTA][2][d] (NULL: not wanted)
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
__device__ __forceinline__ int position_of(const Params &p, int t, long long row) {
    int pos = p.positions ? __ldg(p.positions + t) : t % p.seq_len;
    if ((unsigned)pos >= (unsigned)p.max_pos) {
        if (in_cache(p, row)) atomicExch(p.err, 0x701);
        pos = pos < 0 ? 0 : p.max_pos - 1;
    }
    return pos;
}

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
// The E elements turned.  `row`: d floats of shared memory of the group's own.
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
    const int half = p.rot / 2;
    __syncwarp(mask);                     // the row's last readers are done
    if (there) {
#pragma unroll
        for (int i = 0; i < E; i++) row[e0 + i] = x[i];
    }
    __syncwarp(mask);
    if (there) {
#pragma unroll
        for (int i = 0; i < E; i++) {
            const int e = e0 + i;
            if (e < p.rot) x[i] = fmaf(x[i], c[i], s[i] * row[e < half ? e + half : e - half]);
        }
    }
}

// CODES: k and v into an INT8 cache, quantised as quantize_int8_kernel does (kv.cu).
template <typename T, bool WIDE, bool CODES>
__global__ void __launch_bounds__(kThreads, 2)
norm_rope_kernel(const __grid_constant__ Params p)
{
    pdl_begin();                          // launched by launch_pdl
    using V = Vec<T, WIDE>;
    constexpr int E = V::E;
    extern __shared__ float exchange[];   // d floats per group
    const Place x = place_of<kHeads>(p, (int)blockIdx.y * kThreads + (int)threadIdx.x);
    if (!x.there) return;
    const int e0 = x.item * E;
    const bool there = e0 < p.d;          // lanes past the head take part in the sums alone
    float *row_buf = exchange + threadIdx.x / p.lanes * p.d;
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

// Each CTA's part of the weights' gradients: the groups' sums of a column, in
// the order of the groups.  sums: d floats of each group, at their columns.
__device__ __forceinline__ void write_partial(const Params &p, const float *sums) {
    for (int col = threadIdx.x; col < 2 * p.d; col += kThreads) {
        const int kind = col >= p.d, e = col - kind * p.d;
        float sum = 0.f;
        for (int u = 0; u < kThreads; u += p.lanes) {
            const Place y = place_of<kHeadsBwd>(p, (int)blockIdx.y * kThreads + u);
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
    extern __shared__ float exchange[];   // d floats per group
    const Place x = place_of<kHeadsBwd>(p, (int)blockIdx.y * kThreads + (int)threadIdx.x);
    const int e0 = x.item * E;
    const bool there = x.there && e0 < p.d;
    float *row_buf = exchange + threadIdx.x / p.lanes * p.d;
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
    }
    if (!p.partial) return;
    __syncthreads();
    if (there) {
#pragma unroll
        for (int i = 0; i < E; i++) row_buf[e0 + i] = dw[i];
    }
    __syncthreads();
    write_partial(p, exchange);
}

// ---------------------------------------------------------------------------
// The direct kernels: both elements of every pair in one lane, so nothing is
// exchanged but the sums.  Rotation in halves: an item is 16 bytes of the first
// half and the 16 bytes rot/2 behind them, or 16 bytes that do not turn;
// interleaved: 16 bytes.
// ---------------------------------------------------------------------------
template <bool PAIRS, int E> struct Item {
    static constexpr int C = PAIRS ? E / 2 : E;               // pairs of an item
    int off;                              // of its first element in the head
    bool turns;
    __device__ __forceinline__ Item(const Params &p, int item) {
        turns = item < p.turned;
        off = PAIRS || turns ? item * E : p.rot + (item - p.turned) * E;
    }
    // cosines and sines of its pairs
    __device__ __forceinline__ void angles(const Params &p, int pos, int item, float (&c)[C], float (&s)[C]) const {
        const float4 *row = reinterpret_cast<const float4 *>(p.table + ((long long)pos * (p.rot / 2) + item * C) * 2);
#pragma unroll
        for (int i = 0; i < C; i += 2) {
            const float4 x = __ldg(row + i / 2);
            c[i] = x.x; s[i] = x.y; c[i + 1] = x.z; s[i + 1] = x.w;
        }
    }
};

template <typename T, bool PAIRS, bool CODES>
__global__ void __launch_bounds__(kThreads, direct_ctas(PAIRS))
norm_rope_direct_kernel(const __grid_constant__ Params p)
{
    pdl_begin();                          // launched by launch_pdl
    using V = Vec<T, true>;
    constexpr int E = V::E, C = Item<PAIRS, E>::C;
    __shared__ float weights[2][128];
    for (int i = threadIdx.x; i < 2 * p.d; i += kThreads) {
        const float *from = i < p.d ? p.q_weight : p.k_weight;
        weights[i >= p.d][i < p.d ? i : i - p.d] = from ? __ldg(from + (i < p.d ? i : i - p.d)) : 1.f;
    }
    __syncthreads();
    const Place x = place_of<kHeads>(p, (int)blockIdx.y * kThreads + (int)threadIdx.x);
    if (!x.there) return;
    const Item<PAIRS, E> item(p, x.item);
    const bool there = x.item < p.items, turns = item.turns && x.kind < 2;
    const int half = p.rot / 2;
    const float *weight = weights[x.kind & 1] + (there ? item.off : 0), *weight2 = weight + (!PAIRS && item.turns ? half : 0);

    const int in_row = x.head * p.d + item.off;
    const T *from = static_cast<const T *>(x.kind == 0 ? p.q : x.kind == 1 ? p.k : p.v) + in_row;
    const long long from_stride = x.kind == 0 ? p.q_stride : x.kind == 1 ? p.k_stride : p.v_stride;
    const long long to_stride = x.kind == 0 ? p.qo_stride : p.ko_stride;
    void *to = x.kind == 0 ? p.q_out : x.kind == 1 ? p.k_out : p.v_out;
    const bool second = !PAIRS && item.turns;                // a second vector (V's heads are cut up alike)

    const int stride = (int)gridDim.x * p.tokens_per_block;
    int t = (int)blockIdx.x * p.tokens_per_block + x.token;
    auto slot_of = [&](int t) { return p.slots && t < p.tokens ? __ldg(p.slots + t) : (long long)t; };
    auto pos_of = [&](int t, long long slot) { return turns && there && t < p.tokens ? position_of(p, t, slot) : 0; };
    long long next_slot = slot_of(t);
    int next_pos = pos_of(t, next_slot);
    for (; t < p.tokens; t += stride) {
        const long long slot = next_slot;
        const int pos = next_pos;
        next_slot = slot_of(t + stride);
        next_pos = pos_of(t + stride, next_slot);
        if (x.kind > 0 && !in_cache(p, slot)) continue;       // (the whole group)
        V a[kHeads], b[kHeads];
        const T *src = from + t * from_stride;
#pragma unroll
        for (int h = 0; h < kHeads; h++) {
            a[h].raw = b[h].raw = make_uint4(0, 0, 0, 0);
            if (h < x.n && there) {
                a[h].load(src + h * p.d);
                if (second) b[h].load(src + h * p.d + half);
            }
        }
        const long long at = (x.kind == 0 ? (long long)t : slot) * to_stride + in_row;
        if (!CODES && x.kind == 2) {
#pragma unroll
            for (int h = 0; h < kHeads; h++)
                if (h < x.n && there) {
                    a[h].store(static_cast<T *>(to) + at + h * p.d);
                    if (second) b[h].store(static_cast<T *>(to) + at + h * p.d + half);
                }
            continue;
        }
        // a pair (u, v) becomes r (u wc - v vs, v vc + u ws): the weights go into the angles, for all heads
        float wc[C], ws[C], vc[C], vs[C];
        if (x.kind < 2) {
            float c[C], s[C];
#pragma unroll
            for (int i = 0; i < C; i++) { c[i] = 1.f; s[i] = 0.f; }
            if (turns && there) item.angles(p, pos, x.item, c, s);
#pragma unroll
            for (int i = 0; i < C; i++) {
                const float w = weight[PAIRS ? 2 * i : i], v = PAIRS ? weight[2 * i + 1] : weight2[i];
                wc[i] = w * c[i]; ws[i] = w * s[i]; vc[i] = v * c[i]; vs[i] = v * s[i];
            }
        }
        float r[kHeads];
        if (x.kind < 2) {
#pragma unroll
            for (int h = 0; h < kHeads; h++) {
                float u[E], v[E];
                a[h].get(u);
                r[h] = 0.f;
#pragma unroll
                for (int i = 0; i < E; i++) r[h] = fmaf(u[i], u[i], r[h]);
                if constexpr (!PAIRS) {
                    b[h].get(v);
#pragma unroll
                    for (int i = 0; i < E; i++) r[h] = fmaf(v[i], v[i], r[h]);
                }
            }
            group_sums(r, p, x.mask);
#pragma unroll
            for (int h = 0; h < kHeads; h++) r[h] = __frsqrt_rn(fmaf(r[h], p.inv_d, p.eps));
        }
#pragma unroll
        for (int h = 0; h < kHeads; h++) {
            if (h >= x.n) break;
            float u[E], v[E];
            a[h].get(u);
            b[h].get(v);
            if (x.kind < 2) {
                if constexpr (PAIRS) {
#pragma unroll
                    for (int i = 0; i < C; i++) {
                        const float y = u[2 * i], z = u[2 * i + 1];
                        u[2 * i] = r[h] * (turns ? fmaf(y, wc[i], -(z * vs[i])) : y * wc[i]);
                        u[2 * i + 1] = r[h] * (turns ? fmaf(z, vc[i], y * ws[i]) : z * vc[i]);
                    }
                } else {                  // (what does not turn has no v, and sines of 0)
#pragma unroll
                    for (int i = 0; i < C; i++) {
                        const float y = u[i], z = v[i];
                        u[i] = r[h] * fmaf(y, wc[i], -(z * vs[i]));
                        v[i] = r[h] * fmaf(z, vc[i], y * ws[i]);
                    }
                }
            }
            if (CODES && x.kind > 0) {
                float amax = 1e-8f;
#pragma unroll
                for (int i = 0; i < E; i++) amax = fmaxf(amax, fabsf(u[i]));
                if (second) {
#pragma unroll
                    for (int i = 0; i < E; i++) amax = fmaxf(amax, fabsf(v[i]));
                }
                const float scale = __fdiv_rn(group_max(amax, p, x.mask), 127.0f), inv = __fdiv_rn(1.0f, scale);
                if constexpr (CODES) {
                    int8_t *dst = static_cast<int8_t *>(to) + at + h * p.d;
                    if (there) *reinterpret_cast<uint32_t *>(dst) = codes_of(u, inv);
                    if (there && second) *reinterpret_cast<uint32_t *>(dst + half) = codes_of(v, inv);
                }
                if (x.item == 0) (x.kind == 1 ? p.kscale : p.vscale)[slot * p.heads[x.kind] + x.head + h] = scale;
            } else if (there) {
                a[h].set(u);
                a[h].store(static_cast<T *>(to) + at + h * p.d);
                if (second) {
                    b[h].set(v);
                    b[h].store(static_cast<T *>(to) + at + h * p.d + half);
                }
            }
        }
    }
}

template <typename T, bool PAIRS>
__global__ void __launch_bounds__(kThreads, 2)
norm_rope_bwd_direct_kernel(const __grid_constant__ Params p)
{
    pdl_begin();                          // launched by launch_pdl
    using V = Vec<T, true>;
    constexpr int E = V::E, C = Item<PAIRS, E>::C;
    extern __shared__ float sums[];       // d floats per group
    __shared__ float weights[2][128];
    for (int i = threadIdx.x; i < 2 * p.d; i += kThreads) {
        const float *from = i < p.d ? p.q_weight : p.k_weight;
        weights[i >= p.d][i < p.d ? i : i - p.d] = from ? __ldg(from + (i < p.d ? i : i - p.d)) : 1.f;
    }
    __syncthreads();
    const Place x = place_of<kHeadsBwd>(p, (int)blockIdx.y * kThreads + (int)threadIdx.x);
    const Item<PAIRS, E> item(p, x.item);
    const bool there = x.there && x.item < p.items, second = !PAIRS && item.turns;
    const int half = p.rot / 2;
    const float *weight = weights[x.kind & 1] + (there ? item.off : 0), *weight2 = weight + (second ? half : 0);
    const int in_row = x.head * p.d + item.off;
    const T *from = static_cast<const T *>(x.kind == 0 ? p.q : p.k) + in_row;
    const T *grad = static_cast<const T *>(x.kind == 0 ? p.dq_out : p.dk_out) + in_row;
    T *to = static_cast<T *>(x.kind == 0 ? p.dq : p.dk) + in_row;
    const long long from_stride = x.kind == 0 ? p.q_stride : p.k_stride, grad_stride = x.kind == 0 ? p.qo_stride : p.ko_stride;
    const int last = x.there ? p.tokens : 0;
    float dw[E], dv[E];                   // of the item's first and second vector
#pragma unroll
    for (int i = 0; i < E; i++) dw[i] = dv[i] = 0.f;

    const int stride = (int)gridDim.x * p.tokens_per_block;
    int t = (int)blockIdx.x * p.tokens_per_block + x.token;
    auto pos_of = [&](int t) { return item.turns && there && t < last ? position_of(p, t, t) : 0; };
    int next_pos = pos_of(t);
    for (; t < last; t += stride) {
        const int pos = next_pos;
        next_pos = pos_of(t + stride);
        V xa[kHeadsBwd], xb[kHeadsBwd], ga[kHeadsBwd], gb[kHeadsBwd];
#pragma unroll
        for (int h = 0; h < kHeadsBwd; h++) {
            xa[h].raw = xb[h].raw = ga[h].raw = gb[h].raw = make_uint4(0, 0, 0, 0);
            if (h < x.n && there) {
                xa[h].load(from + t * from_stride + h * p.d);
                ga[h].load(grad + t * grad_stride + h * p.d);
                if (second) {
                    xb[h].load(from + t * from_stride + h * p.d + half);
                    gb[h].load(grad + t * grad_stride + h * p.d + half);
                }
            }
        }
        float c[C], s[C];
#pragma unroll
        for (int i = 0; i < C; i++) { c[i] = 1.f; s[i] = 0.f; }
        if (item.turns && there) item.angles(p, pos, x.item, c, s);
        // the gradient turned back: (g c + g' s, g' c - g s)
        auto back = [&](const V &ra, const V &rb, float (&g)[E], float (&f)[E]) {
            ra.get(g);
            if constexpr (PAIRS) {
                if (item.turns) {
#pragma unroll
                    for (int i = 0; i < C; i++) {
                        const float y = g[2 * i], z = g[2 * i + 1];
                        g[2 * i] = fmaf(y, c[i], z * s[i]);
                        g[2 * i + 1] = fmaf(z, c[i], -(y * s[i]));
                    }
                }
            } else {
                rb.get(f);
#pragma unroll
                for (int i = 0; i < C; i++) {
                    const float y = g[i], z = f[i];
                    g[i] = fmaf(y, c[i], z * s[i]);
                    f[i] = fmaf(z, c[i], -(y * s[i]));
                }
            }
        };
        float sq[2 * kHeadsBwd];          // squares; products with the gradient
#pragma unroll
        for (int h = 0; h < kHeadsBwd; h++) {
            float u[E], v[E], g[E], f[E];
            back(ga[h], gb[h], g, f);
            xa[h].get(u);
            float square = 0.f, dot = 0.f;
#pragma unroll
            for (int i = 0; i < E; i++) {
                square = fmaf(u[i], u[i], square);
                dot = fmaf(g[i] * weight[i], u[i], dot);
            }
            if constexpr (!PAIRS) {
                xb[h].get(v);
                if (second) {
#pragma unroll
                    for (int i = 0; i < E; i++) {
                        square = fmaf(v[i], v[i], square);
                        dot = fmaf(f[i] * weight2[i], v[i], dot);
                    }
                }
            }
            sq[2 * h] = square;
            sq[2 * h + 1] = dot;
        }
        group_sums(sq, p, x.mask);
#pragma unroll
        for (int h = 0; h < kHeadsBwd; h++) {
            if (h >= x.n || !there) break;
            const float r = __frsqrt_rn(fmaf(sq[2 * h], p.inv_d, p.eps)), k = r * r * (sq[2 * h + 1] * p.inv_d);
            float u[E], v[E], g[E], f[E];
            back(ga[h], gb[h], g, f);
            xa[h].get(u);
#pragma unroll
            for (int i = 0; i < E; i++) {
                dw[i] = fmaf(g[i], u[i] * r, dw[i]);
                u[i] = r * fmaf(u[i], -k, g[i] * weight[i]);
            }
            xa[h].set(u);
            xa[h].store(to + t * from_stride + h * p.d);
            if (second) {
                xb[h].get(v);
#pragma unroll
                for (int i = 0; i < E; i++) {
                    dv[i] = fmaf(f[i], v[i] * r, dv[i]);
                    v[i] = r * fmaf(v[i], -k, f[i] * weight2[i]);
                }
                xb[h].set(v);
                xb[h].store(to + t * from_stride + h * p.d + half);
            }
        }
    }
    if (!p.partial) return;
    if (there) {
        float *mine = sums + threadIdx.x / p.lanes * p.d + item.off;
#pragma unroll
        for (int i = 0; i < E; i++) {
            mine[i] = dw[i];
            if (second) mine[half + i] = dv[i];
        }
    }
    __syncthreads();
    write_partial(p, sums);
}

// Columns of the CTAs' parts, 32 to a CTA, summed in an order that the sizes alone decide.
__global__ void __launch_bounds__(1024)
norm_weight_kernel(const float *__restrict__ partial, int parts, int d, float *__restrict__ dq_weight,
                   float *__restrict__ dk_weight, int accumulate)
{
    pdl_begin();                          // launched by launch_pdl
    __shared__ double sums[32][33];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, col = (int)blockIdx.x * 32 + lane;
    double sum = 0.0;
    for (int i = warp; i < parts; i += 32) sum += (double)__ldcg(partial + (long long)i * 2 * d + col);
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
// CTAs that are resident, which stride over the tokens (.y: slices of a row).
dim3 divide(Params &p, bool direct, int vec, int heads, int ctas) {
    p.turned = p.interleaved ? p.rot / vec : p.rot / 2 / vec;
    p.items = direct && !p.interleaved ? p.turned + (p.d - p.rot) / vec : p.d / vec;
    int groups = 0;
    for (int i = 0; i < 3; i++) groups += p.chunks[i] = (p.heads[i] + heads - 1) / heads;
    p.lanes = 1;
    while (p.lanes < p.items) p.lanes *= 2;
    p.per_token = groups * p.lanes;
    p.tokens_per_block = std::max(1, kThreads / p.per_token);
    const int slices = (p.per_token + kThreads - 1) / kThreads;
    const int steps = (p.tokens + p.tokens_per_block - 1) / p.tokens_per_block;
    return dim3(std::max(1, std::min(steps, std::max(1, sm_count_here() * ctas / slices))), slices);
}

bool even(const void *ptr) { return ((uintptr_t)ptr & 15) == 0; }
// Both elements of every pair in one lane's vectors?
bool direct_fits(const Params &p, bool wide, int vec) { return wide && even(p.table) && p.rot % (p.interleaved ? vec : 2 * vec) == 0; }

template <typename T, bool CODES>
int launch_forward(Params p, cudaStream_t s) {
    using namespace attn::nrope;
    constexpr int W = 16 / (int)sizeof(T);
    const bool wide = even(p.q) && even(p.k) && even(p.v) && even(p.q_out) && even(p.k_out) && even(p.v_out) && p.q_stride % W == 0 &&
                      p.k_stride % W == 0 && p.v_stride % W == 0 && p.qo_stride % W == 0 && p.ko_stride % W == 0;
    const bool direct = direct_fits(p, wide, W);
    const dim3 grid = divide(p, direct, W, kHeads, direct ? direct_ctas(p.interleaved) : kCtas);
    if (direct)
        return check_pdl(launch_pdl(p.interleaved ? norm_rope_direct_kernel<T, true, CODES> : norm_rope_direct_kernel<T, false, CODES>, grid,
                                    dim3(kThreads), 0, s, p),
                         "norm_rope_direct_kernel");
    const size_t smem = (size_t)kThreads / p.lanes * p.d * 4;
    return check_pdl(launch_pdl(wide ? norm_rope_kernel<T, true, CODES> : norm_rope_kernel<T, false, CODES>, grid, dim3(kThreads), smem, s, p),
                     "norm_rope_kernel");
}

// *parts: the CTAs' parts of the weights' gradients.
template <typename T>
int launch_backward(Params p, int *parts, cudaStream_t s) {
    using namespace attn::nrope;
    constexpr int W = 16 / (int)sizeof(T);
    const bool wide = even(p.q) && even(p.k) && even(p.dq_out) && even(p.dk_out) && even(p.dq) && even(p.dk) && p.q_stride % W == 0 &&
                      p.k_stride % W == 0 && p.qo_stride % W == 0 && p.ko_stride % W == 0;
    const bool direct = direct_fits(p, wide, W);
    const dim3 grid = divide(p, direct, W, kHeadsBwd, kCtas);
    *parts = (int)(grid.x * grid.y);
    const size_t smem = (size_t)kThreads / p.lanes * p.d * 4;
    if (direct)
        return check_pdl(launch_pdl(p.interleaved ? norm_rope_bwd_direct_kernel<T, true> : norm_rope_bwd_direct_kernel<T, false>, grid,
                                    dim3(kThreads), smem, s, p),
                         "norm_rope_bwd_direct_kernel");
    return check_pdl(launch_pdl(wide ? norm_rope_bwd_kernel<T, true> : norm_rope_bwd_kernel<T, false>, grid, dim3(kThreads), smem, s, p),
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
        Params p = norm_params(s, &n, nullptr, nullptr, i & 4 ? s->kv_heads : 0, 0, nullptr);
        const dim3 grid = divide(p, i & 2, i & 1 ? 8 : 4, attn::nrope::kHeadsBwd, attn::nrope::kCtas);
        parts = std::max(parts, (size_t)grid.x * grid.y);
    }
    return (parts * 2 * s->head_dim * 4 + 255) / 256 * 256;
}

int launch_norm_rope_bwd(const attn_rope_shape *s, const attn_head_norm *n, int dtype, const float *table, const int *positions, const void *q,
                         const void *k, const void *dq_out, const void *dk_out, void *dq, void *dk, float *dq_weight, float *dk_weight,
                         int accumulate, void *ws, int *err, cudaStream_t stream) {
    Params p = norm_params(s, n, table, positions, k ? s->kv_heads : 0, 0, err);
    p.q = q; p.k = k; p.dq_out = dq_out; p.dk_out = dk_out; p.dq = dq; p.dk = dk;
    const bool weights = dq_weight || dk_weight;
    p.partial = weights ? static_cast<float *>(ws) : nullptr;
    int parts = 0;
    if (p.tokens > 0) {
        const int st = dtype == ATTN_F32 ? launch_backward<float>(p, &parts, stream) : launch_backward<__nv_bfloat16>(p, &parts, stream);
        if (st) return st;
    }
    if (!weights) return ATTN_OK;
    return check_pdl(launch_pdl(attn::nrope::norm_weight_kernel, dim3(2 * p.d / 32), dim3(1024), 0, stream, (const float *)p.partial, parts, p.d,
                                dq_weight, dk_weight, accumulate),
                     "norm_weight_kernel");
}

}  // namespace attn_host
