// rope.cu -- rotary positions: attn_rope_ex (training forward and gradient),
// attn_rope_append_ex (serving: K turned and V copied into a paged cache) and
// attn_rope_table_ex.
//
// A pair (a, b) of a head becomes (a cos - b sin, b cos + a sin), the product
// of a + ib with cos + i sin; its transpose, which carries gradients back, is
// the same with -sin.  The work is 6 flops per pair, so memory bounds it: q, k
// (and v) are read once and written once, and a token's row of the table is
// read by the few threads that hold its pairs.
//
// A thread owns one vector position within a head (E elements and, in the
// halves layout, the E elements rot/2 behind them) for kHeads heads: it reads
// a token's cosines and sines once for all of them, and its loads are issued
// together and kept as they come until their turn, so that the 768 threads
// of an SM hold 128 bytes each in flight.  It keeps its place in the token's row
// and strides over the tokens, the next token's position and slot read ahead.
// Consecutive threads take consecutive vectors, so a head's row goes out in
// full sectors.
#include <algorithm>

#include "common.cuh"

namespace attn {
namespace rope {

constexpr int kThreads = 256;
// Heads per thread, and CTAs per SM that its registers leave.  32749 tokens of
// 32/8 heads of 128 in bf16 (822 MB): 136 us, 6.06 TB/s; with 2 heads and 4
// CTAs 150 us, with 4 and 2 157 us, 1 and 8 (spilling) 343 us.  64 tokens of
// 16 heads of 64 in fp32 go the other way: 3.3 us, and 2.9 with 2 heads.
constexpr int kHeads = 4;
constexpr int ctas_of(bool pairs) { return pairs ? 4 : 3; }

struct Params {
    const void *q, *k, *v;
    void *q_out, *k_out, *v_out;          // k_out, v_out: cache bases when slots != NULL
    const float *table;
    const int *positions;
    const long long *slots;               // NULL: row t of k_out
    int *err;
    long long q_stride, k_stride, v_stride, qo_stride, ko_stride;
    long long rows;                       // cache rows (slots != NULL)
    int tokens, seq_len, d, rot, max_pos;
    int q_heads, all_heads, kv_heads;     // heads [0, q_heads) q, then kv_heads of k, then of v
    int items, per_token, tokens_per_block;   // vectors of a head; threads of a token
    float sign;                           // -1: transpose
};

// Does a slot lie in the cache?  (Without a slot map every token has its row.)
__device__ __forceinline__ bool in_cache(const Params &p, long long row) { return !p.slots || (row >= 0 && row < p.rows); }

// Row of the table of token t.  A position outside it is reported, unless the
// token has no place in the cache (slot `row`): a request that the page plan
// refuses at its table's end asks for just such positions.
__device__ __forceinline__ int position_of(const Params &p, int t, long long row) {
    int pos = p.positions ? __ldg(p.positions + t) : t % p.seq_len;
    if ((unsigned)pos >= (unsigned)p.max_pos) {
        if (in_cache(p, row)) atomicExch(p.err, 0x701);
        pos = pos < 0 ? 0 : p.max_pos - 1;
    }
    return pos;
}

__device__ __forceinline__ void turn(float &a, float &b, float c, float s) {
    const float x = fmaf(a, c, -(b * s));
    b = fmaf(b, c, a * s);
    a = x;
}

// E elements as they lie in memory, and as floats.
template <typename T, int E> struct Vec {           // one or two elements, of any alignment
    T raw[E];
    __device__ __forceinline__ void load(const T *p) {
#pragma unroll
        for (int i = 0; i < E; i++) raw[i] = p[i];
    }
    __device__ __forceinline__ void store(T *p) const {
#pragma unroll
        for (int i = 0; i < E; i++) p[i] = raw[i];
    }
    __device__ __forceinline__ void get(float (&x)[E]) const {
#pragma unroll
        for (int i = 0; i < E; i++) x[i] = to_f32(raw[i]);
    }
    __device__ __forceinline__ void set(const float (&x)[E]) {
#pragma unroll
        for (int i = 0; i < E; i++) raw[i] = from_f32<T>(x[i]);
    }
};
template <> struct Vec<float, 4> {
    float4 raw;
    __device__ __forceinline__ void load(const float *p) { raw = *reinterpret_cast<const float4 *>(p); }
    __device__ __forceinline__ void store(float *p) const { *reinterpret_cast<float4 *>(p) = raw; }
    __device__ __forceinline__ void get(float (&x)[4]) const { x[0] = raw.x; x[1] = raw.y; x[2] = raw.z; x[3] = raw.w; }
    __device__ __forceinline__ void set(const float (&x)[4]) { raw = make_float4(x[0], x[1], x[2], x[3]); }
};
template <> struct Vec<__nv_bfloat16, 8> {
    uint4 raw;
    __device__ __forceinline__ void load(const __nv_bfloat16 *p) { raw = *reinterpret_cast<const uint4 *>(p); }
    __device__ __forceinline__ void store(__nv_bfloat16 *p) const { *reinterpret_cast<uint4 *>(p) = raw; }
    __device__ __forceinline__ void get(float (&x)[8]) const {
        const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            x[2 * i] = __uint_as_float(w[i] << 16);
            x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
    __device__ __forceinline__ void set(const float (&x)[8]) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t *>(&h);
        }
        raw = make_uint4(w[0], w[1], w[2], w[3]);
    }
};

// E elements per vector: 16 bytes, or 1 (halves) and 2 (interleaved pairs)
// where an address, a stride or rot is not a multiple of that.
template <typename T, int E, bool PAIRS>
__global__ void __launch_bounds__(kThreads, ctas_of(PAIRS))
rope_kernel(const __grid_constant__ Params p)
{
    pdl_begin();                          // launched by launch_pdl
    using V = Vec<T, E>;
    const int half = p.rot / 2;
    const int turned = PAIRS ? p.rot / E : half / E;        // items of a head that turn
    // this thread's place: a token of the block's, a group of heads, a vector of a head
    const int u = blockIdx.y * kThreads + threadIdx.x;
    const int tl = u / p.per_token, r = u - tl * p.per_token;
    if (tl >= p.tokens_per_block) return;
    const int chunk = r / p.items, item = r - chunk * p.items;
    const bool turns = item < turned;
    const int off = PAIRS || turns ? item * E : p.rot + (item - turned) * E;
    constexpr int C = PAIRS ? (E + 1) / 2 : E;              // pairs of this item

    const int stride = (int)gridDim.x * p.tokens_per_block;
    int t = (int)blockIdx.x * p.tokens_per_block + tl;
    auto slot = [&](int t) { return p.slots && t < p.tokens ? __ldg(p.slots + t) : (long long)t; };
    auto position = [&](int t, long long row) { return turns && t < p.tokens ? position_of(p, t, row) : 0; };
    long long next_row = slot(t);
    int next_pos = position(t, next_row);
    for (; t < p.tokens; t += stride) {
        const int pos = next_pos;
        const long long row = in_cache(p, next_row) ? next_row : -1;
        next_row = slot(t + stride);
        next_pos = position(t + stride, next_row);
        float c[C], s[C];
        if (turns) {
            const float *cs = p.table + ((long long)pos * half + item * C) * 2;
            if constexpr (C % 2 == 0) {
#pragma unroll
                for (int i = 0; i < C; i += 2) {
                    const float4 x = __ldg(reinterpret_cast<const float4 *>(cs + 2 * i));
                    c[i] = x.x; s[i] = x.y * p.sign; c[i + 1] = x.z; s[i + 1] = x.w * p.sign;
                }
            } else {
#pragma unroll
                for (int i = 0; i < C; i++) {
                    const float2 x = __ldg(reinterpret_cast<const float2 *>(cs + 2 * i));
                    c[i] = x.x; s[i] = x.y * p.sign;
                }
            }
        }
        V a[kHeads], b[kHeads];
        T *dst[kHeads];
#pragma unroll
        for (int i = 0; i < kHeads; i++) {
            const int h = chunk * kHeads + i;
            dst[i] = nullptr;
            if (h >= p.all_heads) continue;
            const T *src;
            if (h < p.q_heads) {
                src = static_cast<const T *>(p.q) + t * p.q_stride + h * p.d + off;
                dst[i] = static_cast<T *>(p.q_out) + t * p.qo_stride + h * p.d + off;
            } else {
                if (row < 0) continue;
                const int hk = h - p.q_heads;
                if (hk < p.kv_heads) {
                    src = static_cast<const T *>(p.k) + t * p.k_stride + hk * p.d + off;
                    dst[i] = static_cast<T *>(p.k_out) + row * p.ko_stride + hk * p.d + off;
                } else {
                    src = static_cast<const T *>(p.v) + t * p.v_stride + (hk - p.kv_heads) * p.d + off;
                    dst[i] = static_cast<T *>(p.v_out) + row * p.ko_stride + (hk - p.kv_heads) * p.d + off;
                }
            }
            a[i].load(src);
            if (!PAIRS && turns) b[i].load(src + half);
        }
#pragma unroll
        for (int i = 0; i < kHeads; i++) {
            if (!dst[i]) continue;
            if (turns && chunk * kHeads + i < p.q_heads + p.kv_heads) {
                float x[E], y[E];
                a[i].get(x);
                if constexpr (PAIRS) {
#pragma unroll
                    for (int e = 0; e + 1 < E; e += 2) turn(x[e], x[e + 1], c[e / 2], s[e / 2]);
                } else {
                    b[i].get(y);
#pragma unroll
                    for (int e = 0; e < E; e++) turn(x[e], y[e], c[e], s[e]);
                    b[i].set(y);
                }
                a[i].set(x);
            }
            a[i].store(dst[i]);
            if (!PAIRS && turns) b[i].store(dst[i] + half);
        }
    }
}

// K turned and V as it is into an INT8 cache: one warp per (token, head) and
// tensor, quantised as quantize_int8_kernel does (kv.cu).
template <int D>
__global__ void __launch_bounds__(kThreads)
rope_append_i8_kernel(const __grid_constant__ Params p, int interleaved, float *__restrict__ kscale,
                      float *__restrict__ vscale)
{
    pdl_begin();                          // launched by launch_pdl
    constexpr int E = D / 32;
    const long long unit = (long long)blockIdx.x * (kThreads / 32) + threadIdx.x / 32;
    const int lane = threadIdx.x & 31;
    const int per_token = 2 * p.kv_heads;
    const int t = (int)(unit / per_token);
    if (t >= p.tokens) return;
    const int r = (int)(unit % per_token), h = r % p.kv_heads;
    const bool is_v = r >= p.kv_heads;
    const long long row = __ldg(p.slots + t);
    if (!in_cache(p, row)) return;
    const float *src = is_v ? static_cast<const float *>(p.v) + t * p.v_stride + (long long)h * D
                            : static_cast<const float *>(p.k) + t * p.k_stride + (long long)h * D;
    const int half = p.rot / 2;
    const int pos = is_v || !p.rot ? 0 : position_of(p, t, row);
    float x[E];
    float amax = 1e-8f;
#pragma unroll
    for (int i = 0; i < E; i++) {
        const int e = lane + 32 * i;
        x[i] = src[e];
        if (!is_v && e < p.rot) {
            const int pair = interleaved ? e >> 1 : e % half;
            const bool second = interleaved ? (e & 1) : e >= half;
            const float2 cs = __ldg(reinterpret_cast<const float2 *>(p.table) + (long long)pos * half + pair);
            float a = second ? src[interleaved ? e - 1 : e - half] : x[i];
            float b = second ? x[i] : src[interleaved ? e + 1 : e + half];
            turn(a, b, cs.x, cs.y);
            x[i] = second ? b : a;
        }
        amax = fmaxf(amax, fabsf(x[i]));
    }
    amax = warp_max(amax);
    const float scale = __fdiv_rn(amax, 127.0f);
    const float inv = __fdiv_rn(1.0f, scale);
    int8_t *dst = static_cast<int8_t *>(is_v ? p.v_out : p.k_out) + row * p.ko_stride + (long long)h * D;
#pragma unroll
    for (int i = 0; i < E; i++) {
        const float c = roundf(__fmul_rn(x[i], inv));
        dst[lane + 32 * i] = (int8_t)(int)fminf(127.f, fmaxf(-127.f, c));
    }
    if (lane == 0) (is_v ? vscale : kscale)[row * p.kv_heads + h] = scale;
}

// cos and sin of position x frequency.  The angle is formed and reduced in
// fp64: in fp32 a position of 10^5 leaves it 4e-3 off.
__global__ void rope_table_kernel(const attn_rope_config c, double low, double high, float2 *__restrict__ table)
{
    const int half = c.rot_dim / 2;
    const long long n = (long long)c.max_pos * half;
    for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (long long)gridDim.x * blockDim.x) {
        const int pair = (int)(i % half);
        double f = pow(c.base, -2.0 * pair / c.rot_dim);
        if (c.scaling == ATTN_ROPE_LINEAR) f /= c.factor;
        if (c.scaling == ATTN_ROPE_RAMP) {
            // share of the interpolated frequency: 0 up to pair `low`, 1 from pair `high`
            const double w = fmin(1.0, fmax(0.0, (pair - low) / (high - low)));
            f = f * (1.0 - w) + f / c.factor * w;
        }
        double s, co;
        sincos((double)(i / half) * f, &s, &co);
        table[i] = make_float2((float)(co * c.magnitude), (float)(s * c.magnitude));
    }
}

}  // namespace rope
}  // namespace attn

namespace attn_host {

int sm_count_here();

int launch_rope_table(const attn_rope_config *c, float *table, cudaStream_t s) {
    attn_rope_config k = *c;
    double low = 0, high = 1;
    if (k.scaling == ATTN_ROPE_BASE) k.base *= pow(k.factor, (double)k.rot_dim / (k.rot_dim - 2));
    if (k.scaling == ATTN_ROPE_RAMP) {
        // pair i turns trained_len * base^(-2i/rot) / 2 pi times within the trained context; solved for i
        auto pair_of = [&](double turns) {
            return k.rot_dim * log(k.trained_len / (turns * 2.0 * 3.14159265358979323846)) / (2.0 * log(k.base));
        };
        low = pair_of(k.fast);
        high = pair_of(k.slow);
    }
    if (k.magnitude == 0.0) k.magnitude = 1.0;
    const long long n = (long long)k.max_pos * (k.rot_dim / 2);
    const unsigned blocks = (unsigned)std::min<long long>((n + 255) / 256, 148LL * 8);
    attn::rope::rope_table_kernel<<<blocks, 256, 0, s>>>(k, low, high, reinterpret_cast<float2 *>(table));
    return check_launch("rope_table_kernel");
}

template <typename T>
static int launch_rope_typed(attn::rope::Params p, bool interleaved, cudaStream_t s) {
    using namespace attn::rope;
    constexpr int W = 16 / (int)sizeof(T);
    // 16-byte vectors where every address, stride and part of a head allows them
    auto even = [](const void *ptr) { return ((uintptr_t)ptr & 15) == 0; };
    const bool wide = p.rot % (interleaved ? W : 2 * W) == 0 && even(p.q) && even(p.k) && even(p.v) && even(p.q_out) &&
                      even(p.k_out) && even(p.v_out) && even(p.table) && p.q_stride % W == 0 && p.k_stride % W == 0 &&
                      p.v_stride % W == 0 && p.qo_stride % W == 0 && p.ko_stride % W == 0;
    const int E = wide ? W : interleaved ? 2 : 1;
    p.items = interleaved ? p.d / E : p.rot / 2 / E + (p.d - p.rot) / E;
    p.per_token = p.items * ((p.all_heads + kHeads - 1) / kHeads);
    p.tokens_per_block = std::max(1, kThreads / p.per_token);
    // as many CTAs as are resident, which stride over the tokens
    const int slices = (p.per_token + kThreads - 1) / kThreads;
    const int groups = (p.tokens + p.tokens_per_block - 1) / p.tokens_per_block;
    const dim3 grid(std::min(groups, std::max(1, sm_count_here() * ctas_of(interleaved) / slices)), slices);
    cudaError_t e;
    if (interleaved)
        e = wide ? launch_pdl(rope_kernel<T, W, true>, grid, dim3(kThreads), 0, s, p)
                 : launch_pdl(rope_kernel<T, 2, true>, grid, dim3(kThreads), 0, s, p);
    else
        e = wide ? launch_pdl(rope_kernel<T, W, false>, grid, dim3(kThreads), 0, s, p)
                 : launch_pdl(rope_kernel<T, 1, false>, grid, dim3(kThreads), 0, s, p);
    return check_pdl(e, "rope_kernel");
}

// Fills the strides that are 0 (dense) and the shape; q, k and outputs by the callers.
static attn::rope::Params rope_params(const attn_rope_shape *s, const float *table, const int *positions, int *err) {
    attn::rope::Params p = {};
    const long long qw = (long long)s->heads * s->head_dim, kw = (long long)s->kv_heads * s->head_dim;
    p.q_stride = s->q_row_stride ? s->q_row_stride : qw;
    p.k_stride = s->k_row_stride ? s->k_row_stride : kw;
    p.v_stride = s->v_row_stride ? s->v_row_stride : kw;
    p.qo_stride = s->q_out_row_stride ? s->q_out_row_stride : qw;
    p.ko_stride = s->k_out_row_stride ? s->k_out_row_stride : kw;
    p.table = table; p.positions = positions; p.err = err;
    p.tokens = s->tokens; p.seq_len = s->seq_len; p.d = s->head_dim; p.rot = s->rot_dim; p.max_pos = s->max_pos;
    p.q_heads = s->heads; p.kv_heads = s->kv_heads;
    p.sign = 1.f;
    return p;
}

int launch_rope(const attn_rope_shape *s, int dtype, const float *table, const int *positions, const void *q,
                const void *k, void *q_out, void *k_out, int transpose, int *err, cudaStream_t stream) {
    attn::rope::Params p = rope_params(s, table, positions, err);
    p.q = q; p.k = k; p.q_out = q_out; p.k_out = k_out;
    if (!k) p.kv_heads = 0;
    p.all_heads = p.q_heads + p.kv_heads;
    if (transpose) p.sign = -1.f;
    return dtype == ATTN_F32 ? launch_rope_typed<float>(p, s->interleaved, stream)
                             : launch_rope_typed<__nv_bfloat16>(p, s->interleaved, stream);
}

int launch_rope_append(const attn_rope_shape *s, const attn_paged_kv *c, int dtype, const float *table,
                       const int *positions, const long long *slots, const void *q, const void *k, const void *v,
                       void *q_out, int *err, cudaStream_t stream) {
    using namespace attn::rope;
    Params p = rope_params(s, table, positions, err);
    p.q = q; p.k = k; p.v = v; p.q_out = q_out;
    p.k_out = c->k; p.v_out = c->v;
    p.ko_stride = c->row_stride ? c->row_stride : (long long)s->kv_heads * s->head_dim;
    p.slots = slots;
    p.rows = c->rows;
    if (c->kv_dtype != ATTN_I8) {
        p.all_heads = p.q_heads + 2 * p.kv_heads;
        return dtype == ATTN_F32 ? launch_rope_typed<float>(p, s->interleaved, stream)
                                 : launch_rope_typed<__nv_bfloat16>(p, s->interleaved, stream);
    }
    const long long warps = (long long)s->tokens * 2 * s->kv_heads;
    const long long blocks = (warps + kThreads / 32 - 1) / (kThreads / 32);
    if (blocks > 0x7fffffffLL) return set_error(ATTN_ERR_UNSUPPORTED, "rope append: %d tokens of %d heads", s->tokens, s->kv_heads);
    const dim3 grid((unsigned)blocks), block(kThreads);
    cudaError_t e;
    switch (s->head_dim) {
        case 32: e = launch_pdl(rope_append_i8_kernel<32>, grid, block, 0, stream, p, s->interleaved, c->kscale, c->vscale); break;
        case 64: e = launch_pdl(rope_append_i8_kernel<64>, grid, block, 0, stream, p, s->interleaved, c->kscale, c->vscale); break;
        case 96: e = launch_pdl(rope_append_i8_kernel<96>, grid, block, 0, stream, p, s->interleaved, c->kscale, c->vscale); break;
        default: e = launch_pdl(rope_append_i8_kernel<128>, grid, block, 0, stream, p, s->interleaved, c->kscale, c->vscale); break;
    }
    const int st = check_pdl(e, "rope_append_i8_kernel");
    if (st) return st;
    p.k = p.v = nullptr;                  // q alone
    p.kv_heads = 0;
    p.all_heads = p.q_heads;
    p.k_out = p.v_out = nullptr;
    p.ko_stride = 0;
    return launch_rope_typed<float>(p, s->interleaved, stream);
}

}  // namespace attn_host
