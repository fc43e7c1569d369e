// prefix_decode.cu -- attn_prefix_decode_ex: one query token per request over
// the rows that its group shares and its own, both in a paged cache.
//
// With keys j over prefix and own rows, out = sum_j p_j v_j / sum_j p_j and
// p_j = 2^(x_j - m), x_j = scale log2(e) q.k_j, m = max_j x_j.  Any split of
// the keys gives triples (m, l, o) that join exactly: with M = max m_i,
// l = sum l_i 2^(m_i - M) and o likewise.
#include "prefix.cuh"

namespace attn {
namespace prefix {

constexpr int kThreads = 128;

template <typename KV> struct Elem;
template <> struct Elem<float> { static __device__ float get(const float *p) { return *p; } };
template <> struct Elem<__nv_bfloat16> { static __device__ float get(const __nv_bfloat16 *p) { return to_f32(*p); } };
template <> struct Elem<int8_t> { static __device__ float get(const int8_t *p) { return (float)*p; } };

// One CTA per (request, query head): each warp takes every fourth row, a lane
// holds D/32 elements of it, and the four running softmaxes join at the end.
template <typename T, typename KV, int D>
__global__ void __launch_bounds__(kThreads)
prefix_simple_kernel(const __grid_constant__ Params p)
{
    pdl_begin();                          // launched by launch_pdl
    constexpr int E = D / 32;
    __shared__ float s_m[4], s_l[4], s_o[4][D];
    const int s = blockIdx.y, h = blockIdx.x, hk = h / p.ratio;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int plen = 0, group = 0;
    for (int g = 0; g < p.n_groups; g++)
        if (s >= group_first(p, g) && s < group_first(p, g + 1)) { plen = prefix_len(p, g); group = g; }
    const int total = plen + own_len(p, s);
    float q[E], o[E], m = -INFINITY, l = 0.f;
#pragma unroll
    for (int i = 0; i < E; i++) {
        q[i] = to_f32(static_cast<const T *>(p.q)[s * p.q_stride + h * D + lane + 32 * i]) * p.scale_log2;
        o[i] = 0.f;
    }
    const int *pline = p.prefix_table + (long long)group * p.max_prefix_pages;
    const int *line = p.block_table + (long long)s * p.max_pages;
    for (int t = warp; t < total; t += 4) {
        const long long row = t < plen ? cache_row(p, pline, t) : cache_row(p, line, t - plen);
        if (row < 0) continue;
        const KV *k = static_cast<const KV *>(p.k) + row * p.row_stride + hk * D;
        const KV *v = static_cast<const KV *>(p.v) + row * p.row_stride + hk * D;
        float x = 0.f;
#pragma unroll
        for (int i = 0; i < E; i++) x = fmaf(q[i], Elem<KV>::get(k + lane + 32 * i), x);
        x = warp_sum(x);
        float vs = 1.f;
        if constexpr (sizeof(KV) == 1) {
            x *= p.kscale[row * p.kv_heads + hk];
            vs = p.vscale[row * p.kv_heads + hk];
        }
        const float mx = fmaxf(m, x), a = exp2f(m - mx), w = exp2f(x - mx);
        l = l * a + w;
#pragma unroll
        for (int i = 0; i < E; i++) o[i] = o[i] * a + w * vs * Elem<KV>::get(v + lane + 32 * i);
        m = mx;
    }
    if (lane == 0) { s_m[warp] = m; s_l[warp] = l; }
#pragma unroll
    for (int i = 0; i < E; i++) s_o[warp][lane + 32 * i] = o[i];
    __syncthreads();
    const float M = fmaxf(fmaxf(s_m[0], s_m[1]), fmaxf(s_m[2], s_m[3]));
    float w[4], L = 0.f;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        w[i] = M == -INFINITY ? 0.f : exp2f(s_m[i] - M);
        L += s_l[i] * w[i];
    }
    if (threadIdx.x < D) {
        float r = 0.f;
#pragma unroll
        for (int i = 0; i < 4; i++) r += s_o[i][threadIdx.x] * w[i];
        static_cast<T *>(p.out)[s * p.out_stride + h * D + threadIdx.x] = from_f32<T>(L > 0.f ? r / L : 0.f);
    }
    if (p.lse && threadIdx.x == 0) p.lse[(long long)s * p.heads + h] = L > 0.f ? (M + log2f(L)) * kLn2 : -INFINITY;
}

}  // namespace prefix
}  // namespace attn

namespace attn_host {

template <typename T, typename KV>
static int launch_typed(const attn::prefix::Params &p, int d, cudaStream_t s) {
    using namespace attn::prefix;
    const dim3 grid(p.heads, p.n_seq), block(kThreads);
    cudaError_t e;
    switch (d) {
        case 32: e = launch_pdl(prefix_simple_kernel<T, KV, 32>, grid, block, 0, s, p); break;
        case 64: e = launch_pdl(prefix_simple_kernel<T, KV, 64>, grid, block, 0, s, p); break;
        case 96: e = launch_pdl(prefix_simple_kernel<T, KV, 96>, grid, block, 0, s, p); break;
        default: e = launch_pdl(prefix_simple_kernel<T, KV, 128>, grid, block, 0, s, p); break;
    }
    return check_pdl(e, "prefix_simple_kernel");
}

size_t prefix_decode_workspace(const attn_prefix_shape *, int) { return 256; }

int launch_prefix_decode(const attn::prefix::Params &p, int d, int kv_dtype, void *, cudaStream_t s) {
    if (kv_dtype == ATTN_BF16) return launch_typed<__nv_bfloat16, __nv_bfloat16>(p, d, s);
    if (kv_dtype == ATTN_I8) return launch_typed<float, int8_t>(p, d, s);
    return launch_typed<float, float>(p, d, s);
}

}  // namespace attn_host
