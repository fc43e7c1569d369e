// prefix_tile_sm100.cu -- the prefix part of attn_prefix_decode_ex on the
// Blackwell tensor cores, for bf16 caches whose groups have many query rows
// (requests x query heads per key head).
//
// With r rows a prefix costs r flops per byte, so past about 250 rows the
// tensor cores bound it and not HBM; mma.sync, at a quarter of their rate,
// already from 64 (two 32768-row prefixes of 512 rows each, 8 x 128: 957 us on
// mma.sync, %TILE% us here).
//
// One CTA per SM walks its range of steps (prefix.cuh) of 128 keys.  A slot is
// 256 query rows: with more than 128, warpgroup w takes rows [128 w, 128 w + 128)
// of every step; with fewer, both take the same rows and every other step, and
// the merge finds two pieces in the slot.  12 warps:
//   warps 0-1   copy Q rows and the keys' K and V rows, found through the page
//               table, into the tensor cores' 128-byte swizzled layout, 16 bytes
//               a lane; rows of no key are filled with zeros, so that a
//               probability of 0 never meets a NaN.  They report a copied half
//               (K or V of a step) when kLag more are on their way.
//   warp 2      S_w = Q_w K^T, M = N = 128, both operands in shared memory
//   warp 3      O_w += P_w V (P from TMEM, V as it lies, MN-major)
//   warps 4-7   softmax of warpgroup 0, warps 8-11 of warpgroup 1: a thread owns
//               a row (a TMEM lane), keeps its maximum and sum, writes its bf16
//               probabilities to TMEM, and rescales O when the maximum grew by
//               more than 2^8 (a stale one leaves P <= 256, and the piece's
//               (m, l, o) stay consistent).  All exponentials on MUFU: lse is an
//               output.
// At d 64 TMEM holds two S, two P and two O (512 columns), and S of a step may
// follow as soon as its predecessor is in registers.  At d 128 P lies over its
// own S, so S waits for the product that reads P; the two warpgroups then fill
// each other's gaps.
//
// Every wait is bounded; a timeout records a code in the device error word and
// raises a CTA-wide flag, on which all roles fall through to the teardown.
#include <algorithm>

#include "prefix.cuh"
#include "sm100.cuh"

namespace attn {
namespace ptile {

using namespace sm100;
using namespace prefix;

constexpr int BM = 128, BN = 128;
constexpr int kThreads = 384;
constexpr int kLag = 2;                   // halves on their way when one is reported

template <int D>
struct Cfg {
    static constexpr int STAGES = D == 64 ? 4 : 2;
    static constexpr bool OVER = D == 128;                    // P over S
    static constexpr int TILE = BM * D * 2;                   // Q tile, K or V tile: D / 64 blocks of 128 rows x 128 bytes
    static constexpr int OFF_K = 2 * TILE, STAGE = 2 * TILE;
    static constexpr int OFF_BAR = OFF_K + STAGES * STAGE;
    static constexpr int OFF_MASK = OFF_BAR + 256;
    static constexpr int SMEM = OFF_MASK + STAGES * 16 + 1024;
    static constexpr int S0 = 0, S1 = 128, O0 = 256, O1 = 256 + D;
    static constexpr int P0 = OVER ? S0 : 256 + 2 * D, P1 = OVER ? S1 : P0 + 64;
};

enum {
    B_QF = 0, B_QE = 1,                   // Q copied; its last S finished
    B_SF = 2, B_SE = 4,                   // per warpgroup: S ready; S in registers
    B_PF = 6, B_OD = 8, B_OF = 10,        // P written; PV finished; O read out
    B_KF = 12, B_VF = 16, B_KVE = 20,     // per stage: K, V copied; both used
    B_COUNT = 24
};

__device__ __forceinline__ void copy16(uint32_t dst, const void *src, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}

template <int D>
__global__ void __launch_bounds__(kThreads, 1)
prefix_tile_kernel(const __grid_constant__ Params p, const __grid_constant__ Part w)
{
    using C = Cfg<D>;
    constexpr int CPR = D / 8;            // 16-byte pieces of a row
    extern __shared__ uint8_t smem_raw[];
    __shared__ long long sums[kEntries + 1];
    __shared__ long long warp_sums[32];
    const uint32_t raw = smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
    uint8_t *sb = smem_raw + (base - raw);
    const uint32_t sQ = base, sKV = base + C::OFF_K, bar0 = base + C::OFF_BAR;
#define BAR(i) (bar0 + 8u * (uint32_t)(i))
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(sb + C::OFF_BAR + 224);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(sb + C::OFF_BAR + 228);
    volatile uint32_t *masks = reinterpret_cast<volatile uint32_t *>(sb + C::OFF_MASK);   // [stage][4]: keys with a row

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        mbar_init(BAR(B_QF), 64);
        mbar_init(BAR(B_QE), 1);
        for (int i = 0; i < 2; i++) {
            mbar_init(BAR(B_SF + i), 1);
            mbar_init(BAR(B_SE + i), 128);
            mbar_init(BAR(B_PF + i), 128);
            mbar_init(BAR(B_OD + i), 1);
            mbar_init(BAR(B_OF + i), 128);
        }
        for (int s = 0; s < C::STAGES; s++) {
            mbar_init(BAR(B_KF + s), 64);
            mbar_init(BAR(B_VF + s), 64);
            mbar_init(BAR(B_KVE + s), 2);
        }
        *abort_flag = 0;
        fence_mbar_init();
    }
    if (warp == 0) {
        tmem_alloc(smem_u32(tmem_slot), 512);
        tmem_relinquish();
    }
    // The own rows' launch may start once this one's CTAs have all seen the work before them finished.
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const long long total = sum_lines<true>(p, w, sums, warp_sums);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    Walk<true> walk(p, w, sums, total, (int)blockIdx.x);
    Piece x;

    // 384 x 168 registers at launch: 128 x 72 + 256 x 216
    if (warp < 4) regs_dec<72>();
    if (warp < 2) {
        // ------------------------------------------------------------ copies
        auto wait = [&](int b, int parity, int code) -> bool {
            return __all_sync(0xffffffffu, mbar_wait(BAR(b), parity & 1, abort_flag, p.err, code));
        };
        int due[kLag] = {}, n_due = 0;        // barriers of the halves on their way, oldest first
        auto report = [&](int b) {
            fence_async_smem();           // this thread's copies, for the tensor cores
            mbar_arrive(BAR(b));
        };
        auto copied = [&](int b) {
            asm volatile("cp.async.commit_group;" ::: "memory");
            if (n_due == kLag) {
                asm volatile("cp.async.wait_group %0;" ::"n"(kLag) : "memory");
                report(due[0]);
#pragma unroll
                for (int i = 0; i + 1 < kLag; i++) due[i] = due[i + 1];
                due[kLag - 1] = b;
            } else {
#pragma unroll
                for (int i = 0; i < kLag; i++)
                    if (i == n_due) due[i] = b;
                n_due++;
            }
        };
        auto flush = [&] {
            asm volatile("cp.async.wait_group 0;" ::: "memory");
#pragma unroll
            for (int i = 0; i < kLag; i++)
                if (i < n_due) report(due[i]);
            n_due = 0;
        };
        constexpr int RPI = 32 / CPR;     // rows per copy instruction of a warp
        const int lr = lane / CPR, ch = lane % CPR;
        // a 16-byte piece's place in a tile: 64-column block, row, piece XOR row % 8
        auto place = [&](int r) { return (uint32_t)((ch / 8) * BM * 128 + r * 128 + (((ch % 8) ^ (r & 7)) << 4)); };
        bool ok = true;
        int g = 0;                        // steps copied
        for (int k = 0; ok && walk.next(x); k++) {
            const bool two = x.rows > BM;
            flush();                      // the S that frees Q may wait for what is due
            if (k > 0 && !(ok = wait(B_QE, k - 1, 0x801))) break;
            for (int t = 0; t < (two ? 2 : 1); t++)
#pragma unroll 4
                for (int r0 = 0; r0 < 64; r0 += RPI) {
                    const int r = warp * 64 + r0 + lr, row = x.row0 + t * BM + r;
                    const bool there = t * BM + r < x.rows;
                    const int s = x.first_req + row / p.ratio, h = x.hb * p.ratio + row % p.ratio;
                    const __nv_bfloat16 *src = static_cast<const __nv_bfloat16 *>(p.q) +
                                               (there ? s * p.q_stride + (long long)h * D : 0) + ch * 8;
                    copy16(sQ + t * C::TILE + place(r), src, there);
                }
            copied(B_QF);
            for (int j = x.a; j < x.b; j++, g++) {
                const int st = g % C::STAGES;
                // cache rows of this warp's 64 keys, two per lane
                int row[2];
                bool valid[2];
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const int t = j * BN + warp * 64 + 32 * i + lane;
                    long long at = -1;
                    if (t < x.keys) at = cache_row(p, x.table, t);
                    valid[i] = at >= 0;
                    row[i] = max((int)at, 0);
                }
                if (g >= C::STAGES && !(ok = wait(B_KVE + st, g / C::STAGES + 1, 0x802))) break;
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const unsigned m = __ballot_sync(0xffffffffu, valid[i]);
                    if (lane == 0) masks[st * 4 + 2 * warp + i] = m;
                }
#pragma unroll
                for (int kv = 0; kv < 2; kv++) {
                    const __nv_bfloat16 *from = static_cast<const __nv_bfloat16 *>(kv ? p.v : p.k) + (long long)x.hb * D + ch * 8;
                    const uint32_t to = sKV + st * C::STAGE + kv * C::TILE;
#pragma unroll
                    for (int i = 0; i < 2; i++)
#pragma unroll 4
                        for (int r0 = 0; r0 < 32; r0 += RPI) {
                            const int r = __shfl_sync(0xffffffffu, row[i], r0 + lr);
                            const bool there = __shfl_sync(0xffffffffu, (int)valid[i], r0 + lr);
                            copy16(to + place(warp * 64 + 32 * i + r0 + lr), from + (long long)r * p.row_stride, there);
                        }
                    copied((kv ? B_VF : B_KF) + st);
                }
            }
        }
        if (ok) flush();
        asm volatile("cp.async.wait_all;" ::: "memory");
    } else if (warp == 2) {
        // ------------------------------------------------------------ S = Q K^T
        const bool leader = elect_one();
        auto wait = [&](int b, int parity, int code) -> bool {
            return __all_sync(0xffffffffu, mbar_wait(BAR(b), parity & 1, abort_flag, p.err, code));
        };
        constexpr uint32_t id = idesc_bf16(BM, BN, 0, 0);
        int g = 0, t[2] = {0, 0};         // steps; S products per warpgroup
        bool ok = true;
        for (int k = 0; ok && walk.next(x); k++) {
            const bool two = x.rows > BM;
            if (!(ok = wait(B_QF, k, 0x811))) break;
            for (int j = x.a; ok && j < x.b; j++, g++) {
                const int st = g % C::STAGES;
                if (!(ok = wait(B_KF + st, g / C::STAGES, 0x812))) break;
#pragma unroll
                for (int wg = 0; wg < 2; wg++) {
                    if (!two && ((j - x.a) & 1) != wg) continue;
                    if (t[wg] > 0 && !(ok = wait((C::OVER ? B_OD : B_SE) + wg, t[wg] - 1, 0x813 + wg))) break;
                    tc_fence_after();
                    if (leader) {
                        const uint64_t qd = sw128_desc(sQ + (two ? wg : 0) * C::TILE, 16, 1024);
                        const uint64_t kd = sw128_desc(sKV + st * C::STAGE, 16, 1024);
#pragma unroll
                        for (int kk = 0; kk < D / 16; kk++) {   // 32 bytes on per step, a block of 16 KB on per 64 dims
                            const uint32_t off = (kk / 4) * (BM * 128 >> 4) + (kk % 4) * 2;
                            mma_bf16_ss(tmem + (wg ? C::S1 : C::S0), qd + off, kd + off, id, kk > 0);
                        }
                        mma_commit(BAR(B_SF + wg));
                    }
                    __syncwarp();
                    t[wg]++;
                }
                if (!ok) break;
                if (leader) {
                    mma_commit(BAR(B_KVE + st));
                    if (j == x.b - 1) mma_commit(BAR(B_QE));
                }
                __syncwarp();
            }
        }
    } else if (warp == 3) {
        // ------------------------------------------------------------ O += P V
        const bool leader = elect_one();
        auto wait = [&](int b, int parity, int code) -> bool {
            return __all_sync(0xffffffffu, mbar_wait(BAR(b), parity & 1, abort_flag, p.err, code));
        };
        constexpr uint32_t id = idesc_bf16(BM, D, 0, 1);
        int g = 0, t[2] = {0, 0}, done[2] = {0, 0};   // steps; products and pieces per warpgroup
        bool ok = true;
        while (ok && walk.next(x)) {
            const bool two = x.rows > BM;
            for (int j = x.a; ok && j < x.b; j++, g++) {
                const int st = g % C::STAGES;
                if (!(ok = wait(B_VF + st, g / C::STAGES, 0x821))) break;
#pragma unroll
                for (int wg = 0; wg < 2; wg++) {
                    if (!two && ((j - x.a) & 1) != wg) continue;
                    const bool first = j - x.a < (two ? 1 : 2);   // of this warpgroup in this piece
                    if (first && done[wg] > 0 && !(ok = wait(B_OF + wg, done[wg] - 1, 0x822 + wg))) break;
                    if (!(ok = wait(B_PF + wg, t[wg], 0x824 + wg))) break;
                    tc_fence_after();
                    if (leader) {
                        const uint64_t vd = sw128_desc(sKV + st * C::STAGE + C::TILE, BM * 128, 1024);
#pragma unroll
                        for (int kk = 0; kk < BN / 16; kk++)      // 16 keys: 8 columns of P, 2 KB of V
                            mma_bf16_ts(tmem + (wg ? C::O1 : C::O0), tmem + (wg ? C::P1 : C::P0) + kk * 8, vd + 128 * kk, id,
                                        !first || kk > 0);
                        mma_commit(BAR(B_OD + wg));
                    }
                    __syncwarp();
                    t[wg]++;
                }
                if (!ok) break;
                if (leader) mma_commit(BAR(B_KVE + st));
                __syncwarp();
            }
            done[0]++;
            if (two || x.b - x.a > 1) done[1]++;
        }
    } else {
        // ------------------------------------------------------------ softmax
        regs_inc<216>();
        const int wg = (warp - 4) >> 2, quad = warp & 3, row = quad * 32 + lane;
        const uint32_t lane_base = (uint32_t)(quad * 32) << 16;
        const uint32_t tS = tmem + lane_base + (wg ? C::S1 : C::S0), tP = tmem + lane_base + (wg ? C::P1 : C::P0);
        const uint32_t tO = tmem + lane_base + (wg ? C::O1 : C::O0);
        int g = 0, t = 0;                 // steps of the CTA; of this warpgroup
        bool ok = true;
        while (ok && walk.next(x)) {
            const bool two = x.rows > BM;
            const int mine = two ? x.rows - wg * BM : x.rows;     // query rows of this warpgroup
            const bool idle = quad * 32 >= mine;                  // none of them in this warp: it only keeps step
            float m = -INFINITY, l = 0.f;
            bool any = false;
            for (int j = x.a; j < x.b; j++) {
                if (!two && ((j - x.a) & 1) != wg) continue;
                const int at = g + j - x.a, st = at % C::STAGES;
                // S is ready; then K's barrier, for the copying warps' masks, is past its phase too
                ok = mbar_wait(BAR(B_SF + wg), t & 1, abort_flag, p.err, 0x831) &&
                     mbar_wait(BAR(B_KF + st), at / C::STAGES & 1, abort_flag, p.err, 0x832);
                if (!(ok = __all_sync(0xffffffffu, ok))) break;
                tc_fence_after();
                if (idle) {
                    if (!C::OVER) mbar_arrive(BAR(B_SE + wg));
                    if (t > 0) ok = mbar_wait(BAR(B_OD + wg), (t - 1) & 1, abort_flag, p.err, 0x833);
                    if (!(ok = __all_sync(0xffffffffu, ok))) break;
                    mbar_arrive(BAR(B_PF + wg));
                    t++;
                    any = true;
                    continue;
                }
                uint32_t s[128];
#pragma unroll
                for (int q4 = 0; q4 < 4; q4++) {
                    uint32_t tt[32];
                    tmem_ld32(tS + 32 * q4, tt);
#pragma unroll
                    for (int c = 0; c < 32; c++) s[32 * q4 + c] = tt[c];
                }
                uint32_t valid[4];
#pragma unroll
                for (int i = 0; i < 4; i++) valid[i] = masks[st * 4 + i];
                tmem_wait_ld();
                if (!C::OVER) {
                    tc_fence_before();
                    mbar_arrive(BAR(B_SE + wg));                  // S may be overwritten
                }
                if ((valid[0] & valid[1] & valid[2] & valid[3]) != 0xffffffffu) {
#pragma unroll
                    for (int c = 0; c < 128; c++)
                        if (!(valid[c >> 5] >> (c & 31) & 1)) s[c] = __float_as_uint(-INFINITY);
                }
                float mp[8];
#pragma unroll
                for (int i = 0; i < 8; i++) mp[i] = -INFINITY;
#pragma unroll
                for (int c = 0; c < 128; c += 2)
                    mp[(c >> 1) & 7] = max3(mp[(c >> 1) & 7], __uint_as_float(s[c]), __uint_as_float(s[c + 1]));
                float mx = max3(max3(mp[0], mp[1], mp[2]), max3(mp[3], mp[4], mp[5]), fmaxf(mp[6], mp[7]));
                mx *= p.scale_log2;
                float alpha = 1.f;
                const bool grow = mx > m + 8.f;                   // also at the first step with a key
                if (grow) {
                    alpha = ex2(m - mx);
                    m = mx;
                    l *= alpha;
                }
                const float neg = m == -INFINITY ? 0.f : -m;
                const uint64_t scale2 = f2(p.scale_log2, p.scale_log2), neg2 = f2(neg, neg);
                uint64_t l2[4] = {0ull, 0ull, 0ull, 0ull};
                uint32_t pk[64];
#pragma unroll
                for (int c = 0; c < 64; c++) {
                    float a, b;
                    f2_split(fma2(f2(__uint_as_float(s[2 * c]), __uint_as_float(s[2 * c + 1])), scale2, neg2), a, b);
                    a = ex2(a);
                    b = ex2(b);
                    l2[c & 3] = add2(l2[c & 3], f2(a, b));
                    pk[c] = pack_bf16(a, b);
                }
                {
                    float a, b;
                    f2_split(add2(add2(l2[0], l2[1]), add2(l2[2], l2[3])), a, b);
                    l += a + b;
                }
                // P and O belong to the previous product until it is done
                if (t > 0) ok = mbar_wait(BAR(B_OD + wg), (t - 1) & 1, abort_flag, p.err, 0x834);
                if (!(ok = __all_sync(0xffffffffu, ok))) break;
                tc_fence_after();
#pragma unroll
                for (int half = 0; half < 2; half++) {
                    uint32_t tt[32];
#pragma unroll
                    for (int c = 0; c < 32; c++) tt[c] = pk[32 * half + c];
                    tmem_st32(tP + 32 * half, tt);
                }
                if (__any_sync(0xffffffffu, any && grow)) {
                    uint32_t o[32];
#pragma unroll
                    for (int c0 = 0; c0 < D; c0 += 32) {
                        tmem_ld32(tO + c0, o);
                        tmem_wait_ld();
#pragma unroll
                        for (int c = 0; c < 32; c++) o[c] = __float_as_uint(__uint_as_float(o[c]) * alpha);
                        tmem_st32(tO + c0, o);
                    }
                }
                tmem_wait_st();
                tc_fence_before();
                mbar_arrive(BAR(B_PF + wg));
                t++;
                any = true;
            }
            if (!ok) break;
            g += x.b - x.a;
            // the piece: this warpgroup's half of the slot
            const long long at = x.slot * w.rows + wg * BM + row;
            if (any) {
                ok = mbar_wait(BAR(B_OD + wg), (t - 1) & 1, abort_flag, p.err, 0x835);
                if (!(ok = __all_sync(0xffffffffu, ok))) break;
                tc_fence_after();
                if (!idle) {
#pragma unroll
                    for (int c0 = 0; c0 < D; c0 += 32) {
                        uint32_t o[32];
                        tmem_ld32(tO + c0, o);
                        tmem_wait_ld();
                        if (row < mine) {
                            float4 *out = reinterpret_cast<float4 *>(w.o + at * D + c0);
#pragma unroll
                            for (int c = 0; c < 8; c++)
                                out[c] = make_float4(__uint_as_float(o[4 * c]), __uint_as_float(o[4 * c + 1]),
                                                     __uint_as_float(o[4 * c + 2]), __uint_as_float(o[4 * c + 3]));
                        }
                    }
                    tc_fence_before();
                }
                mbar_arrive(BAR(B_OF + wg));      // the next piece's first product may overwrite O
            }
            if (row < mine) w.ml[at] = make_float2(m, l);
        }
    }

    // ---------------------------------------------------------------- teardown
    tc_fence_before();
    __syncthreads();
    if (*abort_flag) {
        // let what is in flight finish before the CTA releases its memory
        for (int i = 0; i < 1000; i++) __nanosleep(1000);
    }
    if (warp == 0) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
#undef BAR
}

}  // namespace ptile
}  // namespace attn

namespace attn_host {

bool ensure_smem_attr(const void *func, size_t bytes);

template <int D>
static int launch_d(const attn::prefix::Params &p, const attn::prefix::Part &w, cudaStream_t s) {
    using namespace attn::ptile;
    if (!ensure_smem_attr((const void *)prefix_tile_kernel<D>, Cfg<D>::SMEM))
        return set_error(ATTN_ERR_CUDA, "prefix decode: cannot set shared-memory size");
    return check_pdl(launch_pdl(prefix_tile_kernel<D>, dim3(w.teams), dim3(kThreads), Cfg<D>::SMEM, s, p, w), "prefix_tile_kernel");
}

int launch_prefix_tile(const attn::prefix::Params &p, const attn::prefix::Part &w, int d, cudaStream_t s) {
    return d == 64 ? launch_d<64>(p, w, s) : launch_d<128>(p, w, s);
}

}  // namespace attn_host
