// prefix_tile_sm100.cu -- the prefix part of attn_prefix_decode_ex on the
// Blackwell tensor cores, for bf16 caches whose groups have many query rows
// (requests x query heads per key head).
//
// With r rows a prefix costs r flops per byte, so past about 250 rows the
// tensor cores bound it and not HBM; mma.sync, at a quarter of their rate,
// already from 64 (two 32768-row prefixes of 512 rows each, 8 x 128, called with
// one own row a request: 174 us, merge included: 742 TFLOP/s; 957 us on mma.sync
// with probabilities in one part).  The times in brackets below were taken with
// one part too, when the same call took 143 us.
//
// One CTA per SM walks its range of steps (prefix.cuh) of 128 keys.  A slot is
// 256 query rows: with more than 128, warpgroup w takes rows [128 w, 128 w + 128)
// of every step; with fewer, both take the same rows and every other step, and
// the merge finds two pieces in the slot.  12 warps:
//   warp 0      K rows, warp 1 V rows.  A step whose 128 keys all have rows is a
//               TMA box of 64 dims for each page (or 128 rows of one), a lane
//               per box.  At a line's end, with pages of fewer than 8 rows or
//               outside the cache, the lanes copy 16 bytes each into the same
//               128-byte swizzled layout, with zeros for keys without a row, so
//               that a probability of 0 never meets a NaN; they report such a
//               half (K or V of a step) when their next one is on its way.
//               (All steps by lanes: 299 us, the copying instructions setting the pace.)
//   warp 2      S_wu = Q_w K_u^T for the two halves u of a step's keys, M = 128,
//               N = 64, both operands in shared memory
//   warp 3      O_w += P_wu V_u (P in two bf16 parts from TMEM, V as it lies, MN-major)
//   warps 4-7   softmax of warpgroup 0, warps 8-11 of warpgroup 1: a warp
//               brings 32 query rows in, a thread keeps the maximum and sum of its row
//               (a TMEM lane), writes its probabilities to TMEM, and rescales O when the maximum grew by
//               more than 2^8 (a stale one leaves P <= 256, and the piece's
//               (m, l, o) stay consistent).  All exponentials on MUFU: lse is an
//               output.
// A probability goes in as two bf16 parts, its rounding and the rest, which leaves
// no error but that of rounding the output (one part: 1.4 times it).  The second
// product and its packing took that call from 143 to 174 us.
// TMEM: four S of 64 columns, each overwritten by the two parts of its P, and two
// O (512 columns at d 128).  S_w1 is formed while S_w0 is in the softmax, so a warpgroup does
// not wait for its own products.  (With 128 keys in one S per warpgroup the
// chain softmax, PV, next S took 5,300 cycles a step, of which the exponentials
// of both warpgroups are 2,048; with P in halves but S in one product 171 us, the
// warpgroup waiting for its last PV and the S after it.  One warp for both products
// in a fixed order: 217 us, its own instructions and waits take 1,730 cycles a pair;
// four, one per product and warpgroup: no faster than two.)
//
// Every wait is bounded; a timeout records a code in the device error word and
// raises a CTA-wide flag, on which all roles fall through to the teardown.
#include <algorithm>
#include <cudaTypedefs.h>

#include "prefix.cuh"
#include "sm100.cuh"

namespace attn {
namespace ptile {

using namespace sm100;
using namespace prefix;

constexpr int BM = 128, BN = 128, BH = 64;   // query rows; keys of a step, of an S
constexpr int kThreads = 384;
constexpr int kMasks = 8;                 // steps whose key masks are kept: more than K's ring holds, and the ones at work

template <int D>
struct Cfg {
    // rings of K and V tiles (V waits longer for its use); one ring for both would be ambiguous to parity
    // waits once one of the two copying warps runs ahead of the other
    static constexpr int KS = D == 64 ? 4 : 2, VS = D == 64 ? 4 : 3, SLOTS = KS + VS;
    static constexpr int TILE = BM * D * 2;                   // Q tile, K or V tile: D / 64 blocks of 128 rows x 128 bytes
    static constexpr int OFF_KV = 2 * TILE;
    static constexpr int OFF_BAR = OFF_KV + SLOTS * TILE;
    static constexpr int OFF_MASK = OFF_BAR + 320;
    static constexpr int SMEM = OFF_MASK + kMasks * 16 + 1024;
};
// TMEM columns
__device__ __forceinline__ uint32_t col_s(int wg, int u) { return (uint32_t)(wg * 2 + u) * BH; }
template <int D> __device__ __forceinline__ uint32_t col_o(int wg) { return 4 * BH + (uint32_t)wg * D; }

enum {
    B_QF = 0, B_QE = 1,                   // Q there; its last S finished
    B_OF = 2,                             // per warpgroup: O read out
    B_SF = 4, B_PF = 8, B_OD = 12,        // per warpgroup and half (2 w + u): S ready; P written; PV finished
    B_FULL = 16, B_FREE = 24,             // per slot: copied; used
    B_COUNT = 32
};

__device__ __forceinline__ void copy16(uint32_t dst, const void *src, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}

// Place of 16-byte piece ch of row r in a tile: block of 64 dims, row, piece XOR row % 8.
__device__ __forceinline__ uint32_t tile_at(int r, int ch) {
    return (uint32_t)((ch / 8) * BM * 128 + r * 128 + (((ch % 8) ^ (r & 7)) << 4));
}

template <int D>
__global__ void __launch_bounds__(kThreads, 1)
prefix_tile_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv,
                   const __grid_constant__ Params p, const __grid_constant__ Part w, int boxes)
{
    using C = Cfg<D>;
    constexpr int CPR = D / 8;            // 16-byte pieces of a row
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
    uint8_t *sb = smem_raw + (base - raw);
    const uint32_t sQ = base, sKV = base + C::OFF_KV, bar0 = base + C::OFF_BAR;
#define BAR(i) (bar0 + 8u * (uint32_t)(i))
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(sb + C::OFF_BAR + 256);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(sb + C::OFF_BAR + 260);
    volatile uint32_t *masks = reinterpret_cast<volatile uint32_t *>(sb + C::OFF_MASK);   // [step % kMasks][4]: keys with a row

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        mbar_init(BAR(B_QF), 256);
        mbar_init(BAR(B_QE), 1);
        for (int i = 0; i < 2; i++) mbar_init(BAR(B_OF + i), 128);
        for (int i = 0; i < 4; i++) {
            mbar_init(BAR(B_SF + i), 2);
            mbar_init(BAR(B_PF + i), 128);
            mbar_init(BAR(B_OD + i), 1);
        }
        for (int s = 0; s < C::SLOTS; s++) {
            mbar_init(BAR(B_FULL + s), 32);
            mbar_init(BAR(B_FREE + s), 1);
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
    // (the sums lie where the query rows come after the next barrier)
    long long *sums = reinterpret_cast<long long *>(sb);
    static_assert((kEntries + 1 + 32) * 8 <= 2 * C::TILE, "sums in the query tiles");
    const long long of_team = sum_lines<true>(p, w, sums, sums + kEntries + 1);
    Walk<true> walk(p, w, sums, of_team, (int)blockIdx.x);
    Piece x;
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    // 384 x 168 registers at launch: 128 x 88 + 256 x 208
    if (warp < 4) regs_dec<88>();
    if (warp < 2) {
        // ------------------------------------------------------------ K, V
        const int kv = warp;
        const CUtensorMap *map = kv ? &tv : &tk;
        if (lane == 0) prefetch_tmap(map);
        int due = -1;                     // slot of a half that the lanes have on its way
        auto flush = [&] {
            if (due < 0) return;
            asm volatile("cp.async.wait_group 0;" ::: "memory");
            fence_async_smem();           // this thread's copies, for the tensor cores
            mbar_arrive(BAR(B_FULL + due));
            due = -1;
        };
        constexpr int RPI = 32 / CPR;     // rows per copy instruction
        const int lr = lane / CPR, ch = lane % CPR;
        bool ok = true;
        int g = 0;                        // steps
        while (ok && walk.next(x)) {
            const __nv_bfloat16 *from = static_cast<const __nv_bfloat16 *>(kv ? p.v : p.k) + (long long)x.hb * D + ch * 8;
            // cache rows of a step's 128 keys (-1: none), four per lane, read a step ahead
            int next[4];
            auto look_up = [&](int j) {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int t = j * BN + 32 * i + lane;
                    next[i] = j < x.b && t < x.keys ? (int)cache_row(p, x.table, t) : -1;
                }
            };
            look_up(x.a);
            for (int j = x.a; j < x.b; j++, g++) {
                int row[4];
                unsigned valid[4];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    row[i] = next[i];
                    valid[i] = __ballot_sync(0xffffffffu, next[i] >= 0);
                }
                look_up(j + 1);
                const bool whole = boxes && (valid[0] & valid[1] & valid[2] & valid[3]) == 0xffffffffu;
                const int ring = kv ? C::VS : C::KS, slot = kv ? C::KS + g % C::VS : g % C::KS;
                const uint32_t to = sKV + slot * C::TILE;
                if (g >= ring) {
                    flush();              // nothing may stay due behind the wait
                    ok = mbar_wait(BAR(B_FREE + slot), (g / ring + 1) & 1, abort_flag, p.err, 0x801 + kv);
                    if (!(ok = __all_sync(0xffffffffu, ok))) break;
                }
                if (kv == 0 && lane == 0) {
#pragma unroll
                    for (int i = 0; i < 4; i++) masks[g % kMasks * 4 + i] = valid[i];
                }
                __syncwarp();
                if (whole) {
                    const int rows = BN / boxes, key = lane * rows & 127;     // of lane n's box
                    int r = 0;
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const int y = __shfl_sync(0xffffffffu, row[i], key & 31);
                        if (key >> 5 == i) r = y;
                    }
                    if (lane == 0) mbar_arrive_expect_tx(BAR(B_FULL + slot), C::TILE);
                    else mbar_arrive(BAR(B_FULL + slot));
                    __syncwarp();
                    if (lane < boxes) {
#pragma unroll
                        for (int d = 0; d < D / 64; d++)
                            tma_load_3d(to + d * BN * 128 + key * 128, map, BAR(B_FULL + slot), x.hb * D + 64 * d, r, 0);
                    }
                    __syncwarp();
                    continue;
                }
                flush();
#pragma unroll
                for (int i = 0; i < 4; i++)
#pragma unroll 4
                    for (int r0 = 0; r0 < 32; r0 += RPI) {
                        const int r = __shfl_sync(0xffffffffu, row[i], r0 + lr);
                        copy16(to + tile_at(32 * i + r0 + lr, ch), from + (long long)max(r, 0) * p.row_stride, r >= 0);
                    }
                asm volatile("cp.async.commit_group;" ::: "memory");
                due = slot;
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
        constexpr uint32_t id = idesc_bf16(BM, BH, 0, 0);
        int g = 0, t[2] = {0, 0};         // steps; steps per warpgroup
        bool ok = true;
        for (int k = 0; ok && walk.next(x); k++) {
            const bool two = x.rows > BM;
            if (!(ok = wait(B_QF, k, 0x811))) break;
            for (int j = x.a; ok && j < x.b; j++, g++) {
                const int slot = g % C::KS;
                if (!(ok = wait(B_FULL + slot, g / C::KS, 0x812))) break;
#pragma unroll
                for (int n = 0; n < 4; n++) {
                    const int u = n >> 1, wg = n & 1, b = 2 * wg + u;
                    if (!two && ((j - x.a) & 1) != wg) continue;
                    // the product that reads this half's last P is done
                    if (ok && t[wg] > 0) ok = wait(B_OD + b, t[wg] - 1, 0x813 + n);
                    if (!ok) break;
                    tc_fence_after();
                    if (leader) {
                        const uint64_t qd = sw128_desc(sQ + (two ? wg : 0) * C::TILE, 16, 1024);
                        const uint64_t kd = sw128_desc(sKV + slot * C::TILE + u * BH * 128, 16, 1024);
#pragma unroll
                        for (int kk = 0; kk < D / 16; kk++) {   // 32 bytes on per step, a block of 16 KB on per 64 dims
                            const uint32_t off = (kk / 4) * (BM * 128 >> 4) + (kk % 4) * 2;
                            mma_bf16_ss(tmem + col_s(wg, u), qd + off, kd + off, id, kk > 0);
                        }
                        mma_commit(BAR(B_SF + b));
                        mbar_arrive(BAR(B_SF + b));               // (hands on the copying warps' masks)
                    }
                    __syncwarp();
                    if (u == 1) t[wg]++;
                }
                if (!ok) break;
                if (leader) {
                    mma_commit(BAR(B_FREE + slot));
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
        int g = 0, t[2] = {0, 0}, done[2] = {0, 0};   // steps; steps and pieces per warpgroup
        bool ok = true;
        while (ok && walk.next(x)) {
            const bool two = x.rows > BM;
            for (int j = x.a; ok && j < x.b; j++, g++) {
                const int slot = C::KS + g % C::VS;
                if (!(ok = wait(B_FULL + slot, g / C::VS, 0x821))) break;
#pragma unroll
                for (int n = 0; n < 4; n++) {
                    const int u = n >> 1, wg = n & 1, b = 2 * wg + u;
                    if (!two && ((j - x.a) & 1) != wg) continue;
                    const bool first = u == 0 && j - x.a < (two ? 1 : 2);   // of this warpgroup in this piece
                    if (ok && first && done[wg] > 0) ok = wait(B_OF + wg, done[wg] - 1, 0x822 + wg);
                    if (ok) ok = wait(B_PF + b, t[wg], 0x824 + n);
                    if (!ok) break;
                    tc_fence_after();
                    if (leader) {
                        const uint64_t vd = sw128_desc(sKV + slot * C::TILE + u * BH * 128, BM * 128, 1024);
#pragma unroll
                        for (int kk = 0; kk < 2 * BH / 16; kk++)  // 16 keys: 8 columns of a part of P, 2 KB of V
                            mma_bf16_ts(tmem + col_o<D>(wg), tmem + col_s(wg, u) + kk * 8, vd + 128 * (kk % (BH / 16)), id, !first || kk > 0);
                        mma_commit(BAR(B_OD + b));
                    }
                    __syncwarp();
                    if (u == 1) t[wg]++;
                }
                if (!ok) break;
                if (leader) mma_commit(BAR(B_FREE + slot));
                __syncwarp();
            }
            done[0]++;
            if (two || x.b - x.a > 1) done[1]++;
        }
    } else {
        // ------------------------------------------------------------ softmax
        regs_inc<208>();
        const int wg = (warp - 4) >> 2, quad = warp & 3, row = quad * 32 + lane;
        const uint32_t lanes = tmem + ((uint32_t)(quad * 32) << 16), tO = lanes + col_o<D>(wg);
        int g = 0, t = 0;                 // steps of the CTA; of this warpgroup
        bool ok = true;
        for (int k = 0; ok && walk.next(x); k++) {
            const bool two = x.rows > BM;
            // the warp's 32 query rows, CPR lanes a row (with up to 128 rows, warpgroup 0 brings them in for both);
            // a lane to a row, 16 bytes of 32 rows an instruction, took 2.5 us instead of 1.1
            if (two || wg == 0) {
                constexpr int RPI = 32 / CPR;
                const int r = wg * BM + row, at = x.row0 + min(r, x.rows - 1);
                const int s = x.first_req + at / p.ratio, h = x.hb * p.ratio + at % p.ratio;
                const long long mine = s * p.q_stride + (long long)h * D;
#pragma unroll
                for (int r0 = 0; r0 < 32; r0 += RPI) {
                    const int n = r0 + lane / CPR, to = quad * 32 + n, ch = lane % CPR;
                    const __nv_bfloat16 *src = static_cast<const __nv_bfloat16 *>(p.q) + __shfl_sync(0xffffffffu, mine, n) + 8 * ch;
                    copy16(sQ + wg * C::TILE + tile_at(to, ch), src, wg * BM + to < x.rows);
                }
                asm volatile("cp.async.wait_all;" ::: "memory");
                fence_async_smem();
            }
            mbar_arrive(BAR(B_QF));
            const int mine = two ? x.rows - wg * BM : x.rows;     // query rows of this warpgroup
            const bool idle = quad * 32 >= mine;                  // none of them in this warp: it only keeps step
            float m = -INFINITY, l = 0.f;
            bool any = false, ready = false;
            for (int j = x.a; ok && j < x.b; j++) {
                if (!two && ((j - x.a) & 1) != wg) continue;
#pragma unroll 1
                for (int u = 0; u < 2; u++) {
                    const int b = 2 * wg + u;
                    const uint32_t tS = lanes + col_s(wg, u);
                    if (!__all_sync(0xffffffffu, ready)) {
                        ok = mbar_wait(BAR(B_SF + b), t & 1, abort_flag, p.err, 0x831 + u);
                        if (!(ok = __all_sync(0xffffffffu, ok))) break;
                    }
                    tc_fence_after();
                    if (!idle) {
                        uint32_t s[BH];
#pragma unroll
                        for (int q = 0; q < BH / 32; q++) {
                            uint32_t tt[32];
                            tmem_ld32(tS + 32 * q, tt);
#pragma unroll
                            for (int c = 0; c < 32; c++) s[32 * q + c] = tt[c];
                        }
                        uint32_t valid[2];
#pragma unroll
                        for (int i = 0; i < 2; i++) valid[i] = masks[(g + j - x.a) % kMasks * 4 + 2 * u + i];
                        tmem_wait_ld();
                        if ((valid[0] & valid[1]) != 0xffffffffu) {
#pragma unroll
                            for (int c = 0; c < BH; c++)
                                if (!(valid[c >> 5] >> (c & 31) & 1)) s[c] = __float_as_uint(-INFINITY);
                        }
                        float mp[4];
#pragma unroll
                        for (int i = 0; i < 4; i++) mp[i] = -INFINITY;
#pragma unroll
                        for (int c = 0; c < BH; c += 2)
                            mp[(c >> 1) & 3] = max3(mp[(c >> 1) & 3], __uint_as_float(s[c]), __uint_as_float(s[c + 1]));
                        const float mx = fmaxf(max3(mp[0], mp[1], mp[2]), mp[3]) * p.scale_log2;
                        float alpha = 1.f;
                        const bool grow = mx > m + 8.f;           // also at the first half with a key
                        if (grow) {
                            alpha = ex2(m - mx);
                            m = mx;
                            l *= alpha;
                        }
                        const float neg = m == -INFINITY ? 0.f : -m;
                        const uint64_t scale2 = f2(p.scale_log2, p.scale_log2), neg2 = f2(neg, neg);
                        uint64_t l2[4] = {0ull, 0ull, 0ull, 0ull};
                        uint32_t hi[32], lo[32];
#pragma unroll
                        for (int c = 0; c < 32; c++) {
                            float e, f;
                            f2_split(fma2(f2(__uint_as_float(s[2 * c]), __uint_as_float(s[2 * c + 1])), scale2, neg2), e, f);
                            e = ex2(e);
                            f = ex2(f);
                            l2[c & 3] = add2(l2[c & 3], f2(e, f));
                            bf16_parts(e, f, hi[c], lo[c]);
                        }
                        {
                            float e, f;
                            f2_split(add2(add2(l2[0], l2[1]), add2(l2[2], l2[3])), e, f);
                            l += e + f;
                        }
                        tmem_st32(tS, hi);                        // over S, which is in registers
                        tmem_st32(tS + 32, lo);
                        if (__any_sync(0xffffffffu, any && grow)) {
                            // O is the previous half's product's until that is done
                            ok = mbar_wait(BAR(B_OD + 2 * wg + 1 - u), (t - 1 + u) & 1, abort_flag, p.err, 0x833 + u);
                            if (!(ok = __all_sync(0xffffffffu, ok))) break;
                            tc_fence_after();
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
                        // the next half's S, looked for while P is on its way to TMEM (P in one part: 143 us so, 146.5 after it)
                        ready = mbar_test_wait(BAR(B_SF + 2 * wg + 1 - u), (t + u) & 1);
                        tmem_wait_st();
                        tc_fence_before();
                    }
                    mbar_arrive(BAR(B_PF + b));
                    any = true;
                }
                t++;
            }
            if (!ok) break;
            g += x.b - x.a;
            ok = mbar_wait(BAR(B_QE), k & 1, abort_flag, p.err, 0x830);
            if (!(ok = __all_sync(0xffffffffu, ok))) break;
            // The piece: this warpgroup's half of the slot.  A warp turns 32 dims of its 32 rows
            // over in what was the place of their queries and writes them 128 bytes at a time.
            // (Each thread writing its own row, 512 bytes apart: 6.4 us from a piece's last P to the next piece, 3.4 so.)
            const long long at = x.slot * w.rows + wg * BM + row;
            if (any) {
                ok = mbar_wait(BAR(B_OD + 2 * wg), (t - 1) & 1, abort_flag, p.err, 0x835) &&
                     mbar_wait(BAR(B_OD + 2 * wg + 1), (t - 1) & 1, abort_flag, p.err, 0x836);
                if (!(ok = __all_sync(0xffffffffu, ok))) break;
                tc_fence_after();
                if (!idle) {
#pragma unroll
                    for (int c0 = 0; c0 < D; c0 += 32) {
                        uint32_t o[32];
                        tmem_ld32(tO + c0, o);
                        tmem_wait_ld();
                        float4 *turn = reinterpret_cast<float4 *>(sb + wg * C::TILE + quad * 32 * 128);
#pragma unroll
                        for (int c = 0; c < 8; c++)
                            turn[lane * 8 + (c ^ (lane & 7))] = make_float4(__uint_as_float(o[4 * c]), __uint_as_float(o[4 * c + 1]),
                                                                            __uint_as_float(o[4 * c + 2]), __uint_as_float(o[4 * c + 3]));
                        __syncwarp();
#pragma unroll
                        for (int i = 0; i < 8; i++) {
                            const int r = 4 * i + lane / 8, c = lane % 8;
                            const float4 f = turn[r * 8 + (c ^ (r & 7))];
                            if (quad * 32 + r < mine)
                                *reinterpret_cast<float4 *>(w.o + (at - lane + r) * D + c0 + 4 * c) = f;
                        }
                        __syncwarp();
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

static PFN_cuTensorMapEncodeTiled_v12000 tensor_map_encoder() {
    void *ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
        return nullptr;
    return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(ptr);
}

// {key heads x D, rows} of a bf16 cache in boxes of 64 dims x `box` rows, 128-byte swizzle.
static bool cache_map(CUtensorMap *m, const void *ptr, int cols, long long rows, long long stride, int box) {
    static const PFN_cuTensorMapEncodeTiled_v12000 encode = tensor_map_encoder();
    if (!encode) return false;
    const cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, 1};
    const cuuint64_t strides[2] = {(cuuint64_t)stride * 2, (cuuint64_t)stride * 2 * (cuuint64_t)rows};
    const cuuint32_t extent[3] = {64, (cuuint32_t)box, 1}, steps[3] = {1, 1, 1};
    return encode(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void *>(ptr), dims, strides, extent, steps,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int D>
static int launch_d(const attn::prefix::Params &p, const attn::prefix::Part &w, cudaStream_t s) {
    using namespace attn::ptile;
    if (!ensure_smem_attr((const void *)prefix_tile_kernel<D>, Cfg<D>::SMEM))
        return set_error(ATTN_ERR_CUDA, "prefix decode: cannot set shared-memory size");
    // A step is BN / box boxes; a box of the swizzled layout begins on 8 rows.
    CUtensorMap tk = {}, tv = {};
    const int box = std::min(1 << p.log_page, BN);
    const long long rows = (long long)p.n_pages << p.log_page;
    const bool maps = box >= 8 && cache_map(&tk, p.k, p.kv_heads * D, rows, p.row_stride, box) &&
                      cache_map(&tv, p.v, p.kv_heads * D, rows, p.row_stride, box);
    return check_pdl(launch_pdl(prefix_tile_kernel<D>, dim3(w.teams), dim3(kThreads), Cfg<D>::SMEM, s, tk, tv, p, w,
                                maps ? BN / box : 0),
                     "prefix_tile_kernel");
}

int launch_prefix_tile(const attn::prefix::Params &p, const attn::prefix::Part &w, int d, cudaStream_t s) {
    return d == 64 ? launch_d<64>(p, w, s) : launch_d<128>(p, w, s);
}

}  // namespace attn_host
