// Gradient of softmax attention on the 5th-gen tensor cores (sm_100a): the
// probabilities are recomputed from q, k and the forward's L.
//
//   P = exp2(c S - L2)                 c = scale log2(e), L2 = L log2(e)
//   dS = P (dP - delta),  dP = dO V',  delta = rowsum(dO * O)
//   dV = P' dO,   dK = scale dS' Q,   dQ = scale dS K
//
// Two walks, each a sum in a fixed order with no atomics, so repeated calls
// give the same bits: one over the queries of a key tile (dK, dV; four products
// a step), one over the keys of a query tile (dQ; three).  Seven products where
// one walk with scattered sums of dQ would need five.
//
// Bound: the chain of a step (scores, exponentials, dS, products) with the two
// groups of warps taking turns on it.  Measured, 2 x 6144 tokens, 32 heads of 128,
// bf16: dK and dV 1.80 ms (4 products, 1374 TFLOP/s), dQ 1.34 ms (3, 1385), of
// which five of the seven are the least there is (990 TFLOP/s of those).
//
// P and dS enter their products in the tensors' 16-bit type; that rounding (half
// a step, independent from term to term) and the result's own make an error of
// sqrt(2) times the latter.  delta is taken from the forward's rounded out, as
// the caller has it, in fp32, which makes it 1.5 for dQ.  (dS in two parts, what
// its rounding leaves as a second operand: 1.1, and 12% more time for forward and
// backward of 2 x 6144 tokens, 32 heads of 128.)
//
// Registers: 216 a thread for the elementwise warps; beyond them the compiler
// keeps 20 to 40 bytes a thread of dK, dV and of dQ at heads of 128 in local memory.
//
// In both, the second product's operand (P', dS', dS) is written by the CUDA
// cores into tensor memory over the scores it came from, which the issuing
// thread overwrites only behind that product.
#pragma once
#include "attn_common.cuh"

namespace reels {

constexpr int AB_THREADS = 32 * 12;  // 8 elementwise warps, loads, MMA issue, two idle
using AbRegisters = AtRegisters<216>;

// fp16: exponent e with |dS| 2^e <= 2^15, from |dP|, |delta| <= |dO row| |v row|:
// `top` is the largest |dO row| times the largest |v row| of what shares e.
// That is a sample's key head for dK, whose sums run over the rows, and a row
// for dQ.  (What lies 2^-40 and more below the bound rounds to 0.)
template <int DT>
__device__ __forceinline__ int attn_grad_exp(float top) {
    if (DT != DT_F16 || !(top > 1e-30f) || !(top < 1e30f)) return 0;
    return 13 - ilogbf(top);
}

// ------------------------------------------------------------ dK and dV
// Unit: a tile of 128 keys of one key head and a range of the walk over the
// query tiles of the heads that share it.  Everything is computed transposed
// (lanes are keys):
//   S' = K Q',  dP' = V dO'   (128 x 128),   dV += P' dO,  dK += dS' Q
// TMEM: S'/P', dP'/dS', dV, dK, 128 columns each.  The elementwise warps come
// in two groups, one per 64 queries; each overwrites its own half of S' with
// its half of P' (columns 0.. and 64..).
template <int DP>
struct AttnKvGeom {
    static constexpr int TILE = AT_TILE * DP * 2;
    static constexpr int NST = DP == 128 ? 2 : 4;
    static constexpr int STAGE = 2 * TILE;        // Q and dO
    static constexpr int RING_OFF = 2 * TILE;     // behind K and V
    static constexpr int STAT_OFF = RING_OFF + NST * STAGE;  // per stage: L2[128], delta[128]
    static constexpr int BAR_OFF = STAT_OFF + NST * 1024;
    // kv_full, kv_empty, s_full, p_full, dp_full, ds_full, acc_full, acc_empty, mma_done; q_full, q_empty, g_full, g_empty
    static constexpr int NBAR = 9 + 4 * NST;
    static constexpr int MISC_OFF = BAR_OFF + NBAR * 8;
    static constexpr int SMEM_BYTES = MISC_OFF + 16 + 1024;
    static_assert(SMEM_BYTES <= 232448, "shared memory plan exceeds 227 KB");
};

struct AttnKvUnit {
    int b, hk, k0, rows, split;  // rows: keys of the tile before the sample's length
    int it0, n;                  // steps: head it / nqt of the group, query tile it % nqt
};

__device__ __forceinline__ AttnKvUnit attn_kv_unit(const AttnArgs &a, long long u) {
    const int kt = (a.Sk + AT_TILE - 1) / AT_TILE;
    AttnKvUnit w;
    w.k0 = (int)(u % kt) * AT_TILE;
    u /= kt;
    w.hk = (int)(u % a.HK);
    u /= a.HK;
    w.b = (int)(u % a.B);
    w.split = (int)(u / a.B);
    const int total = a.H / a.HK * (a.Sqp / AT_TILE), per = (total + a.red_splits - 1) / a.red_splits;
    w.rows = min(AT_TILE, attn_keys(a, w.b) - w.k0);
    w.it0 = min(total, w.split * per);
    w.n = w.rows > 0 ? min(total, w.it0 + per) - w.it0 : 0;
    return w;
}

template <int DT, int DP>
__device__ __forceinline__ void attn_dkdv(const CUtensorMap &tmQ, const CUtensorMap &tmK, const CUtensorMap &tmV,
                                          const CUtensorMap &tmG, const AttnArgs &a, uint8_t *smem, long long u0,
                                          long long units, unsigned step) {
    using G = AttnKvGeom<DP>;
    const uint32_t sbase = smem_u32(smem);
    uint64_t *bars = reinterpret_cast<uint64_t *>(smem + G::BAR_OFF);
    uint64_t *kv_full = bars, *kv_empty = bars + 1, *s_full = bars + 2, *p_full = bars + 3, *dp_full = bars + 4,
             *ds_full = bars + 5, *acc_full = bars + 6, *acc_empty = bars + 7, *mma_done = bars + 8,
             *q_full = bars + 9, *q_empty = q_full + G::NST, *g_full = q_empty + G::NST, *g_empty = g_full + G::NST;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(smem + G::MISC_OFF);
    volatile int *abort = reinterpret_cast<volatile int *>(smem + G::MISC_OFF + 4);
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        mbar_init(kv_full, 1);
        mbar_init(kv_empty, 1);
        mbar_init(s_full, 1);
        mbar_init(p_full, 8);
        mbar_init(dp_full, 1);
        mbar_init(ds_full, 8);
        mbar_init(acc_full, 1);
        mbar_init(acc_empty, 8);
        mbar_init(mma_done, 1);
        for (int s = 0; s < G::NST; ++s) {
            mbar_init(&q_full[s], 1);
            mbar_init(&q_empty[s], 1);
            mbar_init(&g_full[s], 1);
            mbar_init(&g_empty[s], 1);
        }
        *abort = 0;
        fence_mbar_init();
    }
    if (warp == 8) {
        if (lane == 0) {
            tma_prefetch_desc(&tmQ);
            tma_prefetch_desc(&tmK);
            tma_prefetch_desc(&tmV);
            tma_prefetch_desc(&tmG);
        }
        __syncwarp();
        tmem_alloc(tmem_slot, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    const int nqt = a.Sqp / AT_TILE, group = a.H / a.HK;

    if (warp == 8) {
        // ------------------------------------------------------------ loads
        AbRegisters::fewer();
        if (lane == 0) {
            uint32_t g = 0, nu = 0;
            bool good = true;
            for (long long u = u0; u < units && good; u += step) {
                const AttnKvUnit w = attn_kv_unit(a, u);
                if (w.n == 0) continue;
                good = wait_bar(kv_empty, (nu++ & 1) ^ 1, abort, a.err, DEVERR_TIMEOUT_W_EMPTY);
                if (!good) break;
                mbar_arrive_expect_tx(kv_full, 2 * G::TILE);
                at_load_tile<DP>(sbase, &tmK, w.k0, w.hk, w.b, kv_full);
                at_load_tile<DP>(sbase + G::TILE, &tmV, w.k0, w.hk, w.b, kv_full);
                for (int i = 0; i < w.n; ++i, ++g) {
                    const int it = w.it0 + i, h = w.hk * group + it / nqt, q0 = it % nqt * AT_TILE;
                    const int s = g % G::NST;
                    const uint32_t ph = ((g / G::NST) & 1) ^ 1;
                    const uint32_t dst = sbase + G::RING_OFF + s * G::STAGE, st = sbase + G::STAT_OFF + s * 1024;
                    const long long at = ((long long)w.b * a.H + h) * a.Sqp + q0;
                    good = wait_bar(&q_empty[s], ph, abort, a.err, DEVERR_TIMEOUT_AB_EMPTY);
                    if (!good) break;
                    mbar_arrive_expect_tx(&q_full[s], G::TILE + 1024);
                    at_load_tile<DP>(dst, &tmQ, q0, h, w.b, &q_full[s]);
                    bulk_load(st, a.stat_l + at, 512, &q_full[s]);
                    bulk_load(st + 512, a.stat_d + at, 512, &q_full[s]);
                    good = wait_bar(&g_empty[s], ph, abort, a.err, DEVERR_TIMEOUT_AB_EMPTY);
                    if (!good) break;
                    mbar_arrive_expect_tx(&g_full[s], G::TILE);
                    at_load_tile<DP>(dst + G::TILE, &tmG, q0, h, w.b, &g_full[s]);
                }
            }
        }
    } else if (warp > 9) {
        AbRegisters::fewer();  // idle: completes the third group of four warps
    } else if (warp == 9) {
        // -------------------------------------------------------------- MMAs
        // In turn: dV(i), S'(i+1) run under the elementwise dS(i), and dK(i),
        // dP'(i+1) under the exponentials of step i+1.
        AbRegisters::fewer();
        const bool leader = at_elect();
        constexpr int ab = DT == DT_BF16 ? 1 : 0;
        constexpr uint32_t id_s = idesc_f16(ab, 0, 0, 128, AT_TILE), id_o = idesc_f16(ab, 0, 1, 128, DP);
        const uint64_t kv0 = at_desc_k(sbase), in0 = at_desc_k(sbase + G::RING_OFF),
                       mn0 = at_desc_mn(sbase + G::RING_OFF);
        uint32_t g = 0, np = 0, nu = 0;
        bool good = true;
        // which = 0: S' = K Q', 1: dP' = V dO'
        auto scores = [&](int which, uint32_t i) {
            const int s = i % G::NST;
            good = good && at_wait(which ? &g_full[s] : &q_full[s], (i / G::NST) & 1, abort, a.err,
                                   DEVERR_TIMEOUT_AB_FULL);
            if (!good) return;
            tc_fence_after();
            const uint64_t A = kv0 + which * (G::TILE / 16), B = in0 + s * (G::STAGE / 16) + which * (G::TILE / 16);
            if (leader) {
#pragma unroll
                for (int kk = 0; kk < DP / 16; ++kk)
                    mma_f16_ss(tmem + 128 * which, A + at_step_k(kk), B + at_step_k(kk), id_s, kk > 0);
                mma_commit(which ? dp_full : s_full);
            }
        };
        // which = 0: dV += P' dO, 1: dK += dS' Q
        auto mix = [&](int which, uint32_t i, bool first) {
            const int s = i % G::NST;
            good = good && at_wait(which ? ds_full : p_full, np & 1, abort, a.err, DEVERR_TIMEOUT_ACC);
            if (!good) return;
            tc_fence_after();
            const uint32_t S = tmem + 128 * which, O = tmem + 256 + 128 * which;
            const uint64_t B = mn0 + s * (G::STAGE / 16) + (which ^ 1) * (G::TILE / 16);
            if (leader) {
#pragma unroll
                for (int kk = 0; kk < AT_TILE / 16; ++kk)
                    at_mma_ts(O, S + (kk >> 2) * 64 + (kk & 3) * 8, B + at_step_mn(kk), id_o, !first || kk > 0);
                mma_commit(which ? &q_empty[s] : &g_empty[s]);  // dK is the last to read Q, dV dO
            }
        };
        for (long long u = u0; u < units && good; u += step) {
            const AttnKvUnit w = attn_kv_unit(a, u);
            if (w.n == 0) continue;
            good = at_wait(kv_full, nu & 1, abort, a.err, DEVERR_TIMEOUT_W_FULL);
            scores(0, g);
            scores(1, g);
            if (good) good = at_wait(acc_empty, (nu & 1) ^ 1, abort, a.err, DEVERR_TIMEOUT_ACC);
            for (int i = 0; i < w.n && good; ++i, ++g, ++np) {
                mix(0, g, i == 0);
                if (i + 1 < w.n) scores(0, g + 1);
                mix(1, g, i == 0);
                if (i + 1 < w.n) scores(1, g + 1);
                else if (leader) mma_commit(kv_empty), mma_commit(acc_full);
            }
            ++nu;
        }
        if (leader) mma_commit(mma_done);
    } else {
        // --------------------------------------------- P', dS' and the output
        AbRegisters::more();
        const int half = warp >> 2;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t S = tmem + lanes + 64 * half, DS = S + 128, O = tmem + lanes + 256 + 128 * half;
        const float c = a.scale * CUDART_L2E_F;
        const F2 c2 = F2(c, c);
        uint32_t g = 0, ns = 0, nu = 0;
        bool good = true;
        for (long long u = u0; u < units && good; u += step) {
            const AttnKvUnit w = attn_kv_unit(a, u);
            int e = 0;
            if (DT == DT_F16) {
                const float2 r = __ldcg(a.range + (long long)w.b * a.HK + w.hk);
                e = attn_grad_exp<DT>(r.x * r.y);
            }
            const float g1 = exp2f((float)e - AtRange<DT>::BWD_SHIFT);
            const F2 grow = F2(g1, g1);
            const float f = half ? a.scale * exp2f(-(float)e) : exp2f(-AtRange<DT>::BWD_SHIFT);
            const int row = (warp & 3) * 32 + lane;
            const bool live = row < w.rows;
            for (int i = 0; i < w.n; ++i, ++g, ++ns) {
                const int s = g % G::NST;
                const uint32_t L = sbase + G::STAT_OFF + s * 1024 + half * 256, Dl = L + 512;
                good = at_wait(&q_full[s], (g / G::NST) & 1, abort, a.err, DEVERR_TIMEOUT_AB_FULL) &&
                       at_wait(s_full, ns & 1, abort, a.err, DEVERR_TIMEOUT_ACC);
                if (!good) break;
                tc_fence_after();
                uint32_t x[64];
                at_tmem_ld32(S, x);
                at_tmem_ld32(S + 32, x + 32);
                tmem_wait_ld();
                uint32_t p[32];
#pragma unroll
                for (int k = 0; k < 32; k += 2) {
                    const float4 l = ld_shared_f4(L + 8 * k);
                    const float2 u = fma2(at_pair(x, k), c2, F2(l.x, l.y)).get();
                    const float2 v = fma2(at_pair(x, k + 1), c2, F2(l.z, l.w)).get();
                    x[2 * k] = __float_as_uint(at_exp2(u.x)), x[2 * k + 1] = __float_as_uint(at_exp2(u.y));
                    x[2 * k + 2] = __float_as_uint(at_exp2(v.x)), x[2 * k + 3] = __float_as_uint(at_exp2(v.y));
                    p[k] = at_pack<DT>(at_pair(x, k)), p[k + 1] = at_pack<DT>(at_pair(x, k + 1));
                }
                if (w.rows < AT_TILE && !live) {
#pragma unroll
                    for (int k = 0; k < 32; ++k) p[k] = 0u;
                }
                at_tmem_st32(S, p);
                at_tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(p_full);
                good = at_wait(dp_full, ns & 1, abort, a.err, DEVERR_TIMEOUT_ACC);
                if (!good) break;
                tc_fence_after();
                uint32_t y[64];
                at_tmem_ld32(DS, y);
                at_tmem_ld32(DS + 32, y + 32);
                tmem_wait_ld();
#pragma unroll
                for (int k = 0; k < 32; k += 2) {
                    const float4 d = ld_shared_f4(Dl + 8 * k);
                    F2 u = mul2(at_pair(x, k), add2(at_pair(y, k), F2(d.x, d.y)));
                    F2 v = mul2(at_pair(x, k + 1), add2(at_pair(y, k + 1), F2(d.z, d.w)));
                    if (DT == DT_F16) u = mul2(u, grow), v = mul2(v, grow);
                    p[k] = at_pack<DT>(u), p[k + 1] = at_pack<DT>(v);
                }
                if (w.rows < AT_TILE && !live) {
#pragma unroll
                    for (int k = 0; k < 32; ++k) p[k] = 0u;
                }
                at_tmem_st32(DS, p);
                at_tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(ds_full);
            }
            if (!good) break;
            if (w.n > 0) {
                good = at_wait(acc_full, nu++ & 1, abort, a.err, DEVERR_TIMEOUT_ACC);
                if (!good) break;
                tc_fence_after();
            }
            const int t = w.k0 + row;
            const long long at = (((long long)w.b * a.Sk + t) * a.HK + w.hk) * a.D;
            float *part = a.red_splits > 1
                              ? (half ? a.part_k : a.part_v) + (long long)w.split * a.B * a.Sk * a.HK * a.D + at
                              : nullptr;
            auto *dst = reinterpret_cast<typename Elem<DT>::T *>(half ? a.dk : a.dv) + at;
            const bool sectors = at_sectors(half ? a.dk : a.dv, a.D);
#pragma unroll
            for (int i = 0; i < DP / 32; ++i) {
                uint32_t o[32];
                if (w.n > 0) {
                    at_tmem_ld32(O + 32 * i, o);
                    tmem_wait_ld();
                }
                if (i == DP / 32 - 1 && w.n > 0) {
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(acc_empty);
                }
                if (w.n == 0 || !live) {
#pragma unroll
                    for (int k = 0; k < 32; ++k) o[k] = 0u;
                }
                if (t < a.Sk) at_store32<DT>(o, f, dst, part, 32 * i, a.D, sectors);
                __syncwarp();
            }
        }
    }

    if (*abort) {
        for (int i = 0; i < 64; ++i) __nanosleep(2000);
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 8) at_finish(tmem, mma_done, 1, a.err);
}

// Adds the partial dK (blockIdx.y = 0) and dV of the split walk in order.
template <int DT>
__global__ void __launch_bounds__(256) attn_sum_kernel(const AttnArgs a, long long n, int splits) {
    griddep_wait();
    const float *part = blockIdx.y ? a.part_v : a.part_k;
    void *out = blockIdx.y ? a.dv : a.dk;
    for (long long i = 4ll * (blockIdx.x * 256ll + threadIdx.x); i < n; i += 1024ll * gridDim.x) {
        float4 s = __ldcg(reinterpret_cast<const float4 *>(part + i));
        for (int k = 1; k < splits; ++k) {
            const float4 v = __ldcg(reinterpret_cast<const float4 *>(part + k * n + i));
            s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
        }
        *reinterpret_cast<uint2 *>(reinterpret_cast<typename Elem<DT>::T *>(out) + i) =
            make_uint2(Elem<DT>::pack2(s.x, s.y), Elem<DT>::pack2(s.z, s.w));
    }
}

// ------------------------------------------------------------------- dQ
// Unit: a tile of 128 queries of one head, walking the keys 128 at a time:
//   S = Q K',  dP = dO V'   (128 x 128),   dQ += dS K
// TMEM: S twice (the scores of the next tile are ready when this one's dS is
// written), dP/dS, dQ.
template <int DP>
struct AttnQGeom {
    static constexpr int TILE = AT_TILE * DP * 2;
    static constexpr int NK = DP == 128 ? 3 : 5, NV = DP == 128 ? 2 : 4;  // tiles in flight
    static constexpr int K_OFF = 2 * TILE;  // behind Q and dO
    static constexpr int V_OFF = K_OFF + NK * TILE;
    static constexpr int BAR_OFF = V_OFF + NV * TILE;
    // q_full, q_empty, s_full[2], s_empty[2], dp_full, ds_full, acc_full, acc_empty, raw, mma_done; rings
    static constexpr int NBAR = 12 + 2 * (NK + NV);
    static constexpr int MISC_OFF = BAR_OFF + NBAR * 8;
    static constexpr int SMEM_BYTES = MISC_OFF + 16 + 1024;
    static_assert(SMEM_BYTES <= 232448, "shared memory plan exceeds 227 KB");
};

struct AttnQUnit {
    int b, h, hk, q0, len, nk;
};
__device__ __forceinline__ AttnQUnit attn_q_unit(const AttnArgs &a, long long u) {
    const int qt = a.Sqp / AT_TILE;
    AttnQUnit w;
    w.q0 = (int)(u % qt) * AT_TILE;
    u /= qt;
    w.h = (int)(u % a.H);
    w.b = (int)(u / a.H);
    w.hk = w.h / (a.H / a.HK);
    w.len = attn_keys(a, w.b);
    w.nk = (w.len + AT_TILE - 1) / AT_TILE;
    return w;
}

template <int DT, int DP>
__device__ __forceinline__ void attn_dq(const CUtensorMap &tmQ, const CUtensorMap &tmK, const CUtensorMap &tmV,
                                        const CUtensorMap &tmG, const AttnArgs &a, uint8_t *smem, long long u0,
                                        long long units, unsigned step) {
    using G = AttnQGeom<DP>;
    const uint32_t sbase = smem_u32(smem);
    uint64_t *bars = reinterpret_cast<uint64_t *>(smem + G::BAR_OFF);
    uint64_t *q_full = bars, *q_empty = bars + 1, *s_full = bars + 2, *s_empty = bars + 4, *dp_full = bars + 6,
             *ds_full = bars + 7, *acc_full = bars + 8, *acc_empty = bars + 9, *raw = bars + 10, *mma_done = bars + 11,
             *k_full = bars + 12, *k_empty = k_full + G::NK, *v_full = k_empty + G::NK, *v_empty = v_full + G::NV;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(smem + G::MISC_OFF);
    volatile int *abort = reinterpret_cast<volatile int *>(smem + G::MISC_OFF + 4);
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        mbar_init(q_full, 1);
        mbar_init(q_empty, 1);
        for (int s = 0; s < 2; ++s) {
            mbar_init(&s_full[s], 1);
            mbar_init(&s_empty[s], 8);
        }
        mbar_init(dp_full, 1);
        mbar_init(ds_full, 8);
        mbar_init(acc_full, 1);
        mbar_init(acc_empty, 8);
        mbar_init(mma_done, 1);
        mbar_init(raw, 1);
        for (int s = 0; s < G::NK; ++s) {
            mbar_init(&k_full[s], 1);
            mbar_init(&k_empty[s], 1);
        }
        for (int s = 0; s < G::NV; ++s) {
            mbar_init(&v_full[s], 1);
            mbar_init(&v_empty[s], 1);
        }
        *abort = 0;
        fence_mbar_init();
    }
    if (warp == 8) {
        if (lane == 0) {
            tma_prefetch_desc(&tmQ);
            tma_prefetch_desc(&tmK);
            tma_prefetch_desc(&tmV);
            tma_prefetch_desc(&tmG);
        }
        __syncwarp();
        tmem_alloc(tmem_slot, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    if (warp == 8) {
        // ------------------------------------------------------------ loads
        AbRegisters::fewer();
        uint32_t g = 0, nu = 0, nraw = 0;
        bool good = true;
        for (long long u = u0; u < units && good; u += step) {
            const AttnQUnit w = attn_q_unit(a, u);
            if (w.nk == 0) continue;
            good = at_wait(q_empty, (nu++ & 1) ^ 1, abort, a.err, DEVERR_TIMEOUT_AB_EMPTY);
            if (!good) break;
            if (lane == 0) {
                mbar_arrive_expect_tx(q_full, 2 * G::TILE);
                at_load_tile<DP>(sbase, &tmQ, w.q0, w.h, w.b, q_full);
                at_load_tile<DP>(sbase + G::TILE, &tmG, w.q0, w.h, w.b, q_full);
            }
            for (int j = 0; j < w.nk; ++j, ++g) {
                const int s = g % G::NK, t = g % G::NV;
                good = at_wait(&k_empty[s], ((g / G::NK) & 1) ^ 1, abort, a.err, DEVERR_TIMEOUT_W_EMPTY);
                if (!good) break;
                // keys behind the length: zeroed in K (in V they only make values that are replaced)
                const int rows = w.len - j * AT_TILE;
                const bool fix = rows < AT_TILE && w.len < a.Sk;
                uint64_t *bar = fix ? raw : &k_full[s];
                if (lane == 0) {
                    mbar_arrive_expect_tx(bar, G::TILE);
                    at_load_tile<DP>(sbase + G::K_OFF + s * G::TILE, &tmK, j * AT_TILE, w.hk, w.b, bar);
                }
                if (fix) {
                    good = at_wait(raw, nraw++ & 1, abort, a.err, DEVERR_TIMEOUT_W_FULL);
                    at_zero_rows<DP>(smem + G::K_OFF + s * G::TILE, rows);
                    if (lane == 0) mbar_arrive(&k_full[s]);
                }
                good = good && at_wait(&v_empty[t], ((g / G::NV) & 1) ^ 1, abort, a.err, DEVERR_TIMEOUT_W_EMPTY);
                if (!good) break;
                if (lane == 0) {
                    mbar_arrive_expect_tx(&v_full[t], G::TILE);
                    at_load_tile<DP>(sbase + G::V_OFF + t * G::TILE, &tmV, j * AT_TILE, w.hk, w.b, &v_full[t]);
                }
            }
        }
    } else if (warp > 9) {
        AbRegisters::fewer();  // idle: completes the third group of four warps
    } else if (warp == 9) {
        // -------------------------------------------------------------- MMAs
        // In turn: dQ(j), dP(j+1), S(j+2); the scores run two tiles ahead of
        // the elementwise warps' dS.
        AbRegisters::fewer();
        const bool leader = at_elect();
        constexpr int ab = DT == DT_BF16 ? 1 : 0;
        constexpr uint32_t id_s = idesc_f16(ab, 0, 0, 128, AT_TILE), id_o = idesc_f16(ab, 0, 1, 128, DP);
        const uint32_t DS = tmem + 256, O = tmem + 384;
        const uint64_t Q = at_desc_k(sbase), dO = at_desc_k(sbase + G::TILE), k0 = at_desc_k(sbase + G::K_OFF),
                       v0 = at_desc_k(sbase + G::V_OFF), mn0 = at_desc_mn(sbase + G::K_OFF);
        uint32_t g = 0, nu = 0, np = 0;
        bool good = true;
        auto scores = [&](uint32_t i) {
            const int s = i % G::NK, t = i & 1;
            good = good && at_wait(&k_full[s], (i / G::NK) & 1, abort, a.err, DEVERR_TIMEOUT_W_FULL) &&
                   at_wait(&s_empty[t], ((i >> 1) & 1) ^ 1, abort, a.err, DEVERR_TIMEOUT_ACC);
            if (!good) return;
            tc_fence_after();
            const uint64_t K = k0 + s * (G::TILE / 16);
            if (leader) {
#pragma unroll
                for (int kk = 0; kk < DP / 16; ++kk)
                    mma_f16_ss(tmem + 128 * t, Q + at_step_k(kk), K + at_step_k(kk), id_s, kk > 0);
                mma_commit(&s_full[t]);
            }
        };
        auto grads = [&](uint32_t i) {  // dP
            const int t = i % G::NV;
            good = good && at_wait(&v_full[t], (i / G::NV) & 1, abort, a.err, DEVERR_TIMEOUT_W_FULL);
            if (!good) return;
            tc_fence_after();
            const uint64_t V = v0 + t * (G::TILE / 16);
            if (leader) {
#pragma unroll
                for (int kk = 0; kk < DP / 16; ++kk)
                    mma_f16_ss(DS, dO + at_step_k(kk), V + at_step_k(kk), id_s, kk > 0);
                mma_commit(dp_full);
                mma_commit(&v_empty[t]);
            }
        };
        for (long long u = u0; u < units && good; u += step) {
            const AttnQUnit w = attn_q_unit(a, u);
            if (w.nk == 0) continue;
            good = at_wait(q_full, nu & 1, abort, a.err, DEVERR_TIMEOUT_AB_FULL);
            scores(g);
            grads(g);
            if (w.nk > 1) scores(g + 1);
            if (good) good = at_wait(acc_empty, (nu & 1) ^ 1, abort, a.err, DEVERR_TIMEOUT_ACC);
            for (int j = 0; j < w.nk && good; ++j, ++g, ++np) {
                const int s = g % G::NK;
                good = at_wait(ds_full, np & 1, abort, a.err, DEVERR_TIMEOUT_ACC);
                if (!good) break;
                tc_fence_after();
                const uint64_t K = mn0 + s * (G::TILE / 16);
                if (leader) {
#pragma unroll
                    for (int kk = 0; kk < AT_TILE / 16; ++kk)
                        at_mma_ts(O, DS + (kk >> 2) * 64 + (kk & 3) * 8, K + at_step_mn(kk), id_o, j > 0 || kk > 0);
                    mma_commit(&k_empty[s]);  // dQ is the last to read K
                }
                if (j + 1 < w.nk) grads(g + 1);
                else if (leader) mma_commit(q_empty), mma_commit(acc_full);
                if (j + 2 < w.nk) scores(g + 2);
            }
            ++nu;
        }
        if (leader) mma_commit(mma_done);
    } else {
        // ----------------------------------------------------- dS and the output
        AbRegisters::more();
        const int half = warp >> 2;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t DS = tmem + lanes + 256 + 64 * half, O = tmem + lanes + 384;
        const float c = a.scale * CUDART_L2E_F;
        const F2 c2 = F2(c, c);
        uint32_t g = 0, nu = 0;
        bool good = true;
        for (long long u = u0; u < units && good; u += step) {
            const AttnQUnit w = attn_q_unit(a, u);
            const int row = w.q0 + (warp & 3) * 32 + lane;
            const long long st = ((long long)w.b * a.H + w.h) * a.Sqp + row;
            const float sl = __ldcg(a.stat_l + st), sd = __ldcg(a.stat_d + st);
            const F2 L = F2(sl, sl), delta = F2(sd, sd);
            int e = 0;
            if (DT == DT_F16)
                e = attn_grad_exp<DT>(__ldcg(a.stat_n + st) * __ldcg(a.range + (long long)w.b * a.HK + w.hk).y);
            const float g1 = exp2f((float)e - AtRange<DT>::BWD_SHIFT), f = a.scale * exp2f(-(float)e);
            const F2 grow = F2(g1, g1);
            for (int j = 0; j < w.nk; ++j, ++g) {
                const int t = g & 1;
                good = at_wait(&s_full[t], (g >> 1) & 1, abort, a.err, DEVERR_TIMEOUT_ACC);
                if (!good) break;
                tc_fence_after();
                uint32_t x[64];
                at_tmem_ld32(tmem + lanes + 128 * t + 64 * half, x);
                at_tmem_ld32(tmem + lanes + 128 * t + 64 * half + 32, x + 32);
                tmem_wait_ld();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&s_empty[t]);
#pragma unroll
                for (int k = 0; k < 32; ++k) {
                    const float2 u = fma2(at_pair(x, k), c2, L).get();
                    x[2 * k] = __float_as_uint(at_exp2(u.x)), x[2 * k + 1] = __float_as_uint(at_exp2(u.y));
                }
                good = at_wait(dp_full, g & 1, abort, a.err, DEVERR_TIMEOUT_ACC);
                if (!good) break;
                tc_fence_after();
                uint32_t y[64];
                at_tmem_ld32(DS, y);
                at_tmem_ld32(DS + 32, y + 32);
                tmem_wait_ld();
                const int rows = w.len - j * AT_TILE - 64 * half;
                uint32_t p[32];
#pragma unroll
                for (int k = 0; k < 32; ++k) {
                    F2 u = mul2(at_pair(x, k), add2(at_pair(y, k), delta));
                    if (DT == DT_F16) u = mul2(u, grow);
                    p[k] = at_pack<DT>(u);
                }
                if (rows < 64) {
#pragma unroll
                    for (int k = 0; k < 32; ++k) {  // keys 2k, 2k + 1
                        if (2 * k >= rows) p[k] = 0u;
                        else if (2 * k + 1 >= rows) p[k] &= 0xffffu;
                    }
                }
                at_tmem_st32(DS, p);
                at_tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(ds_full);
            }
            if (!good) break;
            if (w.nk > 0) {
                good = at_wait(acc_full, nu++ & 1, abort, a.err, DEVERR_TIMEOUT_ACC);
                if (!good) break;
                tc_fence_after();
            }
            // the two groups of warps write half of the features each
            auto *dst = reinterpret_cast<typename Elem<DT>::T *>(a.dq) +
                        (((long long)w.b * a.Sq + row) * a.H + w.h) * a.D;
            const bool sectors = at_sectors(a.dq, a.D);
            const int c0 = half * (DP / 2);
            uint32_t o[DP / 2];
            if (w.nk > 0) {
#pragma unroll
                for (int i = 0; i < DP / 64; ++i) at_tmem_ld32(O + c0 + 32 * i, o + 32 * i);
                tmem_wait_ld();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(acc_empty);
            } else {
#pragma unroll
                for (int k = 0; k < DP / 2; ++k) o[k] = 0u;
            }
            if (row < a.Sq) {
#pragma unroll
                for (int i = 0; i < DP / 64; ++i)
                    at_store32<DT>(o + 32 * i, f, dst, nullptr, c0 + 32 * i, a.D, sectors);
            }
            __syncwarp();
        }
    }

    if (*abort) {
        for (int i = 0; i < 64; ++i) __nanosleep(2000);
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 8) at_finish(tmem, mma_done, 1, a.err);
}

// One launch for both: kv_blocks blocks for the units of dK and dV, the long
// ones, then blocks for those of dQ, which fill the SMs that come free.  A block
// takes every kv_blocks-th unit (likewise for dQ), so that blocks running side by
// side are at neighbouring units and read the same keys or queries from L2 (a
// run of neighbouring units for each block instead: 3213 to 3460 us at
// 2 x 6144 tokens, 32 heads).
template <int DP>
struct AttnBwdGeom {
    static constexpr int SMEM_BYTES = AttnKvGeom<DP>::SMEM_BYTES > AttnQGeom<DP>::SMEM_BYTES
                                          ? AttnKvGeom<DP>::SMEM_BYTES
                                          : AttnQGeom<DP>::SMEM_BYTES;
};
struct AttnBwdUnits {
    long long kv, q;  // units
    unsigned kv_blocks;
};

// PART: 0 both, 1 dK and dV alone, 2 dQ alone (large calls, where nothing is
// left to even out and each walk compiled by itself is 2% faster).
template <int DT, int DP, int PART>
__global__ void __launch_bounds__(AB_THREADS, 1)
    attn_bwd_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                    const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CUtensorMap tmG, const AttnArgs a,
                    const AttnBwdUnits n) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    griddep_wait();
    if constexpr (PART == 1) attn_dkdv<DT, DP>(tmQ, tmK, tmV, tmG, a, smem, blockIdx.x, n.kv, gridDim.x);
    else if constexpr (PART == 2) attn_dq<DT, DP>(tmQ, tmK, tmV, tmG, a, smem, blockIdx.x, n.q, gridDim.x);
    else if (blockIdx.x < n.kv_blocks)
        attn_dkdv<DT, DP>(tmQ, tmK, tmV, tmG, a, smem, blockIdx.x, n.kv, n.kv_blocks);
    else
        attn_dq<DT, DP>(tmQ, tmK, tmV, tmG, a, smem, blockIdx.x - n.kv_blocks, n.q, gridDim.x - n.kv_blocks);
}

}  // namespace reels
