// Softmax attention forward on the 5th-gen tensor cores (sm_100a).
//
// A work unit is 256 queries of one head (two tiles of 128) against a range
// of its keys, walked 128 at a time with a running maximum and sum:
//   S_t = Q_t K'   (128 x 128, fp32 in tensor memory)
//   P_t = exp2(S_t c - m)      c = scale log2(e)
//   O_t += P_t V   (P_t as 16-bit operand in tensor memory, over S_t)
// The two tiles share every K and V tile and alternate: while one tile's
// softmax runs on the CUDA cores, the other's two products run on the tensor
// core.  At D = 128 the two sides take about as long as each other.
//
// Bound: a tile's softmax.  Its 16384 exponentials, maxima and conversions take
// the four warps of a tile about as long as the tensor core needs for both
// products, and a step ends with whichever is later.  Measured, bf16: 2 x 6144
// tokens, 32 heads of 128, 925 to 960 us (1290 to 1338 TFLOP/s, a library product
// reaches 1672); heads of 64, where the products take half as long and the
// exponentials do not, 820 us (752 TFLOP/s; 1030 on another card).  Tensor pipe
// active 58% of the time at heads of 128, 31% at 64, the exponential unit 68 and 74%.
//
// P enters its product in the tensors' 16-bit type, as the tensor core takes it;
// its row sum is taken in fp32 before that rounding.
//
// The running maximum lags: O is rescaled only when a row's maximum outgrows
// the one in use by 2^8, which leaves every term below 2^8 (exact in the fp32
// sums' range) and makes rescaling rare.  S_t(j) is issued behind PV_t(j-1) by
// the same thread, so its completion also means that O_t may be rescaled.
//
// Warps: 0-3 and 4-7 softmax and output of tile 0 and 1 (a thread a row),
// 8 loads, 9 and 10 issue the tiles' MMAs.
// TMEM: S0, S1, O0, O1, 128 columns each.  Persistent, one CTA per SM.
#pragma once
#include "attn_common.cuh"

namespace reels {

constexpr int AF_THREADS = 32 * 12;
using AfRegisters = AtRegisters<224>;

template <int DP>
struct AttnFwdGeom {
    static constexpr int TILE = AT_TILE * DP * 2;
    static constexpr int NST = DP == 128 ? 5 : 8;  // K and V tiles in flight
    static constexpr int KV_OFF = 2 * TILE;
    static constexpr int BAR_OFF = KV_OFF + NST * TILE;
    // q_full[2], q_empty[2], s_full[2], p_full[2][2], o_full[2], o_empty[2], mma_done[2], turn[2], raw, kv_full, kv_empty
    static constexpr int NBAR = 19 + 2 * NST;
    static constexpr int MISC_OFF = BAR_OFF + NBAR * 8;
    static constexpr int SMEM_BYTES = MISC_OFF + 16 + 1024;
    static_assert(SMEM_BYTES <= 232448, "shared memory plan exceeds 227 KB");
};

struct AttnUnit {
    int b, h, hk, q0, tiles, split;
    int k0, kn;  // first key, keys (0: nothing to do but write the empty result)
    int nk;      // key tiles
};

// Unit u: query tile pairs fastest, so that neighbouring CTAs read the same keys.
// Each role decodes a unit while it ends the one before, so that no unit begins
// with the divisions and the load of its length (32760 queries over 384 keys, 12
// heads, replayed from a graph: 111 to 106 us).
__device__ __forceinline__ AttnUnit attn_unit(const AttnArgs &a, long long unit) {
    const unsigned pairs = (unsigned)(a.Sq + 2 * AT_TILE - 1) / (2 * AT_TILE);
    unsigned u = (unsigned)unit;  // the host keeps units below 2^31
    AttnUnit w;
    w.q0 = (int)(u % pairs) * 2 * AT_TILE;
    u /= pairs;
    w.h = (int)(u % (unsigned)a.H);
    u /= (unsigned)a.H;
    w.b = (int)(u % (unsigned)a.B);
    w.split = (int)(u / (unsigned)a.B);
    w.hk = (int)((unsigned)w.h / (unsigned)(a.H / a.HK));
    w.tiles = a.Sq - w.q0 > AT_TILE ? 2 : 1;
    const int len = attn_keys(a, w.b);
    int end;
    w.k0 = attn_split(a, len, w.split, end);
    w.kn = end - w.k0;
    w.nk = (w.kn + AT_TILE - 1) / AT_TILE;
    return w;
}

template <int DT, int DP>
__global__ void __launch_bounds__(AF_THREADS, 1)
    attn_fwd_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                    const __grid_constant__ CUtensorMap tmV, const AttnArgs a, const long long units) {
    using G = AttnFwdGeom<DP>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const uint32_t sbase = smem_u32(smem);
    uint64_t *bars = reinterpret_cast<uint64_t *>(smem + G::BAR_OFF);
    uint64_t *q_full = bars, *q_empty = bars + 2, *s_full = bars + 4, *p_full = bars + 6, *o_full = bars + 10,
             *o_empty = bars + 12, *mma_done = bars + 14, *turn = bars + 16, *raw = bars + 18, *kv_full = bars + 19,
             *kv_empty = bars + 19 + G::NST;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(smem + G::MISC_OFF);
    volatile int *abort = reinterpret_cast<volatile int *>(smem + G::MISC_OFF + 4);
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int t = 0; t < 2; ++t) {
            mbar_init(&q_full[t], 1);
            mbar_init(&q_empty[t], 1);
            mbar_init(&s_full[t], 1);
            mbar_init(&p_full[2 * t], 4);
            mbar_init(&p_full[2 * t + 1], 4);
            mbar_init(&turn[t], 1);
            mbar_init(&mma_done[t], 1);
            mbar_init(&o_full[t], 1);
            mbar_init(&o_empty[t], 4);
        }
        mbar_init(raw, 1);
        for (int s = 0; s < G::NST; ++s) {
            mbar_init(&kv_full[s], 1);
            mbar_init(&kv_empty[s], 2);
        }
        *abort = 0;
        fence_mbar_init();
    }
    if (warp == 8) {
        if (lane == 0) {
            tma_prefetch_desc(&tmQ);
            tma_prefetch_desc(&tmK);
            tma_prefetch_desc(&tmV);
        }
        __syncwarp();
        tmem_alloc(tmem_slot, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    griddep_wait();

    if (warp == 8) {
        // ------------------------------------------------------------ loads
        AfRegisters::fewer();
        uint32_t g = 0, qn[2] = {0, 0}, nraw = 0;
        bool good = true;
        AttnUnit next = attn_unit(a, blockIdx.x);
        for (long long u = blockIdx.x; u < units && good; u += gridDim.x) {
            const AttnUnit w = next;
            next = attn_unit(a, min(u + gridDim.x, units - 1));
            if (w.nk == 0) continue;
            auto load_q = [&](int t) {
                good = good && at_wait(&q_empty[t], (qn[t] & 1) ^ 1, abort, a.err, DEVERR_TIMEOUT_AB_EMPTY);
                if (!good) return;
                ++qn[t];
                if (lane == 0) {
                    mbar_arrive_expect_tx(&q_full[t], G::TILE);
                    at_load_tile<DP>(sbase + t * G::TILE, &tmQ, w.q0 + t * AT_TILE, w.h, w.b, &q_full[t]);
                }
            };
            auto load_kv = [&](int j, bool is_v) {
                const int s = g % G::NST;
                good = good && at_wait(&kv_empty[s], ((g / G::NST) & 1) ^ 1, abort, a.err, DEVERR_TIMEOUT_W_EMPTY);
                if (!good) return;
                ++g;
                // keys behind the range: zeroed in V (in K they only make scores that are replaced)
                const int rows = w.kn - j * AT_TILE;
                const bool fix = is_v && rows < AT_TILE && w.k0 + w.kn < a.Sk;
                const uint32_t dst = sbase + G::KV_OFF + s * G::TILE;
                uint64_t *bar = fix ? raw : &kv_full[s];
                if (lane == 0) {
                    mbar_arrive_expect_tx(bar, G::TILE);
                    at_load_tile<DP>(dst, is_v ? &tmV : &tmK, w.k0 + j * AT_TILE, w.hk, w.b, bar);
                }
                if (fix) {
                    good = at_wait(raw, nraw++ & 1, abort, a.err, DEVERR_TIMEOUT_W_FULL);
                    at_zero_rows<DP>(smem + G::KV_OFF + s * G::TILE, rows);
                    if (lane == 0) mbar_arrive(&kv_full[s]);
                }
            };
            load_q(0);
            load_kv(0, false);
            if (w.tiles == 2) load_q(1);
            load_kv(0, true);
            for (int j = 1; j < w.nk && good; ++j) {
                load_kv(j, false);
                load_kv(j, true);
            }
        }
    } else if (warp == 11) {
        AfRegisters::fewer();  // idle: completes the third group of four warps
    } else if (warp > 8) {
        // -------------------------------------------------------------- MMAs
        // An issuer for each tile, so that one's waits run beside the other's
        // products, and in turn: products of both tiles issued side by side
        // would share the tensor core and end together, and then both
        // softmaxes would run, and wait, at the same time.
        AfRegisters::fewer();
        const int t = warp - 9;
        const bool leader = at_elect();
        constexpr int ab = DT == DT_BF16 ? 1 : 0;
        constexpr uint32_t id_s = idesc_f16(ab, 0, 0, 128, AT_TILE), id_o = idesc_f16(ab, 0, 1, 128, DP);
        const uint32_t S = tmem + t * 128, O = tmem + 256 + t * 128;
        const uint64_t Q = at_desc_k(sbase + t * G::TILE), k0 = at_desc_k(sbase + G::KV_OFF),
                       v0 = at_desc_mn(sbase + G::KV_OFF);
        uint32_t g = 0, np = 0, nu = 0, nt = 0;
        bool good = true;
        auto wait = [&](uint64_t *bar, uint32_t parity, unsigned code) {
            good = good && at_wait(bar, parity, abort, a.err, code);
        };
        auto wait_kv = [&](uint32_t i) { wait(&kv_full[i % G::NST], (i / G::NST) & 1, DEVERR_TIMEOUT_W_FULL); };
        auto scores = [&](uint32_t i) {
            const uint64_t K = k0 + (i % G::NST) * (G::TILE / 16);
            if (leader) {
#pragma unroll
                for (int kk = 0; kk < DP / 16; ++kk)
                    mma_f16_ss(S, Q + at_step_k(kk), K + at_step_k(kk), id_s, kk > 0);
                mma_commit(&s_full[t]);
                mma_commit(&kv_empty[i % G::NST]);
            }
        };
        auto take_turn = [&](bool two) {
            if (two) wait(&turn[t], (nt & 1) ^ (t == 0), DEVERR_TIMEOUT_ACC);
        };
        auto pass_turn = [&](bool two) {
            if (!two) return;
            if (leader) mbar_arrive(&turn[t ^ 1]);
            ++nt;
        };
        AttnUnit next = attn_unit(a, blockIdx.x);
        for (long long u = blockIdx.x; u < units && good; u += gridDim.x) {
            const AttnUnit w = next;
            next = attn_unit(a, min(u + gridDim.x, units - 1));
            if (w.nk == 0) continue;
            const bool two = w.tiles == 2;
            if (t >= w.tiles) {  // no second tile: only pass the ring on
                for (int j = 0; j < 2 * w.nk && good; ++j, ++g) {
                    wait_kv(g);
                    if (leader && good) mbar_arrive(&kv_empty[g % G::NST]);
                }
                continue;
            }
            wait(&q_full[t], nu & 1, DEVERR_TIMEOUT_AB_FULL);
            wait_kv(g);
            take_turn(two);
            if (!good) break;
            tc_fence_after();
            scores(g);
            pass_turn(two);
            for (int j = 0; j < w.nk; ++j, g += 2) {
                const int sv = (g + 1) % G::NST;
                const bool more = j + 1 < w.nk;
                const uint64_t V = v0 + sv * (G::TILE / 16);
                if (leader && !more) mma_commit(&q_empty[t]);  // the last scores were issued
                wait_kv(g + 1);
                if (more) wait_kv(g + 2);
                if (j == 0) wait(&o_empty[t], (nu & 1) ^ 1, DEVERR_TIMEOUT_ACC);
                // O += P V, each half of P when it is there
                wait(&p_full[2 * t], np & 1, DEVERR_TIMEOUT_ACC);
                take_turn(two);
                if (!good) break;
                tc_fence_after();
                if (leader) {
#pragma unroll
                    for (int kk = 0; kk < 4; ++kk)
                        at_mma_ts(O, S + kk * 8, V + at_step_mn(kk), id_o, j > 0 || kk > 0);
                }
                wait(&p_full[2 * t + 1], np++ & 1, DEVERR_TIMEOUT_ACC);
                if (!good) break;
                tc_fence_after();
                if (leader) {
#pragma unroll
                    for (int kk = 4; kk < AT_TILE / 16; ++kk) at_mma_ts(O, S + kk * 8, V + at_step_mn(kk), id_o, 1);
                    mma_commit(more ? &kv_empty[sv] : &o_full[t]);
                    if (!more) mma_commit(&kv_empty[sv]);
                }
                if (more) scores(g + 2);
                pass_turn(two);
            }
            ++nu;
        }
        if (leader) mma_commit(&mma_done[t]);
    } else {
        // ------------------------------------------------- softmax and output
        AfRegisters::more();
        const int t = warp >> 2;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t S = tmem + t * 128 + lanes, O = tmem + 256 + t * 128 + lanes;
        const float c = a.scale * CUDART_L2E_F;
        const F2 c2 = F2(c, c);
        const bool sectors = at_sectors(a.out, a.D);
        uint32_t ns = 0, nu = 0;
        bool good = true;
        AttnUnit next = attn_unit(a, blockIdx.x);
        for (long long u = blockIdx.x; u < units && good; u += gridDim.x) {
            const AttnUnit w = next;
            if (t >= w.tiles) {
                next = attn_unit(a, min(u + gridDim.x, units - 1));
                continue;
            }
            const int row = w.q0 + t * AT_TILE + (warp & 3) * 32 + lane;
            float m = 0.0f, l = 0.0f;  // m: the maximum in use, in log2 units, less the fp16 shift
            for (int j = 0; j < w.nk; ++j) {
                good = at_wait(&s_full[t], ns++ & 1, abort, a.err, DEVERR_TIMEOUT_ACC);
                if (!good) break;
                tc_fence_after();
                uint32_t s[AT_TILE];
#pragma unroll
                for (int i = 0; i < 4; ++i) at_tmem_ld32(S + 32 * i, s + 32 * i);
                tmem_wait_ld();
                const int rows = w.kn - j * AT_TILE;
                if (rows < AT_TILE) {
#pragma unroll
                    for (int i = 0; i < AT_TILE; ++i)
                        if (i >= rows) s[i] = 0xff800000u;  // -inf
                }
                float mx[8];
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    mx[i] = at_max3(__uint_as_float(s[i]), __uint_as_float(s[i + 8]), __uint_as_float(s[i + 16]));
#pragma unroll
                for (int i = 24; i < 120; i += 16)
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        mx[e] = at_max3(mx[e], __uint_as_float(s[i + e]), __uint_as_float(s[i + 8 + e]));
#pragma unroll
                for (int e = 0; e < 8; ++e) mx[e] = fmaxf(mx[e], __uint_as_float(s[120 + e]));
                mx[0] = at_max3(mx[0], mx[1], mx[2]);
                mx[3] = at_max3(mx[3], mx[4], mx[5]);
                // Scores of -infinity alone have no maximum: the lowest number stands for it,
                // below every live tile's (0 would cost a row of low scores its sum), and
                // still leaves exp2(-inf - m) = 0.
                const float top = fmaxf(fmaxf(at_max3(mx[0], mx[3], mx[6]), mx[7]) * c, -CUDART_MAX_NORMAL_F) -
                                  AtRange<DT>::FWD_SHIFT;
                if (j == 0) m = top;
                else if (__any_sync(0xffffffffu, top - m > 8.0f)) {
                    const float to = top - m > 8.0f ? top : m, keep = at_exp2(m - to);
                    m = to;
                    l *= keep;
#pragma unroll
                    for (int i = 0; i < DP / 32; ++i) {
                        uint32_t o[32];
                        at_tmem_ld32(O + 32 * i, o);
                        tmem_wait_ld();
#pragma unroll
                        for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * keep);
                        at_tmem_st32(O + 32 * i, o);
                    }
                }
                const F2 m2 = F2(-m, -m);
                F2 sum[2] = {F2(0.0f, 0.0f), F2(0.0f, 0.0f)};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    uint32_t p[16];
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const float2 u = fma2(at_pair(s + 32 * i, e), c2, m2).get();
                        const F2 v = F2(at_exp2(u.x), at_exp2(u.y));
                        p[e] = at_pack<DT>(v);
                        sum[e & 1] = add2(sum[e & 1], v);
                    }
                    at_tmem_st16(S + 16 * i, p);
                    if (i & 1) {  // half of P: its products may start
                        at_tmem_wait_st();
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&p_full[2 * t + (i >> 1)]);
                    }
                }
                const float2 total = add2(sum[0], sum[1]).get();
                l += total.x + total.y;
            }
            if (!good) break;
            next = attn_unit(a, min(u + gridDim.x, units - 1));
            const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
            const float lse = w.nk > 0 ? (m + log2f(l)) * CUDART_LN2_F : -CUDART_INF_F;
            const long long at = ((long long)w.split * a.B + w.b) * a.H + w.h;
            const bool in = row < a.Sq;
            if (in) (a.splits > 1 ? a.part_lse : a.lse)[at * a.Sq + row] = lse;
            if (w.nk > 0) {
                good = at_wait(&o_full[t], nu++ & 1, abort, a.err, DEVERR_TIMEOUT_ACC);
                if (!good) break;
                tc_fence_after();
            }
            typename Elem<DT>::T *out = reinterpret_cast<typename Elem<DT>::T *>(a.out) +
                                        (((long long)w.b * a.Sq + row) * a.H + w.h) * a.D;
            float *part = a.splits > 1 ? a.part_o + (at * a.Sq + row) * a.D : nullptr;
            uint32_t o[DP];
            if (w.nk > 0) {
#pragma unroll
                for (int i = 0; i < DP / 32; ++i) at_tmem_ld32(O + 32 * i, o + 32 * i);
                tmem_wait_ld();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&o_empty[t]);
            } else {
#pragma unroll
                for (int e = 0; e < DP; ++e) o[e] = 0u;
            }
            if (in) {
#pragma unroll
                for (int i = 0; i < DP / 32; ++i)
                    at_store32<DT>(o + 32 * i, inv, out, part, 32 * i, a.D, sectors);
            }
            __syncwarp();
        }
    }

    if (*abort) {  // give the copies in flight time to land before the CTA's shared memory goes
        for (int i = 0; i < 64; ++i) __nanosleep(2000);
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 8) at_finish(tmem, mma_done, 2, a.err);
}

}  // namespace reels
