// Host side of the block's attention stretch: argument checks, plans and
// launches of the q/k norm with rotary positions (norm_rope.cuh) and of
// softmax attention and its gradient (attn_fwd.cuh, attn_bwd.cuh,
// attn_simt.cuh), behind the C ABI of include/reels_lowvram.h.
#include <algorithm>
#include <atomic>
#include <cmath>
#include <mutex>
#include <type_traits>

#include "../../include/reels_lowvram.h"
#include "attn_bwd.cuh"
#include "attn_fwd.cuh"
#include "host.h"
#include "norm_rope.cuh"

using namespace reels;

namespace {

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
size_t up256(size_t x) { return (x + 255) & ~size_t(255); }
bool known_dtype(int dt) { return dt == REELS_F32 || dt == REELS_F16 || dt == REELS_BF16; }
int bytes_of(int dt) { return dt == REELS_F32 ? 4 : 2; }
bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

template <typename F>
void with_dtype(int dt, F &&f) {
    if (dt == REELS_BF16) f(std::integral_constant<int, DT_BF16>{});
    else if (dt == REELS_F16) f(std::integral_constant<int, DT_F16>{});
    else f(std::integral_constant<int, DT_F32>{});
}

#define RA_LAUNCH(expr)                                                                              \
    do {                                                                                             \
        cudaError_t e_ = (expr);                                                                     \
        if (e_ == cudaSuccess) e_ = cudaGetLastError();                                              \
        if (e_ != cudaSuccess) return host_fail_dev(std::string("kernel launch: ") + cudaGetErrorString(e_)); \
        host_count_launch();                                                                         \
    } while (0)

// ------------------------------------------------------- norm and rotation
int check_norm_rope(const void *x, int64_t M, int64_t heads, int64_t D, const reels_rope *rope, int64_t tps, float eps,
                    int dt) {
    if (M < 0 || heads <= 0 || D <= 0 || heads > NR_MAX_C || D > NR_MAX_C || heads * D > NR_MAX_C)
        return host_fail("rms_norm_rope needs 0 <= M and 0 < heads * head_dim <= " + std::to_string(NR_MAX_C));
    if (!x && M > 0) return host_fail("null x");
    if (tps <= 0 || tps > INT32_MAX) return host_fail("tokens_per_sample must be positive");
    if (!(eps >= 0.0f) || !std::isfinite(eps)) return host_fail("epsilon must be finite and non-negative");
    if (!known_dtype(dt)) return host_fail("unknown act_dtype");
    if (!rope) return REELS_OK;
    if (!rope->table) return host_fail("null rotary table");
    if ((reinterpret_cast<uintptr_t>(rope->table) & 7) != 0) return host_fail("the rotary table must be 8-byte aligned");
    if (D & 1) return host_fail("rotary positions need an even head_dim");
    int64_t feats = 0, entries = 0, grid = 1;
    for (int i = 0; i < NR_AXES; ++i) {
        if (rope->size[i] <= 0 || rope->dim[i] < 0 || (rope->dim[i] & 1))
            return host_fail("a rotary axis needs a positive size and an even number of features");
        feats += rope->dim[i];
        entries += (int64_t)rope->size[i] * (rope->dim[i] / 2);
        grid *= rope->size[i];
        if (entries > INT32_MAX || grid > INT32_MAX) return host_fail("the rotary table is too large");
    }
    if (feats != D) return host_fail("the rotary axes' features must sum to head_dim");
    if (rope->pairing != REELS_ROPE_INTERLEAVED && rope->pairing != REELS_ROPE_HALF)
        return host_fail("unknown rotary pairing");
    return REELS_OK;
}

constexpr int kNormRopeSmem = 220 * 1024;  // of an SM's 228 KB, 1 KB a block is the system's

template <int DT, bool BWD, bool ROPE, bool HALF, int UPT, bool W32>
cudaError_t launch_norm_rope(const NormRopeArgs &a, int threads, const HostCall &call, cudaStream_t st) {
    static_assert(!(BWD && UPT == 2) && !(W32 && (!BWD || DT == DT_F32)), "a form that no call takes");
    // Blocks that fit beside each other with a ring of at least two rows, then
    // as many rows as the shared memory holds.
    const int budget = kNormRopeSmem, fixed = nr_smem_bytes(a.C, bytes_of(DT), BWD, W32, 0, a.D) + 1024;
    const int step = a.C * bytes_of(DT) * (BWD ? 2 : 1);
    const int blocks = std::max(1, std::min({(UPT == 1 ? 1024 : UPT == 2 ? 768 : 256) / threads, 24, budget / (fixed + 2 * step)}));
    const int stages = std::max(2, std::min(NR_STAGES, (budget / blocks - fixed) / step));  // (two rows were checked to fit)
    const int smem = nr_smem_bytes(a.C, bytes_of(DT), BWD, W32, stages, a.D);
    auto kern = norm_rope_kernel<DT, BWD, ROPE, HALF, UPT, W32>;
    // the most any call asks for, once per device: calls of several threads agree on it
    static std::atomic<uint64_t> ready{0};
    if (!(ready.load() >> call.device & 1)) {
        cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kNormRopeSmem);
        if (e != cudaSuccess) return e;
        ready.fetch_or(uint64_t(1) << call.device);
    }
    const dim3 grid((unsigned)std::min<int64_t>(a.M, (int64_t)call.sms * blocks));
    return host_launch_pdl(kern, grid, dim3((unsigned)threads), smem, st, a, stages);
}

int norm_rope(const void *x, const void *dout, bool bwd, int64_t M, int64_t heads, int64_t D, const void *weight,
              const reels_rope *rope, int64_t tps, float eps, int dt, void *out, void *stream) {
    const bool w32 = (dt & REELS_NORM_WEIGHT_F32) != 0;
    dt &= ~REELS_NORM_WEIGHT_F32;
    int rc = check_norm_rope(x, M, heads, D, rope, tps, eps, dt);
    if (rc) return rc;
    if (M == 0) return host_ok(REELS_PATH_NONE);
    if (!out) return host_fail(bwd ? "null dx" : "null out");
    if (bwd && !dout) return host_fail("null dout");
    HostCall call;
    rc = call.bind(x);
    if (rc) return rc;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    NormRopeArgs a = {};
    a.x = x, a.dout = dout, a.weight = weight, a.w32 = w32, a.out = out;
    a.M = M, a.C = (int)(heads * D), a.D = (int)D, a.tps = (int)tps, a.eps = eps, a.inv_c = 1.0f / (float)a.C;
    a.err = call.status;
    if (rope) {
        a.table = reinterpret_cast<const float2 *>(rope->table);
        a.pos = rope->positions;
        for (int i = 0; i < NR_AXES; ++i) a.size[i] = rope->size[i], a.pairs[i] = rope->dim[i] / 2;
        a.half = rope->pairing == REELS_ROPE_HALF;
        a.by_hw = NrDivide::by((uint32_t)a.size[1] * (uint32_t)a.size[2]);
        a.by_w = NrDivide::by((uint32_t)a.size[2]);
    }
    const int64_t units = a.C / 16;
    const bool heads_fit = !rope || (D % 16 == 0 && 32 % (D / 16) == 0);
    const bool vec = a.C % 16 == 0 && heads_fit && aligned16(x) && aligned16(out) && aligned16(weight) &&
                     (!bwd || aligned16(dout)) &&
                     // two rows have to fit the shared memory beside the weight
                     nr_smem_bytes(a.C, bytes_of(dt), bwd, w32, 2, a.D) <= kNormRopeSmem;
    if (!vec) {
        const dim3 grid((unsigned)std::min<int64_t>(M, 8ll * call.sms));
        with_dtype(dt, [&](auto t) {
            constexpr int DT = decltype(t)::value;
            if (bwd) host_launch_pdl(norm_rope_any_kernel<DT, true>, grid, dim3(256), 0, st, a);
            else host_launch_pdl(norm_rope_any_kernel<DT, false>, grid, dim3(256), 0, st, a);
        });
        RA_LAUNCH(cudaSuccess);
        return host_ok(REELS_PATH_CUDACORE);
    }
    if (!rope) a.D = 16;
    // Units a thread, and a thread for each pair of a head.  Forward, two (the
    // angles, waits and sums are shared); backward one, whose registers leave
    // room for twice the warps: 8190 x 5120 forward 31 us with two and 37 with
    // one, backward 54 and 49.  Forward rows of up to 512 features fill no more
    // than a warp with one.  Past 512 units (8192 features) neither fits a
    // block: four.
    const int upt = units > 512 ? 4 : bwd || units <= 32 ? 1 : 2;
    const int threads = (int)ceil_div(std::max<int64_t>(ceil_div(units, upt), rope ? D / 2 : 1), 32) * 32;
    cudaError_t e = cudaSuccess;
    with_dtype(dt, [&](auto t) {
        constexpr int DT = decltype(t)::value;
        auto form = [&](auto b, auto r, auto h) {
            constexpr bool B = decltype(b)::value, R = decltype(r)::value, H = decltype(h)::value;
            if constexpr (B && DT != DT_F32)
                if (w32 && weight) {
                    e = upt == 1 ? launch_norm_rope<DT, B, R, H, 1, true>(a, threads, call, st)
                                 : launch_norm_rope<DT, B, R, H, 4, true>(a, threads, call, st);
                    return;
                }
            if (upt == 1) e = launch_norm_rope<DT, B, R, H, 1, false>(a, threads, call, st);
            else if (upt == 4) e = launch_norm_rope<DT, B, R, H, 4, false>(a, threads, call, st);
            else if constexpr (!B) e = launch_norm_rope<DT, B, R, H, 2, false>(a, threads, call, st);
        };
        auto dir = [&](auto b) {
            if (!rope) form(b, std::false_type{}, std::false_type{});
            else if (a.half) form(b, std::true_type{}, std::true_type{});
            else form(b, std::true_type{}, std::false_type{});
        };
        if (bwd) dir(std::true_type{});
        else dir(std::false_type{});
    });
    RA_LAUNCH(e);
    return host_ok(REELS_PATH_CUDACORE);
}

// ---------------------------------------------------------------- attention
constexpr int kPlanSms = 148;
constexpr int kStatBlocks = 8 * kPlanSms;  // most blocks of the statistics kernel

struct AttnPlan {
    bool tc = false;
    int few = 0;                     // > 0: rows of a key head, few enough for attn_rows_kernel (forward)
    int tile = 32;                   // of the CUDA-core kernels: 64 where the blocks fill the GPU twice
    int splits = 1, split_keys = 1;  // forward
    int red_splits = 1;              // backward, dK and dV
    int Sqp = 0;
};

bool tma_strides(const int64_t (&stride)[3], const int64_t (&n)[3]) {
    for (int i = 0; i < 3; ++i)
        if (n[i] > 1 && (stride[i] <= 0 || stride[i] % 8 != 0 || stride[i] >= (int64_t(1) << 38))) return false;
    return true;
}

int check_shape(const reels_attn_shape *s, int dt) {
    if (!s) return host_fail("null attention shape");
    if (s->batch < 0 || s->q_tokens < 0 || s->k_tokens < 0 || s->heads <= 0 || s->kv_heads <= 0)
        return host_fail("attention needs non-negative batch and tokens and positive heads");
    if (s->heads % s->kv_heads != 0) return host_fail("heads must be a multiple of kv_heads");
    if (s->head_dim <= 0 || s->head_dim > AT_MAX_D)
        return host_fail("head_dim must be between 1 and " + std::to_string(AT_MAX_D));
    const int64_t lim = INT32_MAX - 256;
    if (s->batch > lim || s->heads > lim || s->q_tokens > lim || s->k_tokens > lim ||
        s->batch * s->heads > lim || ceil_div(std::max(s->q_tokens, s->k_tokens), 32) > lim / 2 / std::max<int64_t>(1, s->batch * s->heads))
        return host_fail("attention shape too large");
    for (int i = 0; i < 3; ++i)
        if (s->q_stride[i] < 0 || s->k_stride[i] < 0 || s->v_stride[i] < 0) return host_fail("negative stride");
    if (!known_dtype(dt)) return host_fail("unknown act_dtype");
    return REELS_OK;
}

// The tensor-core kernels take 16-bit tensors, heads of up to 128 features in
// multiples of 8 (one 16-byte piece) and strides TMA can follow.
AttnPlan plan_attention(const reels_attn_shape &s, int dt, const void *q, const void *k, const void *v) {
    AttnPlan p;
    const int64_t nq[3] = {s.batch, s.q_tokens, s.heads}, nk[3] = {s.batch, s.k_tokens, s.kv_heads};
    p.tc = dt != REELS_F32 && s.head_dim % 8 == 0 && s.head_dim <= 128 && tma_strides(s.q_stride, nq) &&
           tma_strides(s.k_stride, nk) && tma_strides(s.v_stride, nk) && aligned16(q) && aligned16(k) && aligned16(v);
    p.Sqp = (int)(ceil_div(s.q_tokens, AT_TILE) * AT_TILE);
    const int64_t shared = s.q_tokens * (s.heads / s.kv_heads);
    if (p.tc && shared <= 8) p.few = (int)std::max<int64_t>(shared, 1);
    // Forward: few rows leave SMs idle, so the keys are split over them and
    // joined; a split keeps at least four tiles of keys (two on the CUDA cores).
    // Blocks beside each other on an SM: 1 of the tensor-core kernel, 2 of the
    // few-row kernel with one or two rows, 1 with more (their registers; planned
    // for two, the splits ran one behind the other: 8 rows over 32760 keys of 12
    // heads 104 us against 96, 4 rows 86.5 against 82.3), 4 others.
    if (s.head_dim <= 128 && ceil_div(s.q_tokens, 64) * s.batch * s.heads >= 2 * kPlanSms) p.tile = 64;
    const int tile = p.few ? 64 : p.tc ? AT_TILE : p.tile;
    const int64_t rows = p.few ? (int64_t)s.batch * s.kv_heads
                               : ceil_div(s.q_tokens, p.tc ? 2 * AT_TILE : p.tile) * s.batch * s.heads;
    const int64_t tiles = std::max<int64_t>(1, ceil_div(s.k_tokens, tile));
    int64_t want = rows > 0 ? std::min<int64_t>((p.few == 1 || p.few == 2 ? 2 : p.tc ? 1 : 4) * kPlanSms / rows, tiles / (p.tc ? 4 : 2)) : 1;
    want = std::max<int64_t>(1, std::min<int64_t>(want, 1024));
    const int64_t per = ceil_div(tiles, want);
    p.splits = (int)ceil_div(tiles, per);
    p.split_keys = (int)std::min<int64_t>(per * tile, INT32_MAX - 256);
    // Backward: one launch of the dK, dV walks and then the dQ walks, about 1.9
    // and 1.35 us a step of 128 features (only their ratio to the ends counts).  The first are split where a whole one would outlast the
    // average SM: the launch ends about half a unit behind the average, and the
    // partial sums pass through memory twice (about 5 TB/s) and a launch.
    if (p.tc && s.q_tokens > 0 && s.k_tokens > 0) {
        const double q_tiles = (double)(p.Sqp / AT_TILE), k_tiles = (double)ceil_div(s.k_tokens, AT_TILE);
        const int64_t steps = s.heads / s.kv_heads * (p.Sqp / AT_TILE);
        const double work = (double)(s.batch * s.heads) * q_tiles * k_tiles * (1.9 + 1.35) / kPlanSms;
        const double part = 2.0 * 2.0 * 4.0 * (double)(s.batch * s.k_tokens * s.kv_heads * s.head_dim) / 5e6;
        double best = 1e300;
        for (int64_t n = 1; n <= std::min<int64_t>(steps, 32); ++n) {
            const double unit = 1.9 * (double)ceil_div(steps, n) + 4.0;
            const double cost = std::max(work, unit) + 0.5 * unit + (n > 1 ? 4.0 + part * (double)n : 0.0);
            if (cost < best * 0.97) best = cost, p.red_splits = (int)n;
        }
        p.red_splits = (int)ceil_div(steps, ceil_div(steps, p.red_splits));
    }
    return p;
}

struct AttnWs {
    size_t part_o = 0, part_lse = 0, stat_l = 0, stat_d = 0, stat_n = 0, v_n = 0, range = 0, part_k = 0, part_v = 0,
           total = 0;
};
AttnWs attn_ws(const reels_attn_shape &s, const AttnPlan &p, int dt, bool bwd) {
    AttnWs w;
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t r = at;
        at += up256(bytes);
        return r;
    };
    if (!bwd) {
        if (p.splits > 1) {
            const size_t rows = (size_t)p.splits * s.batch * s.heads * s.q_tokens;
            w.part_o = take(rows * s.head_dim * 4);
            w.part_lse = take(rows * 4);
        }
    } else {
        const size_t rows = (size_t)s.batch * s.heads * p.Sqp;
        w.stat_l = take(rows * 4);
        w.stat_d = take(rows * 4);
        if (p.tc && dt == REELS_F16) {
            w.stat_n = take(rows * 4);
            w.v_n = take((size_t)s.batch * s.kv_heads * s.k_tokens * 4);
            w.range = take((size_t)s.batch * s.kv_heads * 8);
        }
        if (p.red_splits > 1) {
            const size_t n = (size_t)p.red_splits * s.batch * s.k_tokens * s.kv_heads * s.head_dim * 4;
            w.part_k = take(n);
            w.part_v = take(n);
        }
    }
    w.total = at;
    return w;
}

int check_workspace(const void *ws, size_t have, size_t need) {
    if (need == 0) return REELS_OK;
    if (!ws) return host_fail("null workspace; size it with reels_attention_workspace_bytes");
    if ((reinterpret_cast<uintptr_t>(ws) & 255u) != 0) return host_fail("workspace must be 256-byte aligned");
    if (have < need) return host_fail("workspace too small; size it with reels_attention_workspace_bytes");
    return REELS_OK;
}

AttnArgs attn_args(const reels_attn_shape &s, const AttnPlan &p, const void *q, const void *k, const void *v,
                   const int32_t *lengths, float scale) {
    AttnArgs a = {};
    a.q = q, a.k = k, a.v = v, a.lengths = lengths, a.scale = scale;
    for (int i = 0; i < 3; ++i) a.qs[i] = s.q_stride[i], a.ks[i] = s.k_stride[i], a.vs[i] = s.v_stride[i];
    a.B = (int)s.batch, a.H = (int)s.heads, a.HK = (int)s.kv_heads;
    a.Sq = (int)s.q_tokens, a.Sk = (int)s.k_tokens, a.D = (int)s.head_dim;
    a.splits = p.splits, a.split_keys = p.split_keys, a.red_splits = p.red_splits, a.Sqp = p.Sqp;
    return a;
}

// [batch][tokens][heads][D] by strides, boxes of 64 features x 128 tokens
int attn_map(CUtensorMap *tm, const void *base, int dt, int64_t B, int64_t S, int64_t H, int64_t D,
             const int64_t (&stride)[3]) {
    const uint64_t n[4] = {(uint64_t)D, (uint64_t)S, (uint64_t)H, (uint64_t)B};
    auto st = [&](int64_t n_, int64_t s_) { return (uint64_t)(n_ > 1 ? s_ : ceil_div(D, 8) * 8) * 2; };
    const uint64_t b[3] = {st(S, stride[1]), st(H, stride[2]), st(B, stride[0])};
    const uint32_t box[4] = {64, AT_TILE, 1, 1};
    return host_tmap_4d(tm, base, dt == REELS_BF16, n, b, box);
}

template <typename K>
cudaError_t big_smem(K kern, int bytes) {
    return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
}
template <int DT, int DP, int T>
cudaError_t simt_tile_attrs() {
    cudaError_t e = big_smem(attn_simt_fwd_kernel<DT, DP, T>, as_smem_bytes(DP, T, 3));
    if (e == cudaSuccess) e = big_smem(attn_simt_bwd_kernel<DT, DP, T>, as_smem_bytes(DP, T, 4));
    return e;
}
template <int DT, int DP>
cudaError_t simt_attrs() {
    cudaError_t e = simt_tile_attrs<DT, DP, 32>();
    if constexpr (DP <= 128)
        if (e == cudaSuccess) e = simt_tile_attrs<DT, DP, 64>();
    return e;
}
template <int DT, int DP>
cudaError_t tc_attrs() {
    cudaError_t e = big_smem(attn_fwd_kernel<DT, DP>, AttnFwdGeom<DP>::SMEM_BYTES);
    if (e == cudaSuccess) e = big_smem(attn_bwd_kernel<DT, DP, 0>, AttnBwdGeom<DP>::SMEM_BYTES);
    if (e == cudaSuccess) e = big_smem(attn_bwd_kernel<DT, DP, 1>, AttnBwdGeom<DP>::SMEM_BYTES);
    if (e == cudaSuccess) e = big_smem(attn_bwd_kernel<DT, DP, 2>, AttnBwdGeom<DP>::SMEM_BYTES);
    return e;
}
// Shared-memory sizes of the kernels, once per device (which is current).
int attn_ready(int device) {
    static std::mutex mu;
    static bool ready[64];
    std::lock_guard<std::mutex> lock(mu);
    if (ready[device]) return REELS_OK;
    cudaError_t e = cudaSuccess;
    auto also = [&](cudaError_t x) {
        if (e == cudaSuccess) e = x;
    };
    also(simt_attrs<DT_F32, 64>()), also(simt_attrs<DT_F32, 128>()), also(simt_attrs<DT_F32, 256>());
    also(simt_attrs<DT_F16, 64>()), also(simt_attrs<DT_F16, 128>()), also(simt_attrs<DT_F16, 256>());
    also(simt_attrs<DT_BF16, 64>()), also(simt_attrs<DT_BF16, 128>()), also(simt_attrs<DT_BF16, 256>());
    also(tc_attrs<DT_F16, 64>()), also(tc_attrs<DT_F16, 128>());
    also(tc_attrs<DT_BF16, 64>()), also(tc_attrs<DT_BF16, 128>());
    if (e != cudaSuccess) return host_fail_dev(std::string("cudaFuncSetAttribute: ") + cudaGetErrorString(e));
    ready[device] = true;
    return REELS_OK;
}

template <typename F>
void with_simt_dim(int64_t D, F &&f) {
    if (D <= 64) f(std::integral_constant<int, 64>{});
    else if (D <= 128) f(std::integral_constant<int, 128>{});
    else f(std::integral_constant<int, 256>{});
}
// The head size as the kernels' and the tile of the CUDA-core kernels.
template <typename F>
void with_simt_tile(int64_t D, int tile, F &&f) {
    using T32 = std::integral_constant<int, 32>;
    using T64 = std::integral_constant<int, 64>;
    if (D <= 64) tile == 64 ? f(std::integral_constant<int, 64>{}, T64{}) : f(std::integral_constant<int, 64>{}, T32{});
    else if (D <= 128)
        tile == 64 ? f(std::integral_constant<int, 128>{}, T64{}) : f(std::integral_constant<int, 128>{}, T32{});
    else f(std::integral_constant<int, 256>{}, T32{});
}
template <typename F>
void with_tc_type(int dt, int64_t D, F &&f) {
    auto dim = [&](auto t) {
        if (D <= 64) f(t, std::integral_constant<int, 64>{});
        else f(t, std::integral_constant<int, 128>{});
    };
    if (dt == REELS_BF16) dim(std::integral_constant<int, DT_BF16>{});
    else dim(std::integral_constant<int, DT_F16>{});
}

}  // namespace

extern "C" {

int reels_rms_norm_rope(const void *x, int64_t M, int64_t heads, int64_t head_dim, const void *weight,
                        const reels_rope *rope, int64_t tokens_per_sample, float epsilon, int act_dtype, void *out,
                        void *stream) {
    return norm_rope(x, nullptr, false, M, heads, head_dim, weight, rope, tokens_per_sample, epsilon, act_dtype, out,
                     stream);
}

int reels_rms_norm_rope_backward(const void *x, const void *dout, int64_t M, int64_t heads, int64_t head_dim,
                                 const void *weight, const reels_rope *rope, int64_t tokens_per_sample, float epsilon,
                                 int act_dtype, void *dx, void *stream) {
    return norm_rope(x, dout, true, M, heads, head_dim, weight, rope, tokens_per_sample, epsilon, act_dtype, dx,
                     stream);
}

size_t reels_attention_workspace_bytes(const reels_attn_shape *shape, int act_dtype, int pass) {
    if (check_shape(shape, act_dtype) != REELS_OK) return 0;
    // The larger of the two paths: which one runs also depends on the pointers.
    AttnPlan p = plan_attention(*shape, act_dtype, nullptr, nullptr, nullptr);
    size_t n = attn_ws(*shape, p, act_dtype, pass == REELS_PASS_BACKWARD).total;
    p = plan_attention(*shape, act_dtype, reinterpret_cast<const void *>(1), nullptr, nullptr);
    return std::max(n, attn_ws(*shape, p, act_dtype, pass == REELS_PASS_BACKWARD).total);
}

int reels_attention_plan(const reels_attn_shape *shape, int act_dtype, int64_t *info) {
    int rc = check_shape(shape, act_dtype);
    if (rc) return rc;
    if (!info) return host_fail("null info");
    const AttnPlan p = plan_attention(*shape, act_dtype, nullptr, nullptr, nullptr);
    info[0] = p.tc && !p.few ? REELS_PATH_TENSORCORE : REELS_PATH_CUDACORE;
    info[1] = p.splits;
    info[2] = p.split_keys;
    info[3] = p.red_splits;
    return host_ok(REELS_PATH_NONE);
}

int reels_attention_forward(const reels_attn_shape *shape, const void *q, const void *k, const void *v,
                            const int32_t *kv_lengths, float scale, int act_dtype, void *out, float *lse,
                            void *workspace, size_t ws_bytes, void *stream) {
    int rc = check_shape(shape, act_dtype);
    if (rc) return rc;
    const reels_attn_shape &s = *shape;
    if (!(scale > 0.0f) || !std::isfinite(scale)) return host_fail("scale must be finite and positive");
    if (s.batch == 0 || s.q_tokens == 0) return host_ok(REELS_PATH_NONE);
    if (!q || !out || !lse) return host_fail("null q, out or lse");
    if (s.k_tokens > 0 && (!k || !v)) return host_fail("null k or v");
    const AttnPlan p = plan_attention(s, act_dtype, q, k, v);
    const bool tc = p.tc && aligned16(out) && s.k_tokens > 0;
    AttnPlan plan = p;
    if (!tc && p.tc) plan = plan_attention(s, act_dtype, reinterpret_cast<const void *>(1), k, v);
    const AttnWs w = attn_ws(s, plan, act_dtype, false);
    rc = check_workspace(workspace, ws_bytes, w.total);
    if (rc) return rc;
    HostCall call;
    rc = call.bind(q);
    if (rc) return rc;
    rc = attn_ready(call.device);
    if (rc) return rc;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    AttnArgs a = attn_args(s, plan, q, k, v, kv_lengths, scale);
    a.out = out, a.lse = lse, a.err = call.status;
    if (plan.splits > 1) {
        a.part_o = reinterpret_cast<float *>(reinterpret_cast<char *>(workspace) + w.part_o);
        a.part_lse = reinterpret_cast<float *>(reinterpret_cast<char *>(workspace) + w.part_lse);
    }
    cudaError_t e = cudaSuccess;
    if (tc && plan.few) {
        const dim3 grid((unsigned)(s.batch * s.kv_heads), (unsigned)plan.splits);
        with_tc_type(act_dtype, s.head_dim, [&](auto t, auto d) {
            constexpr int DT = decltype(t)::value, G = decltype(d)::value / 8;
            if (plan.few == 1) e = host_launch_pdl(attn_rows_kernel<DT, G, 1>, grid, dim3(256), 0, st, a);
            else if (plan.few == 2) e = host_launch_pdl(attn_rows_kernel<DT, G, 2>, grid, dim3(256), 0, st, a);
            else if (plan.few <= 4) e = host_launch_pdl(attn_rows_kernel<DT, G, 4>, grid, dim3(256), 0, st, a);
            else e = host_launch_pdl(attn_rows_kernel<DT, G, 8>, grid, dim3(256), 0, st, a);
        });
    } else if (tc) {
        CUtensorMap mq, mk, mv;
        if ((rc = attn_map(&mq, q, act_dtype, s.batch, s.q_tokens, s.heads, s.head_dim, s.q_stride)) ||
            (rc = attn_map(&mk, k, act_dtype, s.batch, s.k_tokens, s.kv_heads, s.head_dim, s.k_stride)) ||
            (rc = attn_map(&mv, v, act_dtype, s.batch, s.k_tokens, s.kv_heads, s.head_dim, s.v_stride)))
            return rc;
        const long long units = ceil_div(s.q_tokens, 2 * AT_TILE) * s.batch * s.heads * plan.splits;
        with_tc_type(act_dtype, s.head_dim, [&](auto t, auto d) {
            constexpr int DT = decltype(t)::value, DP = decltype(d)::value;
            e = host_launch_pdl(attn_fwd_kernel<DT, DP>, dim3((unsigned)std::min<long long>(units, call.sms)),
                                dim3(AF_THREADS), AttnFwdGeom<DP>::SMEM_BYTES, st, mq, mk, mv, a, units);
        });
    } else {
        const dim3 grid((unsigned)(ceil_div(s.q_tokens, plan.tile) * s.batch * s.heads), (unsigned)plan.splits);
        with_dtype(act_dtype, [&](auto t) {
            with_simt_tile(s.head_dim, plan.tile, [&](auto d, auto tile) {
                constexpr int DT = decltype(t)::value, DP = decltype(d)::value, T = decltype(tile)::value;
                e = host_launch_pdl(attn_simt_fwd_kernel<DT, DP, T>, grid, dim3(AS_THREADS), as_smem_bytes(DP, T, 3),
                                    st, a);
            });
        });
    }
    RA_LAUNCH(e);
    if (plan.splits > 1) {
        const int64_t rows = s.batch * s.heads * s.q_tokens;
        with_dtype(act_dtype, [&](auto t) {
            with_simt_dim(s.head_dim, [&](auto d) {
                e = host_launch_pdl(attn_join_kernel<decltype(t)::value, decltype(d)::value / 32>,
                                    dim3((unsigned)std::min<int64_t>(ceil_div(rows, 4), 16ll * call.sms)), dim3(128), 0,
                                    st, a);
            });
        });
        RA_LAUNCH(e);
    }
    return host_ok(tc && !plan.few ? REELS_PATH_TENSORCORE : REELS_PATH_CUDACORE);
}

int reels_attention_backward(const reels_attn_shape *shape, const void *q, const void *k, const void *v,
                             const void *out, const float *lse, const void *dout, const int32_t *kv_lengths,
                             float scale, int act_dtype, void *dq, void *dk, void *dv, void *workspace,
                             size_t ws_bytes, void *stream) {
    int rc = check_shape(shape, act_dtype);
    if (rc) return rc;
    const reels_attn_shape &s = *shape;
    if (!(scale > 0.0f) || !std::isfinite(scale)) return host_fail("scale must be finite and positive");
    if (s.batch == 0 || (s.q_tokens == 0 && s.k_tokens == 0)) return host_ok(REELS_PATH_NONE);
    if (s.q_tokens > 0 && (!q || !out || !lse || !dout || !dq)) return host_fail("null q, out, lse, dout or dq");
    if (s.k_tokens > 0 && (!k || !v || !dk || !dv)) return host_fail("null k, v, dk or dv");
    HostCall call;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    if (s.q_tokens == 0 || s.k_tokens == 0) {  // nothing attends: zero gradients
        rc = call.bind(s.q_tokens ? dq : dk);
        if (rc) return rc;
        const size_t row = (size_t)s.head_dim * bytes_of(act_dtype);
        cudaError_t e = cudaSuccess;
        if (s.q_tokens) e = cudaMemsetAsync(dq, 0, (size_t)s.batch * s.q_tokens * s.heads * row, st);
        if (s.k_tokens) {
            e = cudaMemsetAsync(dk, 0, (size_t)s.batch * s.k_tokens * s.kv_heads * row, st);
            if (e == cudaSuccess) e = cudaMemsetAsync(dv, 0, (size_t)s.batch * s.k_tokens * s.kv_heads * row, st);
        }
        if (e != cudaSuccess) return host_fail_dev(std::string("cudaMemsetAsync: ") + cudaGetErrorString(e));
        return host_ok(REELS_PATH_NONE);
    }
    AttnPlan plan = plan_attention(s, act_dtype, q, k, v);
    if (plan.tc && !(aligned16(out) && aligned16(dout) && aligned16(dq) && aligned16(dk) && aligned16(dv)))
        plan = plan_attention(s, act_dtype, reinterpret_cast<const void *>(1), k, v);
    const AttnWs w = attn_ws(s, plan, act_dtype, true);
    rc = check_workspace(workspace, ws_bytes, w.total);
    if (rc) return rc;
    rc = call.bind(q);
    if (rc) return rc;
    rc = attn_ready(call.device);
    if (rc) return rc;
    char *ws = reinterpret_cast<char *>(workspace);
    AttnArgs a = attn_args(s, plan, q, k, v, kv_lengths, scale);
    a.out = const_cast<void *>(out), a.lse = const_cast<float *>(lse), a.dout = dout;
    a.dq = dq, a.dk = dk, a.dv = dv, a.err = call.status;
    float *stat_l = reinterpret_cast<float *>(ws + w.stat_l), *stat_d = reinterpret_cast<float *>(ws + w.stat_d);
    a.stat_l = stat_l, a.stat_d = stat_d;
    a.part_k = reinterpret_cast<float *>(ws + w.part_k), a.part_v = reinterpret_cast<float *>(ws + w.part_v);
    cudaError_t e = cudaSuccess;
    const int64_t rows = s.batch * s.heads * plan.Sqp, keys = s.batch * s.kv_heads * s.k_tokens;
    if (!plan.tc)
        with_dtype(act_dtype, [&](auto t) {
            e = host_launch_pdl(attn_stat_kernel<decltype(t)::value>,
                                dim3((unsigned)std::min<int64_t>(ceil_div(rows, 8), 8ll * call.sms)), dim3(256), 0, st,
                                a, stat_l, stat_d);
        });
    else
        with_tc_type(act_dtype, s.head_dim, [&](auto t, auto d) {
            constexpr int DT = decltype(t)::value, G = decltype(d)::value / 8;
            // for fp16 the rows of v are read too, and there may be many more of them
            const int64_t read = std::max(s.batch * s.q_tokens * s.heads, DT == DT_F16 ? keys : 0);
            const int64_t blocks = ceil_div(read, 256 / G * 4);
            float *stat_n = reinterpret_cast<float *>(ws + w.stat_n), *v_n = reinterpret_cast<float *>(ws + w.v_n);
            float2 *range = reinterpret_cast<float2 *>(ws + w.range);
            a.stat_n = stat_n, a.range = range;
            e = host_launch_pdl(attn_stat_vec_kernel<DT, G>, dim3((unsigned)std::min<int64_t>(blocks, kStatBlocks)),
                                dim3(256), 0, st, a, stat_l, stat_d, stat_n, v_n, AtRange<DT>::BWD_SHIFT);
            if (DT == DT_F16 && e == cudaSuccess) {
                host_count_launch();
                e = host_launch_pdl(attn_range_kernel, dim3((unsigned)(s.batch * s.kv_heads)), dim3(1024), 0, st, a,
                                    static_cast<const float *>(v_n), range);
            }
        });
    RA_LAUNCH(e);
    if (!plan.tc) {
        with_dtype(act_dtype, [&](auto t) {
            with_simt_tile(s.head_dim, plan.tile, [&](auto d, auto tile) {
                constexpr int DT = decltype(t)::value, DP = decltype(d)::value, T = decltype(tile)::value;
                const int64_t blocks =
                    ceil_div(s.k_tokens, T) * s.batch * s.kv_heads + ceil_div(s.q_tokens, T) * s.batch * s.heads;
                e = host_launch_pdl(attn_simt_bwd_kernel<DT, DP, T>, dim3((unsigned)blocks), dim3(AS_THREADS),
                                    as_smem_bytes(DP, T, 4), st, a);
            });
        });
        RA_LAUNCH(e);
        return host_ok(REELS_PATH_CUDACORE);
    }
    const int64_t og[3] = {s.q_tokens * s.heads * s.head_dim, s.heads * s.head_dim, s.head_dim};
    CUtensorMap mq, mk, mv, mg;
    if ((rc = attn_map(&mq, q, act_dtype, s.batch, s.q_tokens, s.heads, s.head_dim, s.q_stride)) ||
        (rc = attn_map(&mk, k, act_dtype, s.batch, s.k_tokens, s.kv_heads, s.head_dim, s.k_stride)) ||
        (rc = attn_map(&mv, v, act_dtype, s.batch, s.k_tokens, s.kv_heads, s.head_dim, s.v_stride)) ||
        (rc = attn_map(&mg, dout, act_dtype, s.batch, s.q_tokens, s.heads, s.head_dim, og)))
        return rc;
    AttnBwdUnits n = {};
    const int64_t q_tiles = plan.Sqp / AT_TILE, k_tiles = ceil_div(s.k_tokens, AT_TILE);
    n.kv = k_tiles * s.batch * s.kv_heads * plan.red_splits;
    n.q = q_tiles * s.batch * s.heads;
    // A block's start and end take some 3 us.  With many units of each kind a
    // block stays on its SM and the walks are launched one after the other (both
    // ways measured at 2 x 6144 tokens, 32 heads: 3160 us, against 3274 together
    // in blocks of two units); with few, blocks of about 32 steps of both let
    // the SMs even out (8190 queries over 512 keys, 40 heads: 352 us together,
    // 381 one by one).
    const bool apart = std::min(n.kv, n.q) >= 8ll * call.sms;
    const int64_t fill = ceil_div(n.kv + n.q, call.sms);
    auto blocks_of = [&](int64_t units, int64_t steps) {
        return ceil_div(units, std::max<int64_t>(1, std::min<int64_t>(32 / std::max<int64_t>(steps, 1), fill)));
    };
    n.kv_blocks = (unsigned)blocks_of(n.kv, ceil_div(s.heads / s.kv_heads * q_tiles, plan.red_splits));
    const int64_t blocks = n.kv_blocks + blocks_of(n.q, k_tiles);
    with_tc_type(act_dtype, s.head_dim, [&](auto t, auto d) {
        constexpr int DT = decltype(t)::value, DP = decltype(d)::value, SM = AttnBwdGeom<DP>::SMEM_BYTES;
        const dim3 block(AB_THREADS), all((unsigned)call.sms);
        if (apart) {
            e = host_launch_pdl(attn_bwd_kernel<DT, DP, 1>, all, block, SM, st, mq, mk, mv, mg, a, n);
            if (e == cudaSuccess)
                e = host_launch_pdl(attn_bwd_kernel<DT, DP, 2>, all, block, SM, st, mq, mk, mv, mg, a, n);
        } else {
            e = host_launch_pdl(attn_bwd_kernel<DT, DP, 0>, dim3((unsigned)blocks), block, SM, st, mq, mk, mv, mg, a,
                                n);
        }
    });
    RA_LAUNCH(e);
    if (apart) host_count_launch();
    if (plan.red_splits > 1) {
        const long long values = (long long)keys * s.head_dim;
        const dim3 grid((unsigned)std::min<long long>(ceil_div(values, 1024), 4ll * call.sms), 2);
        if (act_dtype == REELS_BF16)
            e = host_launch_pdl(attn_sum_kernel<DT_BF16>, grid, dim3(256), 0, st, a, values, plan.red_splits);
        else
            e = host_launch_pdl(attn_sum_kernel<DT_F16>, grid, dim3(256), 0, st, a, values, plan.red_splits);
        RA_LAUNCH(e);
    }
    return host_ok(REELS_PATH_TENSORCORE);
}

}  // extern "C"
