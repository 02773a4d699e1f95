// Root-mean-square norm of q or k over all heads, its weight and the rotary
// positions of a video, in one pass per token (sm_100a).
//
//   r = 1 / sqrt(mean(x^2) + eps),  n = x r w,  y = R n
// R turns feature pair i of every head by the angle of its axis: pair i
// belongs to the axis whose columns hold it, and (cos, sin) are looked up at
// the token's position on that axis.  The tables are fp32 (a few KB, served
// by L2), computed once by the caller in 64 bits, so far positions lose
// nothing here.  Pullback, with g = R' dout and h = g w:
//   dx = r (h - x r^2 mean(h x))
// whose two sums (x^2 and h x) come from the same pass over x and dout.
// All arithmetic is fp32, each output is rounded once.
//
// Bound: HBM, 2 passes of the row forward (x, y), 3 backward (x, dout, dx),
// with issue slots next to it on short rows.  Measured, bf16: 32760 x 1536
// forward 43 us (4.6 TB/s) and backward 56 (5.4), 8190 x 5120 forward 33 us (5.1
// TB/s) and backward 46 (5.4); fp16, 12288 x 4096: 40 us (5.1) and 59 (5.1); fp32,
// 32760 x 1536: 75 us (5.4) and 101 (6.0).  A copy runs at 6.5 TB/s.
#pragma once
#include "common.cuh"

namespace reels {

constexpr int NR_MAX_C = 16384;
constexpr int NR_AXES = 3;

// Division of n < 2^31 by a constant d: n / d = n m >> (31 + s) with
// s = ceil(log2 d) and m = ceil(2^(31 + s) / d), whose error m d - 2^(31 + s)
// < d <= 2^s is too small to reach the next quotient.
struct NrDivide {
    uint32_t d, m, s;
    static NrDivide by(uint32_t d) {
        NrDivide v = {d, 0, 0};
        while ((1ull << v.s) < d) ++v.s;
        v.m = (uint32_t)(((1ull << (31 + v.s)) + d - 1) / d);
        return v;
    }
    __device__ __forceinline__ uint32_t operator()(uint32_t n) const {
        return (uint32_t)(((uint64_t)n * m) >> 31) >> s;
    }
};

struct NormRopeArgs {
    const void *x;
    const void *dout;     // backward only
    const void *weight;   // [C], nullable, of x's type or (w32) fp32
    int w32;
    void *out;            // y, or dx
    const float2 *table;  // (cos, sin): axis after axis, [size][pairs]
    const int *pos;       // [M][3], nullable: raster order of the grid
    long long M;
    int C, D;
    int tps;              // tokens per sample (raster order restarts with every sample)
    int size[NR_AXES];    // positions of an axis
    int pairs[NR_AXES];   // feature pairs of an axis
    int half;             // pairs (i, i + D/2) instead of (2i, 2i + 1)
    float eps, inv_c;
    NrDivide by_hw, by_w;  // positions of a token in raster order
    unsigned *err;
};

struct NrToken {
    int p[NR_AXES];
    bool turn;
};

// The position on each axis of row `row`, token `tok` of its sample.  Raster
// order: width fastest; tokens behind the grid are padding.  A negative
// position marks padding, one behind its table is reported in the status
// word; neither is turned.
__device__ __forceinline__ NrToken nr_token(const NormRopeArgs &a, long long row, uint32_t tok) {
    NrToken t;
    if (a.pos) {
        t.turn = true;
#pragma unroll
        for (int i = 0; i < NR_AXES; ++i) {
            t.p[i] = __ldcg(a.pos + row * NR_AXES + i);
            if (t.p[i] < 0) t.turn = false;
        }
        if (t.turn && (t.p[0] >= a.size[0] || t.p[1] >= a.size[1] || t.p[2] >= a.size[2])) {
            if (threadIdx.x == 0) atomicOr(a.err, DEVERR_ROPE_POSITION);
            t.turn = false;
        }
    } else {
        const uint32_t t0 = a.by_hw(tok), rest = tok - t0 * a.by_hw.d, t1 = a.by_w(rest);
        t.p[0] = (int)t0;
        t.p[1] = (int)t1;
        t.p[2] = (int)(rest - t1 * a.by_w.d);
        t.turn = t.p[0] < a.size[0];
    }
    return t;
}

// Table entry of feature pair i at position 0 of its axis, and the axis.
__device__ __forceinline__ int nr_axis(const NormRopeArgs &a, int i, int &base) {
    if (i < a.pairs[0]) {
        base = i;
        return 0;
    }
    int off = a.size[0] * a.pairs[0];
    i -= a.pairs[0];
    if (i < a.pairs[1]) {
        base = off + i;
        return 1;
    }
    off += a.size[1] * a.pairs[1];
    base = off + i - a.pairs[1];
    return 2;
}

template <int DT>
__device__ __forceinline__ void nr_read_global(const typename Elem<DT>::T *p, F2 (&v)[4]) {
    __align__(16) typename Elem<DT>::T t[8];
#pragma unroll
    for (int j = 0; j < (int)sizeof(t) / 16; ++j)
        reinterpret_cast<uint4 *>(t)[j] = __ldcg(reinterpret_cast<const uint4 *>(p) + j);
    read8<DT>(t, v);
}
template <int DT>
__device__ __forceinline__ void nr_write(typename Elem<DT>::T *p, const F2 (&v)[4]) {
    const float2 a = v[0].get(), b = v[1].get(), c = v[2].get(), d = v[3].get();
    if constexpr (DT == DT_F32) {
        reinterpret_cast<float4 *>(p)[0] = make_float4(a.x, a.y, b.x, b.y);
        reinterpret_cast<float4 *>(p)[1] = make_float4(c.x, c.y, d.x, d.y);
    } else {
        *reinterpret_cast<uint4 *>(p) = make_uint4(Elem<DT>::pack2(a.x, a.y), Elem<DT>::pack2(b.x, b.y),
                                                   Elem<DT>::pack2(c.x, c.y), Elem<DT>::pack2(d.x, d.y));
    }
}

// (a, b) turned by the angle, or back.
template <bool BACK>
__device__ __forceinline__ void nr_turn(float &a, float &b, float2 cs) {
    const float s = BACK ? -cs.y : cs.y;
    const float u = a * cs.x - b * s;
    b = a * s + b * cs.x;
    a = u;
}

// Sums of two values over the block's warps, the same bits in every thread;
// `buf` alternates between calls, so one barrier a call is enough.  The
// barrier also publishes what the caller left in shared memory before.
template <bool TWO>
__device__ __forceinline__ float2 nr_block_sum(float2 v, float2 *buf) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
        if (TWO) v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
    }
    if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = v;
    __syncthreads();
    v = buf[0];
    for (int w = 1; w < (int)(blockDim.x >> 5); ++w) {
        v.x += buf[w].x;
        if (TWO) v.y += buf[w].y;
    }
    return v;
}

// One block per row at a time.  Rows (x, and dout backward) arrive in a ring of
// `stages` slots of shared memory by bulk copies, so that what is in flight
// does not depend on registers or on how far a block's warps have come; the
// weight is kept beside it.  A row is read twice from its slot (sum, result);
// the barrier of row i's sums also says that row i-1's slot is free.
// A thread owns UPT units; unit u is 8 features at i0 = 8 (u mod D/16) of the
// lower half of head u / (D/16) and the 8 features D/2 above, so that both
// pairings find their partners within a thread.  D/16 divides 32 and the block
// is a multiple of 32 wide, so all units of a thread sit at the same place of
// their heads and share their eight (cos, sin), which the block fetches once
// a row into shared memory, two rows ahead (a barrier lies between its writing
// and its reading, and another before it is written over).
// ROPE = 0 runs with D = 16 (two neighbouring vectors a unit).
// Issue slots come next to HBM here: two units a thread share the angles, the
// waits and the sums' tail, and pairs of values run through packed fp32
// instructions where the pairing allows.
constexpr int NR_THREADS = 512;  // at most
constexpr int NR_STAGES = 4;     // at most
// Shared memory: stages of rows, the weight (forward as fp32, which spares
// conversions; backward as it is, which for 16-bit types leaves room for another
// block), angles of three rows.
__host__ __device__ constexpr int nr_smem_bytes(int C, int elem, bool bwd, bool w32, int stages, int D) {
    return stages * C * elem * (bwd ? 2 : 1) + C * (bwd && !w32 ? elem : 4) + 3 * (D / 2) * 8;
}

// W32: backward with an fp32 weight beside 16-bit rows.
template <int DT, bool BWD, bool ROPE, bool HALF, int UPT, bool W32>
__global__ void __launch_bounds__(UPT == 1 ? 512 : 256, UPT == 1 ? 2 : UPT == 2 ? 3 : 1) norm_rope_kernel(const NormRopeArgs a, const int stages) {
    using T = typename Elem<DT>::T;
    constexpr bool PLANES = !BWD || W32;  // the weight's form in shared memory
    extern __shared__ __align__(128) uint8_t ring[];
    __shared__ float2 buf[2][NR_THREADS / 32];
    __shared__ uint64_t full[NR_STAGES];
    __shared__ int abort_flag;
    const int row_bytes = a.C * (int)sizeof(T), slot_bytes = row_bytes * (BWD ? 2 : 1);
    // fp32 as two planes, the first and second four of every eight features,
    // so that a warp's 16-byte reads meet no bank twice
    uint8_t *const weight = ring + stages * slot_bytes;
    float2 *const turn = reinterpret_cast<float2 *>(weight + a.C * (PLANES ? 4 : (int)sizeof(T)));
    volatile int *const abort = &abort_flag;
    if (threadIdx.x == 0) {
        for (int s = 0; s < stages; ++s) mbar_init(&full[s], 1);
        abort_flag = 0;
        fence_mbar_init();
    }
    __syncthreads();
    griddep_wait();
    auto fill = [&](long long row, int s) {
        mbar_arrive_expect_tx(&full[s], slot_bytes);
        bulk_load(smem_u32(ring + s * slot_bytes), reinterpret_cast<const T *>(a.x) + row * a.C, row_bytes, &full[s]);
        if (BWD)
            bulk_load(smem_u32(ring + s * slot_bytes + row_bytes), reinterpret_cast<const T *>(a.dout) + row * a.C,
                      row_bytes, &full[s]);
    };
    if (threadIdx.x == 0)
        for (int s = 0; s < stages; ++s)
            if (blockIdx.x + (long long)s * gridDim.x < a.M) fill(blockIdx.x + (long long)s * gridDim.x, s);
    for (int i = threadIdx.x; i < a.C / 8; i += blockDim.x) {
        F2 w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = F2(1.0f, 1.0f);
        if (a.weight && a.w32) nr_read_global<DT_F32>(reinterpret_cast<const float *>(a.weight) + 8 * i, w);
        else if (a.weight) nr_read_global<DT>(reinterpret_cast<const T *>(a.weight) + 8 * i, w);
        if (!PLANES) {
            nr_write<DT>(reinterpret_cast<T *>(weight) + 8 * i, w);
        } else {
            const float2 p = w[0].get(), q = w[1].get(), u = w[2].get(), v = w[3].get();
            reinterpret_cast<float4 *>(weight)[i] = make_float4(p.x, p.y, q.x, q.y);
            reinterpret_cast<float4 *>(weight)[a.C / 8 + i] = make_float4(u.x, u.y, v.x, v.y);
        }
    }
    const int upr = a.C / 16, uph = a.D / 16;  // units of a row, of a head
    const int i0 = 8 * ((int)threadIdx.x % uph);
    // features of unit k of this thread: f, and f + D/2
    int feat[UPT];
#pragma unroll
    for (int k = 0; k < UPT; ++k) feat[k] = ((int)threadIdx.x + k * (int)blockDim.x) / uph * a.D + i0;
    auto owned = [&](int k) { return (int)threadIdx.x + k * (int)blockDim.x < upr; };
    auto read = [&](const T *from, int k, F2 (&lo)[4], F2 (&hi)[4]) {
        read8<DT>(from + feat[k], lo);
        read8<DT>(from + feat[k] + a.D / 2, hi);
    };
    auto weigh = [&](int k, F2 (&lo)[4], F2 (&hi)[4]) {
        F2 wl[4], wh[4];
        if (!PLANES) {
            read(reinterpret_cast<const T *>(weight), k, wl, wh);
        } else {
            const float4 *const w = reinterpret_cast<const float4 *>(weight) + feat[k] / 8;
            const float4 w0 = w[0], w1 = w[a.C / 8], w2 = w[a.D / 16], w3 = w[a.C / 8 + a.D / 16];
            wl[0] = F2(w0.x, w0.y), wl[1] = F2(w0.z, w0.w), wl[2] = F2(w1.x, w1.y), wl[3] = F2(w1.z, w1.w);
            wh[0] = F2(w2.x, w2.y), wh[1] = F2(w2.z, w2.w), wh[2] = F2(w3.x, w3.y), wh[3] = F2(w3.z, w3.w);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) lo[j] = mul2(lo[j], wl[j]), hi[j] = mul2(hi[j], wh[j]);
    };
    // The angles: thread i < D/2 fetches pair i of a row and leaves it where
    // the threads at position l of their heads find pairs 2p, 2p + 1 of their
    // eight side by side: [p][l] (no bank twice in a warp's reads).
    const bool turner = ROPE && (int)threadIdx.x < a.D / 2;
    float2 nt = make_float2(1.0f, 0.0f);
    int base = 0, axis = 0, put = 0;
    if (turner) {
        const int i = threadIdx.x;
        axis = nr_axis(a, i, base);
        const int l = HALF ? i / 8 : (i % (a.D / 4)) / 4, j = HALF ? i % 8 : i % 4 + i / (a.D / 4) * 4;
        put = ((j >> 1) * uph + l) * 2 + (j & 1);
    }
    const uint32_t stride = ROPE ? gridDim.x % (uint32_t)a.tps : 0;
    uint32_t tok = ROPE ? blockIdx.x % (uint32_t)a.tps : 0;  // of the next row to fetch
    auto fetch_angles = [&](long long row) {
        const NrToken t = nr_token(a, row, tok);
        const int p = axis == 0 ? t.p[0] : axis == 1 ? t.p[1] : t.p[2];
        const int step = axis == 0 ? a.pairs[0] : axis == 1 ? a.pairs[1] : a.pairs[2];
        nt = t.turn ? __ldcg(a.table + base + p * step) : make_float2(1.0f, 0.0f);
        tok += stride;
        if (tok >= (uint32_t)a.tps) tok -= a.tps;
    };
    if (turner) {
#pragma unroll
        for (int n = 0; n < 2; ++n)
            if (blockIdx.x + n * (long long)gridDim.x < a.M) {
                fetch_angles(blockIdx.x + n * (long long)gridDim.x);
                turn[n * (a.D / 2) + put] = nt;
            }
    }
    __syncthreads();  // the weight, the first angles
    int flip = 0, slot = 0, at = 0;  // at: the angles' buffer of this row
    uint32_t phase = 0;
    for (long long row = blockIdx.x; row < a.M; row += gridDim.x, flip ^= 1) {
        const long long later = row + 2ll * gridDim.x;
        if (turner && later < a.M) fetch_angles(later);
        wait_bar(&full[slot], phase, abort, a.err, DEVERR_TIMEOUT_AB_FULL);
        const T *const xs = reinterpret_cast<const T *>(ring + slot * slot_bytes);
        // pairs 0-3 of a unit: its features 2j, 2j+1; 4-7 those of its upper
        // vector (HALF: j of both vectors)
        float2 cs[8];
        auto read_angles = [&](float by) {
#pragma unroll
            for (int j = 0; j < 8; j += 2) {
                const float4 v = reinterpret_cast<const float4 *>(turn + at * (a.D / 2))[(j >> 1) * uph + (i0 >> 3)];
                cs[j] = mul2(F2(v.x, v.y), F2(by, by)).get();
                cs[j + 1] = mul2(F2(v.z, v.w), F2(by, by)).get();
            }
        };
        auto rotate = [&](F2 (&lo)[4], F2 (&hi)[4]) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float2 x = lo[j].get(), y = hi[j].get();
                if (HALF) {
                    nr_turn<BWD>(x.x, y.x, cs[2 * j]);
                    nr_turn<BWD>(x.y, y.y, cs[2 * j + 1]);
                } else {
                    nr_turn<BWD>(x.x, x.y, cs[j]);
                    nr_turn<BWD>(y.x, y.y, cs[4 + j]);
                }
                lo[j] = F2(x.x, x.y), hi[j] = F2(y.x, y.y);
            }
        };
        if (ROPE && BWD) read_angles(1.0f);
        F2 xl[UPT][4], xh[UPT][4];  // (backward: read again for the result)
        F2 hl[BWD ? UPT : 1][4], hh[BWD ? UPT : 1][4];  // h = w R' dout
        F2 s0 = F2(0.0f, 0.0f), s1 = F2(0.0f, 0.0f);
#pragma unroll
        for (int k = 0; k < UPT; ++k) {
            if (owned(k)) {
                read(xs, k, xl[k], xh[k]);
#pragma unroll
                for (int j = 0; j < 4; ++j) s0 = fma2(xl[k][j], xl[k][j], fma2(xh[k][j], xh[k][j], s0));
                if (BWD) {
                    read(xs + a.C, k, hl[k], hh[k]);
                    if (ROPE) rotate(hl[k], hh[k]);
                    weigh(k, hl[k], hh[k]);
#pragma unroll
                    for (int j = 0; j < 4; ++j) s1 = fma2(xl[k][j], hl[k][j], fma2(xh[k][j], hh[k][j], s1));
                }
            }
        }
        float2 sum = make_float2(s0.get().x + s0.get().y, BWD ? s1.get().x + s1.get().y : 0.0f);
        // behind this barrier the other row's slot and angles have no readers left
        sum = nr_block_sum<BWD>(sum, buf[flip]);
        if (turner && later < a.M) turn[(at == 0 ? 2 : at - 1) * (a.D / 2) + put] = nt;
        if (threadIdx.x == 0 && row > blockIdx.x) {
            const long long next = row + (long long)(stages - 1) * gridDim.x;
            if (next < a.M) fill(next, slot == 0 ? stages - 1 : slot - 1);
        }
        const float r = rsqrtf(fmaf(sum.x, a.inv_c, a.eps));
        if (ROPE && !BWD) read_angles(r);
        T *const out = reinterpret_cast<T *>(a.out) + row * a.C;
#pragma unroll
        for (int k = 0; k < UPT; ++k) {
            if (owned(k)) {
                F2 lo[4], hi[4];
                if (BWD) {
                    read(xs, k, xl[0], xh[0]);
                    // r^3 would leave fp32 from r = 7e12 on: rows of small values without epsilon
                    const float c2 = -r * (r * (sum.y * a.inv_c));
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        lo[j] = mul2(fma2(xl[0][j], F2(c2, c2), hl[k][j]), F2(r, r));
                        hi[j] = mul2(fma2(xh[0][j], F2(c2, c2), hh[k][j]), F2(r, r));
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < 4; ++j) lo[j] = xl[k][j], hi[j] = xh[k][j];
                    weigh(k, lo, hi);
                    if (ROPE) rotate(lo, hi);  // and times r
                    else {
#pragma unroll
                        for (int j = 0; j < 4; ++j) lo[j] = mul2(lo[j], F2(r, r)), hi[j] = mul2(hi[j], F2(r, r));
                    }
                }
                nr_write<DT>(out + feat[k], lo);
                nr_write<DT>(out + feat[k] + a.D / 2, hi);
            }
        }
        if (++slot == stages) slot = 0, phase ^= 1;
        if (++at == 3) at = 0;
    }
    if (*abort) {  // give the copies in flight time to land before the shared memory goes
        for (int i = 0; i < 64; ++i) __nanosleep(2000);
    }
}

// Any width, alignment and head size: one block of 256 threads a row, scalar
// accesses, the row read a second time (from L1/L2) for the result.  For what
// the vector form cannot take; not tuned.
template <int DT, bool BWD>
__global__ void __launch_bounds__(256) norm_rope_any_kernel(const NormRopeArgs a) {
    __shared__ float2 buf[2][8];
    griddep_wait();
    const bool rope = a.table != nullptr;
    const int step = rope ? 2 : 1;
    int flip = 0;
    for (long long row = blockIdx.x; row < a.M; row += gridDim.x, flip ^= 1) {
        const long long at = row * a.C;
        NrToken t;
        t.turn = false;
        if (rope) t = nr_token(a, row, (uint32_t)(row % a.tps));
        // features of item i: a pair of a head, or one feature
        auto where = [&](int i, int &f0, int &f1, float2 &cs) {
            cs = make_float2(1.0f, 0.0f);
            if (!rope) {
                f0 = f1 = i;
                return;
            }
            const int hp = a.D / 2, head = i / hp, pair = i - head * hp;
            f0 = head * a.D + (a.half ? pair : 2 * pair);
            f1 = f0 + (a.half ? hp : 1);
            if (t.turn) {
                int base;
                const int ax = nr_axis(a, pair, base);
                cs = __ldcg(a.table + base + t.p[ax] * a.pairs[ax]);
            }
        };
        auto w_of = [&](int f) { return a.weight ? load_act(a.weight, f, a.w32 ? DT_F32 : DT) : 1.0f; };
        float2 sum = make_float2(0.0f, 0.0f);
        for (int i = threadIdx.x; i < a.C / step; i += blockDim.x) {
            int f0, f1;
            float2 cs;
            where(i, f0, f1, cs);
            const float x0 = load_act(a.x, at + f0, DT), x1 = rope ? load_act(a.x, at + f1, DT) : 0.0f;
            sum.x += x0 * x0 + x1 * x1;
            if (BWD) {
                float g0 = load_act(a.dout, at + f0, DT), g1 = rope ? load_act(a.dout, at + f1, DT) : 0.0f;
                nr_turn<true>(g0, g1, cs);
                sum.y += x0 * (g0 * w_of(f0)) + x1 * (g1 * w_of(f1));
            }
        }
        sum = nr_block_sum<BWD>(sum, buf[flip]);
        const float r = 1.0f / sqrtf(sum.x / (float)a.C + a.eps);
        const float c2 = BWD ? r * (r * (sum.y / (float)a.C)) : 0.0f;
        for (int i = threadIdx.x; i < a.C / step; i += blockDim.x) {
            int f0, f1;
            float2 cs;
            where(i, f0, f1, cs);
            float x0 = load_act(a.x, at + f0, DT), x1 = rope ? load_act(a.x, at + f1, DT) : 0.0f;
            if (BWD) {
                float g0 = load_act(a.dout, at + f0, DT), g1 = rope ? load_act(a.dout, at + f1, DT) : 0.0f;
                nr_turn<true>(g0, g1, cs);
                x0 = r * (g0 * w_of(f0) - x0 * c2);
                x1 = r * (g1 * w_of(f1) - x1 * c2);
            } else {
                x0 = x0 * r * w_of(f0);
                x1 = x1 * r * w_of(f1);
                nr_turn<false>(x0, x1, cs);
            }
            store_act(a.out, at + f0, DT, x0);
            if (rope) store_act(a.out, at + f1, DT, x1);
        }
    }
}

}  // namespace reels
