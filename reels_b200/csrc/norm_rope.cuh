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
// Bound: HBM, 2 passes of the row forward (x, y), 3 backward (x, dout, dx).
#pragma once
#include "common.cuh"

namespace reels {

constexpr int NR_MAX_C = 16384;
constexpr int NR_AXES = 3;

struct NormRopeArgs {
    const void *x;
    const void *dout;     // backward only
    const void *weight;   // [C], nullable
    void *out;            // y, or dx
    const float2 *table;  // (cos, sin): axis after axis, [size][pairs]
    const int *pos;       // [M][3], nullable: raster order of the grid
    long long M;
    int C, D;
    int tps;              // tokens per sample (raster order restarts with every sample)
    int size[NR_AXES];    // positions of an axis
    int pairs[NR_AXES];   // feature pairs of an axis
    int half;             // pairs (i, i + D/2) instead of (2i, 2i + 1)
    float eps;
    unsigned *err;
};

struct NrToken {
    int p[NR_AXES];
    bool turn;
};

// The token's position on each axis.  Raster order: width fastest; tokens
// behind the grid are padding.  A negative position marks padding, one
// behind its table is reported in the status word; neither is turned.
__device__ __forceinline__ NrToken nr_token(const NormRopeArgs &a, long long row) {
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
        const unsigned i = (unsigned)(row % a.tps);
        const unsigned hw = (unsigned)a.size[1] * (unsigned)a.size[2];
        t.p[0] = (int)(i / hw);
        const unsigned rest = i - (unsigned)t.p[0] * hw;
        t.p[1] = (int)(rest / (unsigned)a.size[2]);
        t.p[2] = (int)(rest - (unsigned)t.p[1] * (unsigned)a.size[2]);
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

// Eight consecutive elements as fp32.
template <int DT>
struct NrVec;
template <>
struct NrVec<DT_F32> {
    float4 a, b;
    __device__ __forceinline__ void load(const void *p, long long i) {
        const float4 *q = reinterpret_cast<const float4 *>(reinterpret_cast<const float *>(p) + i);
        a = __ldcg(q);
        b = __ldcg(q + 1);
    }
    __device__ __forceinline__ void get(float (&v)[8]) const {
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    }
    static __device__ __forceinline__ void store(void *p, long long i, const float (&v)[8]) {
        float4 *q = reinterpret_cast<float4 *>(reinterpret_cast<float *>(p) + i);
        q[0] = make_float4(v[0], v[1], v[2], v[3]);
        q[1] = make_float4(v[4], v[5], v[6], v[7]);
    }
};
template <int DT>
struct NrVec {
    using T = typename Elem<DT>::T;
    uint4 a;
    __device__ __forceinline__ void load(const void *p, long long i) {
        a = __ldcg(reinterpret_cast<const uint4 *>(reinterpret_cast<const T *>(p) + i));
    }
    __device__ __forceinline__ void get(float (&v)[8]) const {
        const T *t = reinterpret_cast<const T *>(&a);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = Elem<DT>::to_f(t[j]);
    }
    static __device__ __forceinline__ void store(void *p, long long i, const float (&v)[8]) {
        uint4 o = make_uint4(Elem<DT>::pack2(v[0], v[1]), Elem<DT>::pack2(v[2], v[3]), Elem<DT>::pack2(v[4], v[5]),
                             Elem<DT>::pack2(v[6], v[7]));
        *reinterpret_cast<uint4 *>(reinterpret_cast<T *>(p) + i) = o;
    }
};

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
__device__ __forceinline__ float2 nr_block_sum(float2 v, float2 *buf) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
        v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
    }
    if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = v;
    __syncthreads();
    v = buf[0];
    for (int w = 1; w < (int)(blockDim.x >> 5); ++w) {
        v.x += buf[w].x;
        v.y += buf[w].y;
    }
    return v;
}

// One block per row at a time, the row and the weight in registers.
// A thread owns UPT units; unit u is 8 features at i0 = 8 (u mod D/16) of the
// lower half of head u / (D/16) and the 8 features D/2 above, so that both
// pairings find their partners within a thread.  D/16 divides 32 and the block
// is a multiple of 32 wide, so all units of a thread sit at the same place of
// their heads and share their eight (cos, sin), which the block fetches once
// a row into shared memory (through L2: half the requests of a row otherwise).
// ROPE = 0 runs with D = 16 (two neighbouring vectors a unit).
template <int DT, bool BWD, bool ROPE, bool HALF, int UPT>
__global__ void __launch_bounds__(256) norm_rope_kernel(const NormRopeArgs a) {
    __shared__ float2 buf[2][8];
    __shared__ __align__(16) float2 turn[2][256];
    griddep_wait();
    const int upr = a.C / 16, uph = a.D / 16;  // units of a row, of a head
    const int i0 = 8 * ((int)threadIdx.x % uph);
    // features of unit k of this thread: f, and f + D/2
    auto feature = [&](int k) { return ((int)threadIdx.x + k * (int)blockDim.x) / uph * a.D + i0; };
    auto owned = [&](int k) { return (int)threadIdx.x + k * (int)blockDim.x < upr; };
    NrVec<DT> wv[UPT][2];
    if (a.weight) {
#pragma unroll
        for (int k = 0; k < UPT; ++k)
            if (owned(k)) {
                wv[k][0].load(a.weight, feature(k));
                wv[k][1].load(a.weight, feature(k) + a.D / 2);
            }
    }
    auto weigh = [&](int k, float (&lo)[8], float (&hi)[8]) {
        if (!a.weight) return;
        float w[8];
        wv[k][0].get(w);
#pragma unroll
        for (int j = 0; j < 8; ++j) lo[j] *= w[j];
        wv[k][1].get(w);
#pragma unroll
        for (int j = 0; j < 8; ++j) hi[j] *= w[j];
    };
    int flip = 0;
    for (long long row = blockIdx.x; row < a.M; row += gridDim.x, flip ^= 1) {
        const long long at = row * a.C;
        NrVec<DT> xv[UPT][2], gv[BWD ? UPT : 1][2];
#pragma unroll
        for (int k = 0; k < UPT; ++k) {
            if (owned(k)) {
                const int f = feature(k);
                xv[k][0].load(a.x, at + f);
                xv[k][1].load(a.x, at + f + a.D / 2);
                if (BWD) {
                    gv[k][0].load(a.dout, at + f);
                    gv[k][1].load(a.dout, at + f + a.D / 2);
                }
            }
        }
        if (ROPE) {
            const NrToken t = nr_token(a, row);
            for (int i = threadIdx.x; i < a.D / 2; i += blockDim.x) {
                int base;
                const int ax = nr_axis(a, i, base);
                const int p = ax == 0 ? t.p[0] * a.pairs[0] : ax == 1 ? t.p[1] * a.pairs[1] : t.p[2] * a.pairs[2];
                turn[flip][i] = t.turn ? __ldcg(a.table + base + p) : make_float2(1.0f, 0.0f);
            }
        }
        // pairs 0-3 of a unit: its features 2j, 2j+1; 4-7 those of its upper
        // vector (HALF: j of both vectors)
        float2 cs[8];
        auto fetch = [&]() {
#pragma unroll
            for (int j = 0; j < 8; j += 2) {
                const int pair = HALF ? i0 + j : i0 / 2 + (j & 3) + (j >> 2) * (a.D / 4);
                const float4 v = *reinterpret_cast<const float4 *>(&turn[flip][pair]);
                cs[j] = make_float2(v.x, v.y);
                cs[j + 1] = make_float2(v.z, v.w);
            }
        };
        auto rotate = [&](float (&lo)[8], float (&hi)[8]) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if (HALF) nr_turn<BWD>(lo[j], hi[j], cs[j]);
                else if (j < 4) nr_turn<BWD>(lo[2 * j], lo[2 * j + 1], cs[j]);
                else nr_turn<BWD>(hi[2 * j - 8], hi[2 * j - 7], cs[j]);
            }
        };
        if (BWD && ROPE) {
            __syncthreads();
            fetch();
        }
        // h = w R' dout
        auto pulled = [&](int k, float (&lo)[8], float (&hi)[8]) {
            gv[k][0].get(lo);
            gv[k][1].get(hi);
            if (ROPE) rotate(lo, hi);
            weigh(k, lo, hi);
        };
        float2 sum = make_float2(0.0f, 0.0f);
#pragma unroll
        for (int k = 0; k < UPT; ++k) {
            if (owned(k)) {
                float lo[8], hi[8];
                xv[k][0].get(lo);
                xv[k][1].get(hi);
#pragma unroll
                for (int j = 0; j < 8; ++j) sum.x += lo[j] * lo[j] + hi[j] * hi[j];
                if (BWD) {
                    float gl[8], gh[8];
                    pulled(k, gl, gh);
#pragma unroll
                    for (int j = 0; j < 8; ++j) sum.y += lo[j] * gl[j] + hi[j] * gh[j];
                }
            }
        }
        sum = nr_block_sum(sum, buf[flip]);
        const float r = 1.0f / sqrtf(sum.x / (float)a.C + a.eps);
        const float c2 = BWD ? r * r * (sum.y / (float)a.C) : 0.0f;
        if (!BWD && ROPE) fetch();
#pragma unroll
        for (int k = 0; k < UPT; ++k) {
            if (owned(k)) {
                const int f = feature(k);
                float lo[8], hi[8];
                xv[k][0].get(lo);
                xv[k][1].get(hi);
                if (BWD) {
                    float gl[8], gh[8];
                    pulled(k, gl, gh);
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        lo[j] = r * (gl[j] - lo[j] * c2);
                        hi[j] = r * (gh[j] - hi[j] * c2);
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < 8; ++j) lo[j] *= r, hi[j] *= r;
                    weigh(k, lo, hi);
                    if (ROPE) rotate(lo, hi);
                }
                NrVec<DT>::store(a.out, at + f, lo);
                NrVec<DT>::store(a.out, at + f + a.D / 2, hi);
            }
        }
    }
}

// Any width, alignment and head size: one block of 256 threads a row, scalar
// accesses, the row read a second time (from L1/L2) for the result.
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
        if (rope) t = nr_token(a, row);
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
        auto w_of = [&](int f) { return a.weight ? load_act(a.weight, f, DT) : 1.0f; };
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
        sum = nr_block_sum(sum, buf[flip]);
        const float r = 1.0f / sqrtf(sum.x / (float)a.C + a.eps);
        const float c2 = BWD ? r * r * (sum.y / (float)a.C) : 0.0f;
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
