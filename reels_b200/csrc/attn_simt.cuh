// Softmax attention and its gradient on the CUDA cores: fp32 tensors, head
// sizes that are no multiple of 8 or above 128, and strides the tensor-core
// kernels (attn_fwd.cuh, attn_bwd.cuh) cannot read.  Also the small kernels
// both share: the join of key splits and the gradient's row statistics.
//
//   S = scale q k',  P = softmax over the keys before the sample's length,
//   O = P v,  L = log sum exp S
//   delta = rowsum(dO * O),  P = exp(S - L),  dS = P * (dO v' - delta)
//   dV = P' dO,  dQ = scale dS k,  dK = scale dS' q
// A row without keys has O = 0, L = -inf and no part in any gradient.
//
// T x T tiles of S in registers (T / 16 squared a thread, 256 threads), operands
// in shared memory as fp32; every sum is fp32 and in a fixed order.  T = 32 for
// small clips, where a block's latency counts, 64 where the blocks fill the GPU
// (half the shared-memory reads a product); dQ runs beside dK and dV in one
// launch.  Bound: shared-memory reads and fp32 arithmetic with T = 64 (600
// tokens, 48 heads of 128, fp32: forward 23 TFLOP/s); latency with T = 32 (189
// tokens, 5 heads of 64, fp32: forward 8 us and its join 3, backward 34 and its
// statistics 3).
#pragma once
#include <math_constants.h>

#include "common.cuh"

namespace reels {

constexpr int AT_MAX_D = 256;  // head size
constexpr int AS_THREADS = 256;

struct AttnArgs {
    const void *q, *k, *v;                   // [batch][token][head][D] by strides, D contiguous
    long long qs[3], ks[3], vs[3];           // batch, token and head strides in elements
    const int *lengths;                      // [B] keys of a sample, nullable
    int B, H, HK, Sq, Sk, D;
    float scale;
    void *out;                               // [B][Sq][H][D]
    float *lse;                              // [B][H][Sq]
    int splits, split_keys;                  // forward: key ranges of a row and their length
    float *part_o, *part_lse;                // [splits][B][H][Sq][D], [splits][B][H][Sq]
    // backward
    const void *dout;                        // [B][Sq][H][D]
    const float *stat_l, *stat_d;            // [B][H][Sqp]: -L in log2 units (-inf: no part), -delta
    int Sqp;                                 // Sq rounded up to whole tiles
    void *dq, *dk, *dv;                      // contiguous, in the layout of q, k and v
    const float *stat_n;                     // fp16: [B][H][Sqp] |dO row|
    const float2 *range;                     // fp16: [B][HK] largest |dO row| of the heads that share it, and |v row|
    int red_splits;                          // dK, dV: ranges of the (head, query tile) walk
    float *part_k, *part_v;                  // [red_splits][B][Sk][HK][D]
    unsigned *err;
};

// Keys of sample b that take part.
__device__ __forceinline__ int attn_keys(const AttnArgs &a, int b) {
    if (!a.lengths) return a.Sk;
    const int n = __ldcg(a.lengths + b);
    return n < 0 ? 0 : (n < a.Sk ? n : a.Sk);
}

// The first key of a split and the end of its keys, of `len` (splits times
// split_keys may lie past 32 bits).
__device__ __forceinline__ int attn_split(const AttnArgs &a, int len, int split, int &end) {
    const int begin = (int)min((long long)len, (long long)split * a.split_keys);
    end = begin + min(len - begin, a.split_keys);
    return begin;
}

// T rows of D elements into dst[T][DP + 4], rows from `n` on and features
// from D on as zeros.  fp32 rows that allow it in 16-byte pieces.
template <int DT, int DP, int T>
__device__ __forceinline__ void as_load(float *dst, const void *src, long long at, long long pitch, int n, int D) {
    if (DT == DT_F32 && ((reinterpret_cast<uintptr_t>(src) & 15) | ((at | pitch | D) & 3)) == 0) {
        const float *p = reinterpret_cast<const float *>(src) + at;
        constexpr int N = T * DP / 4 / AS_THREADS, B = N < 8 ? N : 8;
#pragma unroll
        for (int i0 = 0; i0 < N; i0 += B) {
            float4 v[B];
#pragma unroll
            for (int i = 0; i < B; ++i) {
                const int x = threadIdx.x + (i0 + i) * AS_THREADS, r = x / (DP / 4), d = x % (DP / 4) * 4;
                v[i] = (r < n && d < D) ? __ldcg(reinterpret_cast<const float4 *>(p + r * pitch + d))
                                        : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            }
#pragma unroll
            for (int i = 0; i < B; ++i) {
                const int x = threadIdx.x + (i0 + i) * AS_THREADS, r = x / (DP / 4), d = x % (DP / 4) * 4;
                *reinterpret_cast<float4 *>(dst + r * (DP + 4) + d) = v[i];
            }
        }
        return;
    }
#pragma unroll 8
    for (int i = threadIdx.x; i < T * DP; i += AS_THREADS) {
        const int r = i / DP, d = i - r * DP;
        dst[r * (DP + 4) + d] = (r < n && d < D) ? load_act(src, at + r * pitch + d, DT) : 0.0f;
    }
}
// acc[i][j] = A[N ty + i] . B[tx + 16 j], N = T / 16
template <int DP, int N>
__device__ __forceinline__ void as_dot(const float *A, const float *B, int ty, int tx, float (&acc)[N][N]) {
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int j = 0; j < N; ++j) acc[i][j] = 0.0f;
#pragma unroll 8
    for (int d = 0; d < DP; d += 4) {
        float4 x[N], y[N];
#pragma unroll
        for (int i = 0; i < N; ++i) {
            x[i] = *reinterpret_cast<const float4 *>(A + (N * ty + i) * (DP + 4) + d);
            y[i] = *reinterpret_cast<const float4 *>(B + (tx + 16 * i) * (DP + 4) + d);
        }
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int j = 0; j < N; ++j)
                acc[i][j] += x[i].x * y[j].x + x[i].y * y[j].y + x[i].z * y[j].z + x[i].w * y[j].w;
    }
}
// acc[i][c][.] += sum_n W(N ty + i, n) B[n][4 tx + 64 c ..]; W(r, n) = w[r * rs + n * ns]
template <int DP, int N>
__device__ __forceinline__ void as_mix(const float *w, int rs, int ns, const float *B, int ty, int tx,
                                       float (&acc)[N][DP / 64][4]) {
#pragma unroll 4
    for (int n = 0; n < 16 * N; ++n) {
        float f[N];
#pragma unroll
        for (int i = 0; i < N; ++i) f[i] = w[(N * ty + i) * rs + n * ns];
#pragma unroll
        for (int c = 0; c < DP / 64; ++c) {
            const float4 b = *reinterpret_cast<const float4 *>(B + n * (DP + 4) + 4 * tx + 64 * c);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                acc[i][c][0] += f[i] * b.x, acc[i][c][1] += f[i] * b.y;
                acc[i][c][2] += f[i] * b.z, acc[i][c][3] += f[i] * b.w;
            }
        }
    }
}
__host__ __device__ constexpr int as_smem_bytes(int DP, int T, int tiles) {
    return (tiles * T * (DP + 4) + 2 * T * (T + 1)) * 4;
}

// grid: query tiles * B * H, splits
template <int DT, int DP, int T>
__global__ void __launch_bounds__(AS_THREADS) attn_simt_fwd_kernel(const AttnArgs a) {
    extern __shared__ float sm[];
    constexpr int N = T / 16;
    float *Q = sm, *K = Q + T * (DP + 4), *V = K + T * (DP + 4), *P = V + T * (DP + 4);
    griddep_wait();
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const int tiles = (a.Sq + T - 1) / T, bh = (int)(blockIdx.x / tiles);
    const int q0 = (int)(blockIdx.x % tiles) * T, b = bh / a.H, h = bh % a.H, hk = h / (a.H / a.HK);
    const int len = attn_keys(a, b);
    int k_end;
    const int k_begin = attn_split(a, len, (int)blockIdx.y, k_end);
    as_load<DT, DP, T>(Q, a.q, b * a.qs[0] + q0 * a.qs[1] + h * a.qs[2], a.qs[1], a.Sq - q0, a.D);
    float m[N], l[N] = {}, o[N][DP / 64][4] = {};
#pragma unroll
    for (int i = 0; i < N; ++i) m[i] = -CUDART_INF_F;
    for (int k0 = k_begin; k0 < k_end; k0 += T) {
        __syncthreads();
        as_load<DT, DP, T>(K, a.k, b * a.ks[0] + k0 * a.ks[1] + hk * a.ks[2], a.ks[1], k_end - k0, a.D);
        as_load<DT, DP, T>(V, a.v, b * a.vs[0] + k0 * a.vs[1] + hk * a.vs[2], a.vs[1], k_end - k0, a.D);
        __syncthreads();
        float s[N][N];
        as_dot<DP, N>(Q, K, ty, tx, s);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            float mx = -CUDART_INF_F;
#pragma unroll
            for (int j = 0; j < N; ++j) {
                s[i][j] = k0 + tx + 16 * j < k_end ? s[i][j] * a.scale : -CUDART_INF_F;
                mx = fmaxf(mx, s[i][j]);
            }
#pragma unroll
            for (int w = 1; w < 16; w <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, w));
            mx = fmaxf(m[i], mx);
            const float ref = mx == -CUDART_INF_F ? 0.0f : mx;
            const float keep = expf(m[i] - ref);
            float sum = 0.0f;
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const float p = expf(s[i][j] - ref);
                P[(N * ty + i) * (T + 1) + tx + 16 * j] = p;
                sum += p;
            }
#pragma unroll
            for (int w = 1; w < 16; w <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
            l[i] = l[i] * keep + sum;
            m[i] = mx;
#pragma unroll
            for (int c = 0; c < DP / 64; ++c)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[i][c][e] *= keep;
        }
        __syncwarp();  // the rows of P that a warp reads are its own
        as_mix<DP, N>(P, T + 1, 1, V, ty, tx, o);
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int q = q0 + N * ty + i;
        if (q >= a.Sq) continue;
        const float inv = l[i] > 0.0f || l[i] != l[i] ? 1.0f / l[i] : 0.0f;
        const float lse = (m[i] == -CUDART_INF_F ? 0.0f : m[i]) + logf(l[i]);
        const long long at = ((long long)blockIdx.y * a.B + b) * a.H + h;
        if (tx == 0) (a.splits > 1 ? a.part_lse : a.lse)[at * a.Sq + q] = lse;
#pragma unroll
        for (int c = 0; c < DP / 64; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int d = 4 * tx + 64 * c + e;
                if (d >= a.D) continue;
                const float v = o[i][c][e] * inv;
                if (a.splits > 1) a.part_o[(at * a.Sq + q) * a.D + d] = v;
                else store_act(a.out, (((long long)b * a.Sq + q) * a.H + h) * a.D + d, DT, v);
            }
    }
}

__device__ __forceinline__ float as_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Forward for few rows (up to R = 8 queries and heads that share a key head, as
// with single tokens): the keys and values pass once through registers at HBM
// rate, where the tensor-core kernel would spend a whole 128-row softmax on
// them.  Bound: HBM, as one row over 32760 keys of 12 heads of 128 shows: 201 MB
// in 41 us (4.9 TB/s) and 4 us for the join, against 60 us by the tensor-core
// kernel.  With more rows it is the arithmetic of one block an SM: 2 rows 39 us,
// 4 rows 82, 8 rows 96 (joins included).  A group of G lanes
// takes a key, 16 bytes of it a lane; groups keep a running maximum, sum and
// output of their own over every (256 / G)-th key, four keys at a time, and
// are joined in a fixed order at the end.  P is not rounded here.
// grid: B * HK, splits
template <int DT, int G, int R>
__global__ void __launch_bounds__(256) attn_rows_kernel(const AttnArgs a) {
    using T = typename Elem<DT>::T;
    constexpr int U = 4, GROUPS = 256 / G, DP = 8 * G;
    __shared__ float sm[8][R][DP + 2];
    griddep_wait();
    const int lane = threadIdx.x & 31, sub = lane % G, grp = threadIdx.x / G;
    const int b = blockIdx.x / a.HK, hk = blockIdx.x % a.HK, group = a.H / a.HK, rows = a.Sq * group;
    const int len = attn_keys(a, b);
    int k_end;
    const int k_begin = attn_split(a, len, (int)blockIdx.y, k_end);
    const bool live = 8 * sub < a.D;
    float q[R][8], acc[R][8] = {}, m[R], l[R] = {};
#pragma unroll
    for (int r = 0; r < R; ++r) {
        m[r] = -CUDART_INF_F;
        uint4 x = make_uint4(0, 0, 0, 0);
        if (r < rows && live) {
            const int h = hk * group + r / a.Sq, t = r % a.Sq;
            x = __ldcg(reinterpret_cast<const uint4 *>(reinterpret_cast<const T *>(a.q) + b * a.qs[0] + t * a.qs[1] +
                                                       h * a.qs[2]) + sub);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) q[r][j] = load_act(&x, j, DT) * (a.scale * CUDART_L2E_F);
    }
    const T *K = reinterpret_cast<const T *>(a.k) + b * a.ks[0] + hk * a.ks[2];
    const T *V = reinterpret_cast<const T *>(a.v) + b * a.vs[0] + hk * a.vs[2];
    uint4 nx[U], ny[U];  // the next keys and values, on their way
    auto fetch = [&](int base) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int t = base + u * GROUPS + grp;
            nx[u] = ny[u] = make_uint4(0, 0, 0, 0);
            if (t < k_end && live) {
                nx[u] = __ldcg(reinterpret_cast<const uint4 *>(K + t * a.ks[1]) + sub);
                ny[u] = __ldcg(reinterpret_cast<const uint4 *>(V + t * a.vs[1]) + sub);
            }
        }
    };
    fetch(k_begin);
    for (int base = k_begin; base < k_end; base += U * GROUPS) {
        uint4 x[U], y[U];
#pragma unroll
        for (int u = 0; u < U; ++u) x[u] = nx[u], y[u] = ny[u];
        fetch(base + U * GROUPS);
        float s[U][R];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float k[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) k[j] = load_act(&x[u], j, DT);
#pragma unroll
            for (int r = 0; r < R; ++r) {
                float d = 0.0f;
#pragma unroll
                for (int j = 0; j < 8; ++j) d += q[r][j] * k[j];
#pragma unroll
                for (int w = G / 2; w > 0; w >>= 1) d += __shfl_xor_sync(0xffffffffu, d, w);
                s[u][r] = base + u * GROUPS + grp < k_end ? d : -CUDART_INF_F;
            }
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float mx = m[r];
#pragma unroll
            for (int u = 0; u < U; ++u) mx = fmaxf(mx, s[u][r]);
            const float ref = mx == -CUDART_INF_F ? 0.0f : mx, keep = as_exp2(m[r] - ref);
            m[r] = mx;
            l[r] *= keep;
#pragma unroll
            for (int j = 0; j < 8; ++j) acc[r][j] *= keep;
#pragma unroll
            for (int u = 0; u < U; ++u) s[u][r] = as_exp2(s[u][r] - ref), l[r] += s[u][r];
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float v = load_act(&y[u], j, DT);
#pragma unroll
                for (int r = 0; r < R; ++r) acc[r][j] += s[u][r] * v;
            }
    }
    // the groups of a warp, then the warps
#pragma unroll
    for (int r = 0; r < R; ++r) {
#pragma unroll
        for (int w = G; w < 32; w <<= 1) {
            const float om = __shfl_xor_sync(0xffffffffu, m[r], w), mx = fmaxf(m[r], om);
            const float ref = mx == -CUDART_INF_F ? 0.0f : mx, f = exp2f(m[r] - ref), g = exp2f(om - ref);
            m[r] = mx;
            l[r] = l[r] * f + __shfl_xor_sync(0xffffffffu, l[r], w) * g;
#pragma unroll
            for (int j = 0; j < 8; ++j) acc[r][j] = acc[r][j] * f + __shfl_xor_sync(0xffffffffu, acc[r][j], w) * g;
        }
        if (lane < G) {
            float *at = sm[threadIdx.x >> 5][r];
#pragma unroll
            for (int j = 0; j < 8; ++j) at[8 * sub + j] = acc[r][j];
            if (sub == 0) at[DP] = m[r], at[DP + 1] = l[r];
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < R * DP; i += 256) {
        const int r = i / DP, d = i % DP;
        if (r >= rows || d >= a.D) continue;
        float mx = -CUDART_INF_F, total = 0.0f, o = 0.0f;
#pragma unroll
        for (int w = 0; w < 8; ++w) mx = fmaxf(mx, sm[w][r][DP]);
        const float ref = mx == -CUDART_INF_F ? 0.0f : mx;
#pragma unroll
        for (int w = 0; w < 8; ++w) {
            const float f = exp2f(sm[w][r][DP] - ref);
            total += f * sm[w][r][DP + 1];
            o += f * sm[w][r][d];
        }
        const int h = hk * group + r / a.Sq, t = r % a.Sq;
        const long long at = (((long long)blockIdx.y * a.B + b) * a.H + h) * a.Sq + t;
        o *= total > 0.0f || total != total ? 1.0f / total : 0.0f;
        if (d == 0) (a.splits > 1 ? a.part_lse : a.lse)[at] = (ref + log2f(total)) * CUDART_LN2_F;
        if (a.splits > 1) a.part_o[at * a.D + d] = o;
        else store_act(a.out, (((long long)b * a.Sq + t) * a.H + h) * a.D + d, DT, o);
    }
}

// Joins the key splits of a row: weights exp(L_i - L), splits in order.  One
// warp a row; the lanes hold a weight each and pass them on.  NC: 32-feature
// pieces of a row; eight splits are read at a time.
template <int DT, int NC>
__global__ void __launch_bounds__(128) attn_join_kernel(const AttnArgs a) {
    griddep_wait();
    const int lane = threadIdx.x & 31;
    const long long rows = (long long)a.B * a.H * a.Sq;
    for (long long row = blockIdx.x * 4ll + (threadIdx.x >> 5); row < rows; row += gridDim.x * 4ll) {
        float m = -CUDART_INF_F;
        for (int s = lane; s < a.splits; s += 32) m = fmaxf(m, __ldcg(a.part_lse + s * rows + row));
#pragma unroll
        for (int w = 16; w > 0; w >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, w));
        const float ref = m == -CUDART_INF_F ? 0.0f : m;
        float total = 0.0f, acc[NC] = {}, f = 0.0f;
        for (int s0 = 0; s0 < a.splits; s0 += 8) {
            float v[8][NC];
#pragma unroll
            for (int s = 0; s < 8; ++s)
#pragma unroll
                for (int c = 0; c < NC; ++c)
                    v[s][c] = s0 + s < a.splits && 32 * c + lane < a.D
                                  ? __ldcg(a.part_o + ((s0 + s) * rows + row) * a.D + 32 * c + lane)
                                  : 0.0f;
            if ((s0 & 31) == 0)
                f = s0 + lane < a.splits ? expf(__ldcg(a.part_lse + (s0 + lane) * rows + row) - ref) : 0.0f;
#pragma unroll
            for (int s = 0; s < 8; ++s) {
                const float g = __shfl_sync(0xffffffffu, f, (s0 & 31) + s);
                total += g;
#pragma unroll
                for (int c = 0; c < NC; ++c) acc[c] += g * v[s][c];
            }
        }
        const float inv = total > 0.0f || total != total ? 1.0f / total : 0.0f;
        if (lane == 0) a.lse[row] = ref + logf(total);
        const int q = (int)(row % a.Sq), h = (int)(row / a.Sq % a.H), b = (int)(row / a.Sq / a.H);
        const long long at = (((long long)b * a.Sq + q) * a.H + h) * a.D;
#pragma unroll
        for (int c = 0; c < NC; ++c)
            if (32 * c + lane < a.D) store_act(a.out, at + 32 * c + lane, DT, acc[c] * inv);
    }
}

// Row statistics of the gradient, as the terms that are added: -L in log2
// units and -delta of every query row, padded to Sqp rows a head.  Rows
// without keys and padding get -inf, so that their probabilities come out as
// exp2(-inf) = 0.  One warp a row: for the CUDA-core kernels, any type and width.
template <int DT>
__global__ void __launch_bounds__(256) attn_stat_kernel(const AttnArgs a, float *stat_l, float *stat_d) {
    griddep_wait();
    const int lane = threadIdx.x & 31;
    const long long rows = (long long)a.B * a.H * a.Sqp;
    for (long long row = blockIdx.x * 8ll + (threadIdx.x >> 5); row < rows; row += gridDim.x * 8ll) {
        const int q = (int)(row % a.Sqp), h = (int)(row / a.Sqp % a.H), b = (int)(row / a.Sqp / a.H);
        float2 st = make_float2(-CUDART_INF_F, 0.0f);
        if (q < a.Sq) {
            const long long at = (((long long)b * a.Sq + q) * a.H + h) * a.D;
            float delta = 0.0f;
            for (int d = lane; d < a.D; d += 32) {
                const float g = load_act(a.dout, at + d, DT);
                delta += g * load_act(a.out, at + d, DT);
            }
#pragma unroll
            for (int w = 16; w > 0; w >>= 1) delta += __shfl_xor_sync(0xffffffffu, delta, w);
            const float lse = __ldcg(a.lse + ((long long)b * a.H + h) * a.Sq + q);
            if (lse != -CUDART_INF_F) st = make_float2(-lse * CUDART_L2E_F, -delta);
        }
        if (lane == 0) {
            stat_l[row] = st.x;
            stat_d[row] = st.y;
        }
    }
}

// x . y (with `y`) and, for fp16, |x| of rows of D = 8 n <= 8 G features: G
// lanes a row with 16 bytes each, four rows in flight.
template <int DT, int G, typename At, typename Use>
__device__ __forceinline__ void as_rows(const void *x, const void *y, long long rows, int D, At at, Use use) {
    using T = typename Elem<DT>::T;
    constexpr int R = 4;
    const int sub = threadIdx.x % G;
    const long long step = (long long)gridDim.x * (256 / G) * R;
    // (the bound is the block's first row: a block stays together for its shuffles)
    for (long long first = (long long)blockIdx.x * (256 / G) * R; first < rows; first += step) {
        const long long r0 = first + threadIdx.x / G * R;
        uint4 u[R], v[R];
#pragma unroll
        for (int i = 0; i < R; ++i) {
            u[i] = v[i] = make_uint4(0, 0, 0, 0);
            if (r0 + i < rows && 8 * sub < D) {
                const long long o = at(r0 + i);
                if (o >= 0) {
                    u[i] = __ldcg(reinterpret_cast<const uint4 *>(reinterpret_cast<const T *>(x) + o) + sub);
                    if (y) v[i] = __ldcg(reinterpret_cast<const uint4 *>(reinterpret_cast<const T *>(y) + o) + sub);
                }
            }
        }
        float mine = 0.0f, size = 0.0f;  // lane i of the group keeps row i's
#pragma unroll
        for (int i = 0; i < R; ++i) {
            F2 g[4], h[4], d2 = F2(0.0f, 0.0f), n2 = F2(0.0f, 0.0f);
            read8<DT>(reinterpret_cast<const T *>(&u[i]), g);
            if (y) read8<DT>(reinterpret_cast<const T *>(&v[i]), h);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (y) d2 = fma2(g[j], h[j], d2);
                if (DT == DT_F16) n2 = fma2(g[j], g[j], n2);
            }
            float dot = d2.get().x + d2.get().y, norm = n2.get().x + n2.get().y;
#pragma unroll
            for (int w = G / 2; w > 0; w >>= 1) {
                if (y) dot += __shfl_xor_sync(0xffffffffu, dot, w);
                if (DT == DT_F16) norm += __shfl_xor_sync(0xffffffffu, norm, w);
            }
            if (sub == i) mine = dot, size = norm;
        }
        if (sub < R && r0 + sub < rows) use(r0 + sub, mine, sqrtf(size));
    }
}

// The same for the tensor-core kernels: rows in memory order (the heads of a
// token side by side), `shift` added to -L (fp16, see AtRange), and for fp16
// the rows' |dO| and, for v_n [B][HK][Sk], |v| (0 behind a sample's length).
// Bound: HBM, out and dO once (2 x 6144 tokens, 32 heads of 128: 201 MB in
// 37 us, 5.4 TB/s).
template <int DT, int G>
__global__ void __launch_bounds__(256) attn_stat_vec_kernel(const AttnArgs a, float *stat_l, float *stat_d,
                                                            float *stat_n, float *v_n, float shift) {
    griddep_wait();
    // a row's head, token and sample (64-bit divisions would cost more than the rows)
    auto where = [](long long r, long long rows, int heads, int tokens, int &b, int &t, int &h) {
        if (rows <= 0x7fffffff) {
            const uint32_t tok = (uint32_t)r / (uint32_t)heads;
            h = (int)((uint32_t)r - tok * heads), b = (int)(tok / (uint32_t)tokens);
            t = (int)(tok - b * (uint32_t)tokens);
        } else {
            const long long tok = r / heads;
            h = (int)(r - tok * heads), b = (int)(tok / tokens), t = (int)(tok - (long long)b * tokens);
        }
    };
    const long long rows = (long long)a.B * a.Sq * a.H;
    as_rows<DT, G>(
        a.dout, a.out, rows, a.D, [&](long long r) { return r * a.D; },
        [&](long long r, float delta, float size) {
            int b, q, h;
            where(r, rows, a.H, a.Sq, b, q, h);
            const long long bh = (long long)b * a.H + h, at = bh * a.Sqp + q;
            const float lse = __ldcg(a.lse + bh * a.Sq + q);
            const bool dead = lse == -CUDART_INF_F;
            stat_l[at] = dead ? -CUDART_INF_F : shift - lse * CUDART_L2E_F;
            stat_d[at] = dead ? 0.0f : -delta;
            if (DT == DT_F16) stat_n[at] = size;
        });
    const int pad = a.Sqp - a.Sq;
    for (long long i = blockIdx.x * 256ll + threadIdx.x; i < (long long)a.B * a.H * pad; i += gridDim.x * 256ll) {
        const long long at = i / pad * a.Sqp + a.Sq + i % pad;
        stat_l[at] = -CUDART_INF_F;
        stat_d[at] = 0.0f;
        if (DT == DT_F16) stat_n[at] = 0.0f;
    }
    if (DT == DT_F16) {
        const long long keys = (long long)a.B * a.Sk * a.HK;
        int b, t, h;
        as_rows<DT, G>(
            a.v, nullptr, keys, a.D,
            [&](long long r) {
                where(r, keys, a.HK, a.Sk, b, t, h);
                return t < attn_keys(a, b) ? b * a.vs[0] + t * a.vs[1] + h * a.vs[2] : -1ll;
            },
            [&](long long r, float, float size) {
                where(r, keys, a.HK, a.Sk, b, t, h);
                v_n[((long long)b * a.HK + h) * a.Sk + t] = size;
            });
    }
}

// The largest |dO row| and |v row| of each sample and key head, a block each: a
// gradient's range goes by what its own sums hold, so that nothing of one
// sample or head is lost beside the gradients of another.  (A launch of 3 us
// where a maximum by atomics would need its memory cleared by another.)
__global__ void __launch_bounds__(1024) attn_range_kernel(const AttnArgs a, const float *v_n, float2 *range) {
    __shared__ float2 warps[32];
    griddep_wait();
    const long long rows = (long long)(a.H / a.HK) * a.Sqp;  // the heads of a group lie side by side
    const float *n = a.stat_n + blockIdx.x * rows, *v = v_n + blockIdx.x * (long long)a.Sk;
    float2 top = make_float2(0.0f, 0.0f);
#pragma unroll 8
    for (long long i = threadIdx.x; i < rows; i += 1024) top.x = fmaxf(top.x, __ldcg(n + i));
#pragma unroll 8
    for (long long i = threadIdx.x; i < a.Sk; i += 1024) top.y = fmaxf(top.y, __ldcg(v + i));
#pragma unroll
    for (int w = 16; w > 0; w >>= 1) {
        top.x = fmaxf(top.x, __shfl_xor_sync(0xffffffffu, top.x, w));
        top.y = fmaxf(top.y, __shfl_xor_sync(0xffffffffu, top.y, w));
    }
    if ((threadIdx.x & 31) == 0) warps[threadIdx.x >> 5] = top;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < 32; ++w) top.x = fmaxf(top.x, warps[w].x), top.y = fmaxf(top.y, warps[w].y);
        range[blockIdx.x] = top;
    }
}

// P and dS of one T x T tile into shared memory, [query][key].
template <int DP, int T>
__device__ __forceinline__ void as_grad_tile(const AttnArgs &a, const float *Q, const float *K, const float *V,
                                             const float *G, float *P, float *S, long long stat_at, int k0, int len,
                                             int ty, int tx) {
    constexpr int N = T / 16;
    float s[N][N], dp[N][N];
    as_dot<DP, N>(Q, K, ty, tx, s);
    as_dot<DP, N>(G, V, ty, tx, dp);
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const float2 st = make_float2(__ldcg(a.stat_l + stat_at + N * ty + i), __ldcg(a.stat_d + stat_at + N * ty + i));
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const bool in = k0 + tx + 16 * j < len && st.x != -CUDART_INF_F;
            const float p = in ? exp2f(s[i][j] * a.scale * CUDART_L2E_F + st.x) : 0.0f;
            const int at = (N * ty + i) * (T + 1) + tx + 16 * j;
            P[at] = p;
            S[at] = in ? p * (dp[i][j] + st.y) : 0.0f;
        }
    }
}

// dK and dV of a tile of keys: all query tiles of all heads that share it.
template <int DT, int DP, int T>
__device__ __forceinline__ void as_dkdv(const AttnArgs &a, float *sm, unsigned block) {
    constexpr int N = T / 16, Z = T * (DP + 4);
    float *K = sm, *V = K + Z, *Q = V + Z, *G = Q + Z, *P = G + Z, *S = P + T * (T + 1);
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const int tiles = (a.Sk + T - 1) / T, bh = (int)(block / tiles);
    const int k0 = (int)(block % tiles) * T, b = bh / a.HK, hk = bh % a.HK, group = a.H / a.HK;
    const int len = attn_keys(a, b);
    as_load<DT, DP, T>(K, a.k, b * a.ks[0] + k0 * a.ks[1] + hk * a.ks[2], a.ks[1], len - k0, a.D);
    as_load<DT, DP, T>(V, a.v, b * a.vs[0] + k0 * a.vs[1] + hk * a.vs[2], a.vs[1], len - k0, a.D);
    float dk[N][DP / 64][4] = {}, dv[N][DP / 64][4] = {};
    for (int h = hk * group; h < (hk + 1) * group && k0 < len; ++h)
        for (int q0 = 0; q0 < a.Sq; q0 += T) {
            __syncthreads();
            as_load<DT, DP, T>(Q, a.q, b * a.qs[0] + q0 * a.qs[1] + h * a.qs[2], a.qs[1], a.Sq - q0, a.D);
            as_load<DT, DP, T>(G, a.dout, (((long long)b * a.Sq + q0) * a.H + h) * a.D, (long long)a.H * a.D, a.Sq - q0,
                            a.D);
            __syncthreads();
            as_grad_tile<DP, T>(a, Q, K, V, G, P, S, ((long long)b * a.H + h) * a.Sqp + q0, k0, len, ty, tx);
            __syncthreads();
            as_mix<DP, N>(P, 1, T + 1, G, ty, tx, dv);
            as_mix<DP, N>(S, 1, T + 1, Q, ty, tx, dk);
        }
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int t = k0 + N * ty + i;
        if (t >= a.Sk) continue;
#pragma unroll
        for (int c = 0; c < DP / 64; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int d = 4 * tx + 64 * c + e;
                if (d >= a.D) continue;
                const long long at = (((long long)b * a.Sk + t) * a.HK + hk) * a.D + d;
                store_act(a.dk, at, DT, t < len ? dk[i][c][e] * a.scale : 0.0f);
                store_act(a.dv, at, DT, t < len ? dv[i][c][e] : 0.0f);
            }
    }
}

// dQ of a tile of queries.
template <int DT, int DP, int T>
__device__ __forceinline__ void as_dq(const AttnArgs &a, float *sm, unsigned block) {
    constexpr int N = T / 16, Z = T * (DP + 4);
    float *K = sm, *V = K + Z, *Q = V + Z, *G = Q + Z, *P = G + Z, *S = P + T * (T + 1);
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const int tiles = (a.Sq + T - 1) / T, bh = (int)(block / tiles);
    const int q0 = (int)(block % tiles) * T, b = bh / a.H, h = bh % a.H, hk = h / (a.H / a.HK);
    const int len = attn_keys(a, b);
    as_load<DT, DP, T>(Q, a.q, b * a.qs[0] + q0 * a.qs[1] + h * a.qs[2], a.qs[1], a.Sq - q0, a.D);
    as_load<DT, DP, T>(G, a.dout, (((long long)b * a.Sq + q0) * a.H + h) * a.D, (long long)a.H * a.D, a.Sq - q0, a.D);
    float dq[N][DP / 64][4] = {};
    for (int k0 = 0; k0 < len; k0 += T) {
        __syncthreads();
        as_load<DT, DP, T>(K, a.k, b * a.ks[0] + k0 * a.ks[1] + hk * a.ks[2], a.ks[1], len - k0, a.D);
        as_load<DT, DP, T>(V, a.v, b * a.vs[0] + k0 * a.vs[1] + hk * a.vs[2], a.vs[1], len - k0, a.D);
        __syncthreads();
        as_grad_tile<DP, T>(a, Q, K, V, G, P, S, ((long long)b * a.H + h) * a.Sqp + q0, k0, len, ty, tx);
        __syncwarp();  // the rows of S that a warp reads are its own
        as_mix<DP, N>(S, T + 1, 1, K, ty, tx, dq);
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int t = q0 + N * ty + i;
        if (t >= a.Sq) continue;
#pragma unroll
        for (int c = 0; c < DP / 64; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int d = 4 * tx + 64 * c + e;
                if (d < a.D)
                    store_act(a.dq, (((long long)b * a.Sq + t) * a.H + h) * a.D + d, DT, dq[i][c][e] * a.scale);
            }
    }
}

// grid: key tiles * B * HK blocks for dK and dV, then query tiles * B * H for dQ
template <int DT, int DP, int T>
__global__ void __launch_bounds__(AS_THREADS) attn_simt_bwd_kernel(const AttnArgs a) {
    extern __shared__ float sm[];
    griddep_wait();
    const unsigned first = (unsigned)((a.Sk + T - 1) / T) * a.B * a.HK;
    if (blockIdx.x < first) as_dkdv<DT, DP, T>(a, sm, blockIdx.x);
    else as_dq<DT, DP, T>(a, sm, blockIdx.x - first);
}

}  // namespace reels
