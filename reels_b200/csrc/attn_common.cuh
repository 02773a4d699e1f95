// Pieces the tensor-core attention kernels share (attn_fwd.cuh, attn_bwd.cuh):
// tile geometry, 4-d TMA loads, tensor-memory moves and the exponential.
//
// Operand tiles are 128 tokens of one head as DP/64 "atoms" of 128 rows x 64
// features (128 bytes a row, TMA 128-byte swizzle).  The same tile serves as
// a K-major operand (features are the reduction: rows are M or N) and as an
// MN-major one (tokens are the reduction, features are N).
#pragma once
#include "attn_simt.cuh"

namespace reels {

constexpr int AT_TILE = 128;

// Operand descriptors.  The issuing thread's instructions are the rate of the
// short MMAs here, so descriptors are formed once per tile and a step only
// adds a constant to the address field (bytes / 16; no carry, shared memory
// ends below 2^18).
// K-major: reduction step kk of 16 features; MN-major: step kk of 16 tokens.
__device__ __forceinline__ uint64_t at_desc_k(uint32_t tile) { return sdesc_sw128(tile, 16, 1024); }
__device__ __forceinline__ uint64_t at_desc_mn(uint32_t tile) { return sdesc_sw128(tile, AT_TILE * 128, 1024); }
__device__ __forceinline__ constexpr uint64_t at_step_k(int kk) { return (kk >> 2) * (AT_TILE * 128 / 16) + (kk & 3) * 2; }
__device__ __forceinline__ constexpr uint64_t at_step_mn(int kk) { return kk * 128; }

__device__ __forceinline__ void tma_load_4d(uint32_t smem_dst, const void *tmap, int x, int y, int z, int w,
                                            uint64_t *bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(smem_dst),
        "l"(reinterpret_cast<uint64_t>(tmap)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(smem_u32(bar))
        : "memory");
}
// 128 tokens from `token` on of one head, DP features.
template <int DP>
__device__ __forceinline__ void at_load_tile(uint32_t dst, const void *tmap, int token, int head, int batch,
                                             uint64_t *bar) {
#pragma unroll
    for (int a = 0; a < DP / 64; ++a) tma_load_4d(dst + a * (AT_TILE * 128), tmap, 64 * a, token, head, batch, bar);
}

// D[tmem] (+)= A[tmem] * B[smem].
__device__ __forceinline__ void at_mma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc,
                                          uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
        "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}

// One thread of a converged warp, the same at every call.
__device__ __forceinline__ bool at_elect() {
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(ok));
    return ok != 0;
}

#define AT_R8(r, i) "=r"(r[i]), "=r"(r[i + 1]), "=r"(r[i + 2]), "=r"(r[i + 3]), "=r"(r[i + 4]), "=r"(r[i + 5]), \
                    "=r"(r[i + 6]), "=r"(r[i + 7])
#define AT_W8(r, i) "r"(r[i]), "r"(r[i + 1]), "r"(r[i + 2]), "r"(r[i + 3]), "r"(r[i + 4]), "r"(r[i + 5]), \
                    "r"(r[i + 6]), "r"(r[i + 7])
// 32 lanes x 32 columns, thread t its own lane.
__device__ __forceinline__ void at_tmem_ld32(uint32_t taddr, uint32_t *r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : AT_R8(r, 0), AT_R8(r, 8), AT_R8(r, 16), AT_R8(r, 24)
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void at_tmem_st32(uint32_t taddr, const uint32_t *r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};" ::AT_W8(r, 0),
        AT_W8(r, 8), AT_W8(r, 16), AT_W8(r, 24), "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void at_tmem_st16(uint32_t taddr, const uint32_t *r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::AT_W8(r, 0),
        AT_W8(r, 8), "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void at_tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ float at_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ float at_max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// A pair of neighbouring accumulator columns.
__device__ __forceinline__ F2 at_pair(const uint32_t *r, int k) {
    return F2(__uint_as_float(r[2 * k]), __uint_as_float(r[2 * k + 1]));
}
template <int DT>
__device__ __forceinline__ uint32_t at_pack(F2 v) {
    const float2 f = v.get();
    return Elem<DT>::pack2(f.x, f.y);
}

// Probabilities are at most 1 (2^8 before the running maximum catches up) and
// fall to 2^-15 and below on long rows.  bf16 holds that range as it is; fp16
// gets them multiplied by a power of two that uses its range up to 2^15 and
// is taken out of the fp32 sums again.
template <int DT>
struct AtRange {
    static constexpr float FWD_SHIFT = DT == DT_F16 ? 7.0f : 0.0f;   // with a lag of 8
    static constexpr float BWD_SHIFT = DT == DT_F16 ? 15.0f : 0.0f;  // P <= 1
};

// The kernels are launched with 12 warps of 168 registers a thread.  The
// eight elementwise warps (two groups of four) hold a row of scores each and
// take MORE, the other four keep FEWER: 256 MORE + 128 FEWER = 384 * 168.
// Called at the head of each role, so that the compiler knows which count holds.
template <int MORE>
struct AtRegisters {
    static constexpr int FEWER = 504 - 2 * MORE;
    static_assert(MORE % 8 == 0 && FEWER % 8 == 0 && FEWER >= 24, "register counts come in eights");
    static __device__ __forceinline__ void more() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(MORE)); }
    static __device__ __forceinline__ void fewer() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(FEWER)); }
};

// 32 fp32 values of this thread's row times f, as 16-bit values at dst + c0 up
// to feature D, in whole 32-byte sectors where alignment allows (a warp writes
// 32 rows at once: half the requests), or as they are at part + c0.
template <int DT>
__device__ __forceinline__ void at_store32(const uint32_t *o, float f, typename Elem<DT>::T *dst, float *part, int c0,
                                           int D, bool sectors) {
#pragma unroll
    for (int e = 0; e < 32; e += 16) {
        if (c0 + e >= D) continue;
        F2 v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = mul2(at_pair(o, e / 2 + k), F2(f, f));
        if (part) {
#pragma unroll
            for (int k = 0; k < 8; k += 2)
                if (c0 + e + 2 * k < D) {
                    const float2 x = v[k].get(), y = v[k + 1].get();
                    *reinterpret_cast<float4 *>(part + c0 + e + 2 * k) = make_float4(x.x, x.y, y.x, y.y);
                }
            continue;
        }
        const uint4 lo = make_uint4(at_pack<DT>(v[0]), at_pack<DT>(v[1]), at_pack<DT>(v[2]), at_pack<DT>(v[3]));
        const uint4 hi = make_uint4(at_pack<DT>(v[4]), at_pack<DT>(v[5]), at_pack<DT>(v[6]), at_pack<DT>(v[7]));
        if (sectors) {
            st_global_v8(dst + c0 + e, lo, hi);
        } else {
            *reinterpret_cast<uint4 *>(dst + c0 + e) = lo;
            if (c0 + e + 8 < D) *reinterpret_cast<uint4 *>(dst + c0 + e + 8) = hi;
        }
    }
}
// Whether rows of D 16-bit features from `p` on are whole 32-byte sectors.
__device__ __forceinline__ bool at_sectors(const void *p, int D) {
    return ((reinterpret_cast<uintptr_t>(p) & 31) | (D & 15)) == 0;
}

// A wait of a whole warp on one barrier.
__device__ __forceinline__ bool at_wait(uint64_t *bar, uint32_t parity, volatile int *abort, unsigned *err,
                                        unsigned code) {
    const bool ok = wait_bar(bar, parity, abort, err, code);
    return __all_sync(0xffffffffu, ok);
}

// Waits for the issuers' last commits, then gives the tensor memory back.
__device__ __forceinline__ void at_finish(uint32_t tmem, uint64_t *mma_done, int issuers, unsigned *err) {
    tc_fence_after();
    for (int t = 0; t < issuers; ++t) {
        const long long t0 = clock64();
        while (!mbar_try_wait(&mma_done[t], 0)) {
            if (clock64() - t0 > REELS_WAIT_LIMIT_CYCLES) {
                if ((threadIdx.x & 31) == 0) atomicOr(err, DEVERR_TIMEOUT_ACC);
                break;
            }
        }
    }
    __syncwarp();
    tmem_dealloc(tmem, 512);
}

// Zeroes rows from `first` on of an operand tile: keys behind a sample's
// length have probability 0, but 0 times what padding may hold (NaN, Inf)
// would still reach the sums.  Called by a whole warp before the tile's MMAs.
template <int DP>
__device__ __forceinline__ void at_zero_rows(uint8_t *tile, int first) {
    for (int i = first * 8 + (int)(threadIdx.x & 31); i < AT_TILE * 8; i += 32)
#pragma unroll
        for (int a = 0; a < DP / 64; ++a)
            reinterpret_cast<uint4 *>(tile + a * (AT_TILE * 128))[i] = make_uint4(0, 0, 0, 0);
    fence_proxy_async_smem();
    __syncwarp();
}

}  // namespace reels
