// Matrix products in 8-bit integers with a scale for each token and channel.
//
//   C[m, n] = fp16( a_scale[m] * w_scale[n] * sum_k A[m, k] W[n, k] )  (+ R[m, n])
//   SwiGLU:   C[m, c] = fp16( silu(z[m, 2c]) * z[m, 2c + 1] ),  z the product above before rounding
//
// tcgen05.mma kind::i8: both operands s8 and K-major from shared memory (one
// 128-byte swizzled row = 128 of K), the sums s32 in tensor memory, exact up to
// |sum| < 2^31 (K * 128 * 128, which bounds K).  The scales are applied in fp32
// and the result is rounded to fp16 once.
//
// Two kernels:
//   w8a8_tile_kernel  persistent, 256 channels x 256 tokens (two MMAs share the
//                     channels' tile; the sums fill tensor memory) or x 128
//                     (the sums of two tiles, so that the epilogue runs behind
//                     the next tile's MMAs)
//   w8a8_few_kernel   128 channels x BT tokens in one CTA, the K axis over the
//                     CTAs of a cluster, which add their sums through one
//                     another's shared memory (integers: the order does not
//                     matter); for few tokens, where the weights' bytes bound
//                     it, and for products of few tiles
// and `pick` chooses.
//
// What bounds the tile kernel: an MMA of 128 x 256 x 32 reads 12 KB of shared
// memory in its 128 cycles, and the copies write 64 KB (256 tokens) for 8 of
// them, 48 KB (128) for 4: 160 and 192 bytes a cycle where the SM has 128, so
// 80 % and 67 % of the tensor rate at the same clock.  8192 x 22016 x 4096 runs
// into the power limit first (542 us, 2730 TOP/s at 1.45 - 1.5 GHz; 128 tokens
// 571), 2048 x 4096 x 11008 takes 78 us in one wave of 256 tokens and 85 in two
// of 128, 1024 x 12288 x 4096 59 and 51.5, 256 x 12288 x 4096 33 and 22.  Stages
// of 64 of K instead of 128, twice as many: 569 and 704 us on the first.
#include "common.cuh"
#include "gemm_tc.h"

namespace npub {
namespace w8a8 {

constexpr int BK = 128;       // K per stage: one swizzled row
constexpr int kUmmaK = 32;    // K of one MMA
constexpr int kMaxCluster = 8;

struct Params {
    CUtensorMap tmA, tmW;
    int M, N, k_tiles;
    int m_tiles, n_tiles, band;      // tile kernel
    int per;                         // few kernel: K tiles of a CTA
    const float* sa;
    const __half* sw;
    const __half* R;
    int64_t ldr;
    __half* C;
    int64_t ldc;
    int swiglu;
    int vec;                         // rows of C (and R) and the scales can be read and written 16 bytes at a time
    int* err;
};

__host__ __device__ constexpr uint32_t idesc_i8(int m, int n) {  // s32 sums, s8 x s8, both K-major
    return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
__device__ __forceinline__ void mma_i8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void set_err(int* err, int code) {
    if (err) atomicCAS(err, 0, code);
}
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, int (&r)[32]) {
    __syncwarp();
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
        "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_ld16i(uint32_t taddr, int (&r)[16]) {
    __syncwarp();
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ uint32_t pack_h2(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float2 half2_at(uint32_t u) { return __half22float2(*reinterpret_cast<const __half2*>(&u)); }

// ------------------------------------------------------------- tiles of 256 channels

constexpr int kTileThreads = 384;
// MH halves of 128 tokens.  The sums take all of tensor memory: with MH = 2 one
// tile's two halves, each read by four epilogue warps, with MH = 1 two tiles',
// each read by all eight.
template <int MH>
struct TileSmem {
    static constexpr int kOp = 128 * BK;  // 128 rows of either operand
    static constexpr int kStage = (MH + 2) * kOp;
    static constexpr int kStages = MH == 2 ? 3 : 4;
    static constexpr int kOffBar = kStages * kStage;
    static constexpr int kOffOut = kOffBar + 256;  // epilogue warps: 32 x 32 sums, rows of 33 words
    static constexpr int kTotal = kOffOut + 8 * 32 * 33 * 4 + 1024;
    static_assert((2 * kStages + 5) * 8 + 8 <= 256, "the barriers' part");
};

// Tiles in bands of p.band token tiles, the channels in turn within a band, so
// that the tiles in flight share operands in L2.
struct TileAt {
    int m0, n0;
};
template <int MH>
__device__ __forceinline__ TileAt tile_at(const Params& p, int t) {
    const int per_band = p.band * p.n_tiles, b = t / per_band, r = t - b * per_band;
    const int nb = min(p.band, p.m_tiles - b * p.band), n = r / nb;
    return TileAt{(b * p.band + r - n * nb) * 128 * MH, n * 256};
}

template <int MH>
__global__ void __launch_bounds__(kTileThreads, 1) w8a8_tile_kernel(const __grid_constant__ Params p) {
    using L = TileSmem<MH>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::kOffBar);  // [stages] both operands landed
    uint64_t* empty = full + L::kStages;                              // [stages] the MMAs are done with the stage
    uint64_t* acc_full = empty + L::kStages;                          // [2] sums ready
    uint64_t* acc_empty = acc_full + 2;                               // [2] the epilogue has read them
    uint64_t* drained = acc_empty + 2;                                // after an abort: the MMAs are done
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drained + 1);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int n_all = p.m_tiles * p.n_tiles;

    if (threadIdx.x == 0) {
        for (int s = 0; s < L::kStages; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&acc_full[b], 1);
            mbar_init(&acc_empty[b], MH == 2 ? 4 : 8);
        }
        mbar_init(drained, 1);
        *abort_flag = 0;
        fence_barrier_init();
        prefetch_tmap(&p.tmA);
        prefetch_tmap(&p.tmW);
    }
    if (warp == 1) {
        tmem_alloc(tmem_slot, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    cta_sync_divergent();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    if (warp == 0) {
        if (lane == 0) {  // producer
            uint32_t g = 0;
            bool ok = true;
            for (int t = (int)blockIdx.x; t < n_all && ok; t += (int)gridDim.x) {
                const TileAt at = tile_at<MH>(p, t);
                for (int i = 0; i < p.k_tiles; ++i, ++g) {
                    const int s = (int)(g % L::kStages);
                    ok = mbar_wait_quick(&empty[s], ((g / L::kStages) & 1u) ^ 1u, abort_flag);
                    if (!ok) break;
                    uint8_t* st = smem + s * L::kStage;
                    mbar_arrive_expect_tx(&full[s], (uint32_t)L::kStage);
                    tma_load_3d(st, &p.tmA, &full[s], i * BK, at.m0, 0);
                    tma_load_3d(st + MH * L::kOp, &p.tmW, &full[s], i * BK, at.n0, 0);
                }
            }
            if (!ok) {  // copies in flight land before the CTA leaves (the MMA thread waits for them otherwise)
                *abort_flag = 1;
                set_err(p.err, 0x701);
                int never = 0;
                for (uint32_t j = g < (uint32_t)L::kStages ? 0 : g - L::kStages; j < g; ++j)
                    mbar_wait_bounded(&full[j % L::kStages], (j / L::kStages) & 1u, &never, 100000000ull);
            }
        }
    } else if (warp == 1) {
        if (elect_one()) {  // MMA
            constexpr uint32_t idesc = idesc_i8(128, 256);
            uint32_t g = 0, n = 0;
            int code = 0;
            for (int t = (int)blockIdx.x; t < n_all && !code; t += (int)gridDim.x, ++n) {
                for (int i = 0; i < p.k_tiles && !code; ++i, ++g) {
                    const int s = (int)(g % L::kStages);
                    if (!mbar_wait_quick(&full[s], (g / L::kStages) & 1u, abort_flag)) {
                        code = 0x703;
                        break;
                    }
                    const uint32_t a = smem_u32(smem + s * L::kStage), w = a + MH * L::kOp;
#pragma unroll
                    for (int h = 0; h < MH; ++h) {
                        const uint32_t b = MH == 2 ? h : n & 1u, ph = MH == 2 ? n & 1u : (n >> 1) & 1u;
                        if (i == 0 && !mbar_wait_quick(&acc_empty[b], ph ^ 1u, abort_flag)) {
                            code = 0x702;
                            break;
                        }
                        tc_fence_after();
#pragma unroll
                        for (int k = 0; k < BK / kUmmaK; ++k)
                            mma_i8(tmem + b * 256u, umma_desc_sw128(a + h * L::kOp + k * kUmmaK),
                                   umma_desc_sw128(w + k * kUmmaK), idesc, (i > 0 || k > 0) ? 1u : 0u);
                        if (i == p.k_tiles - 1) tc_commit(&acc_full[b]);
                    }
                    if (!code) tc_commit(&empty[s]);
                }
            }
            if (code) {
                set_err(p.err, code);
                *abort_flag = 1;
                int never = 0;
                tc_commit(drained);
                mbar_wait_bounded(drained, 0, &never, 100000000ull);
                for (uint32_t j = g; j < g + (uint32_t)L::kStages; ++j)  // copies that nobody has waited for
                    mbar_wait_bounded(&full[j % L::kStages], (j / L::kStages) & 1u, &never, 100000000ull);
            }
        }
    } else if (warp >= 4) {
        // -------------------------------------------------------------------- epilogue: one token per lane
        const int wq = warp & 3, group = (warp - 4) >> 2;
        // of this warp: 32 x 32 sums on their way out, or the channels' 256 scales
        int* out = reinterpret_cast<int*>(smem + L::kOffOut) + (warp - 4) * 32 * 33;
        uint32_t n = 0;
        for (int t = (int)blockIdx.x; t < n_all; t += (int)gridDim.x, ++n) {
            const TileAt at = tile_at<MH>(p, t);
            const int b = MH == 2 ? group : (int)(n & 1u);
            const uint32_t sums = tmem + ((uint32_t)(wq * 32) << 16) + (uint32_t)b * 256u;
            const int m = at.m0 + (MH == 2 ? group * 128 : 0) + wq * 32 + lane;
            const bool row = m < p.M;
            const int rows = min(32, p.M - (m - lane));              // of this warp, may be negative
            const int c0 = MH == 2 ? 0 : group * 4;                  // its chunks of 32 channels
            const int chunks = rows > 0 ? min(MH == 2 ? 8 : c0 + 4, (p.N - at.n0 + 31) / 32) : 0;
            const float sa = row ? __ldg(p.sa + m) : 0.0f;
            const __half* res = p.R ? p.R + (int64_t)m * p.ldr + at.n0 : nullptr;
            uint4 r[4];  // the residual of the chunk to come, where it can be read 16 bytes at a time
            auto fetch = [&](int c) {
                if (!p.vec || !res || !row || c >= 8 || at.n0 + c * 32 + 32 > p.N) return;
#pragma unroll
                for (int e = 0; e < 4; ++e) r[e] = *(reinterpret_cast<const uint4*>(res + c * 32) + e);
            };
            fetch(c0);
            if (p.vec) {
                if (at.n0 + lane * 8 + 8 <= p.N)
                    *(reinterpret_cast<uint4*>(out) + lane) = __ldg(reinterpret_cast<const uint4*>(p.sw + at.n0) + lane);
                __syncwarp();
            }
            // sums of 32 channels to C
            auto finish = [&](int c, int (&acc)[32]) {
                const int n0 = at.n0 + c * 32;
                if (p.vec && n0 + 32 <= p.N) {
                    float z[32];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const uint4 w = *(reinterpret_cast<const uint4*>(out) + c * 4 + e);
                        const uint32_t ww[4] = {w.x, w.y, w.z, w.w}, rr[4] = {r[e].x, r[e].y, r[e].z, r[e].w};
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const float2 f = half2_at(ww[i]);
                            z[e * 8 + 2 * i] = (float)acc[e * 8 + 2 * i] * (sa * f.x);
                            z[e * 8 + 2 * i + 1] = (float)acc[e * 8 + 2 * i + 1] * (sa * f.y);
                            if (res) {
                                const float2 g = half2_at(rr[i]);
                                z[e * 8 + 2 * i] += g.x;
                                z[e * 8 + 2 * i + 1] += g.y;
                            }
                        }
                    }
                    fetch(c + 1);
                    if (!row) return;
                    if (p.swiglu) {
                        uint4* dst = reinterpret_cast<uint4*>(p.C + (int64_t)m * p.ldc + n0 / 2);
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            uint32_t o[4];
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const float* g = z + e * 16 + i * 4;
                                o[i] = pack_h2(swiglu_f(g[0], g[1]), swiglu_f(g[2], g[3]));
                            }
                            dst[e] = make_uint4(o[0], o[1], o[2], o[3]);
                        }
                        return;
                    }
                    uint4* dst = reinterpret_cast<uint4*>(p.C + (int64_t)m * p.ldc + n0);
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        dst[e] = make_uint4(pack_h2(z[e * 8], z[e * 8 + 1]), pack_h2(z[e * 8 + 2], z[e * 8 + 3]),
                                            pack_h2(z[e * 8 + 4], z[e * 8 + 5]), pack_h2(z[e * 8 + 6], z[e * 8 + 7]));
                    return;
                }
                // rows that 16 bytes at a time do not fit: through shared memory, so that the lanes store along a row
                __syncwarp();
#pragma unroll
                for (int i = 0; i < 32; ++i) out[lane * 33 + i] = acc[i];
                __syncwarp();
                const int per = p.swiglu ? 2 : 1, n = n0 + lane * per;  // this lane's column, or the first of its two
                const bool on = lane * per < 32 && n < p.N;
                const float sw0 = on ? __half2float(__ldg(p.sw + n)) : 0.0f;
                const float sw1 = on && p.swiglu ? __half2float(__ldg(p.sw + n + 1)) : 0.0f;
                const __half* add = p.R ? p.R + (int64_t)(m - lane) * p.ldr + n : nullptr;
                __half* dst = p.C + (int64_t)(m - lane) * p.ldc + n / per;
#pragma unroll
                for (int q0 = 0; q0 < 32; q0 += 8) {
                    float z[8];
#pragma unroll
                    for (int q = 0; q < 8; ++q) {
                        const float sq = __shfl_sync(0xffffffffu, sa, q0 + q);
                        const int* v = out + (q0 + q) * 33 + (lane * per & 31);
                        z[q] = (float)v[0] * (sq * sw0);
                        if (p.swiglu) z[q] = swiglu_f(z[q], (float)v[1] * (sq * sw1));
                        if (add && on && q0 + q < rows) z[q] += __half2float(add[(int64_t)(q0 + q) * p.ldr]);
                    }
#pragma unroll
                    for (int q = 0; q < 8; ++q)
                        if (on && q0 + q < rows) dst[(int64_t)(q0 + q) * p.ldc] = __float2half_rn(z[q]);
                }
                __syncwarp();
            };
            const bool ok = __all_sync(0xffffffffu, mbar_wait_quick(&acc_full[b], MH == 2 ? n & 1u : (n >> 1) & 1u, abort_flag));
            if (!ok) {
                if (lane == 0) {
                    set_err(p.err, 0x704);
                    *abort_flag = 1;
                }
                break;
            }
            tc_fence_after();
            // the last two chunks go to registers ahead of their turn, and the MMAs may have the sums' place again
            int acc[32], last[32];
#pragma unroll 1
            for (int c = c0; c < chunks - 2; ++c) {
                tmem_ld32(sums + (uint32_t)(c * 32), acc);
                finish(c, acc);
            }
            if (chunks - 2 >= c0) tmem_ld32(sums + (uint32_t)((chunks - 2) * 32), acc);
            if (chunks - 1 >= c0) tmem_ld32(sums + (uint32_t)((chunks - 1) * 32), last);
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&acc_empty[b]);
            if (chunks - 2 >= c0) finish(chunks - 2, acc);
            if (chunks - 1 >= c0) finish(chunks - 1, last);
            __syncwarp();  // `out` is read
        }
    }

    tc_fence_before();
    cta_sync_divergent();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

// ------------------------------------------------ 128 channels x BT tokens, K over a cluster

constexpr int kFewThreads = 192;

template <int BT>
struct FewSmem {
    static constexpr int kW = 128 * BK, kX = BT * BK;
    static constexpr int kStages = BT >= 128 ? 3 : BT >= 64 ? 4 : 5;
    static constexpr int kOffBar = kStages * (kW + kX);
    static constexpr int kTotal = kOffBar + 256 + 1024;
    static_assert(BT * 128 * 4 <= kOffBar, "the sums reuse the ring");
};

// grid (cluster * channel tiles, token tiles); CTA r of a cluster takes K tiles
// [r * per, (r + 1) * per)
template <int BT>
__global__ void __launch_bounds__(kFewThreads) w8a8_few_kernel(const __grid_constant__ Params p) {
    using L = FewSmem<BT>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t *sW = smem, *sX = smem + L::kStages * L::kW;
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::kOffBar);
    uint64_t* empty = full + L::kStages;
    uint64_t* done = empty + L::kStages;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    volatile int* no_sums = abort_flag + 1;  // a CTA of the cluster gave up
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int S = (p.k_tiles + p.per - 1) / p.per;
    const int tile = (int)blockIdx.x / S, r = (int)blockIdx.x - tile * S;
    const int n0 = tile * 128, m0 = (int)blockIdx.y * BT;
    const int kt0 = r * p.per, nk = min(p.per, p.k_tiles - kt0);
    if (threadIdx.x == 0) {
        for (int s = 0; s < L::kStages; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        mbar_init(done, 1);
        *abort_flag = *no_sums = 0;
        fence_barrier_init();
    }
    if (warp == 4 && lane == 0) {
        prefetch_tmap(&p.tmA);
        prefetch_tmap(&p.tmW);
        // the first weight tiles come to L2 while the kernel ahead still runs
        for (int i = 0; i < min(nk, L::kStages); ++i) tma_prefetch_3d(&p.tmW, (kt0 + i) * BK, n0, 0);
    }
    if (warp == 5) {
        tmem_alloc(tmem_slot, BT);
        tmem_relinquish();
    }
    tc_fence_before();
    cta_sync_divergent();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    pdl_trigger();  // behind the allocation: a successor's CTA that waits for this grid may hold columns of its own
    pdl_wait();

    bool ok = true;
    auto give_up = [&](int code) {
        *abort_flag = 1;
        set_err(p.err, code);
        for (int q = 0; q < S; ++q)
            asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(mapa_shared(smem_u32((const void*)no_sums), q)), "r"(1) : "memory");
    };
    if (warp == 4) {
        if (lane == 0) {  // producer
            int i = 0;
            for (; i < nk; ++i) {
                const int s = i % L::kStages;
                ok = mbar_wait_quick(&empty[s], ((uint32_t)(i / L::kStages) & 1u) ^ 1u, abort_flag);
                if (!ok) break;
                mbar_arrive_expect_tx(&full[s], (uint32_t)(L::kW + L::kX));
                tma_load_3d(sW + s * L::kW, &p.tmW, &full[s], (kt0 + i) * BK, n0, 0);
                tma_load_3d(sX + s * L::kX, &p.tmA, &full[s], (kt0 + i) * BK, m0, 0);
            }
            if (!ok) {  // copies in flight land before the CTA leaves
                give_up(0x711);
                int never = 0;
                for (int j = max(0, i - L::kStages); j < i; ++j)
                    mbar_wait_bounded(&full[j % L::kStages], (uint32_t)(j / L::kStages) & 1u, &never, 100000000ull);
            }
        }
    } else if (warp == 5) {
        if (elect_one()) {  // MMA
            constexpr uint32_t idesc = idesc_i8(128, BT);
            int i = 0;
            for (; i < nk; ++i) {
                const int s = i % L::kStages;
                ok = mbar_wait_quick(&full[s], (uint32_t)(i / L::kStages) & 1u, abort_flag);
                if (!ok) break;
                tc_fence_after();
                const uint32_t w = smem_u32(sW + s * L::kW), x = smem_u32(sX + s * L::kX);
#pragma unroll
                for (int k = 0; k < BK / kUmmaK; ++k)
                    mma_i8(tmem, umma_desc_sw128(w + k * kUmmaK), umma_desc_sw128(x + k * kUmmaK), idesc,
                           (i > 0 || k > 0) ? 1u : 0u);
                tc_commit(&empty[s]);
            }
            if (!ok) give_up(0x712);
            tc_commit(done);
            if (!ok) {  // the MMAs end, and the copies that nobody has waited for land, before the CTA leaves
                int never = 0;
                mbar_wait_bounded(done, 0, &never, 100000000ull);
                for (int j = i; j < min(nk, i + L::kStages); ++j)
                    mbar_wait_bounded(&full[j % L::kStages], (uint32_t)(j / L::kStages) & 1u, &never, 100000000ull);
            }
        }
    } else {
        ok = __all_sync(0xffffffffu, mbar_wait_quick(done, 0, abort_flag));
        tc_fence_after();
        if (ok) {  // the ring is free: this CTA's sums [token][channel]
            int* sums = reinterpret_cast<int*>(smem) + warp * 32 + lane;
            const uint32_t t = tmem + ((uint32_t)(warp * 32) << 16);
#pragma unroll 1
            for (int c0 = 0; c0 < BT && m0 + c0 < p.M; c0 += 16) {
                int acc[16];
                tmem_ld16i(t + (uint32_t)c0, acc);
#pragma unroll
                for (int j = 0; j < 16; ++j) sums[(c0 + j) * 128] = acc[j];
            }
        } else if (lane == 0) {
            give_up(0x713);
        }
    }
    tc_fence_before();
    if (S > 1) cluster_sync();
    else cta_sync_divergent();
    if (warp == 5) {
        tc_fence_after();
        tmem_dealloc(tmem, BT);
    }
    if (warp < 4 && !*no_sums) {
        const int tokens = min(BT, p.M - m0);
        const int n = n0 + lane * 4;
        const int left = p.N - n;  // channels of this lane
        const uint32_t base = smem_u32(smem) + (uint32_t)lane * 16u;
        float sw[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) sw[i] = i < left ? __half2float(__ldg(p.sw + n + i)) : 0.0f;
        for (int j = r * 4 + warp; j < tokens; j += S * 4) {
            int4 v = make_int4(0, 0, 0, 0);
            int4 got[kMaxCluster];
#pragma unroll
            for (int q = 0; q < kMaxCluster; ++q)
                if (q < S)
                    asm volatile("ld.shared::cluster.v4.s32 {%0, %1, %2, %3}, [%4];"
                                 : "=r"(got[q].x), "=r"(got[q].y), "=r"(got[q].z), "=r"(got[q].w)
                                 : "r"(mapa_shared(base + (uint32_t)j * 512u, q))
                                 : "memory");
#pragma unroll
            for (int q = 0; q < kMaxCluster; ++q)
                if (q < S) {
                    v.x += got[q].x;
                    v.y += got[q].y;
                    v.z += got[q].z;
                    v.w += got[q].w;
                }
            if (left <= 0) continue;
            const int m = m0 + j;
            const float sa = __ldg(p.sa + m);
            float z[4] = {(float)v.x * (sa * sw[0]), (float)v.y * (sa * sw[1]), (float)v.z * (sa * sw[2]),
                          (float)v.w * (sa * sw[3])};
            if (p.swiglu) {
                __half* dst = p.C + (int64_t)m * p.ldc + n / 2;
                const uint32_t o = pack_h2(swiglu_f(z[0], z[1]), swiglu_f(z[2], z[3]));
                if (p.vec && left >= 4) {
                    *reinterpret_cast<uint32_t*>(dst) = o;
                } else {
                    dst[0] = __ushort_as_half((unsigned short)(o & 0xffffu));
                    if (left >= 4) dst[1] = __ushort_as_half((unsigned short)(o >> 16));
                }
                continue;
            }
            __half* dst = p.C + (int64_t)m * p.ldc + n;
            const __half* res = p.R ? p.R + (int64_t)m * p.ldr + n : nullptr;
            if (p.vec && left >= 4) {
                if (res) {
                    const uint2 w = *reinterpret_cast<const uint2*>(res);
                    const float2 a = half2_at(w.x), b = half2_at(w.y);
                    z[0] += a.x;
                    z[1] += a.y;
                    z[2] += b.x;
                    z[3] += b.y;
                }
                *reinterpret_cast<uint2*>(dst) = make_uint2(pack_h2(z[0], z[1]), pack_h2(z[2], z[3]));
            } else {
                for (int i = 0; i < min(4, left); ++i)
                    dst[i] = __float2half_rn(z[i] + (res ? __half2float(res[i]) : 0.0f));
            }
        }
    }
    if (S > 1) cluster_sync();  // nobody leaves while its sums are read
}

// ---------------------------------------------------------------------- host

constexpr int kTile1 = 1, kTile2 = 2;  // the tile kernel with 128 and 256 tokens
struct Choice {
    int bt;      // kTile1, kTile2, or the tokens of the few-token kernel's tiles
    int splits;
};

// The estimates' terms, in us, are fitted to CUDA graphs of calls of 1 to 8192 tokens: those above; few-token kernel at 12288
// x 4096 with one and two CTAs for a tile, 32 tokens 15.4 and 14.2, 64 in one tile 19.5 and 16.7, 128 in two 20.5 and 26.6;
// 4096 x 4096 at 32 tokens with 1, 2, 4, 8: 12.6, 9.5, 7.7, 7.7.
// Rows that are not written 16 bytes at a time, few-token kernel, tiles of 128 and of 256 tokens: 777 x 1003 x 2064 13.6, 22.6
// and 35.0; tiles alone, 4000 x 1003 x 4096 24 and 41, 4000 x 5001 x 4096 73 and 110, 8000 x 12289 x 4096 319 and 393, with a
// residual 732 and 763.  The two constants for such rows are the first of these sizes', for any number of waves, and the few-token
// kernel's stores count nothing there, so that up to 800 tokens of many channels it is taken where tiles of 128 are better
// (777 x 5001 x 2064 29.5 and 23.3, 777 x 12289 x 11008 168 and 113), and with a residual and K of 11008 tiles of 256 (4000 x 2049
// 115 and 97, 2000 x 12289 317 and 234).
Choice pick(int M, int N, int k_tiles, bool vec) {
    // clusters of 1 .. 8 CTAs that 148 SMs (whole GPCs of them) hold at one CTA per SM; the few-token kernel has two
    static const int held[kMaxCluster + 1] = {0, 148, 74, 45, 33, 26, 22, 15, 15};
    const int sms = num_sms();
    const int64_t wide = (N + 255) / 256, t1 = (int64_t)((M + 127) / 128) * wide, t2 = (int64_t)((M + 255) / 256) * wide;
    const double some1 = t1 < sms ? (double)t1 / sms : 1.0, some2 = t2 < sms ? (double)t2 / sms : 1.0;
    const double us1 = (vec ? 4.1 : 13.0) + (double)((t1 + sms - 1) / sms) * k_tiles * (0.40 + 0.07 * some1);
    const double us2 = (vec ? 4.5 : 22.0) + (double)((t2 + sms - 1) / sms) * (k_tiles * (0.61 + 0.17 * some2) + 4.0);
    Choice c = {us1 <= us2 ? kTile1 : kTile2, 1};
    double best = us1 <= us2 ? us1 : us2;
    for (int bt = 32; bt <= 128; bt *= 2) {
        const int64_t token_tiles = (M + bt - 1) / bt, tiles = (int64_t)((N + 127) / 128) * token_tiles;
        if (token_tiles > 8) continue;
        const int stages = bt == 32 ? FewSmem<32>::kStages : bt == 64 ? FewSmem<64>::kStages : FewSmem<128>::kStages;
        for (int s = 1; s <= kMaxCluster && s <= k_tiles; ++s) {
            const int per = (k_tiles + s - 1) / s;
            if ((k_tiles + per - 1) / per != s) continue;
            int64_t at_once = 2 * (int64_t)held[s] * sms / 148;
            if (at_once < 1) at_once = 1;
            const double waves = (double)((tiles + at_once - 1) / at_once), ctas = (double)(tiles < at_once ? tiles : at_once) * s;
            // a K tile: a ring's latency, which grows with the weights in flight, HBM's rate, or the SM's tensor core
            const double bytes = ctas / (double)token_tiles * 16384.0;
            double unit = (1.0 + 0.45 * bytes / 1.57e6) / stages;
            if (unit < bytes / 6.5e6) unit = bytes / 6.5e6;
            const double mma = (bt < 128 ? 0.13 : 0.17) * (ctas > sms ? ctas / sms : 1.0);
            if (unit < mma) unit = mma;
            const double us = 4.6 + 0.004 * M + waves * (per * unit + 1.0 + bt / 51.0) + (s > 1 ? 0.5 + 0.12 * s : 0.0);
            if (us < best) {
                best = us;
                c = Choice{bt, s};
            }
        }
    }
    return c;
}

template <int BT>
int launch_few(Params& p, int splits, cudaStream_t st) {
    using L = FewSmem<BT>;
    static_assert(L::kTotal <= 232448, "shared memory budget");
    auto kern = w8a8_few_kernel<BT>;
    NPUB_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kTotal));
    p.per = (p.k_tiles + splits - 1) / splits;
    const int S = (p.k_tiles + p.per - 1) / p.per;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(S * ((p.N + 127) / 128)), (unsigned)((p.M + BT - 1) / BT));
    cfg.blockDim = dim3(kFewThreads);
    cfg.dynamicSmemBytes = L::kTotal;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = npub_internal_pdl_enabled() ? 1 : 0;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = S;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    NPUB_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, p));
    return npub_internal_launch_status();
}

template <int MH>
int launch_tile(Params& p, cudaStream_t st) {
    using L = TileSmem<MH>;
    static_assert(L::kTotal <= 232448, "shared memory budget");
    NPUB_CUDA_TRY(cudaFuncSetAttribute(w8a8_tile_kernel<MH>, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kTotal));
    p.m_tiles = (p.M - 1) / (128 * MH) + 1;
    p.n_tiles = (p.N - 1) / 256 + 1;
    p.band = 16 / MH;
    const int64_t tiles = (int64_t)p.m_tiles * p.n_tiles;
    if (tiles > 0x3fffffff) return NPUB_ERR_UNSUPPORTED;
    const int sms = num_sms();
    w8a8_tile_kernel<MH><<<(unsigned)(tiles < sms ? tiles : sms), kTileThreads, L::kTotal, st>>>(p);
    return npub_internal_launch_status();
}

}  // namespace w8a8
}  // namespace npub

extern "C" int npub_w8a8_gemm(const int8_t* A, int64_t lda, const float* a_scale, const int8_t* W, int64_t ldw,
                              const void* w_scale, void* C, int64_t ldc, const void* R, int64_t ldr, int M, int N, int K,
                              int swiglu, void* stream) {
    using namespace npub;
    using namespace npub::w8a8;
    NPUB_CHECK_ARG(M >= 0 && N >= 0 && K > 0 && K % 16 == 0);
    NPUB_CHECK_ARG(!swiglu || (N % 2 == 0 && !R));
    if (M == 0 || N == 0) return NPUB_OK;
    NPUB_CHECK_ARG(A && a_scale && W && w_scale && C);
    NPUB_CHECK_ARG(lda % 16 == 0 && ldw % 16 == 0 && lda >= K && ldw >= K && npub_aligned(A, 16) && npub_aligned(W, 16));
    NPUB_CHECK_ARG(ldc >= (swiglu ? N / 2 : N) && (!R || ldr >= N));
    NPUB_CHECK_ARG(npub_aligned(a_scale, 4) && npub_aligned(w_scale, 2) && npub_aligned(C, 2) && npub_aligned(R, 2));
    if (K > 131056) return NPUB_ERR_UNSUPPORTED;  // 131072 * 128 * 128 = 2^31
    if (M > 0x7fffff00 || N > 0x7fffff00) return NPUB_ERR_UNSUPPORTED;
    Params p;
    memset(&p, 0, sizeof(p));
    p.M = M;
    p.N = N;
    p.k_tiles = (K + BK - 1) / BK;
    p.sa = a_scale;
    p.sw = reinterpret_cast<const __half*>(w_scale);
    p.C = reinterpret_cast<__half*>(C);
    p.ldc = ldc;
    p.R = reinterpret_cast<const __half*>(R);
    p.ldr = ldr;
    p.swiglu = swiglu ? 1 : 0;
    p.vec = ldc % 8 == 0 && npub_aligned(C, 16) && npub_aligned(w_scale, 16) && (!R || (ldr % 8 == 0 && npub_aligned(R, 16)));
    p.err = npub_internal_device_error_word();
    const Choice c = pick(M, N, p.k_tiles, p.vec);
    const bool tile = c.bt < 32;
    const uint32_t rows_a = tile ? 128 * c.bt : c.bt, rows_w = tile ? 256 : 128;
    int rc = make_tmap_3d(&p.tmA, true, A, (uint64_t)K, (uint64_t)M, 1, (uint64_t)lda, (uint64_t)lda * M, rows_a, 1, true, BK);
    if (rc) return rc;
    rc = make_tmap_3d(&p.tmW, true, W, (uint64_t)K, (uint64_t)N, 1, (uint64_t)ldw, (uint64_t)ldw * N, rows_w, 1, true, BK);
    if (rc) return rc;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    switch (c.bt) {
        case 32: return launch_few<32>(p, c.splits, st);
        case 64: return launch_few<64>(p, c.splits, st);
        case 128: return launch_few<128>(p, c.splits, st);
        case kTile1: return launch_tile<1>(p, st);
        default: return launch_tile<2>(p, st);
    }
}
