// Attention of a few new rows per sequence over a paged KV cache held in 8
// bits, K = s_k q_k and V = s_v q_v with one scale for each page and kv head
// (the 8-bit form of paged_decode.cu; the rows' tiles, the key ranges and their
// combination are the same).
//
// What it costs is one read of the 8-bit K and V (HBM bound: 2 * head_dim bytes
// per key and head); beside it the conversion to fp16 has to keep up, about two
// instructions per 4 elements of K and three per 4 of V.  So:
//   * the integers go into the fp16 tensor-core products as they are (exact in
//     fp16); a step of 16 keys lies in one page, so its scales are two numbers.
//   * s_k multiplies the scores; s_v goes into the exponent: with z = s_k (q . k)
//     + log2(s_v) / c the weights 2^((z - m) c) carry s_v, O takes them times
//     the integers, and the row's sum takes them times 1 / s_v.  The running
//     reference m is of z, so a weight's rounding to fp16 (2^-11) is relative to
//     what it adds to the result.  (s_v below 2^-40 counts as 2^-40: what it
//     adds to a result is below 2^-33.)
//   * an element's place in the product's inner dimension is free, as long as
//     both operands agree: a lane takes 16 neighbouring columns of a key with one
//     16-byte load, which are 4 steps of the K product, or 16 of the columns of
//     the V product; the swizzle of the tile keeps the loads free of bank
//     conflicts.
//
// Rows: 16 of a kv head (token x grouped head) per CTA, more in further CTAs
// (blockIdx.z), which find K and V in L2.
#include "common.cuh"
#include "gemm_tc.h"
#include "paged_decode.h"

#ifndef NPUB_Q8_STEP
#define NPUB_Q8_STEP 32
#endif
#ifndef NPUB_Q8_RING
#define NPUB_Q8_RING 96
#endif
#ifndef NPUB_Q8_CTAS8
#define NPUB_Q8_CTAS8 3
#endif
#ifndef NPUB_Q8_RING8
#define NPUB_Q8_RING8 64
#endif
#ifndef NPUB_Q8_CTAS
#define NPUB_Q8_CTAS 2
#endif
namespace npub {
namespace pdq8 {

constexpr int kWarps = 4;               // consumers
constexpr int kThreads = kWarps * 32 + 32;
constexpr int kStep = NPUB_Q8_STEP;     // keys of a stage that a warp takes
constexpr int kKeys = kWarps * kStep;   // keys per stage
constexpr int kGroups = kKeys / 16;     // runs of keys with the same scales

template <int HD, int kMaxRows>
struct Smem {
    static constexpr int kTile = kKeys * HD;  // K or V of a stage
    static constexpr int kStages = (kMaxRows == 8 ? NPUB_Q8_RING8 : NPUB_Q8_RING) * 1024 / (2 * kTile);
    static constexpr int kOffScale = kStages * 2 * kTile;  // [stage][group]: s_k, log2(s_v) / c, 1 / s_v
    static constexpr int kOffBar = kOffScale + kStages * kGroups * 16;
    static constexpr int kTotal = kOffBar + 256;
    // The merge reuses the ring: the warps' partials, then (clusters) the CTA's own.  A lane writes runs of HD / 8
    // columns; 4 words behind each run and 4 behind a row spread the lanes over the banks.
    static constexpr int kRun = HD / 8;
    static constexpr int kRow = 8 * (kRun + 4) + 4;
    static constexpr int kOffMl = kWarps * kMaxRows * kRow * 4;
    static constexpr int kOffOwn = kOffMl + kWarps * kMaxRows * 8;
    static constexpr int kOffOwnMl = kOffOwn + kMaxRows * HD * 4;
    static_assert(kOffOwnMl + kMaxRows * 8 <= kOffScale, "layout");
};

struct Params {
    CUtensorMap tmK, tmV;
    const float *ks, *vs;
    const __half* q;
    int64_t ldq;
    const int32_t *cu, *lens, *table;
    int64_t ldt;
    int max_keys, page_shift, box_rows, n_pages;
    int total_q, heads, kv_heads, group, head_dim, causal;
    int splits, cluster;
    float c;
    __half* out;
    int64_t ldo;
    float* part_o;
    float2* part_ml;
    int* err;
};

__device__ __forceinline__ void set_err(int* err, int code) {
    if (err) atomicCAS(err, 0, code);
}
__device__ __forceinline__ void consumer_bar() { asm volatile("barrier.sync 1, %0;" ::"n"(kWarps * 32) : "memory"); }
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// The transpose of an 8 x 8 matrix of fp16 held by a warp, row lane / 4, columns 2 (lane & 3) and the next.
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ float2 ld_cluster_f2(uint32_t a) {
    float2 v;
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ float4 ld_cluster_f4(uint32_t a) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"(a)
                 : "memory");
    return v;
}
__device__ __forceinline__ uint32_t h2(float a, float b) {
    __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&h);
}
__device__ __forceinline__ void no_keys(const Params& p, bool part, int split, int row, int head) {
    if (part) {
        p.part_ml[((int64_t)split * p.total_q + row) * p.heads + head] = make_float2(-INFINITY, 0.0f);
    } else {
        for (int d = 0; d < p.head_dim; d += 4)
            *reinterpret_cast<uint2*>(p.out + (int64_t)row * p.ldo + (int64_t)head * p.head_dim + d) = make_uint2(0, 0);
    }
}

// grid (kv_heads * splits, batch, tiles of kMaxRows rows)
//
// kMaxRows 16: S = Q K^T and O = P V with the rows on the product's 16-side.
// kMaxRows 8: transposed, S^T = K Q^T and O^T = V^T P^T with the rows on its
// 8-side: half of the products, exponentials and sums.  A lane's integers of K
// and V are the same in both.
template <int HD, int kMaxRows>
__global__ void __launch_bounds__(kThreads, kMaxRows == 8 ? NPUB_Q8_CTAS8 : NPUB_Q8_CTAS)
    paged_decode_q8_kernel(const __grid_constant__ Params p) {
    using L = Smem<HD, kMaxRows>;
    constexpr bool kT = kMaxRows == 8;
    pdl_trigger();
    extern __shared__ __align__(1024) uint8_t smem[];
    if (smem_u32(smem) & 1023u) {
        if (threadIdx.x == 0) set_err(p.err, 0x720);
        pdl_wait();
        return;
    }
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::kOffBar);
    uint64_t* empty = full + L::kStages;
    volatile int* abort_flag = reinterpret_cast<volatile int*>(empty + L::kStages);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int kvh = (int)blockIdx.x / p.splits, split = (int)blockIdx.x - kvh * p.splits, b = blockIdx.y;
    const bool part = p.part_o != nullptr;
    pdl_wait();
    // this CTA's rows, the sequence's keys, and the range of them
    int row0 = b, nseq = 1, nrow = 1, first = 0;
    if (p.cu) {
        const int per_tile = kMaxRows / p.group;
        row0 = max(0, min(p.total_q, p.cu[b]));
        nseq = max(0, min(p.total_q, p.cu[b + 1]) - row0);
        first = (int)blockIdx.z * per_tile;
        nrow = max(0, min(nseq - first, per_tile));
        const int covered = (int)gridDim.z * per_tile;
        if (blockIdx.z == gridDim.z - 1 && covered < nseq && (part || split == 0)) {
            // a caller's max_new below the sequence's rows: the rest are zeros
            const int rest = (nseq - covered) * p.group;
            for (int i = threadIdx.x; i < rest; i += kThreads) {
                const int t = i / p.group;
                no_keys(p, part, split, row0 + covered + t, kvh * p.group + i - t * p.group);
            }
        }
        row0 += first;
    }
    const int R = nrow * p.group;
    const int len = max(0, min(p.lens[b], p.max_keys));
    const int per = max(128 / kKeys, ((len + kKeys - 1) / kKeys + p.splits - 1) / p.splits) * kKeys;
    const int k0 = R == 0 ? 0 : min(len, split * per);
    const int k1 = R == 0 ? 0 : min(len, split * per + per);
    const int nst = (k1 - k0 + kKeys - 1) / kKeys;
    if (nst == 0) {
        for (int r = threadIdx.x; r < R; r += kThreads) {
            const int t = r / p.group;
            if (part || split == 0) no_keys(p, part, split, row0 + t, kvh * p.group + r - t * p.group);
        }
        return;
    }
    if (threadIdx.x == 0) {
        for (int i = 0; i < L::kStages; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], kWarps);
        }
        *abort_flag = 0;
        fence_barrier_init();
    }
    if (warp == kWarps && lane == 0) {
        prefetch_tmap(&p.tmK);
        prefetch_tmap(&p.tmV);
    }
    cta_sync_divergent();

    if (warp == kWarps) {
        // -------------------------------------------------------------------- producer
        // One lane per page piece of K or V.  Its page id is read two stages ahead, the page's scale one.
        const int nbox = kKeys / p.box_rows, groups = p.box_rows / 16;
        const int kv = lane & 1, box = lane >> 1;
        const float* scales = kv ? p.vs : p.ks;
        const float inv_c = 1.0f / p.c;
        auto page_of = [&](int j) {
            const int key = k0 + j * kKeys + box * p.box_rows;
            int page = p.n_pages;  // past the keys: outside the pool, filled with zeros
            if (box < nbox && j < nst && key < k1) {
                const int id = __ldg(p.table + (int64_t)b * p.ldt + (key >> p.page_shift));
                if (id >= 0 && id < p.n_pages) page = id;
            }
            return page;
        };
        auto scale_of = [&](int page) { return page < p.n_pages ? __ldg(scales + (int64_t)page * p.kv_heads + kvh) : 0.0f; };
        int page = page_of(0), next = page_of(1);
        float scale = scale_of(page);
        bool ok = true;
        int j = 0;
        for (; j < nst; ++j) {
            const int s = j % L::kStages;
            const int key = k0 + j * kKeys + box * p.box_rows;
            const int after = page_of(j + 2);
            const float next_scale = scale_of(next);
            ok = mbar_wait_warp(&empty[s], ((uint32_t)(j / L::kStages) & 1u) ^ 1u, abort_flag);
            if (!ok) break;
            if (box < nbox) {
                float* sc = reinterpret_cast<float*>(smem + L::kOffScale) + (s * kGroups + box * groups) * 4;
                float v = isfinite(scale) ? scale : NAN;
                if (kv) {
                    v = page < p.n_pages ? (v < 9.094947e-13f ? 9.094947e-13f : v) : 1.0f;  // 2^-40; NaN stays
                    const float lb = log2f(v) * inv_c, inv = 1.0f / v;
                    for (int g = 0; g < groups; ++g) {
                        sc[g * 4 + 1] = lb;
                        sc[g * 4 + 2] = inv;
                    }
                } else {
                    for (int g = 0; g < groups; ++g) sc[g * 4] = v;
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive_expect_tx(&full[s], 2u * L::kTile);
            __syncwarp();
            if (box < nbox)
                tma_load_4d(smem + (s * 2 + kv) * L::kTile + box * p.box_rows * HD, kv ? &p.tmV : &p.tmK, &full[s], 0,
                            key & ((1 << p.page_shift) - 1), kvh, page);
            page = next;
            next = after;
            scale = next_scale;
        }
        if (!ok && lane == 0) {  // copies in flight land before the CTA leaves
            *abort_flag = 1;
            set_err(p.err, 0x721);
            int never = 0;
            for (int i = max(0, j - L::kStages); i < j; ++i)
                mbar_wait_bounded(&full[i % L::kStages], (uint32_t)(i / L::kStages) & 1u, &never, 200000000ull);
        }
        return;
    }

    // ------------------------------------------------------------------------ consumers
    const int g8 = lane >> 2, t4 = lane & 3;  // the lane's place among eight and among four
    // rows whose scores and output this lane holds
    const int ra = kT ? 2 * t4 : g8, rb = kT ? ra + 1 : ra + 8;
    constexpr int kQ = kT ? 1 : 2;  // rows of Q that a lane holds: g8 (and g8 + 8)
    uint32_t qf[HD / 16][2 * kQ];
#pragma unroll
    for (int i = 0; i < kQ; ++i) {
        const int row = g8 + 8 * i, t = row / p.group;
        const __half* src = p.q + (int64_t)(row0 + t) * p.ldq + (int64_t)(kvh * p.group + row - t * p.group) * p.head_dim;
#pragma unroll
        for (int kk = 0; kk < HD / 16; ++kk) {  // step kk of the lane's HD / 4 columns: 4 of them
            const int d = t4 * (HD / 4) + kk * 4;
            const uint2 w = d < p.head_dim && row < R ? *reinterpret_cast<const uint2*>(src + d) : make_uint2(0, 0);
            qf[kk][i] = w.x;
            qf[kk][kQ + i] = w.y;
        }
    }
    int lim[2] = {len, len};  // keys of rows ra and rb end here
    if (p.causal) {
        lim[0] = len - nseq + first + ra / p.group + 1;
        lim[1] = len - nseq + first + rb / p.group + 1;
    }
    lim[0] = min(lim[0], k1);
    lim[1] = min(lim[1], k1);
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
    // output: kT: tile n has columns g8 HD / 8 + 2 n (e < 2) and the next (e >= 2), rows ra (even e) and rb; else tile n has
    // column (2 t4 + (e & 1)) HD / 8 + n, rows ra (e < 2) and rb
    constexpr int kO = kT ? HD / 16 : HD / 8;
    float o[kO][4];
#pragma unroll
    for (int n = 0; n < kO; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[n][e] = 0.0f;
    const float c = p.c;
    // scores of 16 keys, [2 u + i][e]: kT: x[2 u] are keys g8 (e < 2) and g8 + 8 of rows ra (even e) and rb; else x[2 u + i]
    // is key 8 i + 2 t4 + (e & 1) of row ra (e < 2) or rb
    constexpr int kX = kT ? kStep / 16 : kStep / 8;
    auto row_of = [](int e) { return kT ? e & 1 : e >> 1; };
    auto key_of = [&](int n, int e) { return kT ? n * 16 + g8 + (e >> 1) * 8 : n * 8 + t4 * 2 + (e & 1); };
    bool ok = true;
    for (int j = 0; j < nst; ++j) {
        const int s = j % L::kStages;
        ok = mbar_wait_warp(&full[s], (uint32_t)(j / L::kStages) & 1u, abort_flag);
        if (!ok) break;
        const int kb = k0 + j * kKeys + warp * kStep;  // first key of this warp
        if (kb < k1) {
            const uint8_t* kt = smem + s * 2 * L::kTile + warp * kStep * HD;
            const uint8_t* vt = kt + L::kTile;
            const float4* sc = reinterpret_cast<const float4*>(smem + L::kOffScale + (s * kGroups + warp * (kStep / 16)) * 16);
            float x[kX][4];
#pragma unroll
            for (int u = 0; u < kStep / 16; ++u) {
#pragma unroll
                for (int n = u * kX * 16 / kStep; n < (u + 1) * kX * 16 / kStep; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[n][e] = 0.0f;
#pragma unroll
                for (int h = 0; h < HD / 64; ++h) {
                    // keys g8 and g8 + 8 at columns t4 * HD / 4 + 16 h and the 15 behind them
                    uint32_t f[2][8];
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const int key = u * 16 + i * 8 + g8;
                        const int at = HD == 128 ? key * 128 + (((2 * t4 + h) ^ (key & 7)) << 4)
                                                 : key * 64 + ((t4 ^ ((key >> 1) & 3)) << 4);
                        i8x16_to_f16x2(*reinterpret_cast<const uint4*>(kt + at), f[i]);
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint32_t(&q)[2 * kQ] = qf[h * 4 + i];
                        if constexpr (kT) {
                            const uint32_t a[4] = {f[0][2 * i], f[1][2 * i], f[0][2 * i + 1], f[1][2 * i + 1]};
                            mma16816(x[u], a, q[0], q[1]);
                        } else {
                            mma16816(x[2 * u], q, f[0][2 * i], f[0][2 * i + 1]);
                            mma16816(x[2 * u + 1], q, f[1][2 * i], f[1][2 * i + 1]);
                        }
                    }
                }
            }
            float inv[kStep / 16];
#pragma unroll
            for (int u = 0; u < kStep / 16; ++u) {
                const float4 v = sc[u];
                inv[u] = v.z;
#pragma unroll
                for (int n = u * kX * 16 / kStep; n < (u + 1) * kX * 16 / kStep; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[n][e] = fmaf(x[n][e], v.x, v.y);
            }
            if (kb + kStep > min(lim[0], lim[1])) {
#pragma unroll
                for (int n = 0; n < kX; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[n][e] = kb + key_of(n, e) < lim[row_of(e)] ? x[n][e] : -INFINITY;
            }
            float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
            for (int n = 0; n < kX; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) mx[row_of(e)] = fmaxf(mx[row_of(e)], x[n][e]);
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], kT ? 4 : 1));
                mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], kT ? 8 : 2));
                if (kT) mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 16));
            }
            const bool need[2] = {(mx[0] - m[0]) * c > 8.0f, (mx[1] - m[1]) * c > 8.0f};
            if (__any_sync(0xffffffffu, need[0] || need[1])) {
                float corr[2];
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    corr[r] = need[r] ? ex2_approx((m[r] - mx[r]) * c) : 1.0f;
                    if (need[r]) m[r] = mx[r];
                    l[r] *= corr[r];
                }
#pragma unroll
                for (int n = 0; n < kO; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[n][e] *= corr[row_of(e)];
            }
            const float ref[2] = {m[0] == -INFINITY ? 0.0f : m[0], m[1] == -INFINITY ? 0.0f : m[1]};
#pragma unroll
            for (int n = 0; n < kX; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float pv = ex2_approx((x[n][e] - ref[row_of(e)]) * c);
                    x[n][e] = pv;
                    l[row_of(e)] = fmaf(pv, inv[n * (kStep / 16) / kX], l[row_of(e)]);
                }
#pragma unroll
            for (int u = 0; u < kStep / 16; ++u) {
                uint32_t pf[4];
                if constexpr (kT) {
                    pf[0] = transpose8(h2(x[u][0], x[u][1]));  // keys 2 t4, 2 t4 + 1 of row g8
                    pf[1] = transpose8(h2(x[u][2], x[u][3]));  // 2 t4 + 8, 2 t4 + 9
                } else {
                    pf[0] = h2(x[2 * u][0], x[2 * u][1]);
                    pf[1] = h2(x[2 * u][2], x[2 * u][3]);
                    pf[2] = h2(x[2 * u + 1][0], x[2 * u + 1][1]);
                    pf[3] = h2(x[2 * u + 1][2], x[2 * u + 1][3]);
                }
                // V rows 2 t4, 2 t4 + 1, 2 t4 + 8, 2 t4 + 9 of the 16 at the HD / 8 columns from g8 * HD / 8 on
                uint32_t v[4][HD / 32];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int key = u * 16 + 2 * t4 + (i & 1) + (i >> 1) * 8;
                    if constexpr (HD == 128) {
                        const uint4 r = *reinterpret_cast<const uint4*>(vt + key * 128 + ((g8 ^ (key & 7)) << 4));
                        v[i][0] = r.x ^ 0x80808080u;
                        v[i][1] = r.y ^ 0x80808080u;
                        v[i][2] = r.z ^ 0x80808080u;
                        v[i][3] = r.w ^ 0x80808080u;
                    } else {
                        const uint2 r = *reinterpret_cast<const uint2*>(
                            vt + key * 64 + (((g8 >> 1) ^ ((key >> 1) & 3)) << 4) + (g8 & 1) * 8);
                        v[i][0] = r.x ^ 0x80808080u;
                        v[i][1] = r.y ^ 0x80808080u;
                    }
                }
#pragma unroll
                for (int w = 0; w < HD / 32; ++w) {  // 4 columns: the two keys of a pair side by side
                    uint32_t a[4], b[4];
                    const uint32_t a0 = __byte_perm(v[0][w], v[1][w], 0x5140), a1 = __byte_perm(v[0][w], v[1][w], 0x7362);
                    const uint32_t b0 = __byte_perm(v[2][w], v[3][w], 0x5140), b1 = __byte_perm(v[2][w], v[3][w], 0x7362);
                    a[0] = f16x2_sub1152(i8_perm_lo(a0));
                    a[1] = f16x2_sub1152(i8_perm_hi(a0));
                    a[2] = f16x2_sub1152(i8_perm_lo(a1));
                    a[3] = f16x2_sub1152(i8_perm_hi(a1));
                    b[0] = f16x2_sub1152(i8_perm_lo(b0));
                    b[1] = f16x2_sub1152(i8_perm_hi(b0));
                    b[2] = f16x2_sub1152(i8_perm_lo(b1));
                    b[3] = f16x2_sub1152(i8_perm_hi(b1));
                    if constexpr (kT) {
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            const uint32_t f[4] = {a[2 * i], a[2 * i + 1], b[2 * i], b[2 * i + 1]};
                            mma16816(o[2 * w + i], f, pf[0], pf[1]);
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; ++i) mma16816(o[4 * w + i], pf, a[i], b[i]);
                    }
                }
            }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[s]);
    }
    if (!ok) {
        *abort_flag = 1;
        if (lane == 0) set_err(p.err, 0x722);
    }
    // ---- merge of the four warps
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        l[r] += __shfl_xor_sync(0xffffffffu, l[r], kT ? 4 : 1);
        l[r] += __shfl_xor_sync(0xffffffffu, l[r], kT ? 8 : 2);
        if (kT) l[r] += __shfl_xor_sync(0xffffffffu, l[r], 16);
    }
    consumer_bar();  // nobody reads the ring any more
    float* so = reinterpret_cast<float*>(smem);                 // [warp][row][8 runs]
    float2* sml = reinterpret_cast<float2*>(smem + L::kOffMl);  // [warp][row]
    if ((kT ? g8 : t4) == 0) {
        sml[warp * kMaxRows + ra] = make_float2(m[0], l[0]);
        sml[warp * kMaxRows + rb] = make_float2(m[1], l[1]);
    }
    if constexpr (kT) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            float* dst = so + (warp * kMaxRows + ra + r) * L::kRow + g8 * (L::kRun + 4);
#pragma unroll
            for (int n = 0; n < kO; n += 2)
                *reinterpret_cast<float4*>(dst + 2 * n) = make_float4(o[n][r], o[n][2 + r], o[n + 1][r], o[n + 1][2 + r]);
        }
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            float* dst = so + (warp * kMaxRows + (e < 2 ? ra : rb)) * L::kRow + (2 * t4 + (e & 1)) * (L::kRun + 4);
#pragma unroll
            for (int n = 0; n < kO; n += 4)
                *reinterpret_cast<float4*>(dst + n) = make_float4(o[n][e], o[n + 1][e], o[n + 2][e], o[n + 3][e]);
        }
    }
    consumer_bar();
    const int cols = p.head_dim >> 2;
    for (int i = threadIdx.x; i < R * cols; i += kWarps * 32) {
        const int r = i / cols, d = (i - r * cols) * 4;
        float mm = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) mm = fmaxf(mm, sml[w * kMaxRows + r].x);
        float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f}, sum = 0.0f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float2 ml = sml[w * kMaxRows + r];
            if (ml.y == 0.0f) continue;  // no key of this warp
            const float f = ex2_approx((ml.x - mm) * c);
            const float4 v = *reinterpret_cast<const float4*>(so + (w * kMaxRows + r) * L::kRow + d + d / L::kRun * 4);
            sum += f * ml.y;
            acc[0] += f * v.x;
            acc[1] += f * v.y;
            acc[2] += f * v.z;
            acc[3] += f * v.w;
        }
        const int t = r / p.group, head = kvh * p.group + r - t * p.group;
        // keys, but all scores -inf: 0 / 0 in the formula, (-inf, 1) for a combination
        const bool flat = mm == -INFINITY && sum == 0.0f && (p.causal ? min(k1, len - nseq + first + t + 1) : k1) > k0;
        if (flat) sum = 1.0f;
        if (p.cluster) {
            if (d == 0) *reinterpret_cast<float2*>(smem + L::kOffOwnMl + r * 8) = make_float2(mm, sum);
            *reinterpret_cast<float4*>(smem + L::kOffOwn + (r * HD + d) * 4) =
                make_float4(acc[0], acc[1], acc[2], acc[3]);
        } else if (part) {
            const int64_t at = ((int64_t)split * p.total_q + row0 + t) * p.heads + head;
            if (d == 0) p.part_ml[at] = make_float2(mm, sum);
            if (sum != 0.0f && !flat)
                *reinterpret_cast<float4*>(p.part_o + at * p.head_dim + d) = make_float4(acc[0], acc[1], acc[2], acc[3]);
        } else {
            const float inv = flat ? NAN : sum != 0.0f ? 1.0f / sum : 0.0f;
            uint2 w;
            w.x = sum != 0.0f ? h2(acc[0] * inv, acc[1] * inv) : 0u;
            w.y = sum != 0.0f ? h2(acc[2] * inv, acc[3] * inv) : 0u;
            *reinterpret_cast<uint2*>(p.out + (int64_t)(row0 + t) * p.ldo + (int64_t)head * p.head_dim + d) = w;
        }
    }
    if (p.cluster) {
        // the CTAs of the cluster with keys (the producers and the CTAs without have left, and do not count) each
        // combine a part of the rows from all of their shared memories
        const int n = (len + per - 1) / per;
        cluster_arrive();
        cluster_wait();
        for (int i = split * (kWarps * 32) + threadIdx.x; i < R * cols; i += n * (kWarps * 32)) {
            const int r = i / cols, d = (i - r * cols) * 4;
            const uint32_t ml_at = smem_u32(smem + L::kOffOwnMl + r * 8);
            const uint32_t o_at = smem_u32(smem + L::kOffOwn + (r * HD + d) * 4);
            float mm = -INFINITY;
            for (int t = 0; t < n; ++t) mm = fmaxf(mm, ld_cluster_f2(mapa_shared(ml_at, t)).x);
            float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f}, sum = 0.0f;
            for (int t = 0; t < n; ++t) {
                const float2 ml = ld_cluster_f2(mapa_shared(ml_at, t));
                if (ml.y == 0.0f) continue;
                const float f = ex2_approx((ml.x - mm) * c);
                const float4 v = ld_cluster_f4(mapa_shared(o_at, t));
                sum += f * ml.y;
                acc[0] += f * v.x;
                acc[1] += f * v.y;
                acc[2] += f * v.z;
                acc[3] += f * v.w;
            }
            const float inv = 1.0f / sum;
            uint2 w;
            w.x = sum != 0.0f ? h2(acc[0] * inv, acc[1] * inv) : 0u;
            w.y = sum != 0.0f ? h2(acc[2] * inv, acc[3] * inv) : 0u;
            const int t = r / p.group, head = kvh * p.group + r - t * p.group;
            *reinterpret_cast<uint2*>(p.out + (int64_t)(row0 + t) * p.ldo + (int64_t)head * p.head_dim + d) = w;
        }
        cluster_arrive();  // nobody leaves while its shared memory is read
        cluster_wait();
    }
}

template <int HD, int kMaxRows>
int launch(const Params& p, int batch, int tiles, cudaStream_t st) {
    auto kern = paged_decode_q8_kernel<HD, kMaxRows>;
    constexpr int kTotal = Smem<HD, kMaxRows>::kTotal;
    NPUB_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kTotal));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(p.kv_heads * p.splits, batch, tiles);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = kTotal;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = npub_internal_pdl_enabled() ? 1 : 0;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = p.splits;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = p.cluster ? 2 : 1;
    NPUB_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, p));
    return npub_internal_launch_status();
}

// 16 columns of a key per thread and step: s q in fp16 (2^-11; the products with fp16 take no more), one block per
// (key block of 128, kv head, sequence).
__global__ void __launch_bounds__(256) expand_q8_kernel(const int8_t* __restrict__ kp, const int8_t* __restrict__ vp,
                                                        const float* __restrict__ ks, const float* __restrict__ vs,
                                                        const int32_t* __restrict__ table, int64_t ldt, int n_pages,
                                                        int page_shift, int max_keys, const int32_t* __restrict__ lens,
                                                        int kv_heads, int head_dim, int width, __half* __restrict__ k_out,
                                                        __half* __restrict__ v_out, int32_t* __restrict__ table_out,
                                                        int32_t* __restrict__ lens_out) {
    pdl_trigger();
    pdl_wait();
    const int w = blockIdx.x, kvh = blockIdx.y, b = blockIdx.z;
    int len = max(0, min(lens[b], max_keys));
    if (len > width * 128) len = 0;  // more than the caller's ctx_len: no keys, rows of zeros
    if (kvh == 0 && threadIdx.x == 0) {
        table_out[(int64_t)b * width + w] = b * width + w;
        if (w == 0) lens_out[b] = len;
    }
    const int n = min(128, len - w * 128);
    const int units = head_dim / 16;
    const int64_t to = ((int64_t)(b * (int64_t)width + w) * kv_heads + kvh) * 128 * head_dim;
    for (int i = threadIdx.x; i < n * units * 2; i += 256) {
        const bool v = i >= n * units;
        const int u = v ? i - n * units : i, row = u / units, col = (u - row * units) * 16;
        const int key = w * 128 + row;
        const int id = __ldg(table + (int64_t)b * ldt + (key >> page_shift));
        uint4 o[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
        if (id >= 0 && id < n_pages) {
            const int64_t at = (int64_t)id * kv_heads + kvh;
            const float s = __ldg((v ? vs : ks) + at);
            const uint4 r = *reinterpret_cast<const uint4*>(
                (v ? vp : kp) + ((at << page_shift) + (key & ((1 << page_shift) - 1))) * head_dim + col);
            const uint32_t x[4] = {r.x, r.y, r.z, r.w};
            uint32_t* y = reinterpret_cast<uint32_t*>(o);
            const float fs = isfinite(s) ? s : NAN;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                y[2 * e] = h2((float)(int8_t)x[e] * fs, (float)(int8_t)(x[e] >> 8) * fs);
                y[2 * e + 1] = h2((float)(int8_t)(x[e] >> 16) * fs, (float)(int8_t)(x[e] >> 24) * fs);
            }
        }
        uint4* dst = reinterpret_cast<uint4*>((v ? v_out : k_out) + to + (int64_t)row * head_dim + col);
        dst[0] = o[0];
        dst[1] = o[1];
    }
}

}  // namespace pdq8

int paged_decode_q8(const PackedArgs& a, const float* k_scales, const float* v_scales, int rows, int tiles,
                    cudaStream_t st) {
    using namespace pdq8;
    Params p;
    memset(&p, 0, sizeof(p));
    p.box_rows = a.kv.page_size < kKeys ? a.kv.page_size : kKeys;
    int rc = make_tmap_pages_q8(&p.tmK, a.kv.k, a.kv.n_pages, a.kv_heads, a.kv.page_size, a.head_dim, p.box_rows);
    if (rc) return rc;
    rc = make_tmap_pages_q8(&p.tmV, a.kv.v, a.kv.n_pages, a.kv_heads, a.kv.page_size, a.head_dim, p.box_rows);
    if (rc) return rc;
    while ((1 << p.page_shift) < a.kv.page_size) ++p.page_shift;
    const int64_t mk = (int64_t)a.kv.max_pages << p.page_shift;
    p.max_keys = mk > 0x7ff00000 ? 0x7ff00000 : (int)mk;
    p.n_pages = a.kv.n_pages;
    p.ks = k_scales;
    p.vs = v_scales;
    p.table = a.kv.table;
    p.ldt = a.kv.ldt;
    p.lens = a.lens;
    p.cu = a.cu;
    p.q = reinterpret_cast<const __half*>(a.q);
    p.ldq = a.ldq;
    p.total_q = a.total_q;
    p.heads = a.heads;
    p.kv_heads = a.kv_heads;
    p.group = a.heads / a.kv_heads;
    p.head_dim = a.head_dim;
    p.causal = a.causal ? 1 : 0;
    p.splits = a.splits;
    p.cluster = !a.part_o && a.splits > 1;
    p.c = a.scale * 1.4426950408889634f;
    p.out = reinterpret_cast<__half*>(a.out);
    p.ldo = a.ldo;
    p.part_o = a.part_o;
    p.part_ml = a.part_ml;
    p.err = npub_internal_device_error_word();
    const bool small = a.head_dim <= 64;
    if (rows <= 8) return small ? launch<64, 8>(p, a.batch, tiles, st) : launch<128, 8>(p, a.batch, tiles, st);
    return small ? launch<64, 16>(p, a.batch, tiles, st) : launch<128, 16>(p, a.batch, tiles, st);
}

int expand_q8(const PackedArgs& a, const float* k_scales, const float* v_scales, int width, void* k_out, void* v_out,
              int32_t* table_out, int32_t* lens_out, cudaStream_t st) {
    int shift = 0;
    while ((1 << shift) < a.kv.page_size) ++shift;
    const int64_t mk = (int64_t)a.kv.max_pages << shift;
    return launch_pdl(pdq8::expand_q8_kernel, dim3(width, a.kv_heads, a.batch), dim3(256), 0, st,
                      reinterpret_cast<const int8_t*>(a.kv.k), reinterpret_cast<const int8_t*>(a.kv.v), k_scales, v_scales,
                      a.kv.table, a.kv.ldt, a.kv.n_pages, shift, (int)(mk > 0x7ff00000 ? 0x7ff00000 : mk), a.lens,
                      a.kv_heads, a.head_dim, width, reinterpret_cast<__half*>(k_out), reinterpret_cast<__half*>(v_out),
                      table_out, lens_out);
}

}  // namespace npub
