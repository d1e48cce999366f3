// Attention of a few new rows per sequence (up to 16 rows per kv head: the
// decode step of a grouped-query model, or a handful of drafted tokens) over a
// paged KV cache, and the combination of partial results.
//
// One CTA takes one (sequence, kv head, range of keys): every K and V byte of
// the range is read once, and what it costs is that read (HBM bound: per key
// 2 * head_dim * 2 bytes against 4 * 16 * head_dim MACs of which rows/16 are
// useful).  So the rows of the group share an m16n8k16 tile (mma.sync: at 16
// rows a 128-row tcgen05 tile would be one eighth full and its softmax would
// run in 16 lanes of one warp), and the design is about keeping loads in
// flight: a producer warp streams stages of 64 keys (K and V, 32 KB at
// head_dim 128) through a ring by TMA, its lanes issuing one page piece each;
// four consumer warps take 16 keys of every stage, each with its own running
// maximum and sum, and meet only at the end.  Up to eight ranges of one item
// are a cluster and combine through one another's shared memory; more of them,
// or a shared prefix, leave partials for a second kernel.
//
// As in fmha_packed.cu the running maximum moves only when it has grown by
// more than 2^8, and the weights are rounded to fp16 (2^-11 of each) for the
// product with V, all else is fp32; keys past the sequence's end are masked by a select and their
// V rows zeroed, so stale slots of the last page never reach a result.
#include "common.cuh"
#include "fmha_packed.h"
#include "gemm_tc.h"
#include "paged_decode.h"

namespace npub {
namespace pdec {

constexpr int kWarps = 4;               // consumers
constexpr int kThreads = kWarps * 32 + 32;
constexpr int kKeys = kWarps * 16;      // keys per stage
constexpr int kMaxRows = 16;

template <int HD>
struct Smem {
    static constexpr int kChunks = HD / 64;
    static constexpr int kChunk = kKeys * 128;
    static constexpr int kTile = kChunks * kChunk;  // K or V of a stage
    static constexpr int kStages = HD == 128 ? 3 : 6;
    static constexpr int kOffBar = kStages * 2 * kTile;
    static constexpr int kTotal = kOffBar + 256;
    // the merge reuses the ring: the warps' partials, then (clusters) the CTA's own
    static constexpr int kOffMl = kWarps * kMaxRows * HD * 4;
    static constexpr int kOffOwn = kOffMl + kWarps * kMaxRows * 8;
    static constexpr int kOffOwnMl = kOffOwn + kMaxRows * HD * 4;
    static_assert(kOffOwnMl + kMaxRows * 8 <= kOffBar, "layout");
};

struct Params {
    CUtensorMap tmK, tmV;
    const __half* q;
    int64_t ldq;
    const int32_t *cu, *lens, *table;
    int64_t ldt;
    int max_keys, page_shift, box_rows, n_pages, common;
    int total_q, heads, kv_heads, group, head_dim, causal;
    int first, splits;         // every sequence's keys from `first` on in `splits` equal ranges
    int split0;                // index of split 0 among the partials
    int cluster;               // the splits of an item are a cluster, which combines them itself
    int beside;                // launched behind a shared-prefix phase, which has waited for all earlier work
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

__device__ __forceinline__ void ldsm_x4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void ldsm_x4_t(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
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

// What a row and head without keys in this range leaves: an empty partial, or a row of zeros.
__device__ __forceinline__ void no_keys(const Params& p, bool part, int split, int row, int head) {
    if (part) {
        p.part_ml[((int64_t)(p.split0 + split) * p.total_q + row) * p.heads + head] = make_float2(-INFINITY, 0.0f);
    } else {
        for (int d = 0; d < p.head_dim; d += 4)
            *reinterpret_cast<uint2*>(p.out + (int64_t)row * p.ldo + (int64_t)head * p.head_dim + d) = make_uint2(0, 0);
    }
}

// grid (kv_heads * splits, batch)
template <int HD>
__global__ void __launch_bounds__(kThreads, 2) paged_decode_kernel(const __grid_constant__ Params p) {
    using L = Smem<HD>;
    pdl_trigger();
    extern __shared__ __align__(1024) uint8_t smem[];
    if (smem_u32(smem) & 1023u) {
        if (threadIdx.x == 0) set_err(p.err, 0x600);
        pdl_wait();
        return;
    }
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::kOffBar);
    uint64_t* empty = full + L::kStages;
    volatile int* abort_flag = reinterpret_cast<volatile int*>(empty + L::kStages);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int kvh = (int)blockIdx.x / p.splits, split = (int)blockIdx.x - kvh * p.splits, b = blockIdx.y;
    const bool part = p.part_o != nullptr;
    // Beside a prefix phase the last CTA waits for that phase at its end: this grid's completion then means the prefix's
    // to the combination behind it.  (All CTAs waiting would keep their slots from the CTAs behind them.)
    const bool holds = p.beside && blockIdx.x == gridDim.x - 1 && blockIdx.y == gridDim.y - 1;
    if (!p.beside) pdl_wait();
    // rows of this sequence, its keys, and this CTA's range of them
    int row0 = b, nseq = 1, nrow = 1;
    if (p.cu) {
        row0 = max(0, min(p.total_q, p.cu[b]));
        nseq = max(0, min(p.total_q, p.cu[b + 1]) - row0);
        nrow = min(nseq, kMaxRows / p.group);
        if (nrow < nseq && (part || split == 0)) {  // a caller's max_new below the sequence's rows: the rest are zeros
            const int rest = (nseq - nrow) * p.group;
            for (int i = threadIdx.x; i < rest; i += kThreads) {
                const int t = i / p.group;
                no_keys(p, part, split, row0 + nrow + t, kvh * p.group + i - t * p.group);
            }
        }
    }
    const int R = nrow * p.group;
    const int len = max(0, min(p.lens[b], p.max_keys));
    const int own = max(0, len - p.first);
    // whole stages, at least 128 keys: the CTAs that a short sequence does not fill end at once
    const int per = max(2, ((own + kKeys - 1) / kKeys + p.splits - 1) / p.splits) * kKeys;
    const int k0 = R == 0 ? 0 : p.first + min(own, split * per);
    const int k1 = R == 0 ? 0 : p.first + min(own, split * per + per);
    const int nst = (k1 - k0 + kKeys - 1) / kKeys;
    if (nst == 0) {
        for (int r = threadIdx.x; r < R; r += kThreads) {
            const int t = r / p.group;
            if (part || split == 0) no_keys(p, part, split, row0 + t, kvh * p.group + r - t * p.group);
        }
        if (holds) pdl_wait();
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
        const int nbox = kKeys / p.box_rows;
        const int kv = lane & 1, ch = (lane >> 1) % L::kChunks, box = (lane >> 1) / L::kChunks;
        bool ok = true;
        int j = 0;
        for (; j < nst; ++j) {
            const int s = j % L::kStages;
            const int key = k0 + j * kKeys + box * p.box_rows;
            int page = p.n_pages;  // past the keys: outside the pool, filled with zeros
            if (box < nbox && key < k1) {
                const int64_t row = key < p.common ? 0 : b;
                const int id = __ldg(p.table + row * p.ldt + (key >> p.page_shift));
                if (id >= 0 && id < p.n_pages) page = id;
            }
            ok = mbar_wait_warp(&empty[s], ((uint32_t)(j / L::kStages) & 1u) ^ 1u, abort_flag);
            if (!ok) break;
            if (lane == 0) mbar_arrive_expect_tx(&full[s], 2u * L::kTile);
            __syncwarp();
            if (box < nbox)
                tma_load_4d(smem + (s * 2 + kv) * L::kTile + ch * L::kChunk + box * p.box_rows * 128,
                            kv ? &p.tmV : &p.tmK, &full[s], ch * 64, key & ((1 << p.page_shift) - 1), kvh, page);
        }
        if (!ok && lane == 0) {  // copies in flight land before the CTA leaves
            *abort_flag = 1;
            set_err(p.err, 0x601);
            int never = 0;
            for (int i = max(0, j - L::kStages); i < j; ++i)
                mbar_wait_bounded(&full[i % L::kStages], (uint32_t)(i / L::kStages) & 1u, &never, 200000000ull);
        }
        if (holds) pdl_wait();
        return;
    }

    // ------------------------------------------------------------------------ consumers
    const int ra = lane >> 2, rb = ra + 8, cq = (lane & 3) * 2;  // rows and column pair of this lane's fragments
    uint32_t qf[HD / 16][4];
    {
        const int ta = ra / p.group, tb = rb / p.group;
        const __half* qa = p.q + (int64_t)(row0 + ta) * p.ldq + (int64_t)(kvh * p.group + ra - ta * p.group) * p.head_dim;
        const __half* qb = p.q + (int64_t)(row0 + tb) * p.ldq + (int64_t)(kvh * p.group + rb - tb * p.group) * p.head_dim;
#pragma unroll
        for (int kk = 0; kk < HD / 16; ++kk) {
            const bool in = kk * 16 < p.head_dim;
            const int d = kk * 16 + cq;
            qf[kk][0] = in && ra < R ? *reinterpret_cast<const uint32_t*>(qa + d) : 0u;
            qf[kk][1] = in && rb < R ? *reinterpret_cast<const uint32_t*>(qb + d) : 0u;
            qf[kk][2] = in && ra < R ? *reinterpret_cast<const uint32_t*>(qa + d + 8) : 0u;
            qf[kk][3] = in && rb < R ? *reinterpret_cast<const uint32_t*>(qb + d + 8) : 0u;
        }
    }
    int lim[2] = {len, len};  // keys of rows ra and rb end here
    if (p.causal) {
        lim[0] = len - nseq + ra / p.group + 1;
        lim[1] = len - nseq + rb / p.group + 1;
    }
    lim[0] = min(lim[0], k1);
    lim[1] = min(lim[1], k1);
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
    float o[HD / 8][4];
#pragma unroll
    for (int n = 0; n < HD / 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[n][e] = 0.0f;
    const float c = p.c;
    bool ok = true;
    for (int j = 0; j < nst; ++j) {
        const int s = j % L::kStages;
        ok = mbar_wait_warp(&full[s], (uint32_t)(j / L::kStages) & 1u, abort_flag);
        if (!ok) break;
        const int kb = k0 + j * kKeys + warp * 16;  // first key of this warp
        if (kb < k1) {
            const uint32_t kt = smem_u32(smem + s * 2 * L::kTile), vt = kt + L::kTile;
            if (kb + 16 > k1) {  // V rows behind the last key
                uint8_t* vz = smem + (s * 2 + 1) * L::kTile;
                for (int i = lane; i < (16 - (k1 - kb)) * 8 * L::kChunks; i += 32) {
                    const int ch = i / ((16 - (k1 - kb)) * 8), e = i - ch * ((16 - (k1 - kb)) * 8);
                    *reinterpret_cast<uint4*>(vz + ch * L::kChunk + (warp * 16 + k1 - kb) * 128 + e * 16) =
                        make_uint4(0, 0, 0, 0);
                }
                __syncwarp();
            }
            float x[2][4] = {{0.0f, 0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}};
            {
                const int key = warp * 16 + (lane >> 4) * 8 + (lane & 7);
                const uint32_t base = kt + (uint32_t)key * 128u;
#pragma unroll
                for (int kk = 0; kk < HD / 16; ++kk) {
                    uint32_t f[4];
                    const int piece = (2 * kk + ((lane >> 3) & 1)) & 7;
                    ldsm_x4(base + (uint32_t)((kk >> 2) * L::kChunk + ((piece ^ (key & 7)) << 4)), f);
                    mma16816(x[0], qf[kk], f[0], f[1]);
                    mma16816(x[1], qf[kk], f[2], f[3]);
                }
            }
            if (kb + 16 > min(lim[0], lim[1])) {
#pragma unroll
                for (int n = 0; n < 2; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[n][e] = kb + n * 8 + cq + (e & 1) < lim[e >> 1] ? x[n][e] : -INFINITY;
            }
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                float mx = fmaxf(fmaxf(x[0][2 * r], x[0][2 * r + 1]), fmaxf(x[1][2 * r], x[1][2 * r + 1]));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                const bool need = (mx - m[r]) * c > 8.0f;
                if (__any_sync(0xffffffffu, need)) {
                    const float corr = need ? ex2_approx((m[r] - mx) * c) : 1.0f;
                    if (need) m[r] = mx;
                    l[r] *= corr;
#pragma unroll
                    for (int n = 0; n < HD / 8; ++n) {
                        o[n][2 * r] *= corr;
                        o[n][2 * r + 1] *= corr;
                    }
                }
                const float ref = m[r] == -INFINITY ? 0.0f : m[r];
#pragma unroll
                for (int n = 0; n < 2; ++n)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const float pv = ex2_approx((x[n][2 * r + e] - ref) * c);
                        x[n][2 * r + e] = pv;
                        l[r] += pv;
                    }
            }
            const uint32_t pf[4] = {h2(x[0][0], x[0][1]), h2(x[0][2], x[0][3]), h2(x[1][0], x[1][1]),
                                    h2(x[1][2], x[1][3])};
            {
                const int key = warp * 16 + ((lane >> 3) & 1) * 8 + (lane & 7);
                const uint32_t base = vt + (uint32_t)key * 128u;
#pragma unroll
                for (int n = 0; n < HD / 16; ++n) {
                    uint32_t f[4];
                    const int piece = (2 * n + (lane >> 4)) & 7;
                    ldsm_x4_t(base + (uint32_t)((n >> 2) * L::kChunk + ((piece ^ (key & 7)) << 4)), f);
                    mma16816(o[2 * n], pf, f[0], f[1]);
                    mma16816(o[2 * n + 1], pf, f[2], f[3]);
                }
            }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[s]);
    }
    if (!ok) {
        *abort_flag = 1;
        if (lane == 0) set_err(p.err, 0x602);
    }
    // ---- merge of the four warps
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
        l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
    }
    consumer_bar();  // nobody reads the ring any more
    float* so = reinterpret_cast<float*>(smem);                                    // [warp][row][HD]
    float2* sml = reinterpret_cast<float2*>(smem + L::kOffMl);                      // [warp][row]
    if ((lane & 3) == 0) {
        sml[warp * kMaxRows + ra] = make_float2(m[0], l[0]);
        sml[warp * kMaxRows + rb] = make_float2(m[1], l[1]);
    }
#pragma unroll
    for (int n = 0; n < HD / 8; ++n) {
        const int d = n * 8 + cq;
        if (ra < R) *reinterpret_cast<float2*>(so + (warp * kMaxRows + ra) * HD + d) = make_float2(o[n][0], o[n][1]);
        if (rb < R) *reinterpret_cast<float2*>(so + (warp * kMaxRows + rb) * HD + d) = make_float2(o[n][2], o[n][3]);
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
            const float4 v = *reinterpret_cast<const float4*>(so + (w * kMaxRows + r) * HD + d);
            sum += f * ml.y;
            acc[0] += f * v.x;
            acc[1] += f * v.y;
            acc[2] += f * v.z;
            acc[3] += f * v.w;
        }
        const int t = r / p.group, head = kvh * p.group + r - t * p.group;
        // keys, but all scores -inf: 0 / 0 in the formula, (-inf, 1) for a combination
        const bool flat = mm == -INFINITY && sum == 0.0f && (p.causal ? min(k1, len - nseq + t + 1) : k1) > k0;
        if (flat) sum = 1.0f;
        if (p.cluster) {
            if (d == 0)
                *reinterpret_cast<float2*>(smem + L::kOffOwnMl + r * 8) =
                    make_float2(mm, sum);
            *reinterpret_cast<float4*>(smem + L::kOffOwn + (r * HD + d) * 4) =
                make_float4(acc[0], acc[1], acc[2], acc[3]);
        } else if (part) {
            const int64_t at = ((int64_t)(p.split0 + split) * p.total_q + row0 + t) * p.heads + head;
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
        const int n = (own + per - 1) / per;
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
    if (holds) pdl_wait();
}

// out[row, head] = sum_s 2^((m_s - m) c) o_s / sum_s 2^((m_s - m) c) l_s over the
// splits that saw a key; one warp per (row, head).  Rows outside
// [cu[0], cu[batch]) are left as they are.
__global__ void __launch_bounds__(128) paged_combine_kernel(const float* __restrict__ part_o,
                                                            const float2* __restrict__ part_ml, int splits, int rows,
                                                            int heads, int hd, const int32_t* __restrict__ cu,
                                                            int batch, float c, __half* __restrict__ out,
                                                            int64_t ldo) {
    pdl_trigger();
    pdl_wait();
    const int lane = threadIdx.x & 31;
    const int64_t id = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5), n = (int64_t)rows * heads;
    if (id >= n) return;
    const int64_t row = id / heads;
    if (cu && (row < cu[0] || row >= cu[batch])) return;
    float m = -INFINITY;
    for (int s = lane; s < splits; s += 32) m = fmaxf(m, part_ml[(int64_t)s * n + id].x);
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
    float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f}, sum = 0.0f;
    const bool act = lane * 4 < hd;
    for (int s0 = 0; s0 < splits; s0 += 32) {
        // lane s: the weight of split s0 + s (0 where it saw no key and has no partial)
        float f = 0.0f;
        if (s0 + lane < splits) {
            const float2 ml = part_ml[(int64_t)(s0 + lane) * n + id];
            if (ml.y != 0.0f) f = ex2_approx((ml.x - m) * c);
            sum += f * ml.y;
        }
        const float* src = part_o + ((int64_t)s0 * n + id) * hd + lane * 4;
        const int cnt = min(32, splits - s0);
        for (int s = 0; s < cnt; s += 8) {  // eight loads in flight
            float4 v[8];
            float w[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                w[i] = __shfl_sync(0xffffffffu, f, (s + i) & 31);
                if (s + i >= cnt) w[i] = 0.0f;
                v[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                if (act && w[i] != 0.0f) v[i] = __ldcs(reinterpret_cast<const float4*>(src + (int64_t)(s + i) * n * hd));
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                acc[0] += w[i] * v[i].x;
                acc[1] += w[i] * v[i].y;
                acc[2] += w[i] * v[i].z;
                acc[3] += w[i] * v[i].w;
            }
        }
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    if (!act) return;
    const float inv = 1.0f / sum;
    uint2 w;
    w.x = sum != 0.0f ? h2(acc[0] * inv, acc[1] * inv) : 0u;
    w.y = sum != 0.0f ? h2(acc[2] * inv, acc[3] * inv) : 0u;
    *reinterpret_cast<uint2*>(out + row * ldo + (id - row * heads) * hd + lane * 4) = w;
}

template <int HD>
int launch(const Params& p, int batch, cudaStream_t st) {
    auto kern = paged_decode_kernel<HD>;
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Smem<HD>::kTotal);
    if (e != cudaSuccess) {
        npub_internal_set_cuda_error(e);
        return NPUB_ERR_CUDA;
    }
    if (!p.cluster)
        return launch_pdl(kern, dim3(p.kv_heads * p.splits, batch), dim3(kThreads), Smem<HD>::kTotal, st, p);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(p.kv_heads * p.splits, batch);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = Smem<HD>::kTotal;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = npub_internal_pdl_enabled() ? 1 : 0;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = p.splits;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    const cudaError_t le = cudaLaunchKernelEx(&cfg, kern, p);
    if (le != cudaSuccess) {
        npub_internal_set_cuda_error(le);
        return NPUB_ERR_CUDA;
    }
    return npub_internal_launch_status();
}

}  // namespace pdec

int paged_decode(const PackedArgs& a, cudaStream_t st) {
    using namespace pdec;
    Params p;
    memset(&p, 0, sizeof(p));
    p.box_rows = a.kv.page_size < kKeys ? a.kv.page_size : kKeys;
    int rc = make_tmap_pages(&p.tmK, a.kv.k, a.kv.n_pages, a.kv_heads, a.kv.page_size, a.head_dim, p.box_rows);
    if (rc) return rc;
    rc = make_tmap_pages(&p.tmV, a.kv.v, a.kv.n_pages, a.kv_heads, a.kv.page_size, a.head_dim, p.box_rows);
    if (rc) return rc;
    while ((1 << p.page_shift) < a.kv.page_size) ++p.page_shift;
    const int64_t mk = (int64_t)a.kv.max_pages << p.page_shift;
    p.max_keys = mk > 0x7ff00000 ? 0x7ff00000 : (int)mk;
    p.n_pages = a.kv.n_pages;
    p.common = a.kv.common;
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
    p.first = a.first;
    p.splits = a.splits;
    p.cluster = !a.part_o && a.splits > 1;
    p.split0 = a.split0;
    p.beside = a.first > 0;
    p.c = a.scale * 1.4426950408889634f;
    p.out = reinterpret_cast<__half*>(a.out);
    p.ldo = a.ldo;
    p.part_o = a.part_o;
    p.part_ml = a.part_ml;
    p.err = npub_internal_device_error_word();
    return a.head_dim <= 64 ? launch<64>(p, a.batch, st) : launch<128>(p, a.batch, st);
}

int paged_combine(const PackedArgs& a, int splits, cudaStream_t st) {
    const int64_t n = (int64_t)a.total_q * a.heads;
    if ((n + 3) / 4 > 0x7fffffff) return NPUB_ERR_UNSUPPORTED;
    return launch_pdl(pdec::paged_combine_kernel, dim3((unsigned)((n + 3) / 4)), dim3(128), 0, st, a.part_o,
                      a.part_ml, splits, a.total_q, a.heads, a.head_dim, a.cu, a.batch, a.scale * 1.4426950408889634f,
                      reinterpret_cast<__half*>(a.out), a.ldo);
}

}  // namespace npub
