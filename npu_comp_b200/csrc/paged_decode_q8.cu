// Attention of a few new rows per sequence over a paged KV cache held in 8
// bits, K = s_k q_k and V = s_v q_v with one scale for each page and kv head
// (the 8-bit form of paged_decode.cu; the rows' tiles, the key ranges and their
// combination are the same).
//
// What it costs is one read of the 8-bit K and V (HBM bound: 2 * head_dim bytes
// per key and head); beside it the conversion to fp16 has to keep up.  So:
//   * the integers go into the fp16 tensor-core products as they are (exact in
//     fp16); a step of 16 keys lies in one page, so its scales are two numbers.
//   * an integer q of K goes in as the byte q + 128, which as the bits of an fp16
//     is the subnormal (q + 128) 2^-24: one byte permutation for two of them, and
//     128 sum(q_row) is taken off the score (whose fp32 sums round relative to
//     255 sum |q_row| for it).  (Not for V: the weights' sum times 128 would drown
//     an average over many keys.  There it is two instructions.)
//   * s_k multiplies the scores; s_v goes into the exponent: with z = c s_k (q . k)
//     + log2(s_v), c = scale log2(e), the weights 2^(z - m) carry s_v, O takes them
//     times the integers, and the row's sum takes them times 1 / s_v.  The running
//     reference m is of z, so a weight's rounding to fp16 (2^-11, for the product
//     with V) is relative to what it adds to the result: off by 0.00023 to 0.00029
//     against 64 bits, where the output's rounding alone is 0.00021.  (s_v below
//     2^-40 counts as 2^-40: what it adds to a result is below 2^-33.)
//   * a scale that is not finite makes the scores of its keys NaN, and with them
//     the sum of every row that sees one; a part of an item whose sum is NaN is
//     never left out of a merge.
//   * an element's place in the product's inner dimension is free, as long as
//     both operands agree: a lane takes 16 neighbouring columns of a key with one
//     16-byte load, which are 4 steps of the K product, or 16 of the columns of
//     the V product; the swizzle of the tile keeps the loads free of bank
//     conflicts.
//
// Rows: a tile is 8 or 16 of a kv head, (token, grouped head) in order; more in
// further tiles, which find K and V in L2.
//
// Two kernels.  paged_decode_q8_kernel: one CTA per (sequence, kv head, tile,
// range of keys), up to eight ranges of an item a cluster that combines through
// one another's shared memory: one launch, for small calls.
// paged_list_q8_kernel: all items' steps of 32 keys are one list, cut into equal
// parts for the resident warps, each of which streams its part on its own (its
// ring, its loads, no barrier with another warp) across the items' borders; an
// item that several warps share leaves partials for paged_list_combine_kernel.
// The lengths are on the device, so the list is cut there.
//
// Measured, heads of 128: one row on 777 keys, 32 / 8 heads, 7.5 to 8 us (cluster
// kernel: launch and memory latencies); 32 rows on 65000 keys of 32 heads 97 us,
// 5.5 TB/s (list, tiles of 8 rows: HBM); 96 drafted rows of 24 sequences on 70001
// keys, 32 / 8 heads, 60 us, 2.4 TB/s (list, tiles of 16 rows: the conversions and
// products of 12 warps an SM, at 34 % of the issue slots).
#include "common.cuh"
#include "gemm_tc.h"
#include "paged_decode.h"

namespace npub {
namespace pdq8 {

constexpr int kWarps = 4;               // consumers
constexpr int kThreads = kWarps * 32 + 32;
constexpr int kStep = 32;               // keys that a warp takes at a time
constexpr int kKeys = kWarps * kStep;   // keys per stage
constexpr int kGroups = kKeys / 16;     // runs of keys with the same scales

template <int HD, int kMaxRows>
struct Smem {
    static constexpr int kTile = kKeys * HD;  // K or V of a stage
    static constexpr int kStages = (kMaxRows == 8 ? 64 : 96) * 1024 / (2 * kTile);
    static constexpr int kOffScale = kStages * 2 * kTile;  // [stage][group]: c s_k, log2(s_v), 1 / s_v
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
    // list kernel: partials [2 workers][rows of a tile][64 or 128] and (reference score, sum); of each item [batch][kv_heads]
    // [tiles] where its partials are, and how many (1: none, the item is whole)
    float* part_o;
    float2* part_ml;
    int2* parts;
    int batch, tiles;  // tiles of a sequence at most
    int slots;         // of partials, two for each warp
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
// What a scale is to the kernels: K's as it is (NaN where it is not finite), V's held at 2^-40 or more (NaN stays).  A page
// outside the pool is zeros, its scale 1.
__device__ __forceinline__ float usable(float scale, bool v, bool in_pool) {
    if (!in_pool) return v ? 1.0f : 0.0f;
    if (!isfinite(scale)) return NAN;
    return v && scale < 9.094947e-13f ? 9.094947e-13f : scale;
}

// A score's integer sum is its products' sum 2^24 - 128 sum(q), in one rounding; the scales come behind it, so that scores
// are right as far as fp32 holds them (2^24 in the scale ran over from c s_k = 2e31 on).
// log2 and reciprocal of a usable V scale (to 2^-22 and 2^-23: as close as the scores).  The
// reciprocal of NaN is 1: the scores carry the NaN to the rows that see the page, and masked ones weigh 0 times this.
constexpr float kSubnormal = 16777216.0f;
__device__ __forceinline__ float log2_of(float v) {
    float r;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ float inverse_of(float v) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return isnan(v) ? 1.0f : r;
}
// 16 int8 as fp16 pairs (q + 128) 2^-24.
__device__ __forceinline__ void bytes_to_subnormals(uint4 raw, uint32_t (&f)[8]) {
    const uint32_t w[4] = {raw.x ^ 0x80808080u, raw.y ^ 0x80808080u, raw.z ^ 0x80808080u, raw.w ^ 0x80808080u};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f[2 * i] = __byte_perm(w[i], 0u, 0x4140);
        f[2 * i + 1] = __byte_perm(w[i], 0u, 0x4342);
    }
}

// A warp's tile: scores, running maxima and sums, and output of up to kMaxRows rows over the keys that it has taken.
//
// kMaxRows 16: S = Q K^T and O = P V with the rows on the product's 16-side.
// kMaxRows 8: transposed, S^T = K Q^T and O^T = V^T P^T with the rows on its
// 8-side: half of the products, exponentials and sums.  A lane's integers of K
// and V are the same in both.
template <int HD, int kMaxRows>
struct WarpTile {
    static constexpr bool kT = kMaxRows == 8;
    static constexpr int kQ = kT ? 1 : 2;  // rows of Q that a lane holds: g8 (and g8 + 8)
    // output: kT: tile n has columns g8 HD / 8 + 2 n (e < 2) and the next (e >= 2), rows ra (even e) and rb; else tile n has
    // column (2 t4 + (e & 1)) HD / 8 + n, rows ra (e < 2) and rb
    static constexpr int kO = kT ? HD / 16 : HD / 8;
    // scores of 16 keys, [2 u + i][e]: kT: x[u] are keys g8 (e < 2) and g8 + 8 of rows ra (even e) and rb; else x[2 u + i]
    // is key 8 i + 2 t4 + (e & 1) of row ra (e < 2) or rb
    static constexpr int kX = kT ? kStep / 16 : kStep / 8;
    int g8, t4;  // the lane's place among eight and among four
    int ra, rb;  // rows whose scores and output this lane holds
    uint32_t qf[HD / 16][2 * kQ];
    int lim[2];  // keys of rows ra and rb end here
    float m[2], l[2];
    float bias[2];  // 128 sum(q) of rows ra and rb
    float o[kO][4];

    __device__ __forceinline__ static int row_of(int e) { return kT ? e & 1 : e >> 1; }
    __device__ __forceinline__ int key_of(int n, int e) const {
        return kT ? n * 16 + g8 + (e >> 1) * 8 : n * 8 + t4 * 2 + (e & 1);
    }
    __device__ __forceinline__ WarpTile() {
        const int lane = threadIdx.x & 31;
        g8 = lane >> 2;
        t4 = lane & 3;
        ra = kT ? 2 * t4 : g8;
        rb = kT ? ra + 1 : ra + 8;
    }
    // R rows of head kvh from number f0 on, (token, grouped head) in order, of the sequence of nseq tokens from row0 on and
    // len keys, over keys up to k1.
    __device__ __forceinline__ void start(const Params& p, int row0, int R, int kvh, int f0, int nseq, int len, int k1) {
#pragma unroll
        for (int i = 0; i < kQ; ++i) {
            const int row = g8 + 8 * i, t = (f0 + row) / p.group;
            const __half* src =
                p.q + (int64_t)(row0 + t) * p.ldq + (int64_t)(kvh * p.group + f0 + row - t * p.group) * p.head_dim;
#pragma unroll
            for (int kk = 0; kk < HD / 16; ++kk) {  // step kk of the lane's HD / 4 columns: 4 of them
                const int d = t4 * (HD / 4) + kk * 4;
                const uint2 w = d < p.head_dim && row < R ? *reinterpret_cast<const uint2*>(src + d) : make_uint2(0, 0);
                qf[kk][i] = w.x;
                qf[kk][kQ + i] = w.y;
            }
            float sum = 0.0f;
#pragma unroll
            for (int kk = 0; kk < HD / 16; ++kk) {
                const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&qf[kk][i]));
                const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&qf[kk][kQ + i]));
                sum += (a.x + a.y) + (b.x + b.y);
            }
            sum += __shfl_xor_sync(0xffffffffu, sum, 1);
            sum += __shfl_xor_sync(0xffffffffu, sum, 2);
            bias[i] = sum * 128.0f;
        }
        if (kT) {  // that of row g8 is in its lanes
            bias[1] = __shfl_sync(0xffffffffu, bias[0], rb * 4);
            bias[0] = __shfl_sync(0xffffffffu, bias[0], ra * 4);
        }
        lim[0] = lim[1] = len;
        if (p.causal) {
            lim[0] = len - nseq + (f0 + ra) / p.group + 1;
            lim[1] = len - nseq + (f0 + rb) / p.group + 1;
        }
        lim[0] = min(lim[0], k1);
        lim[1] = min(lim[1], k1);
        m[0] = m[1] = -INFINITY;
        l[0] = l[1] = 0.0f;
#pragma unroll
        for (int n = 0; n < kO; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[n][e] = 0.0f;
    }
    // kStep keys from kb on at kt and vt; sc(u): {c s_k, log2(s_v), 1 / s_v} of its u-th 16 keys.
    template <typename Scales>
    __device__ __forceinline__ void step(const uint8_t* kt, const uint8_t* vt, int kb, Scales sc) {
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
                    bytes_to_subnormals(*reinterpret_cast<const uint4*>(kt + at), f[i]);
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
            const float4 v = sc(u);
            inv[u] = v.z;
#pragma unroll
            for (int n = u * kX * 16 / kStep; n < (u + 1) * kX * 16 / kStep; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) x[n][e] = fmaf(fmaf(x[n][e], kSubnormal, -bias[row_of(e)]), v.x, v.y);
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
        const bool need[2] = {mx[0] - m[0] > 8.0f, mx[1] - m[1] > 8.0f};
        if (__any_sync(0xffffffffu, need[0] || need[1])) {
            float corr[2];
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                corr[r] = need[r] ? ex2_approx(m[r] - mx[r]) : 1.0f;
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
                const float pv = ex2_approx(x[n][e] - ref[row_of(e)]);
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
    // The rows' sums over the lanes that share them.
    __device__ __forceinline__ void sum_lanes() {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], kT ? 4 : 1);
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], kT ? 8 : 2);
            if (kT) l[r] += __shfl_xor_sync(0xffffffffu, l[r], 16);
        }
    }
    // f(row, first column, its HD / 8 outputs) for the runs of columns that this lane holds: of row ra, then rb.
    template <typename F>
    __device__ __forceinline__ void runs(F f) const {
        if constexpr (kT) {
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                float v[HD / 8];
#pragma unroll
                for (int n = 0; n < kO; ++n) {
                    v[2 * n] = o[n][r];
                    v[2 * n + 1] = o[n][2 + r];
                }
                f(r, g8 * (HD / 8), v);
            }
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float v[HD / 8];
#pragma unroll
                for (int n = 0; n < kO; ++n) v[n] = o[n][e];
                f(e >> 1, (2 * t4 + (e & 1)) * (HD / 8), v);
            }
        }
    }
};

__device__ __forceinline__ void zero_row(const Params& p, int row, int head) {
    for (int d = 0; d < p.head_dim; d += 4)
        *reinterpret_cast<uint2*>(p.out + (int64_t)row * p.ldo + (int64_t)head * p.head_dim + d) = make_uint2(0, 0);
}

// grid (kv_heads * splits, batch, tiles of kMaxRows rows)
template <int HD, int kMaxRows>
__global__ void __launch_bounds__(kThreads, kMaxRows == 8 ? 3 : 2)
    paged_decode_q8_kernel(const __grid_constant__ Params p) {
    using L = Smem<HD, kMaxRows>;
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
    pdl_wait();
    // this CTA's rows, the sequence's keys, and the range of them
    int row0 = b, nseq = 1;
    if (p.cu) {
        row0 = max(0, min(p.total_q, p.cu[b]));
        nseq = max(0, min(p.total_q, p.cu[b + 1]) - row0);
    }
    const int f0 = (int)blockIdx.z * kMaxRows;  // (token, grouped head) in order
    const int64_t all = (int64_t)nseq * p.group;
    const int R = (int)max((int64_t)0, min(all - f0, (int64_t)kMaxRows));
    if (blockIdx.z == gridDim.z - 1 && split == 0) {  // a caller's max_new below the sequence's rows: the rest are zeros
        for (int64_t f = (int64_t)gridDim.z * kMaxRows + threadIdx.x; f < all; f += kThreads) {
            const int t = (int)(f / p.group);
            zero_row(p, row0 + t, kvh * p.group + (int)(f - (int64_t)t * p.group));
        }
    }
    const int len = max(0, min(p.lens[b], p.max_keys));
    const int per = max(128 / kKeys, ((len + kKeys - 1) / kKeys + p.splits - 1) / p.splits) * kKeys;
    const int k0 = R == 0 ? 0 : min(len, split * per);
    const int k1 = R == 0 ? 0 : min(len, split * per + per);
    const int nst = (k1 - k0 + kKeys - 1) / kKeys;
    if (nst == 0) {
        for (int r = threadIdx.x; r < R; r += kThreads) {
            const int t = (f0 + r) / p.group;
            if (split == 0) zero_row(p, row0 + t, kvh * p.group + f0 + r - t * p.group);
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
                const float v = usable(scale, kv, page < p.n_pages);
                if (kv) {
                    for (int g = 0; g < groups; ++g) {
                        sc[g * 4 + 1] = log2_of(v);
                        sc[g * 4 + 2] = inverse_of(v);
                    }
                } else {
                    for (int g = 0; g < groups; ++g) sc[g * 4] = v * p.c;
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
    WarpTile<HD, kMaxRows> w;
    w.start(p, row0, R, kvh, f0, nseq, len, k1);
    bool ok = true;
    int j = 0;
    for (; j < nst; ++j) {
        const int s = j % L::kStages;
        ok = mbar_wait_warp(&full[s], (uint32_t)(j / L::kStages) & 1u, abort_flag);
        if (!ok) break;
        const int kb = k0 + j * kKeys + warp * kStep;  // first key of this warp
        if (kb < k1) {
            const uint8_t* kt = smem + s * 2 * L::kTile + warp * kStep * HD;
            const uint8_t* vt = kt + L::kTile;
            const float4* sc = reinterpret_cast<const float4*>(smem + L::kOffScale + (s * kGroups + warp * (kStep / 16)) * 16);
            w.step(kt, vt, kb, [&](int u) { return sc[u]; });
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[s]);
    }
    if (!ok) {  // copies in flight land before the ring is used again and the CTA leaves; the rows are NaN
        *abort_flag = 1;
        if (lane == 0) set_err(p.err, 0x722);
        int never = 0;
        for (int i = j; i < min(nst, j + L::kStages); ++i)
            mbar_wait_bounded(&full[i % L::kStages], (uint32_t)(i / L::kStages) & 1u, &never, 100000000ull);
        __syncwarp();
        w.l[0] = w.l[1] = NAN;
    }
    // ---- merge of the four warps
    w.sum_lanes();
    consumer_bar();  // nobody reads the ring any more
    float* so = reinterpret_cast<float*>(smem);                 // [warp][row][8 runs]
    float2* sml = reinterpret_cast<float2*>(smem + L::kOffMl);  // [warp][row]
    if ((w.kT ? w.g8 : w.t4) == 0) {
        sml[warp * kMaxRows + w.ra] = make_float2(w.m[0], w.l[0]);
        sml[warp * kMaxRows + w.rb] = make_float2(w.m[1], w.l[1]);
    }
    w.runs([&](int r, int col, const float (&v)[HD / 8]) {
        float* dst = so + (warp * kMaxRows + (r ? w.rb : w.ra)) * L::kRow + col / L::kRun * (L::kRun + 4);
#pragma unroll
        for (int n = 0; n < HD / 8; n += 4)
            *reinterpret_cast<float4*>(dst + n) = make_float4(v[n], v[n + 1], v[n + 2], v[n + 3]);
    });
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
            const float f = ex2_approx(ml.x - mm);
            const float4 v = *reinterpret_cast<const float4*>(so + (w * kMaxRows + r) * L::kRow + d + d / L::kRun * 4);
            sum += f * ml.y;
            acc[0] += f * v.x;
            acc[1] += f * v.y;
            acc[2] += f * v.z;
            acc[3] += f * v.w;
        }
        const int t = (f0 + r) / p.group, head = kvh * p.group + f0 + r - t * p.group;
        // keys, but all scores -inf: 0 / 0 in the formula, (-inf, 1) for a combination
        const bool flat = mm == -INFINITY && sum == 0.0f && (p.causal ? min(k1, len - nseq + t + 1) : k1) > k0;
        if (flat) sum = 1.0f;
        if (p.cluster) {
            if (d == 0) *reinterpret_cast<float2*>(smem + L::kOffOwnMl + r * 8) = make_float2(mm, sum);
            *reinterpret_cast<float4*>(smem + L::kOffOwn + (r * HD + d) * 4) =
                make_float4(acc[0], acc[1], acc[2], acc[3]);
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
                const float f = ex2_approx(ml.x - mm);
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
            const int t = (f0 + r) / p.group, head = kvh * p.group + f0 + r - t * p.group;
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

// ------------------------------------------------------------------------ the list of all items' steps

constexpr int kListCtas = 3;  // per SM
template <int HD>
struct ListSmem {
    static constexpr int kTile = kStep * HD;                   // K or V of a step
    static constexpr int kStages = HD == 128 ? 2 : 4;          // a warp's ring: 16 KB
    static constexpr int kRing = kStages * 2 * kTile;
    static constexpr int kOffBar = kWarps * kRing;
    static constexpr int kTotal = kOffBar + kWarps * kStages * 8;
};

// A sequence as the list sees it: `items` of `steps` steps each, item i = kv head i / tiles, tile i % tiles of its rows.
struct Seq {
    int row0, rows, len, tiles, steps, items;
};
__device__ __forceinline__ Seq seq_at(const Params& p, int rows_of_tile, int b) {
    Seq s = {b, 1, 0, 0, 0, 0};
    if (b >= p.batch) return s;
    if (p.cu) {
        s.row0 = max(0, min(p.total_q, __ldg(p.cu + b)));
        s.rows = max(0, min(p.total_q, __ldg(p.cu + b + 1)) - s.row0);
    }
    s.len = max(0, min(__ldg(p.lens + b), p.max_keys));
    s.tiles = (int)min((int64_t)p.tiles, ((int64_t)s.rows * p.group + rows_of_tile - 1) / rows_of_tile);
    s.steps = (int)(((int64_t)s.len + kStep - 1) / kStep);
    s.items = s.steps > 0 ? s.tiles * p.kv_heads : 0;
    return s;
}
__device__ __forceinline__ int64_t scan_up(int64_t v) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int64_t u = __shfl_up_sync(0xffffffffu, v, d);
        if (lane >= d) v += u;
    }
    return v;
}
// Warps that share the list: all of them, or one for every four steps.
__device__ __forceinline__ int64_t workers_of(int64_t steps, int64_t warps) {
    const int64_t w = (steps + 3) / 4;
    return w < warps ? w : warps;
}
// The first step of worker w, and the worker that has step g.
__device__ __forceinline__ int64_t first_step(int64_t w, int64_t steps, int64_t workers) { return steps * w / workers; }
__device__ __forceinline__ int64_t worker_of(int64_t g, int64_t steps, int64_t workers) {
    return ((g + 1) * workers + steps - 1) / steps - 1;
}

template <int HD, int kMaxRows>
__global__ void __launch_bounds__(kWarps * 32, kListCtas) paged_list_q8_kernel(const __grid_constant__ Params p) {
    using L = ListSmem<HD>;
    constexpr int kD = L::kStages;
    pdl_trigger();
    extern __shared__ __align__(1024) uint8_t smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::kOffBar) + warp * kD;
    uint8_t* ring = smem + warp * L::kRing;
    if (smem_u32(smem) & 1023u) {
        if (threadIdx.x == 0) set_err(p.err, 0x730);
        pdl_wait();
        return;
    }
    if (lane == 0) {
        for (int i = 0; i < kD; ++i) mbar_init(&full[i], 1);
        fence_barrier_init();
        prefetch_tmap(&p.tmK);
        prefetch_tmap(&p.tmV);
    }
    __syncwarp();
    pdl_wait();
    // ---- this warp's part of the list
    const int64_t id = (int64_t)blockIdx.x * kWarps + warp;
    int64_t total = 0;
    for (int b = lane; b < p.batch; b += 32) {
        const Seq s = seq_at(p, kMaxRows, b);
        total += (int64_t)s.steps * s.items;
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) total += __shfl_xor_sync(0xffffffffu, total, d);
    const int64_t workers = workers_of(total, (int64_t)gridDim.x * kWarps);
    const int64_t s0 = id < workers ? first_step(id, total, workers) : total;
    const int64_t s1 = id < workers ? first_step(id + 1, total, workers) : total;
    int b = 0, item = 0, step = 0;
    Seq seq = {};
    {
        int64_t ahead = 0;
        bool found = s0 >= s1;
        for (int base = 0; base < p.batch && !found; base += 32) {
            const Seq s = seq_at(p, kMaxRows, base + lane);
            const int64_t n = (int64_t)s.steps * s.items, end = ahead + scan_up(n);
            const uint32_t vote = __ballot_sync(0xffffffffu, end > s0);
            if (vote) {
                const int l = __ffs(vote) - 1;
                const int64_t in = s0 - __shfl_sync(0xffffffffu, end - n, l);
                found = true;
                b = base + l;
                seq = seq_at(p, kMaxRows, b);
                item = (int)(in / seq.steps);
                step = (int)(in - (int64_t)item * seq.steps);
            }
            ahead = __shfl_sync(0xffffffffu, end, 31);
        }
    }
    const int n = (int)min(s1 - s0, (int64_t)0x7fffffff);
    if (n == 0) return;

    // ---- loads: the lane of (K or V, page piece) looks its page up, copies it and keeps its scale until the step is taken
    const int kv = lane & 1, piece = lane >> 1;
    const bool loads = piece * p.box_rows < kStep;
    const int ahead_of = piece * p.box_rows;  // keys of the step ahead of the piece
    const float* scales = kv ? p.vs : p.ks;
    const CUtensorMap* tm = kv ? &p.tmV : &p.tmK;
    uint8_t* to = ring + kv * L::kTile + ahead_of * HD;
    const int slot_mask = (1 << p.page_shift) - 1;
    struct At {  // a step of the list
        int b, kvh, tile, step;
        int tiles, steps, len;  // of sequence b
    };
    auto next = [&](At& t) {
        if (++t.step < t.steps) return;
        t.step = 0;
        if (++t.tile < t.tiles) return;
        t.tile = 0;
        if (++t.kvh < p.kv_heads) return;
        t.kvh = 0;
        Seq s;
        do {
            s = seq_at(p, kMaxRows, ++t.b);
        } while (s.items == 0 && t.b < p.batch);
        t.tiles = s.tiles;
        t.steps = s.steps;
        t.len = s.len;
    };
    At now = {b, item / seq.tiles, item % seq.tiles, step, seq.tiles, seq.steps, seq.len};
    At then = now;  // the step to load next
    const int32_t* ids = p.table + (int64_t)then.b * p.ldt;
    float scale[kD];
    bool pool[kD];
    auto load = [&](int slot, float& sc, bool& in) {
        const int key = then.step * kStep + ahead_of;
        int page = p.n_pages;  // past the keys: outside the pool, filled with zeros
        if (loads && key < then.len) {
            const int id = __ldg(ids + (key >> p.page_shift));
            if (id >= 0 && id < p.n_pages) page = id;
        }
        if (lane == 0) mbar_arrive_expect_tx(&full[slot], 2u * L::kTile);
        __syncwarp();
        if (loads) tma_load_4d(to + slot * 2 * L::kTile, tm, &full[slot], 0, key & slot_mask, then.kvh, page);
        in = page < p.n_pages;
        sc = in ? __ldg(scales + (int64_t)page * p.kv_heads + then.kvh) : 0.0f;
        const int was = then.b;
        next(then);
        if (then.b != was) ids = p.table + (int64_t)then.b * p.ldt;
    };
#pragma unroll
    for (int d = 0; d < kD; ++d) {
        scale[d] = 0.0f;
        pool[d] = false;
        if (d < n) load(d, scale[d], pool[d]);
    }

    // ---- the steps
    WarpTile<HD, kMaxRows> w;
    int src[kStep / 16];  // the lane of the K piece that holds 16 keys (V's is the next)
#pragma unroll
    for (int u = 0; u < kStep / 16; ++u) src[u] = 2 * (u * 16 / p.box_rows);
    int begun = now.step;  // first step of the current item that is this warp's
    int row0 = 0, f0 = 0, R = 0;
    bool fresh = true;  // the current item is the first of this warp's
    // j: steps of this warp ahead of the item's
    auto open = [&](int j) {
        if (now.step == 0 && lane == 0) {  // the warp with an item's first step says where its parts will be
            const int64_t g0 = s0 + j;
            const int last = (int)worker_of(g0 + now.steps - 1, total, workers);
            p.parts[((int64_t)now.b * p.kv_heads + now.kvh) * p.tiles + now.tile] =
                make_int2(2 * (int)id + (fresh ? 0 : 1), last - (int)id + 1);
        }
        const Seq s = seq_at(p, kMaxRows, now.b);
        row0 = s.row0;
        f0 = now.tile * kMaxRows;
        R = (int)min((int64_t)kMaxRows, (int64_t)s.rows * p.group - f0);
        w.start(p, row0, R, now.kvh, f0, s.rows, s.len, s.len);
    };
    open(0);
    int never = 0;
    volatile int* no_abort = &never;
    for (int j = 0; j < n; ++j) {
        const int slot = j % kD;
        if (!mbar_wait_warp(&full[slot], (uint32_t)(j / kD) & 1u, no_abort)) {
            if (lane == 0) {
                set_err(p.err, 0x731);
                for (int i = j + 1; i < min(n, j + kD); ++i)  // copies in flight land before the warp leaves
                    mbar_wait_bounded(&full[i % kD], (uint32_t)(i / kD) & 1u, &never, 100000000ull);
            }
            return;
        }
        const float v = usable(scale[0], kv, pool[0]);
        const float first_of = kv ? log2_of(v) : v * p.c, inv = inverse_of(v);
        const uint8_t* kt = ring + slot * 2 * L::kTile;
        w.step(kt, kt + L::kTile, now.step * kStep, [&](int u) {
            return make_float4(__shfl_sync(0xffffffffu, first_of, src[u]), __shfl_sync(0xffffffffu, first_of, src[u] + 1),
                               __shfl_sync(0xffffffffu, inv, src[u] + 1), 0.0f);
        });
        __syncwarp();  // every lane has read the slot
#pragma unroll
        for (int d = 0; d + 1 < kD; ++d) {
            scale[d] = scale[d + 1];
            pool[d] = pool[d + 1];
        }
        if (j + kD < n) load(slot, scale[kD - 1], pool[kD - 1]);
        const bool ends = now.step + 1 == now.steps;
        if (ends || j + 1 == n) {
            w.sum_lanes();
            const int k0 = begun * kStep;
            float inv_l[2];
            bool flat[2];
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                // keys, but all scores -inf: 0 / 0 in the formula, (-inf, 1) for the combination
                flat[r] = w.l[r] == 0.0f && w.lim[r] > k0 && w.m[r] == -INFINITY;
                inv_l[r] = flat[r] ? NAN : w.l[r] != 0.0f ? 1.0f / w.l[r] : 0.0f;
            }
            if (begun == 0 && ends) {  // a whole item
                w.runs([&](int r, int col, const float (&o)[HD / 8]) {
                    const int row = r ? w.rb : w.ra;
                    if (row >= R || col >= p.head_dim) return;
                    const int t = (f0 + row) / p.group;
                    __half* dst = p.out + (int64_t)(row0 + t) * p.ldo +
                                  (int64_t)(now.kvh * p.group + f0 + row - t * p.group) * p.head_dim + col;
                    const bool any = w.l[r] != 0.0f || flat[r];
#pragma unroll
                    for (int i = 0; i < HD / 8; i += 8)
                        *reinterpret_cast<uint4*>(dst + i) =
                            any ? make_uint4(h2(o[i] * inv_l[r], o[i + 1] * inv_l[r]), h2(o[i + 2] * inv_l[r], o[i + 3] * inv_l[r]),
                                             h2(o[i + 4] * inv_l[r], o[i + 5] * inv_l[r]), h2(o[i + 6] * inv_l[r], o[i + 7] * inv_l[r]))
                                : make_uint4(0, 0, 0, 0);
                });
            } else {
                const int64_t at = (2 * id + (fresh ? 0 : 1)) * kMaxRows;
                if ((w.kT ? w.g8 : w.t4) == 0) {
                    p.part_ml[at + w.ra] = make_float2(w.m[0], flat[0] ? 1.0f : w.l[0]);
                    p.part_ml[at + w.rb] = make_float2(w.m[1], flat[1] ? 1.0f : w.l[1]);
                }
                w.runs([&](int r, int col, const float (&o)[HD / 8]) {
                    const int row = r ? w.rb : w.ra;
                    if (row >= R) return;
                    float* dst = p.part_o + (at + row) * HD + col;
#pragma unroll
                    for (int i = 0; i < HD / 8; i += 4)
                        *reinterpret_cast<float4*>(dst + i) = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
                });
            }
            fresh = false;
        }
        next(now);
        if (ends && j + 1 < n) {
            begun = 0;
            open(j + 1);
        }
    }
}

// The rows of the items that several warps shared, from their partials; rows without an item are zeros.  One warp per (row,
// head), or (kCoop) a block of eight.
template <int HD, int kMaxRows, bool kCoop>
__global__ void __launch_bounds__(kCoop ? 256 : 128) paged_list_combine_kernel(const Params p) {
    pdl_trigger();
    __shared__ float4 sums[8][32];
    __shared__ float2 tops[8];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int id = kCoop ? (int)blockIdx.x : (int)blockIdx.x * 4 + warp;
    if (id >= p.total_q * p.heads) return;
    const int row = id / p.heads, head = id - row * p.heads;
    pdl_wait();
    int b = row;
    if (p.cu) {
        if (row < __ldg(p.cu) || row >= __ldg(p.cu + p.batch)) return;
        int lo = 0, hi = p.batch;  // the first sequence that ends behind the row
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (__ldg(p.cu + mid + 1) > row) hi = mid;
            else lo = mid + 1;
        }
        b = lo;
    }
    const Seq s = seq_at(p, kMaxRows, b);
    const int kvh = head / p.group;
    const int64_t f = (int64_t)(row - s.row0) * p.group + head - kvh * p.group;  // (token, grouped head) in order
    const int64_t tile = f / kMaxRows;
    __half* dst = p.out + (int64_t)row * p.ldo + (int64_t)head * p.head_dim + lane * 4;
    const bool act = lane * 4 < p.head_dim;
    if (s.items == 0 || tile >= s.tiles || row < s.row0) {
        if (act && (!kCoop || warp == 0)) *reinterpret_cast<uint2*>(dst) = make_uint2(0, 0);
        return;
    }
    const int2 at = p.parts[((int64_t)b * p.kv_heads + kvh) * p.tiles + tile];
    const int n = at.y;
    if (n == 1) return;  // one warp had it whole
    if (at.x < 0 || at.x >= p.slots || n < 1 || n > (p.slots - (at.x & ~1)) / 2) {  // never written: that warp gave up on a wait
        if (act && (!kCoop || warp == 0)) *reinterpret_cast<uint2*>(dst) = make_uint2(0x7fff7fffu, 0x7fff7fffu);  // NaN
        return;
    }
    const int r = (int)(f - tile * kMaxRows);  // row of the tile
    // the first part's warp had other items ahead of this one or not; of the others it is the first
    auto slot = [&](int i) { return (int64_t)(i ? (at.x & ~1) + 2 * i : at.x) * kMaxRows + r; };
    float m = -INFINITY, acc[4] = {0.0f, 0.0f, 0.0f, 0.0f}, sum = 0.0f;
    bool any = false;  // a part with a key
    constexpr int kStride = kCoop ? 8 : 1;
    for (int i0 = kCoop ? warp : 0; i0 < n; i0 += 8 * kStride) {  // eight loads in flight
        float4 v[8];
        float2 ml[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int k = i0 + i * kStride;
            ml[i] = make_float2(-INFINITY, 0.0f);
            v[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (k < n) {
                ml[i] = p.part_ml[slot(k)];
                if (act) v[i] = *reinterpret_cast<const float4*>(p.part_o + slot(k) * HD + lane * 4);
            }
        }
        float mm = m;
#pragma unroll
        for (int i = 0; i < 8; ++i) mm = fmaxf(mm, ml[i].x);
        const float ref = mm == -INFINITY ? 0.0f : mm, f0 = ex2_approx(m - ref);
        m = mm;
        sum *= f0;
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[e] *= f0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            // A part without a finite score weighs nothing beside others, but its sum counts where it is NaN (0 * NaN).
            // O is finite unless the sum is NaN.
            if (ml[i].y == 0.0f) continue;  // no key
            any = true;
            const float f = ex2_approx(ml[i].x - ref);
            sum += f * ml[i].y;
            acc[0] += f * v[i].x;
            acc[1] += f * v[i].y;
            acc[2] += f * v[i].z;
            acc[3] += f * v[i].w;
        }
    }
    if (kCoop) {
        sums[warp][lane] = make_float4(acc[0], acc[1], acc[2], acc[3]);
        if (lane == 0) tops[warp] = make_float2(m, any && sum == 0.0f ? 1.0f : sum);  // (-inf, 1) as the parts are
        __syncthreads();
        if (warp) return;
        m = -INFINITY;
        for (int i = 0; i < 8; ++i) m = fmaxf(m, tops[i].x);
        const float ref = m == -INFINITY ? 0.0f : m;
        sum = acc[0] = acc[1] = acc[2] = acc[3] = 0.0f;
        for (int i = 0; i < 8; ++i) {
            if (tops[i].y == 0.0f) continue;
            any = true;
            const float f = ex2_approx(tops[i].x - ref);
            const float4 v = sums[i][lane];
            sum += f * tops[i].y;
            acc[0] += f * v.x;
            acc[1] += f * v.y;
            acc[2] += f * v.z;
            acc[3] += f * v.w;
        }
    }
    if (any && m == -INFINITY) sum = NAN;  // keys, but all scores -inf: 0 / 0
    if (!act) return;
    const float inv = 1.0f / sum;
    uint2 o;
    o.x = sum != 0.0f ? h2(acc[0] * inv, acc[1] * inv) : 0u;
    o.y = sum != 0.0f ? h2(acc[2] * inv, acc[3] * inv) : 0u;
    *reinterpret_cast<uint2*>(dst) = o;
}

template <int HD, int kMaxRows>
int launch_list(const Params& p, int ctas, cudaStream_t st) {
    auto kern = paged_list_q8_kernel<HD, kMaxRows>;
    constexpr int kTotal = ListSmem<HD>::kTotal;
    NPUB_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kTotal));
    // Not ahead of the kernel before it ends: CTAs placed around that one's do not come out three on every SM (32 sequences
    // on 65000 keys 126 us so, 96 from an empty GPU).
    kern<<<dim3(ctas), dim3(kWarps * 32), kTotal, st>>>(p);
    const int rc = npub_internal_launch_status();
    if (rc) return rc;
    const int64_t n = (int64_t)p.total_q * p.heads;
    if (n > 0x7fffffff) return NPUB_ERR_UNSUPPORTED;
    // few rows: their items are cut into many parts, and there are warps enough
    if (n <= 4 * num_sms())
        return launch_pdl(paged_list_combine_kernel<HD, kMaxRows, true>, dim3((unsigned)n), dim3(256), 0, st, p);
    return launch_pdl(paged_list_combine_kernel<HD, kMaxRows, false>, dim3((unsigned)((n + 3) / 4)), dim3(128), 0, st, p);
}

// 16 columns of a key per thread and step: the whole numbers as fp16, which holds them exactly, and the scales of every 16
// keys; one block per (key block of 128, kv head, sequence).  Bound: HBM, mostly the writes (36000 keys of 8 heads of 128,
// 74 MB to 147 MB: 41 us, 5.4 TB/s).
__global__ void __launch_bounds__(256) expand_q8_kernel(const int8_t* __restrict__ kp, const int8_t* __restrict__ vp,
                                                        const float* __restrict__ ks, const float* __restrict__ vs,
                                                        const int32_t* __restrict__ table, int64_t ldt, int n_pages,
                                                        int page_shift, int max_keys, const int32_t* __restrict__ lens,
                                                        int kv_heads, int head_dim, int width, __half* __restrict__ k_out,
                                                        __half* __restrict__ v_out, int32_t* __restrict__ table_out,
                                                        int32_t* __restrict__ lens_out, float c,
                                                        float2* __restrict__ key_scale) {
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
    if (threadIdx.x < 8 && n > 0) {  // of keys behind the last one too: they weigh nothing times this
        const int key = w * 128 + (int)threadIdx.x * 16;
        const int id = key < len ? __ldg(table + (int64_t)b * ldt + (key >> page_shift)) : -1;
        const bool in = id >= 0 && id < n_pages;
        const float sk = in ? __ldg(ks + (int64_t)id * kv_heads + kvh) : 0.0f;
        const float sv = in ? __ldg(vs + (int64_t)id * kv_heads + kvh) : 0.0f;
        // log2 s_v is an addend of the exponents: within [-60, 60], below which a V is zero in fp16 and above which infinite
        const float e = fminf(fmaxf(log2f(sv), -60.0f), 60.0f);
        const int64_t g = ((int64_t)b * kv_heads + kvh) * width * 8 + w * 8 + threadIdx.x;
        // a scale that is not finite: NaN scores, which a mask replaces, and a finite addend, which it leaves in the sum
        key_scale[g] = isfinite(sk) && isfinite(sv) ? make_float2(c * sk, sv > 0.0f ? e : -60.0f) : make_float2(NAN, 0.0f);
    }
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
            const uint4 r = *reinterpret_cast<const uint4*>(
                (v ? vp : kp) + ((at << page_shift) + (key & ((1 << page_shift) - 1))) * head_dim + col);
            const uint32_t x[4] = {r.x, r.y, r.z, r.w};
            uint32_t* y = reinterpret_cast<uint32_t*>(o);
            if (!v || !(__ldg(vs + at) < 0x1p-60f)) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    y[2 * e] = h2((float)(int8_t)x[e], (float)(int8_t)(x[e] >> 8));
                    y[2 * e + 1] = h2((float)(int8_t)(x[e] >> 16), (float)(int8_t)(x[e] >> 24));
                }
            }
        }
        uint4* dst = reinterpret_cast<uint4*>((v ? v_out : k_out) + to + (int64_t)row * head_dim + col);
        dst[0] = o[0];
        dst[1] = o[1];
    }
}

}  // namespace pdq8

namespace pdq8 {
int fill(Params& p, const PackedArgs& a, const float* k_scales, const float* v_scales, int tiles, int keys) {
    memset(&p, 0, sizeof(p));
    p.box_rows = a.kv.page_size < keys ? a.kv.page_size : keys;
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
    p.cluster = a.splits > 1;
    p.c = a.scale * 1.4426950408889634f;
    p.out = reinterpret_cast<__half*>(a.out);
    p.ldo = a.ldo;
    p.batch = a.batch;
    p.tiles = tiles;
    p.err = npub_internal_device_error_word();
    return NPUB_OK;
}
size_t up256(size_t n) { return (n + 255) / 256 * 256; }
}  // namespace pdq8

int paged_decode_q8(const PackedArgs& a, const float* k_scales, const float* v_scales, int rows, int tiles,
                    cudaStream_t st) {
    using namespace pdq8;
    Params p;
    const int rc = fill(p, a, k_scales, v_scales, tiles, kKeys);
    if (rc) return rc;
    const bool small = a.head_dim <= 64;
    if (rows <= 8) return small ? launch<64, 8>(p, a.batch, tiles, st) : launch<128, 8>(p, a.batch, tiles, st);
    return small ? launch<64, 16>(p, a.batch, tiles, st) : launch<128, 16>(p, a.batch, tiles, st);
}

size_t paged_list_q8_workspace(int batch, int kv_heads, int head_dim, int rows, int tiles) {
    using namespace pdq8;
    const size_t n = (size_t)2 * kListCtas * num_sms() * kWarps * rows;
    return up256(n * (head_dim <= 64 ? 64 : 128) * sizeof(float)) + up256(n * sizeof(float2)) +
           up256((size_t)batch * kv_heads * tiles * sizeof(int2));
}

int paged_list_q8(const PackedArgs& a, const float* k_scales, const float* v_scales, int rows, int tiles, void* workspace,
                  cudaStream_t st) {
    using namespace pdq8;
    Params p;
    const int rc = fill(p, a, k_scales, v_scales, tiles, kStep);
    if (rc) return rc;
    const int ctas = kListCtas * num_sms();
    const size_t n = (size_t)2 * ctas * kWarps * rows;
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    p.part_o = reinterpret_cast<float*>(ws);
    ws += up256(n * (a.head_dim <= 64 ? 64 : 128) * sizeof(float));
    p.part_ml = reinterpret_cast<float2*>(ws);
    p.parts = reinterpret_cast<int2*>(ws + up256(n * sizeof(float2)));
    p.slots = 2 * ctas * kWarps;
    const bool small = a.head_dim <= 64;
    if (rows <= 8) return small ? launch_list<64, 8>(p, ctas, st) : launch_list<128, 8>(p, ctas, st);
    return small ? launch_list<64, 16>(p, ctas, st) : launch_list<128, 16>(p, ctas, st);
}

int expand_q8(const PackedArgs& a, const float* k_scales, const float* v_scales, int width, void* k_out, void* v_out,
              int32_t* table_out, int32_t* lens_out, float2* key_scale, cudaStream_t st) {
    int shift = 0;
    while ((1 << shift) < a.kv.page_size) ++shift;
    const int64_t mk = (int64_t)a.kv.max_pages << shift;
    return launch_pdl(pdq8::expand_q8_kernel, dim3(width, a.kv_heads, a.batch), dim3(256), 0, st,
                      reinterpret_cast<const int8_t*>(a.kv.k), reinterpret_cast<const int8_t*>(a.kv.v), k_scales, v_scales,
                      a.kv.table, a.kv.ldt, a.kv.n_pages, shift, (int)(mk > 0x7ff00000 ? 0x7ff00000 : mk), a.lens,
                      a.kv_heads, a.head_dim, width, reinterpret_cast<__half*>(k_out), reinterpret_cast<__half*>(v_out),
                      table_out, lens_out, a.scale * 1.4426950408889634f, key_scale);
}

}  // namespace npub
