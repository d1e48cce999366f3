// RoPE, per-head RMSNorm and the append to a paged KV cache in one pass over
// the fused QKV rows (decode steps and packed prompts).
//
// Per token t with position p and head x = qkv[t, h]:
//   q and k heads:  x_i <- x_i * gamma_i / sqrt(mean(x^2) + eps)   (when gamma is given)
//                   (a, b) <- (a cos - b sin, b cos + a sin) with angle p * inv_freq[i] for
//                   the R/2 pairs (i, i + R/2), or (2i, 2i + 1) when interleaved;
//                   columns past R pass through
//   q -> q_out[t, h], k and v -> pages[table[seq(t), p / ps], h, p % ps, :]
// All of it in fp32 with one rounding to fp16 at the store.  The rotation is
// the rope_Q / rope_Kt macros of b_program_examples/llama_layer.py:96-112; the
// reference has no cache and no per-head norm.
//
// The angle: at position 100000 an fp32 product p * f is off by up to 4e-3
// rad, more than a fp16 step of the result, so the product and its reduction
// to one turn are in fp64 (R/2 of them per token, shared by all heads) and
// only the remainder in [-1/2, 1/2) turns goes to sincospif.
//
// Bound: HBM, every row read and written once.
#include "common.cuh"
#include "f32x2.cuh"
#include "gemm_tc.h"

namespace npub {
namespace {

constexpr int kAppThreads = 128;
constexpr int kMaxHalf = 256;  // rot_dim / 2

struct AppendArgs {
    const __half* x;
    int64_t ldx;
    __half* q;
    int64_t ldq;
    int hq, hk, hd, half, interleaved;
    int units, units_p2, units_log2;  // 16-element units per head, padded to a power of two
    const int32_t* pos;
    const float* inv_freq;
    const __half *gq, *gk;
    float eps, inv_hd;
    __half *kp, *vp;
    int n_pages, page_shift;
    const int32_t* table;
    int64_t ldt;
    int max_pages;
    const int32_t* cu;
    int batch;
};

// Eight fp16 as four pairs of fp32, and back.
__device__ __forceinline__ void unpack8(const uint4& r, uint64_t (&f)[4]) {
    const __half2* h = reinterpret_cast<const __half2*>(&r);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 t = __half22float2(h[i]);
        f[i] = pack2(t.x, t.y);
    }
}

__device__ __forceinline__ uint4 pack8(const uint64_t (&f)[4]) {
    uint4 r;
    __half2* h = reinterpret_cast<__half2*>(&r);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float a, b;
        unpack2(f[i], a, b);
        h[i] = __floats2half2_rn(a, b);
    }
    return r;
}

// The sequence of packed row t (cu[seq] <= t < cu[seq + 1], empty sequences
// skipped), or -1 for a row outside [cu[0], cu[batch]).  A whole warp: each
// step looks at the ends of 32 parts of the sequences left, the last at 32
// sequences (32 / 8 heads of 128: 20000 sequences of one row 654 -> 87 us, 1000
// of 20 rows 94 -> 84, against a pass over all sequences).
__device__ __forceinline__ int seq_of_row(const int32_t* __restrict__ cu, int batch, int t) {
    const int lane = threadIdx.x & 31;
    if (t < __ldg(cu)) return -1;
    int b0 = 0, n = batch;  // the first sequence that ends behind t is one of b0 .. b0 + n - 1, or none
    while (n > 32) {
        const int step = (n + 31) >> 5;
        const uint32_t vote = __ballot_sync(0xffffffffu, __ldg(cu + b0 + min(n, (lane + 1) * step)) > t);
        if (!vote) return -1;
        const int skip = (__ffs(vote) - 1) * step;
        b0 += skip;
        n = min(step, n - skip);
    }
    const uint32_t vote = __ballot_sync(0xffffffffu, lane < n && __ldg(cu + b0 + min(n, lane + 1)) > t);
    return vote ? b0 + __ffs(vote) - 1 : -1;
}

// Block (x, y): token x, and of its 16-element units every gridDim.y-th run of
// kAppThreads, one unit per thread and step.  A thread loads its first unit
// before the block forms the angles and looks up the page.
//
// Measured at 8192 packed tokens of 32 / 8 heads of 128 with norms (201 MB):
// 38 us with 128 threads, 5.3 TB/s or 0.81 of the copy rate (when it was chosen 37.2; 39.3 and 41.9
// with the heads of a token over two and three blocks); 43 with 96 or
// 192 threads, 39.6 and 45 with two and four tokens per block, 46-48 with two
// or three units in flight per thread (their registers cost more warps than
// they bring loads), 51 with the arithmetic one element at a time: the
// instructions, not the loads, are what competes with HBM here, so it runs on
// pairs (f32x2) and v heads are copied.
__global__ void __launch_bounds__(kAppThreads) rope_paged_append_kernel(const AppendArgs a) {
    pdl_trigger();
    // {cos, cos', sin, sin'} of the pairs 8 u + 2 e and 8 u + 2 e + 1 at [e][u]: the lanes of a head (u = 0, 1, ...)
    // read neighbouring words
    __shared__ float4 turn[kMaxHalf / 2];
    __shared__ int page_of, slot_of;
    pdl_wait();
    const int t = blockIdx.x;
    const int heads = a.hq + 2 * a.hk;
    const int total = ((heads << a.units_log2) + 31) & ~31;  // units of a token, whole warps (the norm's shuffles)
    const int rot_units = a.half >> 3;
    const bool any_norm = a.gq || a.gk;
    bool first = true;
    for (int base = blockIdx.y * kAppThreads; base < total; base += gridDim.y * kAppThreads) {
        const int i = base + threadIdx.x;
        const int h = i >> a.units_log2, u = i & (a.units_p2 - 1);
        const bool act = h < heads && u < a.units;
        // the unit's two 8-element chunks: the two halves of a rotated pair, else neighbours
        const bool split = !a.interleaved && u < rot_units;
        const int c0 = split ? u * 8 : u * 16, c1 = split ? c0 + a.half : c0 + 8;
        uint4 o0 = make_uint4(0, 0, 0, 0), o1 = o0;
        if (act) {
            const __half* x = a.x + (int64_t)t * a.ldx + (int64_t)h * a.hd;
            o0 = *reinterpret_cast<const uint4*>(x + c0);
            o1 = *reinterpret_cast<const uint4*>(x + c1);
        }
        if (first) {
            first = false;
            const int p = a.pos[t];
            for (int k = threadIdx.x; k < a.half; k += kAppThreads) {
                const double turns = (double)p * (double)a.inv_freq[k] * 0.15915494309189535;  // 1 / (2 pi)
                float s, c;
                sincospif((float)(2.0 * (turns - rint(turns))), &s, &c);
                float* w = reinterpret_cast<float*>(&turn[((k & 7) >> 1) * rot_units + (k >> 3)]) + (k & 1);
                w[0] = c;
                w[2] = s;
            }
            if ((threadIdx.x >> 5) == kAppThreads / 32 - 1) {  // the last warp has the fewest angles
                const int seq = a.cu ? seq_of_row(a.cu, a.batch, t) : t;
                // a position outside the table, or a page outside the pool, is not stored (-1); a row of no sequence
                // stays as it is (-2)
                int page = seq < 0 ? -2 : -1;
                if (seq >= 0 && p >= 0 && (p >> a.page_shift) < a.max_pages) {
                    const int id = a.table[(int64_t)seq * a.ldt + (p >> a.page_shift)];
                    if (id >= 0 && id < a.n_pages) page = id;
                }
                if ((threadIdx.x & 31) == 0) {
                    page_of = page;
                    slot_of = p & ((1 << a.page_shift) - 1);
                }
            }
            __syncthreads();
        }
        const bool isq = h < a.hq, isv = h >= a.hq + a.hk;
        const int page = page_of;
        const __half* g = isv ? nullptr : isq ? a.gq : a.gk;
        const bool turns = !isv && u < rot_units;
        if (__any_sync(0xffffffffu, turns || g)) {  // a warp of v heads copies
            uint64_t x0[4], x1[4];
            unpack8(o0, x0);
            unpack8(o1, x1);
            if (any_norm) {
                uint64_t s2 = 0;
#pragma unroll
                for (int e = 0; e < 4; ++e) s2 = fma2(x1[e], x1[e], fma2(x0[e], x0[e], s2));
                float ss, sb;
                unpack2(s2, ss, sb);
                ss += sb;
                for (int m = a.units_p2 >> 1; m > 0; m >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, m);
                if (g && act) {
                    const float inv = rsqrtf(ss * a.inv_hd + a.eps);
                    const uint64_t inv2 = pack2(inv, inv);
                    uint64_t g0[4], g1[4];
                    unpack8(__ldg(reinterpret_cast<const uint4*>(g + c0)), g0);
                    unpack8(__ldg(reinterpret_cast<const uint4*>(g + c1)), g1);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        x0[e] = mul2(x0[e], mul2(inv2, g0[e]));
                        x1[e] = mul2(x1[e], mul2(inv2, g1[e]));
                    }
                }
            }
            if (turns) {
                const float4* cs = &turn[u];
                if (split) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float4 w = cs[e * rot_units];
                        const uint64_t c = pack2(w.x, w.y), s = pack2(w.z, w.w), ns = pack2(-w.z, -w.w);
                        const uint64_t v0 = x0[e], v1 = x1[e];
                        x0[e] = fma2(v0, c, mul2(v1, ns));
                        x1[e] = fma2(v1, c, mul2(v0, s));
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float4 w = cs[(e >> 1) * rot_units], v = cs[((e >> 1) + 2) * rot_units];
                        const float c0 = (e & 1) ? w.y : w.x, s0 = (e & 1) ? w.w : w.z;
                        const float c1 = (e & 1) ? v.y : v.x, s1 = (e & 1) ? v.w : v.z;
                        float p, q;
                        unpack2(x0[e], p, q);
                        x0[e] = pack2(p * c0 - q * s0, q * c0 + p * s0);
                        unpack2(x1[e], p, q);
                        x1[e] = pack2(p * c1 - q * s1, q * c1 + p * s1);
                    }
                }
            }
            if (!isv) {
                o0 = pack8(x0);
                o1 = pack8(x1);
            }
        }
        if (!act || page == -2) continue;
        __half* dst;
        if (isq) {
            dst = a.q + (int64_t)t * a.ldq + (int64_t)h * a.hd;
        } else {
            if (page < 0) continue;
            const int kvh = isv ? h - a.hq - a.hk : h - a.hq;
            dst = (isv ? a.vp : a.kp) + ((((int64_t)page * a.hk + kvh) << a.page_shift) + slot_of) * a.hd;
        }
        *reinterpret_cast<uint4*>(dst + c0) = o0;
        *reinterpret_cast<uint4*>(dst + c1) = o1;
    }
}

}  // namespace
}  // namespace npub

extern "C" int npub_rope_paged_append(const void* qkv, int64_t ldx, void* q_out, int64_t ldq, int tokens, int q_heads,
                                      int kv_heads, int head_dim, int rot_dim, int interleaved,
                                      const int32_t* positions, const float* inv_freq, const void* q_gamma,
                                      const void* k_gamma, float eps, void* k_pages, void* v_pages, int n_pages,
                                      int page_size, const int32_t* page_table, int64_t ldt, int max_pages,
                                      const int32_t* cu_seqlens, int batch, void* stream) {
    using namespace npub;
    NPUB_CHECK_ARG(tokens >= 0 && batch >= 0 && q_heads > 0 && kv_heads > 0 && q_heads + 2 * (int64_t)kv_heads <= 65536);
    if (tokens == 0) return NPUB_OK;
    NPUB_CHECK_ARG(qkv && q_out && positions && inv_freq && k_pages && v_pages && page_table);
    NPUB_CHECK_ARG(head_dim % 16 == 0 && head_dim > 0 && head_dim <= 512);
    NPUB_CHECK_ARG(rot_dim % 16 == 0 && rot_dim > 0 && rot_dim <= head_dim);
    NPUB_CHECK_ARG(ldx % 8 == 0 && ldq % 8 == 0 && ldx >= (int64_t)(q_heads + 2 * kv_heads) * head_dim &&
                   ldq >= (int64_t)q_heads * head_dim);
    NPUB_CHECK_ARG(npub_aligned(qkv, 16) && npub_aligned(q_out, 16) && npub_aligned(k_pages, 16) &&
                   npub_aligned(v_pages, 16) && npub_aligned(q_gamma, 16) && npub_aligned(k_gamma, 16));
    NPUB_CHECK_ARG(page_size >= 1 && page_size <= 65536 && (page_size & (page_size - 1)) == 0 && n_pages > 0);
    NPUB_CHECK_ARG(max_pages > 0 && ldt >= max_pages);
    NPUB_CHECK_ARG(cu_seqlens ? batch > 0 : batch == tokens);
    AppendArgs a;
    a.x = reinterpret_cast<const __half*>(qkv);
    a.ldx = ldx;
    a.q = reinterpret_cast<__half*>(q_out);
    a.ldq = ldq;
    a.hq = q_heads;
    a.hk = kv_heads;
    a.hd = head_dim;
    a.half = rot_dim / 2;
    a.interleaved = interleaved ? 1 : 0;
    a.units = head_dim / 16;
    a.units_log2 = 0;
    while ((1 << a.units_log2) < a.units) ++a.units_log2;
    a.units_p2 = 1 << a.units_log2;
    a.pos = positions;
    a.inv_freq = inv_freq;
    a.gq = reinterpret_cast<const __half*>(q_gamma);
    a.gk = reinterpret_cast<const __half*>(k_gamma);
    a.eps = eps;
    a.inv_hd = 1.0f / (float)head_dim;
    a.kp = reinterpret_cast<__half*>(k_pages);
    a.vp = reinterpret_cast<__half*>(v_pages);
    a.n_pages = n_pages;
    a.page_shift = 0;
    while ((1 << a.page_shift) < page_size) ++a.page_shift;
    a.table = page_table;
    a.ldt = ldt;
    a.max_pages = max_pages;
    a.cu = cu_seqlens;
    a.batch = batch;
    const int total = (((q_heads + 2 * kv_heads) << a.units_log2) + 31) & ~31;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    // few tokens: blocks over the heads too, one unit per thread
    const int groups = tokens < 4 * num_sms() ? (total + kAppThreads - 1) / kAppThreads : 1;
    return launch_pdl(rope_paged_append_kernel, dim3(tokens, groups), dim3(kAppThreads), 0, st, a);
}
