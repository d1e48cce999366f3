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
#include "gemm_tc.h"

namespace npub {
namespace {

constexpr int kAppThreads = 256;
constexpr int kMaxHalf = 256;  // rot_dim / 2

struct AppendArgs {
    const __half* x;
    int64_t ldx;
    __half* q;
    int64_t ldq;
    int tokens, hq, hk, hd, half, interleaved;
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

__device__ __forceinline__ void unpack8f(const uint4& r, float* f) {
    const __half2* h = reinterpret_cast<const __half2*>(&r);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 t = __half22float2(h[i]);
        f[2 * i] = t.x;
        f[2 * i + 1] = t.y;
    }
}

__device__ __forceinline__ uint4 pack8h(const float* f) {
    uint4 r;
    __half2* h = reinterpret_cast<__half2*>(&r);
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
    return r;
}

// The sequence of packed row t (cu[seq] <= t < cu[seq + 1], empty sequences
// skipped), or -1 for a row outside [cu[0], cu[batch]).  A whole warp, 32
// sequence ends per step.
__device__ __forceinline__ int seq_of_row(const int32_t* __restrict__ cu, int batch, int t) {
    const int lane = threadIdx.x & 31;
    if (t < __ldg(cu)) return -1;
    for (int b0 = 0; b0 < batch; b0 += 32) {
        const int b = b0 + lane;
        const bool after = b < batch && __ldg(cu + b + 1) > t;
        const uint32_t vote = __ballot_sync(0xffffffffu, after);
        if (vote) return b0 + __ffs(vote) - 1;
    }
    return -1;
}

__global__ void __launch_bounds__(kAppThreads) rope_paged_append_kernel(const AppendArgs a) {
    pdl_trigger();
    __shared__ float cs[kMaxHalf], sn[kMaxHalf];
    pdl_wait();
    const int t = blockIdx.x;
    int seq = t;
    if (a.cu) {
        seq = seq_of_row(a.cu, a.batch, t);
        if (seq < 0) return;  // block-uniform: a row of no sequence stays as it is
    }
    const int p = a.pos[t];
    for (int i = threadIdx.x; i < a.half; i += kAppThreads) {
        const double turns = (double)p * (double)a.inv_freq[i] * 0.15915494309189535;  // 1 / (2 pi)
        float s, c;
        sincospif((float)(2.0 * (turns - rint(turns))), &s, &c);
        cs[i] = c;
        sn[i] = s;
    }
    int page = -1;  // a position outside the table, or a page outside the pool, is not stored
    if (p >= 0 && (p >> a.page_shift) < a.max_pages) {
        const int id = a.table[(int64_t)seq * a.ldt + (p >> a.page_shift)];
        if (id >= 0 && id < a.n_pages) page = id;
    }
    __syncthreads();
    const int slot = p & ((1 << a.page_shift) - 1);
    const __half* row = a.x + (int64_t)t * a.ldx;
    const int heads = a.hq + 2 * a.hk;
    const int total = ((heads << a.units_log2) + 31) & ~31;  // whole warps: the norm's shuffles
    const int rot_units = a.half >> 3;
    const bool any_norm = a.gq || a.gk;
    for (int i = blockIdx.y * kAppThreads + threadIdx.x; i < total; i += gridDim.y * kAppThreads) {
        const int h = i >> a.units_log2, u = i & (a.units_p2 - 1);
        const bool act = h < heads && u < a.units;
        const bool isq = h < a.hq, isv = h >= a.hq + a.hk;
        // the unit's two 8-element chunks: the two halves of a rotated pair, else neighbours
        const bool split = !a.interleaved && u < rot_units;
        const int c0 = split ? u * 8 : u * 16;
        const int c1 = split ? c0 + a.half : c0 + 8;
        uint4 r0 = make_uint4(0, 0, 0, 0), r1 = r0;
        if (act) {
            r0 = *reinterpret_cast<const uint4*>(row + (int64_t)h * a.hd + c0);
            r1 = *reinterpret_cast<const uint4*>(row + (int64_t)h * a.hd + c1);
        }
        float x0[8], x1[8];
        unpack8f(r0, x0);
        unpack8f(r1, x1);
        const __half* g = isv ? nullptr : isq ? a.gq : a.gk;
        if (any_norm) {
            float ss = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; ++e) ss += x0[e] * x0[e] + x1[e] * x1[e];
            for (int m = a.units_p2 >> 1; m > 0; m >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, m);
            if (g && act) {
                const float inv = 1.0f / sqrtf(ss * a.inv_hd + a.eps);
                float g0[8], g1[8];
                unpack8f(__ldg(reinterpret_cast<const uint4*>(g + c0)), g0);
                unpack8f(__ldg(reinterpret_cast<const uint4*>(g + c1)), g1);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    x0[e] *= inv * g0[e];
                    x1[e] *= inv * g1[e];
                }
            }
        }
        if (!act) continue;
        if (!isv && u < rot_units) {
            if (split) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float c = cs[c0 + e], s = sn[c0 + e], v0 = x0[e], v1 = x1[e];
                    x0[e] = v0 * c - v1 * s;
                    x1[e] = v1 * c + v0 * s;
                }
            } else {
#pragma unroll
                for (int e = 0; e < 8; e += 2) {
                    const int f0 = u * 8 + (e >> 1), f1 = f0 + 4;
                    const float a0 = x0[e], b0 = x0[e + 1], a1 = x1[e], b1 = x1[e + 1];
                    x0[e] = a0 * cs[f0] - b0 * sn[f0];
                    x0[e + 1] = b0 * cs[f0] + a0 * sn[f0];
                    x1[e] = a1 * cs[f1] - b1 * sn[f1];
                    x1[e + 1] = b1 * cs[f1] + a1 * sn[f1];
                }
            }
        }
        __half* dst;
        if (isq) {
            dst = a.q + (int64_t)t * a.ldq + (int64_t)h * a.hd;
        } else {
            if (page < 0) continue;
            const int kvh = isv ? h - a.hq - a.hk : h - a.hq;
            dst = (isv ? a.vp : a.kp) + ((((int64_t)page * a.hk + kvh) << a.page_shift) + slot) * a.hd;
        }
        *reinterpret_cast<uint4*>(dst + c0) = pack8h(x0);
        *reinterpret_cast<uint4*>(dst + c1) = pack8h(x1);
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
    a.tokens = tokens;
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
    const int total = (q_heads + 2 * kv_heads) << a.units_log2;
    int groups = 1;  // blocks per token: one while the tokens alone fill the GPU
    if (tokens < 2 * num_sms()) groups = (total + kAppThreads - 1) / kAppThreads;
    return launch_pdl(rope_paged_append_kernel, dim3(tokens, groups), dim3(kAppThreads), 0,
                      reinterpret_cast<cudaStream_t>(stream), a);
}
