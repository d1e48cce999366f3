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
#include "gemm_tc.h"
#include "paged_append.cuh"

namespace npub {
namespace {

// Block (x, y): token x, part y of gridDim.y of its heads.
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
    pdl_wait();
    append_token(a, blockIdx.x, blockIdx.y, gridDim.y);
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
    a.turns = nullptr;
    const int total = (((q_heads + 2 * kv_heads) << a.units_log2) + 31) & ~31;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    // few tokens: blocks over the heads too, one unit per thread
    const int groups = tokens < 4 * num_sms() ? (total + kAppThreads - 1) / kAppThreads : 1;
    return launch_pdl(rope_paged_append_kernel, dim3(tokens, groups), dim3(kAppThreads), 0, st, a);
}
