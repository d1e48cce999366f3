// RoPE, per-head RMSNorm and the append to a paged KV cache held in 8 bits,
// with one scale for each page and kv head.
//
// The rows' arithmetic is paged_append.cu's in fp32; q is rounded to fp16, k
// and v go to int8 unrounded:
//   s' = max(s, max|new rows of the page| / 127)   (s = 0 where they start at the page's first slot)
//   new rows  q = rint(y / s'), half a step of s' off at most
//   where s' > s, the rows ahead of them in the page: q <- rint(q s / s'), another half step
// A page's scale only grows (a record of the maxima: of n like rows the n-th
// raises it with probability 1/n, so a page is rewritten about ln(page_size)
// times in its life), and it starts anew with the page.  A value that is not
// finite makes its page's scale, and so all that is read from that page and
// head, NaN.
//
// The rows of a sequence are stored from positions[its first row] on, one slot
// after the other, so that the rows that meet in a page are known from the
// offsets alone: one block (packed rows) or one warp (decode steps) takes a
// page's new rows of one head, finds their maximum, and stores.
//
// Bound: the launch and a few memory latencies for a decode step (250 rows of 32 /
// 8 heads of 128: 5.5 us).  For prompts HBM (the qkv rows read, q and the 8-bit
// rows written) is the floor, 14 us for 4096 rows of those heads with norms; they
// take 34, the query heads' launch about 14 at half of the issue slots, the
// pages' the rest, on 16 warps an SM (a thread holds 64 values) that look for
// their pages again, which the query heads' launch has done for every token.  8192
// rows: 54 us.  The fp16 append (paged_append.cu), one launch, takes 22.5 and 40.
//
// A prompt's q rows are normalised with rsqrtf and sums of pairs (paged_append.cuh),
// a decode step's with 1 / sqrtf: the same row can differ in its last bit.
#include "gemm_tc.h"
#include "paged_append.cuh"

namespace npub {
namespace {

struct Q8Args {
    AppendArgs q;  // the query heads (hk = 0 there), and what both sides use
    int hk, rows;
    int8_t *kp, *vp;
    float *ks, *vs;
    int window, windows;  // packed: rows of a window, windows of the call
};

// The columns that a lane holds of a head, two pairs: (ca, ca + 1) and (cb, cb + 1).
struct Cols {
    int ca, cb, pair;  // pair: first of its two angles, -1 where it has none
    bool on;
};
__device__ __forceinline__ Cols lane_cols(const AppendArgs& a, bool turns) {
    const int u = 2 * (threadIdx.x & 31);
    Cols c;
    c.on = u < a.hd / 2;
    const bool rot = turns && u < a.half;
    const bool split = rot && !a.interleaved;
    c.ca = split ? u : 2 * u;
    c.cb = split ? u + a.half : 2 * u + 2;
    c.pair = rot ? u : -1;
    return c;
}

__device__ __forceinline__ void angle(const AppendArgs& a, int p, int k, float& c, float& s) {
    const double turns = (double)p * (double)__ldg(a.inv_freq + k) * 0.15915494309189535;  // 1 / (2 pi)
    sincospif((float)(2.0 * (turns - rint(turns))), &s, &c);
}

__device__ __forceinline__ void turn(float& a, float& b, float c, float s) {
    const float x = a;
    a = x * c - b * s;
    b = b * c + x * s;
}

// Row t's head (its first column x), by a warp: normalised by g, rotated by the angles of position p.
__device__ __forceinline__ void head_row(const AppendArgs& a, const __half* x, const Cols& c, const __half* g, int p,
                                         float (&y)[4]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = 0.0f;
    if (c.on) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(x + c.ca));
        const float2 h = __half22float2(*reinterpret_cast<const __half2*>(x + c.cb));
        y[0] = f.x;
        y[1] = f.y;
        y[2] = h.x;
        y[3] = h.y;
    }
    if (g) {
        float ss = y[0] * y[0] + y[1] * y[1] + y[2] * y[2] + y[3] * y[3];
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, d);
        const float inv = 1.0f / sqrtf(ss * a.inv_hd + a.eps);
        if (c.on) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(g + c.ca));
            const float2 h = __half22float2(*reinterpret_cast<const __half2*>(g + c.cb));
            y[0] *= inv * f.x;
            y[1] *= inv * f.y;
            y[2] *= inv * h.x;
            y[3] *= inv * h.y;
        }
    }
    if (c.on && c.pair >= 0) {
        float c0, s0, c1, s1;
        angle(a, p, c.pair, c0, s0);
        angle(a, p, c.pair + 1, c1, s1);
        if (a.interleaved) {
            turn(y[0], y[1], c0, s0);
            turn(y[2], y[3], c1, s1);
        } else {
            turn(y[0], y[2], c0, s0);
            turn(y[1], y[3], c1, s1);
        }
    }
}

__device__ __forceinline__ uint32_t max_bits(const float (&y)[4]) {  // as integers NaN is above infinity
    uint32_t m = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) m = max(m, __float_as_uint(y[e]) & 0x7fffffffu);
    return m;
}

// The page's scale behind rows of the largest magnitude `top` (bits), its reciprocal (0 where all is 0), and what the rows
// ahead of them are multiplied with (1: left).
struct Step {
    float scale, inv, old;
};
__device__ __forceinline__ Step step_of(float before, uint32_t top) {
    Step s;
    const float most = __uint_as_float(top);
    s.scale = fmaxf(before, most / 127.0f);
    if (top >= 0x7f800000u || !(before <= 3.4e38f)) s.scale = NAN;
    s.inv = s.scale > 1e-37f ? 1.0f / s.scale : 0.0f;
    s.old = s.scale > before && s.scale > 1e-37f ? before / s.scale : 1.0f;
    return s;
}
// round(y / s') in the low byte: |y / s'| is at most 127 (1 + 2^-22), and adding 1.5 * 2^23 rounds it, halves to even.  The
// quotient y inv is corrected by its remainder: halves are not rare (half of the largest value is 63.5), and with the
// reciprocal's rounding alone they fall to either side (error of a prompt's keys and values against 64 bits a third more).
__device__ __forceinline__ uint32_t q8(float y, const Step& s) {
    const float t = y * s.inv;
    return __float_as_uint(fmaf(fmaf(-t, s.scale, y), s.inv, t) + 12582912.0f);
}
__device__ __forceinline__ uint32_t bytes4(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}
__device__ __forceinline__ uint32_t rescaled(uint32_t w, float f) {
    uint32_t r = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) r |= ((uint32_t)(int)rintf((float)(int8_t)(w >> (8 * e)) * f) & 0xffu) << (8 * e);
    return r;
}

// Where sequence b's key p lives: its page, or -1 outside the table or the pool.
__device__ __forceinline__ int page_at(const AppendArgs& a, int b, int64_t p) {
    if (p < 0 || (p >> a.page_shift) >= a.max_pages) return -1;
    const int id = __ldg(a.table + (int64_t)b * a.ldt + (p >> a.page_shift));
    return id >= 0 && id < a.n_pages ? id : -1;
}

// ------------------------------------------------------------------ decode steps
// One warp per token and head (q, k or v).
constexpr int kDecodeWarps = 4;
__global__ void __launch_bounds__(kDecodeWarps * 32) append_decode_q8_kernel(const Q8Args p) {
    pdl_trigger();
    pdl_wait();
    const AppendArgs& a = p.q;
    const int t = blockIdx.x, lane = threadIdx.x & 31;
    const int h = blockIdx.y * kDecodeWarps + (threadIdx.x >> 5);
    if (h >= a.hq + 2 * p.hk) return;
    const bool isq = h < a.hq, isv = h >= a.hq + p.hk;
    const int pos = __ldg(a.pos + t);
    const Cols c = lane_cols(a, !isv);
    float y[4];
    head_row(a, a.x + (int64_t)t * a.ldx + (int64_t)h * a.hd, c, isv ? nullptr : isq ? a.gq : a.gk, pos, y);
    if (isq) {
        if (c.on) {
            __half* dst = a.q + (int64_t)t * a.ldq + (int64_t)h * a.hd;
            *reinterpret_cast<__half2*>(dst + c.ca) = __floats2half2_rn(y[0], y[1]);
            *reinterpret_cast<__half2*>(dst + c.cb) = __floats2half2_rn(y[2], y[3]);
        }
        return;
    }
    const int page = page_at(a, t, pos);
    if (page < 0) return;
    const int kvh = isv ? h - a.hq - p.hk : h - a.hq, slot = pos & ((1 << a.page_shift) - 1);
    const int64_t at = (int64_t)page * p.hk + kvh;
    float* scale = (isv ? p.vs : p.ks) + at;
    int8_t* rows = (isv ? p.vp : p.kp) + (at << a.page_shift) * a.hd;
    const float before = slot ? *scale : 0.0f;
    const Step s = step_of(before, __reduce_max_sync(0xffffffffu, max_bits(y)));
    if (c.on) {
        int8_t* dst = rows + (int64_t)slot * a.hd;
        const uint32_t w = bytes4(q8(y[0], s), q8(y[1], s), q8(y[2], s), q8(y[3], s));
        *reinterpret_cast<uint16_t*>(dst + c.ca) = (uint16_t)w;
        *reinterpret_cast<uint16_t*>(dst + c.cb) = (uint16_t)(w >> 16);
    }
    if (s.old != 1.0f) {
        uint4* w = reinterpret_cast<uint4*>(rows);
        for (int i = lane; i < slot * a.hd / 16; i += 32) {
            const uint4 v = w[i];
            w[i] = make_uint4(rescaled(v.x, s.old), rescaled(v.y, s.old), rescaled(v.z, s.old), rescaled(v.w, s.old));
        }
    }
    __syncwarp();  // every lane has read the scale
    if (lane == 0) *scale = s.scale;
}

// ------------------------------------------------------------------ packed rows
// One block per token for its query heads, in a launch of their own: they are
// three quarters of the bytes, and need neither the registers nor the shared
// memory of the others.  They leave the angles for the k heads, which would form
// them once for each head and page.
__global__ void __launch_bounds__(kAppThreads) append_query_kernel(const AppendArgs a) {
    pdl_trigger();
    pdl_wait();
    append_token(a, blockIdx.x, 0, 1);
}

// Blocks of (window of p.window packed rows, k or v head): each takes the pages
// whose first new row lies in its window, one after the other.  A thread holds
// one 16-element unit (as in append_token) of up to kUnits rows of the page in
// registers, so that all of a page's loads are in flight at once and its rows
// stay there between the maximum and the store.
constexpr int kUnits = 4;
constexpr int kMaxPackedThreads = 512;  // 256 rows of 8 units
__global__ void __launch_bounds__(kMaxPackedThreads, 1) append_packed_q8_kernel(const Q8Args p) {
    pdl_trigger();
    __shared__ uint32_t part[kMaxPackedThreads / 32];
    pdl_wait();
    const AppendArgs& a = p.q;
    const int heads = 2 * p.hk;
    const int win = (int)blockIdx.x / heads, head = (int)blockIdx.x - win * heads;
    const bool isv = head >= p.hk;
    const int kvh = isv ? head - p.hk : head;
    const int threads = (int)blockDim.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int ps = 1 << a.page_shift;
    // this thread's unit: two 8-element chunks, the halves of a rotated pair or neighbours
    const int u = threadIdx.x & (a.units_p2 - 1), row_of = threadIdx.x >> a.units_log2, stride = threads >> a.units_log2;
    const bool act = u < a.units, turns = !isv && u < a.half >> 3, split = turns && !a.interleaved;
    const int c0 = split ? u * 8 : u * 16, c1 = split ? c0 + a.half : c0 + 8;
    const bool norm = !isv && a.gk;
    const int row_end = min(p.rows, (win + 1) * p.window);
    for (int t0 = win * p.window; t0 < row_end; t0 += 32) {
        // the page that starts with row t0 + lane: its sequence, first slot, rows
        const int t = t0 + lane;
        int page = -1, slot = 0, n = 0;
        if (t < row_end && t >= __ldg(a.cu) && t < __ldg(a.cu + a.batch)) {
            int lo = 0, hi = a.batch;  // the first sequence that ends behind t
            while (lo < hi) {
                const int mid = (lo + hi) >> 1;
                if (__ldg(a.cu + mid + 1) > t) hi = mid;
                else lo = mid + 1;
            }
            const int first = lo < a.batch ? max(0, __ldg(a.cu + lo)) : p.rows;
            if (first <= t) {
                const int64_t at = (int64_t)__ldg(a.pos + first) + (t - first);
                slot = (int)(at & (ps - 1));
                if (slot == 0 || t == first) {
                    page = page_at(a, lo, at);
                    n = min(min(ps - slot, __ldg(a.cu + lo + 1) - t), p.rows - t);
                }
            }
        }
        uint32_t todo = __ballot_sync(0xffffffffu, page >= 0 && n > 0);  // the same in all warps
        while (todo) {
            const int l = __ffs(todo) - 1;
            todo &= todo - 1;
            const int pg = __shfl_sync(0xffffffffu, page, l), sl = __shfl_sync(0xffffffffu, slot, l);
            const int rows = __shfl_sync(0xffffffffu, n, l);
            const int row0 = t0 + l;
            const int64_t at = (int64_t)pg * p.hk + kvh;
            float* scale = (isv ? p.vs : p.ks) + at;
            int8_t* dst = (isv ? p.vp : p.kp) + (at << a.page_shift) * a.hd;
            const float before = sl ? *scale : 0.0f;
            const __half* x = a.x + (int64_t)row0 * a.ldx + (int64_t)(a.hq + head) * a.hd;
            uint4 raw[kUnits][2];
#pragma unroll
            for (int i = 0; i < kUnits; ++i) {
                const int r = row_of + i * stride;
                raw[i][0] = raw[i][1] = make_uint4(0, 0, 0, 0);
                if (act && r < rows) {
                    raw[i][0] = *reinterpret_cast<const uint4*>(x + (int64_t)r * a.ldx + c0);
                    raw[i][1] = *reinterpret_cast<const uint4*>(x + (int64_t)r * a.ldx + c1);
                }
            }
            float y[kUnits][16];
            uint32_t top = 0;
#pragma unroll
            for (int i = 0; i < kUnits; ++i) {
                const int r = row_of + i * stride;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float2 f = __half22float2(reinterpret_cast<const __half2*>(&raw[i][e >> 2])[e & 3]);
                    y[i][2 * e] = f.x;
                    y[i][2 * e + 1] = f.y;
                }
                if (norm) {
                    float ss = 0.0f;
#pragma unroll
                    for (int e = 0; e < 16; ++e) ss = fmaf(y[i][e], y[i][e], ss);
                    for (int m = a.units_p2 >> 1; m > 0; m >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, m);
                    const float inv = 1.0f / sqrtf(ss * a.inv_hd + a.eps);
                    uint4 g[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
                    if (act) {
                        g[0] = __ldg(reinterpret_cast<const uint4*>(a.gk + c0));
                        g[1] = __ldg(reinterpret_cast<const uint4*>(a.gk + c1));
                    }
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const float2 f = __half22float2(reinterpret_cast<const __half2*>(&g[e >> 2])[e & 3]);
                        y[i][2 * e] *= inv * f.x;
                        y[i][2 * e + 1] *= inv * f.y;
                    }
                }
                if (turns && r < rows) {  // pairs (e, e + 8), or (2 e, 2 e + 1), by the angles of the token's pairs 8 u + e
                    const float4* w = reinterpret_cast<const float4*>(a.turns + (int64_t)(row0 + r) * a.half + u * 8);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float4 cs = *(w + e);
                        if (split) {
                            turn(y[i][2 * e], y[i][2 * e + 8], cs.x, cs.y);
                            turn(y[i][2 * e + 1], y[i][2 * e + 9], cs.z, cs.w);
                        } else {
                            turn(y[i][4 * e], y[i][4 * e + 1], cs.x, cs.y);
                            turn(y[i][4 * e + 2], y[i][4 * e + 3], cs.z, cs.w);
                        }
                    }
                }
                if (act && r < rows) {
#pragma unroll
                    for (int e = 0; e < 16; ++e) top = max(top, __float_as_uint(y[i][e]) & 0x7fffffffu);
                }
            }
            top = __reduce_max_sync(0xffffffffu, top);
            if (lane == 0) part[warp] = top;
            __syncthreads();
            for (int w = 0; w < threads >> 5; ++w) top = max(top, part[w]);
            const Step s = step_of(before, top);
#pragma unroll
            for (int i = 0; i < kUnits; ++i) {
                const int r = row_of + i * stride;
                if (!act || r >= rows) continue;
                uint32_t w[4];
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    w[e] = bytes4(q8(y[i][4 * e], s), q8(y[i][4 * e + 1], s), q8(y[i][4 * e + 2], s),
                                  q8(y[i][4 * e + 3], s));
                int8_t* out = dst + (int64_t)(sl + r) * a.hd;
                *reinterpret_cast<uint2*>(out + c0) = make_uint2(w[0], w[1]);
                *reinterpret_cast<uint2*>(out + c1) = make_uint2(w[2], w[3]);
            }
            if (s.old != 1.0f) {
                uint4* old = reinterpret_cast<uint4*>(dst);
                for (int i = threadIdx.x; i < sl * (a.hd / 16); i += threads) {
                    const uint4 v = old[i];
                    old[i] = make_uint4(rescaled(v.x, s.old), rescaled(v.y, s.old), rescaled(v.z, s.old),
                                        rescaled(v.w, s.old));
                }
            }
            if (threadIdx.x == 0) *scale = s.scale;
            __syncthreads();  // part is free
        }
    }
}

}  // namespace
}  // namespace npub

extern "C" size_t npub_rope_paged_append_q8_workspace(int tokens, int rot_dim, int packed) {
    return packed && tokens > 0 && rot_dim > 0 ? (size_t)tokens * (rot_dim / 2) * sizeof(float2) : 0;
}

extern "C" int npub_rope_paged_append_q8(const void* qkv, int64_t ldx, void* q_out, int64_t ldq, int tokens, int q_heads,
                                         int kv_heads, int head_dim, int rot_dim, int interleaved,
                                         const int32_t* positions, const float* inv_freq, const void* q_gamma,
                                         const void* k_gamma, float eps, int8_t* k_pages, int8_t* v_pages,
                                         float* k_scales, float* v_scales, int n_pages, int page_size,
                                         const int32_t* page_table, int64_t ldt, int max_pages,
                                         const int32_t* cu_seqlens, int batch, void* workspace, size_t workspace_bytes,
                                         void* stream) {
    using namespace npub;
    NPUB_CHECK_ARG(tokens >= 0 && batch >= 0 && q_heads > 0 && kv_heads > 0 && q_heads + 2 * (int64_t)kv_heads <= 65536);
    if (tokens == 0) return NPUB_OK;
    NPUB_CHECK_ARG(qkv && q_out && positions && inv_freq && k_pages && v_pages && k_scales && v_scales && page_table);
    NPUB_CHECK_ARG(head_dim % 16 == 0 && head_dim > 0);
    NPUB_CHECK_ARG(rot_dim % 16 == 0 && rot_dim > 0 && rot_dim <= head_dim);
    NPUB_CHECK_ARG(ldx % 8 == 0 && ldq % 8 == 0 && ldx >= (int64_t)(q_heads + 2 * kv_heads) * head_dim &&
                   ldq >= (int64_t)q_heads * head_dim);
    NPUB_CHECK_ARG(npub_aligned(qkv, 16) && npub_aligned(q_out, 16) && npub_aligned(k_pages, 16) &&
                   npub_aligned(v_pages, 16) && npub_aligned(q_gamma, 16) && npub_aligned(k_gamma, 16) &&
                   npub_aligned(k_scales, 4) && npub_aligned(v_scales, 4));
    NPUB_CHECK_ARG(page_size >= 16 && page_size <= 256 && (page_size & (page_size - 1)) == 0 && n_pages > 0);
    NPUB_CHECK_ARG(max_pages > 0 && ldt >= max_pages);
    NPUB_CHECK_ARG(cu_seqlens ? batch > 0 : batch == tokens);
    if (head_dim > 128) return NPUB_ERR_UNSUPPORTED;
    Q8Args p = {};
    AppendArgs& a = p.q;
    a.x = reinterpret_cast<const __half*>(qkv);
    a.ldx = ldx;
    a.q = reinterpret_cast<__half*>(q_out);
    a.ldq = ldq;
    a.hq = q_heads;
    a.hd = head_dim;
    a.half = rot_dim / 2;
    a.interleaved = interleaved ? 1 : 0;
    a.units = head_dim / 16;
    while ((1 << a.units_log2) < a.units) ++a.units_log2;
    a.units_p2 = 1 << a.units_log2;
    a.pos = positions;
    a.inv_freq = inv_freq;
    a.gq = reinterpret_cast<const __half*>(q_gamma);
    a.gk = reinterpret_cast<const __half*>(k_gamma);
    a.eps = eps;
    a.inv_hd = 1.0f / (float)head_dim;
    a.n_pages = n_pages;
    while ((1 << a.page_shift) < page_size) ++a.page_shift;
    a.table = page_table;
    a.ldt = ldt;
    a.max_pages = max_pages;
    a.cu = cu_seqlens;
    a.batch = batch;
    p.hk = kv_heads;
    p.rows = tokens;
    p.kp = k_pages;
    p.vp = v_pages;
    p.ks = k_scales;
    p.vs = v_scales;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    if (!cu_seqlens) {
        const int groups = (q_heads + 2 * kv_heads + kDecodeWarps - 1) / kDecodeWarps;
        return launch_pdl(append_decode_q8_kernel, dim3(tokens, groups), dim3(kDecodeWarps * 32), 0, st, p);
    }
    // short sequences start several pages in the rows of one
    p.window = tokens / batch >= page_size ? page_size : 16;
    p.windows = (tokens + p.window - 1) / p.window;
    const int64_t blocks = (int64_t)p.windows * 2 * kv_heads;
    if (!workspace || workspace_bytes < npub_rope_paged_append_q8_workspace(tokens, rot_dim, 1)) return NPUB_ERR_WORKSPACE;
    NPUB_CHECK_ARG(npub_aligned(workspace, 256));
    a.turns = reinterpret_cast<float2*>(workspace);
    if (blocks > 0x7fffffff) return NPUB_ERR_UNSUPPORTED;
    const int rc = launch_pdl(append_query_kernel, dim3(tokens), dim3(kAppThreads), 0, st, p.q);
    if (rc) return rc;
    int threads = (page_size << a.units_log2) / kUnits;
    if (threads < 32) threads = 32;
    return launch_pdl(append_packed_q8_kernel, dim3((unsigned)blocks), dim3(threads), 0, st, p);
}
