// Rows to 8-bit integers with one scale each, behind the residual add and the
// RMSNorm that precede a projection.
//
//   h = fp16(x + residual)                        (x without a residual; h is stored)
//   t = h * gamma, y = t / sqrt(mean(h^2) + eps)  (y = t = h without gamma)
//   scale = max|y| / 127,  q = rint(127 t / max|t|), halves to even
//
// The norm's factor cancels in q, so one pass over the row collects the sum of
// squares and the largest |t| together, and the row stays in registers for the
// second.  q is exactly the definition's: t is exact in fp32 (a product of two
// fp16), and where the fp32 quotient comes within 1e-4 of a half the remainder
// 127 t - q max|t| is formed in fp64, which holds it exactly.
// A row with a NaN or an infinity gets the scale NaN and q = 0; a row of zeros
// the scale 0.
//
// Bound: HBM, 2 bytes read and 1 written per element (6 and 3 with a residual).
#include "common.cuh"

namespace npub {
namespace {

struct QuantArgs {
    const __half *x, *r, *g;
    __half* h;
    int64_t ldx, ldr, ldh, ldq;
    int8_t* q;
    float* scale;
    int cols;
    float eps;
};

__device__ __forceinline__ void load_h(const QuantArgs& a, int64_t row, int c, uint4& v) {
    v = *reinterpret_cast<const uint4*>(a.x + row * a.ldx + c);
    if (!a.r) return;
    const uint4 w = *reinterpret_cast<const uint4*>(a.r + row * a.ldr + c);
    __half2* p = reinterpret_cast<__half2*>(&v);
    const __half2* s = reinterpret_cast<const __half2*>(&w);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(p[i]), e = __half22float2(s[i]);
        p[i] = __floats2half2_rn(f.x + e.x, f.y + e.y);
    }
    *reinterpret_cast<uint4*>(a.h + row * a.ldh + c) = v;
}

__device__ __forceinline__ void times_gamma(const QuantArgs& a, int c, const uint4& v, float (&t)[8]) {
    const __half2* p = reinterpret_cast<const __half2*>(&v);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(p[i]);
        t[2 * i] = f.x;
        t[2 * i + 1] = f.y;
    }
    if (!a.g) return;
    const uint4 w = __ldg(reinterpret_cast<const uint4*>(a.g + c));
    const __half2* s = reinterpret_cast<const __half2*>(&w);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(s[i]);
        t[2 * i] *= f.x;
        t[2 * i + 1] *= f.y;
    }
}

// rint(127 t / most), halves to even; inv = 127 / most in fp32.
__device__ __forceinline__ int quantised(float t, float most, float inv) {
    const float y = t * inv, n = rintf(y);
    int q = (int)n;
    if (fabsf(y - n) > 0.4999f) {  // near a half: 127 (2^-23 of y's two roundings) is far inside 1e-4
        const double e = 127.0 * (double)t - (double)q * (double)most, half = 0.5 * (double)most;
        if (e > half || (e == half && (q & 1))) ++q;
        else if (e < -half || (e == -half && (q & 1))) --q;
    }
    return q;
}

// One row per block; V 8-element vectors of it in the registers of a thread,
// those behind them (rows of more than 8 V blockDim elements) read again.
template <int V>
__global__ void __launch_bounds__(512) quantize_rows_kernel(const QuantArgs a) {
    pdl_trigger();
    pdl_wait();
    __shared__ float part_ss[16];
    __shared__ uint32_t part_top[16];
    const int64_t row = blockIdx.x;
    const int step = (int)blockDim.x * 8;
    uint4 v[V];
    float ss = 0.0f;
    uint32_t top = 0;  // bits of the largest |t|: ordered as integers, NaN above infinity
    auto look = [&](int c, const uint4& u) {
        float t[8];
        times_gamma(a, c, u, t);
        const __half2* p = reinterpret_cast<const __half2*>(&u);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = __half22float2(p[i]);
            ss = fmaf(f.x, f.x, fmaf(f.y, f.y, ss));
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(t[i]) & 0x7fffffffu);
    };
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int c = j * step + (int)threadIdx.x * 8;
        if (c < a.cols) load_h(a, row, c, v[j]);
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int c = j * step + (int)threadIdx.x * 8;
        if (c < a.cols) look(c, v[j]);
    }
    for (int c = V * step + (int)threadIdx.x * 8; c < a.cols; c += step) {
        uint4 u;
        load_h(a, row, c, u);
        look(c, u);
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, d);
    top = __reduce_max_sync(0xffffffffu, top);
    const int warps = (int)blockDim.x >> 5;
    if ((threadIdx.x & 31) == 0) {
        part_ss[threadIdx.x >> 5] = ss;
        part_top[threadIdx.x >> 5] = top;
    }
    __syncthreads();
    ss = 0.0f;
    for (int w = 0; w < warps; ++w) {
        ss += part_ss[w];
        top = max(top, part_top[w]);
    }
    float most = __uint_as_float(top), y = most;
    if (a.g) y = most * (1.0f / sqrtf(ss / (float)a.cols + a.eps));
    const bool fine = top < 0x7f800000u;
    if (threadIdx.x == 0) a.scale[row] = fine ? y / 127.0f : NAN;
    if (!fine) most = 0.0f;
    // below 127 / FLT_MAX the reciprocal would overflow: all of the row is taken as zero beside what fp16 can hold
    const float inv = most > 1e-30f ? 127.0f / most : 0.0f;
    auto put = [&](int c, const uint4& u) {
        float t[8];
        times_gamma(a, c, u, t);
        uint32_t w[2] = {0, 0};
        if (inv != 0.0f) {
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i >> 2] |= (uint32_t)(quantised(t[i], most, inv) & 0xff) << (8 * (i & 3));
        }
        *reinterpret_cast<uint2*>(a.q + row * a.ldq + c) = make_uint2(w[0], w[1]);
    };
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int c = j * step + (int)threadIdx.x * 8;
        if (c < a.cols) put(c, v[j]);
    }
    for (int c = V * step + (int)threadIdx.x * 8; c < a.cols; c += step) {
        // this thread's own elements again
        put(c, *reinterpret_cast<const uint4*>((a.r ? a.h + row * a.ldh : a.x + row * a.ldx) + c));
    }
}

}  // namespace
}  // namespace npub

extern "C" int npub_quantize_rows(const void* x, int64_t ldx, const void* residual, int64_t ldr, void* h_out, int64_t ldh,
                                  const void* gamma, float eps, int rows, int cols, int8_t* q, int64_t ldq, float* scale,
                                  void* stream) {
    using namespace npub;
    NPUB_CHECK_ARG(rows >= 0 && cols > 0 && cols % 8 == 0);
    if (rows == 0) return NPUB_OK;
    NPUB_CHECK_ARG(x && q && scale && (!residual || h_out));
    NPUB_CHECK_ARG(ldx % 8 == 0 && ldx >= cols && ldq % 8 == 0 && ldq >= cols);
    NPUB_CHECK_ARG(!residual || (ldr % 8 == 0 && ldr >= cols && ldh % 8 == 0 && ldh >= cols));
    NPUB_CHECK_ARG(npub_aligned(x, 16) && npub_aligned(residual, 16) && npub_aligned(h_out, 16) && npub_aligned(gamma, 16) &&
                   npub_aligned(q, 8) && npub_aligned(scale, 4));
    QuantArgs a;
    a.x = reinterpret_cast<const __half*>(x);
    a.r = reinterpret_cast<const __half*>(residual);
    a.g = reinterpret_cast<const __half*>(gamma);
    a.h = reinterpret_cast<__half*>(h_out);
    a.ldx = ldx;
    a.ldr = ldr;
    a.ldh = ldh;
    a.ldq = ldq;
    a.q = q;
    a.scale = scale;
    a.cols = cols;
    a.eps = eps;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    const int vecs = cols / 8;
    if (vecs <= 256) return launch_pdl(quantize_rows_kernel<2>, dim3(rows), dim3(128), 0, st, a);
    if (vecs <= 512) return launch_pdl(quantize_rows_kernel<2>, dim3(rows), dim3(256), 0, st, a);
    if (vecs <= 1024) return launch_pdl(quantize_rows_kernel<4>, dim3(rows), dim3(256), 0, st, a);
    return launch_pdl(quantize_rows_kernel<4>, dim3(rows), dim3(512), 0, st, a);
}
