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
// fp16), and where the fp32 quotient comes within 2e-5 of a half the remainder
// 127 t - q max|t| is formed in fp64, which holds it exactly.
// A row with a NaN or an infinity gets the scale NaN and q = 0; a row of zeros
// the scale 0.
//
// Bound: HBM, 2 bytes read and 1 written per element (6 and 3 with a residual).
#include "common.cuh"
#include "gemm_tc.h"

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

// The eight t = h * gamma (h without gamma).
template <bool GAMMA>
__device__ __forceinline__ void times_gamma(const uint4& v, const uint4& g, float (&t)[8]) {
    const __half2* p = reinterpret_cast<const __half2*>(&v);
    const __half2* s = reinterpret_cast<const __half2*>(&g);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(p[i]);
        t[2 * i] = f.x;
        t[2 * i + 1] = f.y;
        if (GAMMA) {
            const float2 e = __half22float2(s[i]);
            t[2 * i] *= e.x;
            t[2 * i + 1] *= e.y;
        }
    }
}

// The larger magnitude, NaN when one is.
__device__ __forceinline__ float top_of(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(fabsf(b)));
    return r;
}

// rint(127 t / most), halves to even, from the fp32 quotient's q, where that is near a half.
__device__ __forceinline__ int beside_half(float t, float most, int q) {
    const double e = 127.0 * (double)t - (double)q * (double)most, half = 0.5 * (double)most;
    if (e > half || (e == half && (q & 1))) return q + 1;
    if (e < -half || (e == -half && (q & 1))) return q - 1;
    return q;
}

// One row per block; V 8-element vectors of it in the registers of a thread,
// those behind them (rows of more than 8 V THREADS elements) read again.
//
// Measured: 32 rows of 4096 with gamma 2.6 us, 2048 of 11008 17.5 (3.9 TB/s), 8192 of 11008 54 (5.0), 8192 of 4096 with gamma
// 32 (3.1), without 21.5: with gamma the instructions bound it. (rintf, a conversion and the fp64 path as a call: 4.1, 29, 108,
// 40 and 37.)
template <int THREADS, int V, bool GAMMA>
__global__ void __launch_bounds__(THREADS) quantize_rows_kernel(const QuantArgs a) {
    pdl_trigger();
    pdl_wait();
    __shared__ float part_ss[THREADS / 32];
    __shared__ uint32_t part_top[THREADS / 32];
    const int64_t row = blockIdx.x;
    constexpr int step = THREADS * 8;
    uint4 v[V];
    float ss = 0.0f;
    uint32_t top = 0;  // bits of the largest |t|: ordered as integers, NaN above infinity
    float most = 0.0f;
    auto gamma_at = [&](int c) { return GAMMA ? __ldg(reinterpret_cast<const uint4*>(a.g + c)) : make_uint4(0, 0, 0, 0); };
    auto look = [&](int c, const uint4& u) {
        if (GAMMA) {
            float t[8];
            times_gamma<true>(u, gamma_at(c), t);
            const __half2* p = reinterpret_cast<const __half2*>(&u);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 f = __half22float2(p[i]);
                ss = fmaf(f.x, f.x, fmaf(f.y, f.y, ss));
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) most = top_of(most, t[i]);
        } else {  // fp16 magnitudes, two in a word
            const uint32_t m = __vmaxu2(__vmaxu2(u.x & 0x7fff7fffu, u.y & 0x7fff7fffu),
                                        __vmaxu2(u.z & 0x7fff7fffu, u.w & 0x7fff7fffu));
            top = __vmaxu2(top, m);
        }
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
    if (GAMMA) top = __float_as_uint(most);
    else top = __float_as_uint(__half2float(__ushort_as_half((unsigned short)max(top & 0xffffu, top >> 16))));
    if (GAMMA) {
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, d);
    }
    top = __reduce_max_sync(0xffffffffu, top);
    if ((threadIdx.x & 31) == 0) {
        part_ss[threadIdx.x >> 5] = ss;
        part_top[threadIdx.x >> 5] = top;
    }
    __syncthreads();
    ss = 0.0f;
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) {
        ss += part_ss[w];
        top = max(top, part_top[w]);
    }
    most = __uint_as_float(top);
    float y = most;
    if (GAMMA && most > 0.0f) y = most * (1.0f / sqrtf(ss / (float)a.cols + a.eps));  // zeros stay zeros with eps = 0 too
    const bool fine = top < 0x7f800000u;
    if (threadIdx.x == 0) a.scale[row] = fine ? y / 127.0f : NAN;
    // the smallest |t| that is not 0 is 2^-48
    const float inv = fine && most > 0.0f ? 127.0f / most : 0.0f;
    auto put = [&](int c, const uint4& u) {
        float t[8];
        times_gamma<GAMMA>(u, gamma_at(c), t);
        // adding 1.5 * 2^23 rounds to whole numbers, halves to even, and leaves them in the low bits
        uint32_t q[8];
        float off = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float y = t[i] * inv, m = y + 12582912.0f;
            q[i] = __float_as_uint(m);
            off = fmaxf(off, fabsf(y - (m - 12582912.0f)));
        }
        if (off > 0.49998f) {  // near a half: y's two roundings are within 127 * 2^-23 = 1.52e-5
#pragma unroll
            for (int i = 0; i < 8; ++i) q[i] = (uint32_t)beside_half(t[i], most, (int)q[i] - 0x4b400000);
        }
        if (inv == 0.0f) {
#pragma unroll
            for (int i = 0; i < 8; ++i) q[i] = 0;
        }
        uint2 w;
        w.x = __byte_perm(__byte_perm(q[0], q[1], 0x0040), __byte_perm(q[2], q[3], 0x0040), 0x5410);
        w.y = __byte_perm(__byte_perm(q[4], q[5], 0x0040), __byte_perm(q[6], q[7], 0x0040), 0x5410);
        *reinterpret_cast<uint2*>(a.q + row * a.ldq + c) = w;
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

template <int THREADS, int V>
int launch_quantize(const QuantArgs& a, int rows, cudaStream_t st) {
    if (a.g) return launch_pdl(quantize_rows_kernel<THREADS, V, true>, dim3(rows), dim3(THREADS), 0, st, a);
    return launch_pdl(quantize_rows_kernel<THREADS, V, false>, dim3(rows), dim3(THREADS), 0, st, a);
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
    if (rows <= num_sms() && vecs > 256) {  // one block on an SM: a row's latency counts
        if (vecs <= 512) return launch_quantize<512, 1>(a, rows, st);
        return launch_quantize<512, 3>(a, rows, st);
    }
    if (vecs <= 256) return launch_quantize<128, 2>(a, rows, st);
    if (vecs <= 512) return launch_quantize<256, 2>(a, rows, st);
    if (vecs <= 768) return launch_quantize<256, 3>(a, rows, st);
    if (vecs <= 1024) return launch_quantize<256, 4>(a, rows, st);
    return launch_quantize<256, 6>(a, rows, st);
}
