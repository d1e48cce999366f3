// Sampling of one token per row from given random numbers, with temperature,
// top-k, top-p and min-p (the counterpart of npub_argmax_rows for a decoder
// that does not choose greedily; the reference stops at the logits).
//
// Order the row by logit, descending, equal logits by index, ascending;
// w_i = exp((l_i - max) / T).  Kept are the first top_k; of them those i whose
// predecessors' sum is below top_p times the sum of all of them; of those the
// ones with w_i >= min_p; the first always.  The token is the first kept one at
// which the running sum exceeds u times the kept sum.
//
// There are 63,488 different fp16 logits above -inf, so the row is not sorted:
// a histogram over the values in shared memory (16-bit counts, 124 KB; one
// logit is one shared-memory increment) is the sorted row, with one weight for
// each value instead of one for each token.  Sums of weights are fp64 in a
// fixed order, counts are integers: a token at a border of the running sum is
// the one that the formula gives, up to 1e-13 of the sum, and the same on
// every call.  A row of more than 40,960 logits is cut over the CTAs of a
// cluster, which then each take a range of values out of all of their
// histograms.
//
// Bound: the logits are read once (from L1 or L2 a second time for the index);
// what a row takes is the histogram's clearing, filling and scan.
#include "common.cuh"

#include <cmath>

namespace npub {
namespace smp {

constexpr int kThreads = 1024;
constexpr int kZero = 0x7c00;         // bin of the logit 0; bin 0 is +inf
constexpr int kBins = 2 * kZero;      // the last is -65504
constexpr int kGroups = kBins / 8;    // 16 bytes of counts
constexpr int kOwners = kGroups / 8;  // threads that hold a range of values (992)
constexpr uint32_t kNone = 0xffffu;   // -inf and NaN: no bin

struct Args {
    const __half* x;
    int64_t ld;
    int vocab, seg, vec;
    const float *u, *t, *p, *m;
    const int32_t* k;
    float t0, p0, m0;
    int k0;
    int32_t* ids;
};

// The bin of a logit's bits: descending values, both zeros the same.
__device__ __forceinline__ uint32_t bin_of(uint32_t b) {
    const uint32_t mag = b & 0x7fffu;
    if (mag >= 0x7c00u) return b == 0x7c00u ? 0u : kNone;
    return (b & 0x8000u) ? kZero + mag : kZero - mag;
}
__device__ __forceinline__ double value_of(int bin) {
    const uint32_t b = bin <= kZero ? (uint32_t)(kZero - bin) : 0x8000u | (uint32_t)(bin - kZero);
    return (double)__half2float(__ushort_as_half((unsigned short)b));
}

// What the CTAs of a cluster tell one another.
struct Mail {
    double w, w_min;          // this CTA's range of values: weights, and those of at least min_p
    double cut_w;             // a cut's weight
    uint32_t top;             // first bin in use
    uint32_t n, n_min;        // the same, tokens
    uint32_t cut_n;
    uint32_t pos, bin, rank;  // the sampled place in the order, its value, its number among the equal ones
};

template <int C>
__device__ __forceinline__ void sync_all() {
    if (C > 1) cluster_sync();
    else __syncthreads();
}
template <int C>
__device__ __forceinline__ uint32_t addr_in(uint32_t local, int cta) {
    return C > 1 ? mapa_shared(local, (uint32_t)cta) : local;
}
__device__ __forceinline__ uint32_t ld_u32(uint32_t a) {
    uint32_t v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ double ld_f64(uint32_t a) {
    double v;
    asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ uint4 ld_v4(uint32_t a) {
    uint4 v;
    asm volatile("ld.shared::cluster.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "r"(a)
                 : "memory");
    return v;
}
__device__ __forceinline__ void st_u32(uint32_t a, uint32_t v) {
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(a), "r"(v) : "memory");
}
__device__ __forceinline__ void st_f64(uint32_t a, double v) {
    asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(a), "d"(v) : "memory");
}

// Counts of the 8 bins of a group over the cluster's histograms.
template <int C>
__device__ __forceinline__ uint32_t group_counts(uint32_t hist, int g, uint32_t (&c)[8]) {
    uint4 v[C];
#pragma unroll
    for (int q = 0; q < C; ++q) v[q] = ld_v4(addr_in<C>(hist + (uint32_t)g * 16u, q));
#pragma unroll
    for (int e = 0; e < 8; ++e) c[e] = 0;
#pragma unroll
    for (int q = 0; q < C; ++q) {
        const uint32_t w[4] = {v[q].x, v[q].y, v[q].z, v[q].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            c[2 * e] += w[e] & 0xffffu;
            c[2 * e + 1] += w[e] >> 16;
        }
    }
    uint32_t any = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) any |= c[e];
    return any;
}

// Weights of a thread's range of values (64 / C bins inside one binade, evenly
// spaced): exp of a group's first value, then products with the step's ratio
// (7 of them: within 1e-15).  The largest value of the row has weight 1.
struct Weights {
    double top, inv_t, ratio;
    int top_bin;
    __device__ __forceinline__ double first(int g, int& e0) const {
        e0 = 0;
        if (g == (top_bin >> 3)) {
            e0 = top_bin & 7;
            return 1.0;
        }
        return exp((value_of(g * 8) - top) * inv_t);
    }
};

// Walks the tokens of a thread's range in order: f(tokens before, weight before, count, weight) until it returns true.
template <int C, typename F>
__device__ __forceinline__ void walk(uint32_t hist, int g0, const Weights& wt, uint32_t n, double w, F f) {
#pragma unroll 1
    for (int j = 0; j < 8 / C; ++j) {
        uint32_t c[8];
        if (!group_counts<C>(hist, g0 + j, c)) continue;
        int e0;
        double x = wt.first(g0 + j, e0);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if (e < e0) continue;
            if (c[e]) {
                if (f(n, w, c[e], x, (g0 + j) * 8 + e)) return;
                n += c[e];
                w += (double)c[e] * x;
            }
            x *= wt.ratio;
        }
    }
}

template <int C>
__global__ void __launch_bounds__(kThreads, 1) sample_kernel(const Args a) {
    pdl_trigger();
    extern __shared__ __align__(16) uint32_t hist[];  // [kBins / 2], two counts each
    __shared__ Mail mail;
    __shared__ double part_w[32];
    __shared__ uint32_t part_n[32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int rank = C > 1 ? (int)cluster_ctarank() : 0;
    const int64_t row = blockIdx.x / C;
    for (int i = tid; i < kGroups; i += kThreads) reinterpret_cast<uint4*>(hist)[i] = make_uint4(0, 0, 0, 0);
    if (tid == 0) mail.top = kNone;
    __syncthreads();
    pdl_wait();

    // ---- the histogram of this CTA's logits
    const __half* x = a.x + row * a.ld;
    const int i0 = min(a.vocab, rank * a.seg), i1 = min(a.vocab, i0 + a.seg);
    uint32_t top = kNone;
    for (int base = i0; base < i1; base += kThreads * 8) {
        const int i = base + tid * 8;
        uint32_t w[4] = {0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u};
        if (a.vec && i + 8 <= i1) {
            const uint4 v = __ldg(reinterpret_cast<const uint4*>(x + i));
            w[0] = v.x;
            w[1] = v.y;
            w[2] = v.z;
            w[3] = v.w;
        } else {
            for (int e = 0; e < 8; ++e)
                if (i + e < i1) {
                    const uint32_t h = __half_as_ushort(x[i + e]);
                    w[e >> 1] = (e & 1) ? (w[e >> 1] & 0xffffu) | (h << 16) : (w[e >> 1] & 0xffff0000u) | h;
                }
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const uint32_t bin = bin_of((e & 1) ? w[e >> 1] >> 16 : w[e >> 1] & 0xffffu);
            top = min(top, bin);
            // a warp of one value (a mask's) counts it at once
            if (__all_sync(0xffffffffu, bin == __shfl_sync(0xffffffffu, bin, 0))) {
                if (lane == 0 && bin != kNone) atomicAdd(&hist[bin >> 1], 32u << ((bin & 1) * 16));
            } else if (bin != kNone) {
                atomicAdd(&hist[bin >> 1], 1u << ((bin & 1) * 16));
            }
        }
    }
    top = __reduce_min_sync(0xffffffffu, top);
    if (lane == 0 && top != kNone) atomicMin(&mail.top, top);
    sync_all<C>();
    const uint32_t mb = smem_u32(&mail), hb = smem_u32(hist);
    auto at = [&](int q, const void* field) {
        return addr_in<C>(mb + (uint32_t)(reinterpret_cast<const char*>(field) - reinterpret_cast<const char*>(&mail)), q);
    };
    top = kNone;
#pragma unroll
    for (int q = 0; q < C; ++q) top = min(top, ld_u32(at(q, &mail.top)));

    if (top == kNone) {  // nothing left to draw from
        if (rank == 0 && tid == 0) a.ids[row] = -1;
    } else {
        float t = a.t ? a.t[row] : a.t0;
        const float pf = a.p ? a.p[row] : a.p0, mf = a.m ? a.m[row] : a.m0;
        const int k = a.k ? a.k[row] : a.k0;
        const double u = (double)a.u[row];
        const bool greedy = !(t > 0.0f);
        if (top == 0 || greedy) t = 1.0f;  // +inf takes all of the weight
        // ---- tokens and weights of this thread's values, and their running sums
        constexpr int G = 8 / C;
        const bool owner = tid < kOwners;
        const int g0 = (rank * kOwners + tid) * G;
        Weights wt;
        wt.top = value_of((int)top);
        wt.top_bin = (int)top;
        wt.inv_t = 1.0 / (double)t;
        wt.ratio = 0.0;
        const double min_p = (double)mf;
        uint32_t n = 0, nm = 0;
        double w = 0.0, wm = 0.0;
        if (owner) {
            // (between the second and third value: the first of bin 0's group is +inf)
            wt.ratio = top == 0 ? 0.0 : exp((value_of(g0 * 8 + 2) - value_of(g0 * 8 + 1)) * wt.inv_t);
#pragma unroll 1
            for (int j = 0; j < G; ++j) {
                // lanes start at different groups: no two of a quarter warp read the same banks
                const int g = g0 + ((j + (lane >> (C == 8 ? 3 : C == 4 ? 2 : C == 2 ? 1 : 0))) & (G - 1));
                uint32_t c[8];
                if (!group_counts<C>(hb, g, c)) continue;
                int e0;
                double y = wt.first(g, e0);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    if (e < e0) continue;
                    if (c[e]) {
                        const double cy = (double)c[e] * y;
                        n += c[e];
                        w += cy;
                        if (y >= min_p) {
                            nm += c[e];
                            wm += cy;
                        }
                    }
                    y *= wt.ratio;
                }
            }
        }
        uint32_t ni = n;
        double wi = w;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const uint32_t an = __shfl_up_sync(0xffffffffu, ni, d);
            const double aw = __shfl_up_sync(0xffffffffu, wi, d);
            if (lane >= d) {
                ni += an;
                wi = aw + wi;
            }
        }
        if (lane == 31) {
            part_n[warp] = ni;
            part_w[warp] = wi;
        }
        __syncthreads();
        uint32_t bn = 0, tn = 0;
        double bw = 0.0, tw = 0.0;
        for (int q = 0; q < 32; ++q) {  // the warps ahead, and all of them
            if (q == warp) {
                bn = tn;
                bw = tw;
            }
            tn += part_n[q];
            tw += part_w[q];
        }
        __syncthreads();
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) {
            nm += __shfl_xor_sync(0xffffffffu, nm, d);
            wm += __shfl_xor_sync(0xffffffffu, wm, d);
        }
        if (lane == 0) {
            part_n[warp] = nm;
            part_w[warp] = wm;
        }
        __syncthreads();
        if (tid == 0) {
            nm = 0;
            wm = 0.0;
            for (int q = 0; q < 32; ++q) {
                nm += part_n[q];
                wm += part_w[q];
            }
            mail.n = tn;
            mail.w = tw;
            mail.n_min = nm;
            mail.w_min = wm;
        }
        sync_all<C>();
        uint32_t N = 0, Nm = 0;
        double W = 0.0, Wm = 0.0, cta_w = 0.0;
        uint32_t cta_n = 0;
#pragma unroll
        for (int q = 0; q < C; ++q) {
            if (q == rank) {
                cta_n = N;
                cta_w = W;
            }
            N += ld_u32(at(q, &mail.n));
            W += ld_f64(at(q, &mail.w));
            Nm += ld_u32(at(q, &mail.n_min));
            Wm += ld_f64(at(q, &mail.w_min));
        }
        // [n0, n1) tokens and [w0, w1) of the running weight are this thread's.  w0 is the w1 of the thread ahead, the
        // same sum of the same terms, so that the threads' ranges leave no gap.
        const uint32_t n0 = cta_n + bn + ni - n, n1 = n0 + n;
        const double up = __shfl_up_sync(0xffffffffu, wi, 1);
        const double w0 = cta_w + (lane ? bw + up : bw), w1 = cta_w + (bw + wi);
        auto tell = [&](uint32_t cn, double cw) {
#pragma unroll
            for (int q = 0; q < C; ++q) {
                st_u32(at(q, &mail.cut_n), cn);
                st_f64(at(q, &mail.cut_w), cw);
            }
        };
        uint32_t keep = N;
        double mass = W;
        if (greedy) {
            keep = 1;
        } else {
            if (k > 0 && (uint32_t)k < N) {
                if (n && n0 < (uint32_t)k && (uint32_t)k <= n1) {
                    double cw = w1;
                    walk<C>(hb, g0, wt, n0, w0, [&](uint32_t an, double aw, uint32_t c, double y, int) {
                        if (an + c < (uint32_t)k) return false;
                        cw = aw + (double)((uint32_t)k - an) * y;
                        return true;
                    });
                    tell((uint32_t)k, cw);
                }
                sync_all<C>();
                keep = mail.cut_n;
                mass = mail.cut_w;
                sync_all<C>();
            }
            if (pf < 1.0f) {
                const double goal = fmax((double)pf, 0.0) * mass;
                if (tid == 0) {
                    mail.cut_n = keep;
                    mail.cut_w = mass;
                }
                sync_all<C>();
                if (goal <= 0.0 ? n && n0 == 0 : n && w0 < goal && goal <= w1) {
                    uint32_t cn = n1;
                    double cw = w1;
                    walk<C>(hb, g0, wt, n0, w0, [&](uint32_t an, double aw, uint32_t c, double y, int) {
                        if (goal > 0.0 && aw + (double)c * y < goal) return false;
                        const double r = fmin(fmax(ceil((goal - aw) / y), 1.0), (double)c);
                        cn = an + (uint32_t)r;
                        cw = aw + r * y;
                        return true;
                    });
                    if (cn < keep) tell(cn, cw);
                }
                sync_all<C>();
                keep = mail.cut_n;
                mass = mail.cut_w;
            }
            if (Nm < keep) {
                keep = Nm;
                mass = Wm;
            }
        }
        if (keep == 0) keep = 1;  // min_p above 1
        // ---- the place in the order, then its value
        uint32_t pos = 0;
        if (keep > 1) {
            const double goal = u * mass;
            if (tid == 0) mail.pos = goal > 0.0 ? keep - 1 : 0;
            sync_all<C>();
            if (n && w0 <= goal && goal < w1) {
                uint32_t found = n1 - 1;
                walk<C>(hb, g0, wt, n0, w0, [&](uint32_t an, double aw, uint32_t c, double y, int) {
                    if (aw + (double)c * y <= goal) return false;
                    found = an + (uint32_t)fmin(fmax(floor((goal - aw) / y), 0.0), (double)(c - 1));
                    return true;
                });
#pragma unroll
                for (int q = 0; q < C; ++q) st_u32(at(q, &mail.pos), found);
            }
            sync_all<C>();
            pos = min(mail.pos, keep - 1);
        }
        if (n && n0 <= pos && pos < n1) {
            walk<C>(hb, g0, wt, n0, w0, [&](uint32_t an, double, uint32_t c, double, int bin) {
                if (an + c <= pos) return false;
#pragma unroll
                for (int q = 0; q < C; ++q) {
                    st_u32(at(q, &mail.bin), (uint32_t)bin);
                    st_u32(at(q, &mail.rank), pos - an);
                }
                return true;
            });
        }
        sync_all<C>();
        // ---- the rank-th token of that value, by index
        const uint32_t bin = mail.bin;
        uint32_t r = mail.rank;
        uint32_t mine = 0;
        bool here = true;
#pragma unroll
        for (int q = 0; q < C; ++q) {
            const uint32_t c = (ld_u32(addr_in<C>(hb + (bin >> 1) * 4u, q)) >> ((bin & 1) * 16)) & 0xffffu;
            if (q < rank) {
                here = here && r >= c;
                r -= c;  // wraps where a CTA ahead has the token
            } else if (q == rank) {
                mine = c;
            }
        }
        if (here && r < mine) {
            const int per = ((i1 - i0 + kThreads - 1) / kThreads + 7) / 8 * 8;
            const int j0 = min(i1, i0 + tid * per), j1 = min(i1, j0 + per);
            uint32_t c = 0;
            for (int i = j0; i < j1; ++i) c += bin_of(__half_as_ushort(x[i])) == bin;
            uint32_t s = c;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const uint32_t v = __shfl_up_sync(0xffffffffu, s, d);
                if (lane >= d) s += v;
            }
            if (lane == 31) part_n[warp] = s;
            __syncthreads();
            for (int q = 0; q < warp; ++q) s += part_n[q];
            if (s - c <= r && r < s) {
                r -= s - c;
                for (int i = j0; i < j1; ++i)
                    if (bin_of(__half_as_ushort(x[i])) == bin && r-- == 0) {
                        a.ids[row] = i;
                        break;
                    }
            }
        }
    }
    if (C > 1) cluster_sync();  // nobody leaves while its shared memory is read
}

template <int C>
int launch(const Args& a, int rows, cudaStream_t st) {
    auto kern = sample_kernel<C>;
    constexpr int bytes = kBins * 2;
    NPUB_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)rows * C);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = bytes;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = npub_internal_pdl_enabled() ? 1 : 0;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = C;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = C > 1 ? 2 : 1;
    NPUB_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, a));
    return npub_internal_launch_status();
}

}  // namespace smp
}  // namespace npub

extern "C" int npub_sample(const void* logits, int64_t ldl, int rows, int vocab, const float* u, const float* temperature,
                           float temperature_all, const int32_t* top_k, int top_k_all, const float* top_p,
                           float top_p_all, const float* min_p, float min_p_all, int32_t* ids, void* stream) {
    using namespace npub;
    using namespace npub::smp;
    NPUB_CHECK_ARG(rows >= 0 && vocab > 0);
    if (rows == 0) return NPUB_OK;
    NPUB_CHECK_ARG(logits && u && ids && ldl >= vocab && npub_aligned(logits, 2));
    NPUB_CHECK_ARG(npub_aligned(u, 4) && npub_aligned(temperature, 4) && npub_aligned(top_k, 4) && npub_aligned(top_p, 4) &&
                   npub_aligned(min_p, 4) && npub_aligned(ids, 4));
    // 16-bit counts: at most 65535 logits in a CTA's histogram
    if (vocab > 8 * 65528 || rows > 0x0fffffff) return NPUB_ERR_UNSUPPORTED;
    Args a;
    a.x = reinterpret_cast<const __half*>(logits);
    a.ld = ldl;
    a.vocab = vocab;
    a.vec = ldl % 8 == 0 && npub_aligned(logits, 16);
    a.u = u;
    a.t = temperature;
    a.t0 = temperature_all;
    a.k = top_k;
    a.k0 = top_k_all;
    a.p = top_p;
    a.p0 = top_p_all;
    a.m = min_p;
    a.m0 = min_p_all;
    a.ids = ids;
    const int c = vocab <= 40960 ? 1 : vocab <= 2 * 40960 ? 2 : vocab <= 4 * 40960 ? 4 : 8;
    a.seg = ((vocab + c - 1) / c + 7) / 8 * 8;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    switch (c) {
        case 1: return launch<1>(a, rows, st);
        case 2: return launch<2>(a, rows, st);
        case 4: return launch<4>(a, rows, st);
        default: return launch<8>(a, rows, st);
    }
}
