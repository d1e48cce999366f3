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
// every call.  A row may be cut over the CTAs of a cluster, which then each take
// a range of values out of all of their histograms.
//
// Bound: the logits are read once (from L1 or L2 a second time for the index);
// what a row takes is latency: clearing the histogram (0.5 us), filling it (1.9 us
// for 8192 logits), the weights of its values (2 to 5 us), the cuts by one warp (1.5
// to 2 us each: fp64 exp and scans), and the barriers between them.
#include "common.cuh"
#include "gemm_tc.h"

#include <cmath>
#include <cstddef>

namespace npub {
namespace smp {

constexpr int kThreads = 1024;
constexpr int kZero = 0x7c00;         // bin of the logit 0; bin 0 is +inf
constexpr int kBins = 2 * kZero;      // the last is -65504
constexpr int kGroups = kBins / 8;    // 16 bytes of counts
constexpr int kOwners = kGroups / 8;  // threads that hold a range of values (992)
constexpr uint32_t kNone = 0xffffu;   // -inf and NaN: no bin
constexpr int kMaxSegment = 65528;    // logits of a CTA: what a 16-bit count holds
constexpr int kMaxSteps = (kMaxSegment + kThreads * 8 - 1) / (kThreads * 8);

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
    double w[kOwners + 1];    // weight ahead of each thread's values, of the CTA's; their sum
    uint32_t n[kOwners + 1];  // tokens, likewise
    uint32_t top;             // first bin in use
    uint32_t bin, rank;       // the sampled value, and its number among the equal ones
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

// exp in one place: it is long
__device__ __noinline__ double exp_of(double x) { return exp(x); }
__device__ __forceinline__ double double_of(uint32_t c) {  // c < 2^32, by way of 2^52 + c
    return __hiloint2double(0x43300000, (int)c) - 4503599627370496.0;
}

// The row's weights: exp((l - top) / T), 1 at the top.
struct Weights {
    double top, inv_t;
    int top_bin;
    __device__ __forceinline__ double at(int bin) const {
        return bin <= top_bin ? 1.0 : exp_of((value_of(bin) - top) * inv_t);
    }
};

__device__ __forceinline__ double scan_up(double v, int lane) {
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const double u = __shfl_up_sync(0xffffffffu, v, d);
        if (lane >= d) v = u + v;
    }
    return v;
}
__device__ __forceinline__ uint32_t scan_up(uint32_t v, int lane) {
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const uint32_t u = __shfl_up_sync(0xffffffffu, v, d);
        if (lane >= d) v += u;
    }
    return v;
}

// A value of the row: tokens and weight ahead of it, its count, its weight, its bin.
struct Hit {
    uint32_t n;
    double w;
    uint32_t c;
    double y;
    int bin;
};
// By a warp: the first value in use behind which crossed(tokens, weight, bin) holds (none ahead of one behind which it
// does), or the last of the first thread's range behind which it does.  crossed is of running sums, so the search goes from
// the CTA to the thread, 32 at a time, to its values; a sum's rounding may put it at a range's end.
template <int C, typename F>
__device__ __noinline__ Hit locate(uint32_t hist, uint32_t mail_w, uint32_t mail_n, const Weights& wt, F crossed) {
    const int lane = threadIdx.x & 31;
    constexpr int G = 8 / C, kAll = C * kOwners;
    uint32_t n = 0;
    double w = 0.0;
    int cta = 0;
#pragma unroll
    for (int q = 0; q < C - 1; ++q) {
        if (cta != q) continue;
        const uint32_t an = n + ld_u32(addr_in<C>(mail_n + kOwners * 4u, q));
        const double aw = w + ld_f64(addr_in<C>(mail_w + kOwners * 8u, q));
        if (crossed(an, aw, (q + 1) * kOwners * G * 8 - 1)) continue;
        n = an;
        w = aw;
        cta = q + 1;
    }
    int thread = 0;
#pragma unroll
    for (int step = 32; step >= 1; step /= 32) {
        // the first lane's range of `step` threads behind which it holds
        const int end = min(kOwners, thread + (lane + 1) * step);
        const bool hit = end >= kOwners ||
                         crossed(n + ld_u32(addr_in<C>(mail_n + (uint32_t)end * 4u, cta)),
                                 w + ld_f64(addr_in<C>(mail_w + (uint32_t)end * 8u, cta)), (cta * kOwners + end) * G * 8 - 1);
        thread += (__ffs(__ballot_sync(0xffffffffu, hit)) - 1) * step;
    }
    const int g0 = (cta * kOwners + thread) * G;
    n += ld_u32(addr_in<C>(mail_n + (uint32_t)thread * 4u, cta));
    w += ld_f64(addr_in<C>(mail_w + (uint32_t)thread * 8u, cta));
    static_assert(kAll * G * 8 == kBins, "every bin has a thread");
    constexpr int kPer = C == 1 ? 2 : 1;  // bins per lane
    uint32_t c[kPer];
    double y[kPer];
    const int first = g0 * 8 + lane * kPer;
#pragma unroll
    for (int i = 0; i < kPer; ++i) c[i] = 0;
    if (lane * kPer < 64 / C) {
#pragma unroll
        for (int q = 0; q < C; ++q) {
            const uint32_t v = ld_u32(addr_in<C>(hist + (uint32_t)(first >> 1) * 4u, q));
            if constexpr (C == 1) {
                c[0] += v & 0xffffu;
                c[1] += v >> 16;
            } else {
                c[0] += (first & 1) ? v >> 16 : v & 0xffffu;
            }
        }
    }
    uint32_t sn = 0;
    double sw = 0.0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        y[i] = c[i] ? wt.at(first + i) : 0.0;
        sn += c[i];
        sw += double_of(c[i]) * y[i];
    }
    const uint32_t in = scan_up(sn, lane);
    const double iw = scan_up(sw, lane), up = __shfl_up_sync(0xffffffffu, iw, 1);
    Hit h, last;
    h.n = n + in - sn;
    h.w = w + (lane ? up : 0.0);
    bool hit = false;
    last.c = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        if (hit || !c[i]) continue;
        if (last.c) {
            h.n += last.c;
            h.w += double_of(last.c) * last.y;
        }
        last.c = h.c = c[i];
        last.y = h.y = y[i];
        h.bin = first + i;
        hit = crossed(h.n + c[i], h.w + double_of(c[i]) * y[i], first + i);
    }
    const uint32_t hits = __ballot_sync(0xffffffffu, hit), used = __ballot_sync(0xffffffffu, sn != 0);
    const int src = hits ? __ffs(hits) - 1 : 31 - __clz(used | 1u);
    if (!used) h.c = 0, h.y = 0.0, h.bin = 0;
    h.n = __shfl_sync(0xffffffffu, h.n, src);
    h.w = __shfl_sync(0xffffffffu, h.w, src);
    h.c = __shfl_sync(0xffffffffu, h.c, src);
    h.y = __shfl_sync(0xffffffffu, h.y, src);
    h.bin = __shfl_sync(0xffffffffu, h.bin, src);
    return h;
}

// Eight logits from i on (-inf behind the segment's end).
__device__ __forceinline__ uint4 load8(const __half* x, int i, int end, int vec) {
    uint32_t w[4] = {0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u};
    if (vec && i + 8 <= end) return __ldg(reinterpret_cast<const uint4*>(x + i));
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (i + e < end) {
            const uint32_t h = __half_as_ushort(x[i + e]);
            w[e >> 1] = (e & 1) ? (w[e >> 1] & 0xffffu) | (h << 16) : (w[e >> 1] & 0xffff0000u) | h;
        }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

template <int C>
__global__ void __launch_bounds__(kThreads, 1) sample_kernel(const Args a) {
    pdl_trigger();
    extern __shared__ __align__(16) uint32_t hist[];  // [kBins / 2], two counts each
    __shared__ Mail mail;
    __shared__ double part_w[32];
    __shared__ uint32_t part_n[kMaxSteps * 32];
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
        const uint4 v = load8(x, base + tid * 8, i1, a.vec);
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
        // a warp of one value (a mask's) counts it at once
        const bool flat = v.x == v.y && v.x == v.z && v.x == v.w && (v.x >> 16) == (v.x & 0xffffu);
        const uint32_t first = __shfl_sync(0xffffffffu, v.x, 0);
        if (__all_sync(0xffffffffu, flat && v.x == first)) {
            const uint32_t bin = bin_of(v.x & 0xffffu);
            top = min(top, bin);
            if (lane == 0 && bin != kNone) atomicAdd(&hist[bin >> 1], 256u << ((bin & 1) * 16));
            continue;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const uint32_t bin = bin_of((e & 1) ? w[e >> 1] >> 16 : w[e >> 1] & 0xffffu);
            top = min(top, bin);
            if (bin != kNone) atomicAdd(&hist[bin >> 1], 1u << ((bin & 1) * 16));
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
        Weights wt;
        wt.top = value_of((int)top);
        wt.top_bin = (int)top;
        wt.inv_t = 1.0 / (double)t;
        // ---- tokens and weights of this thread's values: 64 / C bins inside one binade, evenly spaced, so that the weights
        // of a group are exp of its first value times powers of the step's ratio, and the groups' first values likewise
        // (products of at most 63 steps: within 2e-14)
        constexpr int G = 8 / C;
        const int g0 = (rank * kOwners + tid) * G;
        uint32_t n = 0;
        double w = 0.0;
        if (tid < kOwners) {
            double ratio = 0.0, begin = 0.0, r2 = 0.0, r4 = 0.0, r8 = 0.0;
            bool ready = false;
#pragma unroll 1
            for (int j = 0; j < G; ++j) {
                // lanes start at different groups: no two of a quarter warp read the same banks
                const int i = (j + (lane >> (C == 8 ? 3 : C == 4 ? 2 : C == 2 ? 1 : 0))) & (G - 1), g = g0 + i;
                uint32_t c[8];
                if (!group_counts<C>(hb, g, c)) continue;
                if (!ready) {
                    ready = true;
                    // (between the second and third value: the first of bin 0's group is +inf)
                    ratio = top == 0 ? 0.0 : exp_of((value_of(g0 * 8 + 2) - value_of(g0 * 8 + 1)) * wt.inv_t);
                    r2 = ratio * ratio;
                    r4 = r2 * r2;
                    r8 = r4 * r4;
                    begin = g0 > wt.top_bin >> 3 ? wt.at(g0 * 8) : 0.0;
                }
                double y;
                if (g0 > wt.top_bin >> 3) {
                    const double r16 = r8 * r8;
                    y = begin * ((i & 1) ? r8 : 1.0) * ((i & 2) ? r16 : 1.0) * ((i & 4) ? r16 * r16 : 1.0);
                } else if (g > wt.top_bin >> 3) {
                    y = wt.at(g * 8);
                } else {  // the top's group: from the top on
                    y = 1.0;
                    const int e0 = wt.top_bin & 7;
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        if (e < e0) continue;
                        n += c[e];
                        w += double_of(c[e]) * y;
                        y *= ratio;
                    }
                    continue;
                }
                // sum of c[e] ratio^e
                double s[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) s[e] = fma(double_of(c[2 * e + 1]), ratio, double_of(c[2 * e]));
                w = fma(fma(fma(s[3], r2, s[2]), r4, fma(s[1], r2, s[0])), y, w);
#pragma unroll
                for (int e = 0; e < 8; ++e) n += c[e];
            }
        }
        // ---- running sums over the threads
        const uint32_t ni = scan_up(n, lane);
        const double wi = scan_up(w, lane);
        if (lane == 31) {
            part_n[warp] = ni;
            part_w[warp] = wi;
        }
        __syncthreads();
        const uint32_t pn = scan_up(part_n[lane], lane);
        const double pw = scan_up(part_w[lane], lane);
        const uint32_t bn = __shfl_sync(0xffffffffu, pn - part_n[lane], warp);
        double bw = __shfl_sync(0xffffffffu, pw, max(warp - 1, 0));
        if (warp == 0) bw = 0.0;
        const double up = __shfl_up_sync(0xffffffffu, wi, 1);
        if (tid <= kOwners) {  // (the thread behind the last owner has the sums)
            mail.n[tid] = bn + ni - n;
            mail.w[tid] = lane ? bw + up : bw;
        }
        sync_all<C>();
        // ---- the cuts, and the place: by one warp
        if (rank == 0 && warp == 0) {
            const uint32_t mn = mb + (uint32_t)offsetof(Mail, n), mw = mb + (uint32_t)offsetof(Mail, w);
            uint32_t keep = 0;
            double mass = 0.0;
#pragma unroll
            for (int q = 0; q < C; ++q) {
                keep += ld_u32(addr_in<C>(mn + kOwners * 4u, q));
                mass += ld_f64(addr_in<C>(mw + kOwners * 8u, q));
            }
            uint32_t m_keep = keep;
            double m_mass = mass;
            if (greedy) {
                keep = 1;
            } else {
                if (k > 0 && (uint32_t)k < keep) {
                    const Hit h = locate<C>(hb, mw, mn, wt, [=](uint32_t an, double, int) { return an >= (uint32_t)k; });
                    keep = (uint32_t)k;
                    mass = h.w + double_of((uint32_t)k - h.n) * h.y;
                }
                if (mf > 0.0f) {
                    // the first bin whose weight is below min_p, in (lo, hi]; the top's is 1
                    int lo = (int)top, hi = kBins;
                    if (1.0 < (double)mf) hi = lo;
                    while (hi - lo > 1) {
                        const int step = (hi - lo + 31) >> 5, bin = min(hi, lo + (lane + 1) * step);
                        const bool below = bin >= hi || wt.at(bin) < (double)mf;
                        const int f = __ffs(__ballot_sync(0xffffffffu, below)) - 1;  // the lanes' bins ascend
                        hi = min(hi, lo + (f + 1) * step);
                        lo += f * step;
                    }
                    if (hi < kBins) {
                        const Hit h = locate<C>(hb, mw, mn, wt, [=](uint32_t, double, int bin) { return bin >= hi; });
                        const bool ahead = h.c && h.bin < hi;  // none of the thread's values is behind the cut
                        m_keep = ahead ? h.n + h.c : h.n;
                        m_mass = ahead ? h.w + double_of(h.c) * h.y : h.w;
                    }
                }
                if (pf < 1.0f) {
                    const double goal = fmax((double)pf, 0.0) * mass;
                    const Hit h = locate<C>(hb, mw, mn, wt, [=](uint32_t an, double aw, int) { return an > 0 && aw >= goal; });
                    const double r = goal > 0.0 ? fmin(fmax(ceil((goal - h.w) / h.y), 1.0), double_of(h.c)) : 1.0;
                    const uint32_t cn = h.n + (uint32_t)r;
                    if (cn < keep) {
                        keep = cn;
                        mass = h.w + r * h.y;
                    }
                }
                if (m_keep < keep) {
                    keep = m_keep;
                    mass = m_mass;
                }
            }
            if (keep == 0) keep = 1;  // min_p above 1
            uint32_t pos = 0;
            Hit h;
            const double goal = keep > 1 ? u * mass : 0.0;
            if (goal > 0.0) {
                h = locate<C>(hb, mw, mn, wt, [=](uint32_t, double aw, int) { return aw > goal; });
                pos = h.n + (h.c ? (uint32_t)fmin(fmax(floor((goal - h.w) / h.y), 0.0), double_of(h.c - 1)) : 0);
            }
            if (!(goal > 0.0) || pos >= keep || !h.c) {  // the first; u of 1 or more, or a sum's rounding
                pos = min(pos, keep - 1);
                h = locate<C>(hb, mw, mn, wt, [=](uint32_t an, double, int) { return an > pos; });
            }
            if (lane < C) {
                st_u32(at(lane, &mail.bin), (uint32_t)h.bin);
                st_u32(at(lane, &mail.rank), pos - h.n);
            }
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
            // matches of every warp in every step of the segment, then the step and warp that hold the r-th, then its place
            const int steps = (i1 - i0 + kThreads * 8 - 1) / (kThreads * 8);
            const uint32_t one = bin <= (uint32_t)kZero ? kZero - bin : 0x8000u | (bin - kZero);
            const uint32_t wanted = one | one << 16, mask = one ? 0xffffffffu : 0x7fff7fffu;  // both zeros
            auto matches = [&](int s, int at_warp) {
                const uint4 v = load8(x, i0 + (s * kThreads + at_warp * 32 + lane) * 8, i1, a.vec);
                const uint32_t h[4] = {v.x, v.y, v.z, v.w};
                uint32_t m = 0;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t eq = __vcmpeq2(h[e] & mask, wanted);
                    m |= ((eq & 1u) | (eq >> 30 & 2u)) << (2 * e);
                }
                return m;
            };
            for (int s = 0; s < steps; ++s) {
                const uint32_t c = __reduce_add_sync(0xffffffffu, __popc(matches(s, warp)));
                if (lane == 0) part_n[s * 32 + warp] = c;
            }
            __syncthreads();
            if (warp == 0) {
                uint32_t before = 0;
                for (int s = 0; s < steps; ++s) {
                    const uint32_t c = part_n[s * 32 + lane], in = before + scan_up(c, lane);
                    const uint32_t vote = __ballot_sync(0xffffffffu, in > r);
                    if (vote) {
                        const int l = __ffs(vote) - 1;
                        before = __shfl_sync(0xffffffffu, in - c, l);
                        const uint32_t m = matches(s, l), cm = __popc(m), im = before + scan_up(cm, lane);
                        if (im - cm <= r && r < im)
                            a.ids[row] = i0 + (s * kThreads + l * 32 + lane) * 8 + (int)__fns(m, 0, (int)(r - (im - cm)) + 1);
                        break;
                    }
                    before = __shfl_sync(0xffffffffu, in, 31);
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
    if (vocab > 8 * kMaxSegment || rows > 0x0fffffff) return NPUB_ERR_UNSUPPORTED;
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
    // CTAs of a row.  Measured, one CTA per SM: 11, 14, 15 and 16.5 us with 1, 2, 4 and 8 of them and 1.9 us for every 8192
    // logits of a CTA (32000: 18.4 us alone, 17.6 in two; 128256: 29, 22.6 and 20.1 in 2, 4 and 8; 64 rows of it 29, 49 and 95).
    // Of clusters of 4 and 8 not quite all SMs hold one.
    static const double start[4] = {11.0, 14.0, 15.0, 16.5};
    int c = 8;
    double best = 1e30;
    for (int i = 0; i < 4; ++i) {
        const int n = 1 << i, at_once = num_sms() / n > 4 ? num_sms() / n - (i > 1 ? 3 : 0) : 1;
        if ((vocab + n - 1) / n > kMaxSegment - 8) continue;
        const double us = (double)((rows + at_once - 1) / at_once) * (start[i] + 1.9 * vocab / n / 8192.0);
        if (us < best) {
            best = us;
            c = n;
        }
    }
    a.seg = ((vocab + c - 1) / c + 7) / 8 * 8;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    switch (c) {
        case 1: return launch<1>(a, rows, st);
        case 2: return launch<2>(a, rows, st);
        case 4: return launch<4>(a, rows, st);
        default: return launch<8>(a, rows, st);
    }
}
