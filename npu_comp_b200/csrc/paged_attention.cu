// C entries of the packed and paged attention: argument checks, the choice of
// kernel (fmha_packed.cu: tcgen05 tiles of 128 rows; paged_decode.cu: up to 16
// rows per kv head) and the split of the keys over CTAs.
#include "common.cuh"
#include "fmha_packed.h"
#include "gemm_tc.h"
#include "paged_decode.h"

#include <cmath>

namespace npub {
namespace {

bool dims_ok(int heads, int kv_heads, int head_dim, float scale) {
    return heads > 0 && kv_heads > 0 && heads % kv_heads == 0 && head_dim > 0 && head_dim % 16 == 0 && scale > 0.0f &&
           std::isfinite(scale);
}

// What the tile kernels implement beyond dims_ok: heads that fit two 64-column
// chunks, groups that fit a tile, and at most 65535 heads.
bool dims_supported(int heads, int kv_heads, int head_dim) {
    return head_dim <= 128 && heads / kv_heads <= 128 && heads <= 65535;
}

bool pool_ok(const void* k, const void* v, int n_pages, int page_size, const int32_t* table, int64_t ldt,
             int max_pages) {
    return k && v && table && n_pages > 0 && page_size >= 16 && page_size <= 256 &&
           (page_size & (page_size - 1)) == 0 && max_pages > 0 && ldt >= max_pages && npub_aligned(k, 16) &&
           npub_aligned(v, 16);
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// How the keys of a call are cut.  The partials are numbered through: the shared prefix's, then those of the sequences'
// own keys.  The ranges are equal parts of what each sequence holds, so ctx_len only decides their number.
struct Phase {
    int tiles, dual;  // tile kernel: rows of an item, and whether its keys go in two halves
    int splits;
    bool cluster;     // paged_decode combines its ranges itself
    double us;        // the estimate
    int64_t ctas;     // tile kernel: items of all ranges
    int partials() const { return splits * (dual ? 2 : 1); }
};
struct Plan {
    bool few;    // own keys on paged_decode (else on the tiles)
    int shared;  // keys of the shared prefix phase (0: none)
    Phase pre, own;
    int total() const { return (shared > 0 ? pre.partials() : 0) + own.partials(); }
    bool part() const { return total() > 1 && !own.cluster; }
};

// What a kernel takes, in us: `first` to start, then per item `item` and `unit_us` for every `unit` keys.
struct Cost {
    double first, item, unit_us;
    int unit;
};

// The number of key ranges s <= most for `items` items of up to `keys` keys on `slots` resident CTAs that makes the
// estimate below smallest.  `range_us`: what one more range's partials cost (written, read); `fixed`: a combination
// pass runs anyway, else it adds `pass_us` where there is more than one partial (`per` of them for a range).
//   equal   items of one length, in waves: first + waves * (item + range)
//   ragged  lengths below `keys` (0.7 of it on average), CTAs taken in order as slots come free: the work over the
//           slots and half of the longest CTA, or that CTA where the slots are not filled
struct Split {
    int s;
    double us;
};
Split pick_splits(int64_t keys, int64_t items, int64_t slots, const Cost& c, bool ragged, int most, double range_us,
                  int per, bool fixed, double pass_us) {
    const int64_t units = ceil_div(keys > 0 ? keys : 1, c.unit);
    Split best = {1, 0.0};
    for (int s = 1; s <= most && s <= units; ++s) {
        const double cta = c.item + (double)ceil_div(units, s) * c.unit_us;
        double t;
        if (ragged) {
            const double bulk = (double)items * (s * c.item + 0.7 * (double)units * c.unit_us) / (double)slots;
            t = bulk + 0.5 * cta > cta ? bulk + 0.5 * cta : cta;
        } else {
            t = (double)ceil_div(items * s, slots) * cta;
        }
        t += c.first;
        if (s * per > 1 || fixed) t += s * per * range_us + (fixed ? 0.0 : pass_us);
        if (s == 1 || t < 0.97 * best.us) best = Split{s, t};
    }
    return best;
}

// A phase on the tile kernel (measured: 7 us to start, 2 us to change items, 1.6 us per 128 keys of a pair of tiles),
// on `slots` SMs: pairs of tiles, or, where the rows fill one tile, one tile on two halves of the keys.
Phase tile_phase(int total, int batch, int heads, int kv_heads, int max_new, int64_t keys, int64_t slots,
                 double part_us, bool fixed) {
    const int64_t one = fmha_packed_items(total, batch, heads, kv_heads, max_new, 1) * kv_heads;
    const int64_t two = fmha_packed_items(total, batch, heads, kv_heads, max_new, 2) * kv_heads;
    Phase a = {}, b = {};
    const double range_us = part_us + 0.15;
    const Split sa = pick_splits(keys, two, slots, Cost{7.0, 2.0, 1.6, 128}, false, 64, range_us, 1, fixed, 4.0);
    const Split sb = pick_splits(keys, one, slots, Cost{7.0, 2.0, 1.6, 256}, false, 64, range_us, 2, fixed, 4.0);
    a.tiles = sa.s == 1 && !fixed ? 0 : 2;
    a.splits = sa.s;
    a.us = sa.us;
    a.ctas = two * sa.s;
    b.tiles = 1;
    b.dual = 1;
    b.splits = sb.s;
    b.us = sb.us;
    b.ctas = one * sb.s;
    return sb.us < sa.us ? b : a;
}

// The few-row kernel on up to `keys` keys of each sequence; behind: a shared
// prefix's partials are combined with its own.  One of its CTAs, two of which
// share an SM, takes 4 us (in a cluster 5) and 3 us per 128 keys of 128 columns.
Phase few_phase(int batch, int kv_heads, int head_dim, int64_t keys, double part_us, bool behind) {
    const Cost c = {0.0, 4.0, head_dim > 64 ? 3.0 : 1.6, 128}, cc = {0.0, 5.0, c.unit_us, 128};
    const bool ragged = batch > 1;
    const int64_t items = (int64_t)batch * kv_heads, slots = 2 * num_sms();
    Phase ph = {};
    const Split sp = pick_splits(keys, items, slots, c, ragged, 64, part_us + 0.15, 1, behind, 4.0);
    ph.splits = sp.s;
    ph.us = sp.us;
    if (!behind) {
        const Split sc = pick_splits(keys, items, slots, cc, ragged, kPagedDecodeCluster, 0.0, 1, true, 0.0);
        if (sc.us <= sp.us) {
            ph.splits = sc.s;
            ph.us = sc.us;
            ph.cluster = true;
        }
    }
    return ph;
}

Plan make_plan(int batch, int total, int max_new, int64_t ctx, int shared, int heads, int kv_heads, int head_dim) {
    Plan pl = {};
    const int group = heads / kv_heads, sms = num_sms();
    pl.few = max_new > 0 && (int64_t)max_new * group <= kPagedDecodeRows && batch <= 65535;
    const double part_us = (double)total * heads * head_dim * 8.0 / 4e6;  // about 4 TB/s: they stay in L2
    auto own = [&](int64_t keys, bool behind) {
        return pl.few ? few_phase(batch, kv_heads, head_dim, keys, part_us, behind)
                      : tile_phase(total, batch, heads, kv_heads, max_new, keys, sms, part_us, behind);
    };
    pl.own = own(ctx, false);
    if (shared <= 0 || batch < 2) return pl;  // nothing to share
    // The prefix phase takes a part of the SMs and the own keys run beside it on the others, then on all: together
    // they take the longer of the prefix's time and the sum of both phases' shares of the SMs, and 4 us to combine.
    // It is left out where the few-row kernel is estimated to read the prefix for every sequence as quickly (through row
    // 0 of the table; the same look-up in the tile kernel costs chunks of prompts 1 %).  Measured, 32 / 8 heads
    // of 128, with the phase and without: 2 sequences of 100 own keys behind 512 keys 9.4 and 6.8 us, 64 of 200 behind
    // 128 22.7 and 18.7, 16 of 200 behind 2048 15.0 and 25.3.  (The estimate without it takes no account of the L2,
    // from which all but the first read the prefix: near the border it keeps the phase, 4 sequences behind 4096 16.6
    // and 13.0.)  Its SMs: 64 sequences of 100 own keys behind 131072 take 213 us on half of them, 163 on all;
    // 64 of 265 behind 8192 36 on half, 46 on all.
    double best = pl.few ? pl.own.us : 1e30;
    const Phase mine = own(ctx > shared ? ctx - shared : 1, true);
    for (int quarters = 2; quarters <= 4; ++quarters) {
        const Phase pre = tile_phase(total, 1, heads, kv_heads, 0, shared, sms * quarters / 4, part_us, true);
        const double both = mine.us + pre.us * (pre.ctas < sms ? (double)pre.ctas / sms : 1.0);
        const double us = 4.0 + (pre.us > both ? pre.us : both);
        if (us < best) {
            best = us;
            pl.shared = shared;
            pl.pre = pre;
            pl.own = mine;
        }
        if (pre.us <= both) break;  // more SMs for the prefix would only take them from the own keys
    }
    return pl;
}

size_t plan_bytes(const Plan& pl, int total, int heads, int head_dim) {
    if (!pl.part()) return 0;
    const size_t n = (size_t)pl.total() * total * heads;
    return (n * sizeof(float2) + 255) / 256 * 256 + n * head_dim * sizeof(float);
}

int run_plan(const Plan& pl, PackedArgs& a, void* workspace, size_t workspace_bytes, cudaStream_t st) {
    const size_t need = plan_bytes(pl, a.total_q, a.heads, a.head_dim);
    if (need) {
        if (!workspace || workspace_bytes < need) return NPUB_ERR_WORKSPACE;
        NPUB_CHECK_ARG(npub_aligned(workspace, 256));
        const size_t n = (size_t)pl.total() * a.total_q * a.heads;
        a.part_ml = reinterpret_cast<float2*>(workspace);
        a.part_o = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + (n * sizeof(float2) + 255) / 256 * 256);
    }
    if (pl.shared > 0) {
        PackedArgs s = a;
        s.shared = pl.shared;
        s.causal = 0;
        s.cu = nullptr;
        s.splits = pl.pre.splits;
        s.tiles = pl.pre.tiles;
        s.dual = pl.pre.dual;
        const int rc = fmha_packed(s, st);
        if (rc) return rc;
    }
    a.first = pl.shared;
    a.splits = pl.own.splits;
    a.tiles = pl.own.tiles;
    a.dual = pl.own.dual;
    a.split0 = pl.shared > 0 ? pl.pre.partials() : 0;
    const int rc = pl.few ? paged_decode(a, st) : fmha_packed(a, st);
    if (rc || !need) return rc;
    return paged_combine(a, pl.total(), st);
}

}  // namespace
}  // namespace npub

extern "C" int npub_attention_packed(const void* q, int64_t ldq, const void* k, int64_t ldk, const void* v,
                                     int64_t ldv, void* out, int64_t ldo, const int32_t* cu_seqlens, int batch,
                                     int total, int heads, int kv_heads, int head_dim, float scale,
                                     int causal, void* stream) {
    using namespace npub;
    NPUB_CHECK_ARG(batch >= 0 && total >= 0 && dims_ok(heads, kv_heads, head_dim, scale));
    if (batch == 0 || total == 0) return NPUB_OK;
    NPUB_CHECK_ARG(q && k && v && out && cu_seqlens);
    if (!dims_supported(heads, kv_heads, head_dim)) return NPUB_ERR_UNSUPPORTED;
    NPUB_CHECK_ARG(ldq % 8 == 0 && ldk % 8 == 0 && ldv % 8 == 0 && ldo % 8 == 0);
    NPUB_CHECK_ARG(ldq >= (int64_t)heads * head_dim && ldk >= (int64_t)kv_heads * head_dim &&
                   ldv >= (int64_t)kv_heads * head_dim && ldo >= (int64_t)heads * head_dim);
    NPUB_CHECK_ARG(npub_aligned(q, 16) && npub_aligned(k, 16) && npub_aligned(v, 16) && npub_aligned(out, 16));
    PackedArgs a = {};
    a.q = q;
    a.ldq = ldq;
    a.out = out;
    a.ldo = ldo;
    a.kv.k = k;
    a.kv.v = v;
    a.kv.ldk = ldk;
    a.kv.ldv = ldv;
    a.cu = cu_seqlens;
    a.total_q = total;
    a.batch = batch;
    a.heads = heads;
    a.kv_heads = kv_heads;
    a.head_dim = head_dim;
    a.scale = scale;
    a.causal = causal;
    return fmha_packed(a, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int npub_attention_paged(const void* q, int64_t ldq, const void* k_pages, const void* v_pages, int n_pages,
                                    int page_size, const int32_t* page_table, int64_t ldt, int max_pages,
                                    const int32_t* lens, const int32_t* cu_seqlens, int batch, int total, int max_new,
                                    int ctx_len, void* out, int64_t ldo, int heads, int kv_heads, int head_dim,
                                    float scale, int causal, void* workspace, size_t workspace_bytes, void* stream) {
    using namespace npub;
    NPUB_CHECK_ARG(batch >= 0 && total >= 0 && max_new >= 0 && ctx_len >= 0 &&
                   dims_ok(heads, kv_heads, head_dim, scale));
    if (batch == 0 || total == 0) return NPUB_OK;
    NPUB_CHECK_ARG(q && out && lens && cu_seqlens &&
                   pool_ok(k_pages, v_pages, n_pages, page_size, page_table, ldt, max_pages));
    if (!dims_supported(heads, kv_heads, head_dim)) return NPUB_ERR_UNSUPPORTED;
    NPUB_CHECK_ARG(ldq % 8 == 0 && ldo % 8 == 0 && ldq >= (int64_t)heads * head_dim &&
                   ldo >= (int64_t)heads * head_dim && npub_aligned(q, 16) && npub_aligned(out, 16));
    PackedArgs a = {};
    a.q = q;
    a.ldq = ldq;
    a.out = out;
    a.ldo = ldo;
    a.kv.k = k_pages;
    a.kv.v = v_pages;
    a.kv.table = page_table;
    a.kv.ldt = ldt;
    a.kv.max_pages = max_pages;
    a.kv.n_pages = n_pages;
    a.kv.page_size = page_size;
    a.cu = cu_seqlens;
    a.lens = lens;
    a.total_q = total;
    a.batch = batch;
    a.heads = heads;
    a.kv_heads = kv_heads;
    a.head_dim = head_dim;
    a.scale = scale;
    a.causal = causal;
    const int64_t cap = (int64_t)max_pages * page_size;
    const Plan pl = make_plan(batch, total, max_new, ctx_len > 0 && ctx_len < cap ? ctx_len : cap, 0, heads, kv_heads,
                              head_dim);
    return run_plan(pl, a, workspace, workspace_bytes, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" size_t npub_attention_paged_workspace(int batch, int total, int max_new, int64_t ctx_len, int heads,
                                                 int kv_heads, int head_dim) {
    using namespace npub;
    if (batch <= 0 || total <= 0 || max_new < 0 || ctx_len < 0 || !dims_ok(heads, kv_heads, head_dim, 1.0f) ||
        !dims_supported(heads, kv_heads, head_dim))
        return 0;
    return plan_bytes(make_plan(batch, total, max_new, ctx_len, 0, heads, kv_heads, head_dim), total, heads, head_dim);
}

extern "C" int npub_attention_paged_decode(const void* q, int64_t ldq, const void* k_pages, const void* v_pages,
                                           int n_pages, int page_size, const int32_t* page_table, int64_t ldt,
                                           int max_pages, const int32_t* lens, int batch, int ctx_len, int shared_len,
                                           void* out, int64_t ldo, int heads, int kv_heads, int head_dim, float scale,
                                           void* workspace, size_t workspace_bytes, void* stream) {
    using namespace npub;
    NPUB_CHECK_ARG(batch >= 0 && ctx_len >= 0 && shared_len >= 0 && dims_ok(heads, kv_heads, head_dim, scale));
    if (batch == 0) return NPUB_OK;
    NPUB_CHECK_ARG(q && out && lens && pool_ok(k_pages, v_pages, n_pages, page_size, page_table, ldt, max_pages));
    NPUB_CHECK_ARG(shared_len % page_size == 0 && shared_len <= (int64_t)max_pages * page_size);
    if (!dims_supported(heads, kv_heads, head_dim) || batch > 65535) return NPUB_ERR_UNSUPPORTED;
    NPUB_CHECK_ARG(ldq % 8 == 0 && ldo % 8 == 0 && ldq >= (int64_t)heads * head_dim &&
                   ldo >= (int64_t)heads * head_dim && npub_aligned(q, 16) && npub_aligned(out, 16));
    PackedArgs a = {};
    a.q = q;
    a.ldq = ldq;
    a.out = out;
    a.ldo = ldo;
    a.kv.k = k_pages;
    a.kv.v = v_pages;
    a.kv.table = page_table;
    a.kv.ldt = ldt;
    a.kv.max_pages = max_pages;
    a.kv.n_pages = n_pages;
    a.kv.page_size = page_size;
    a.kv.common = shared_len;
    a.lens = lens;
    a.total_q = batch;
    a.batch = batch;
    a.heads = heads;
    a.kv_heads = kv_heads;
    a.head_dim = head_dim;
    a.scale = scale;
    a.causal = 1;
    const int64_t cap = (int64_t)max_pages * page_size;
    const Plan pl = make_plan(batch, batch, 1, ctx_len > 0 && ctx_len < cap ? ctx_len : cap, shared_len, heads,
                              kv_heads, head_dim);
    return run_plan(pl, a, workspace, workspace_bytes, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" size_t npub_attention_paged_decode_workspace(int batch, int64_t ctx_len, int shared_len, int heads,
                                                        int kv_heads, int head_dim) {
    using namespace npub;
    if (batch <= 0 || ctx_len < 0 || shared_len < 0 || !dims_ok(heads, kv_heads, head_dim, 1.0f) ||
        !dims_supported(heads, kv_heads, head_dim))
        return 0;
    return plan_bytes(make_plan(batch, batch, 1, ctx_len, shared_len, heads, kv_heads, head_dim), batch, heads, head_dim);
}
