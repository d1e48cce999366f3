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

// Over 8-bit pages: few rows on paged_decode_q8.cu, more of them on the tile kernel behind a pass that writes the keys as
// fp16 pages.  Measured on 70001 keys, 32 / 8 heads of 128, ragged rows, with the tiles of the longest sequence, as they
// are and behind the pass: 24 sequences of 6 tiles 88 and 153 us, of 9 tiles 142 and 169, of 14 tiles 226 and 173; 4
// sequences of 5 tiles 133 and 156, of 10 tiles 220 and 160.
constexpr int kQ8Tiles = 8;
// Bytes of the fp16 copy (one sequence's at least): the sequences take turns in it, each group of them behind the one before.
// Measured, 32 / 8 heads of 128, all sequences at once, groups of 4, 2 and 1 GiB: 16 of 65000 keys (4 GiB at once) 3330, 3391,
// 3339 and 4137 us; one of 65000 and 15 of 3000 697, 669, 735 and 969; 64 of 1000 keys in a table of 131072 (32 GiB) without
// ctx_len 1098, 1650, 2442 and 5200, with it 231.
constexpr int64_t kQ8Copy = (int64_t)1 << 31;
struct PlanQ8 {
    Plan p;
    int tiles, rows;              // paged_decode_q8: tiles of a sequence and kv head, and the rows of one
    int width, seqs;              // tile kernel: fp16 pages of 128 keys per sequence, sequences of a group
    bool list;                    // paged_list_q8 instead
    size_t parts, pages, scales, tables;  // bytes of the partials, of the fp16 K (or V), of two scales for 16 keys, and
                                          // of the table and lengths
    size_t bytes() const { return parts + 2 * pages + scales + tables; }
};

PlanQ8 make_plan_q8(int batch, int total, int max_new, int64_t ctx, int heads, int kv_heads, int head_dim) {
    PlanQ8 pl = {};
    const int group = heads / kv_heads;
    const double part_us = (double)total * heads * head_dim * 8.0 / 4e6;
    if (max_new > 0) {
        const int64_t rows = (int64_t)max_new * group;
        pl.rows = rows <= 8 ? 8 : kPagedDecodeRows;
        if (ceil_div(rows, pl.rows) <= kQ8Tiles) pl.tiles = (int)ceil_div(rows, pl.rows);
    }
    pl.p.few = pl.tiles > 0;
    if (pl.p.few) {
        const int64_t items = (int64_t)batch * kv_heads * pl.tiles, blocks = ceil_div(ctx, 128);
        // resident CTAs of the cluster kernel; ranges while they hold all of it at once
        const int64_t slots = (pl.rows == 8 ? 3 : 2) * num_sms();
        int64_t splits = slots / items;
        if (splits > kPagedDecodeCluster) splits = kPagedDecodeCluster;
        if (splits > blocks) splits = blocks;
        if (splits < 1) splits = 1;
        // The list takes two launches and 12 us for the smallest call, the cluster kernel 6 us and 1 to 1.5 us for each
        // block of 128 keys that its fullest slot takes (the largest sequence's share: it is not balanced).  Measured, 32 / 8
        // heads of 128, cluster and list: one sequence of 4096 keys 8.9 and 12.3 us, of 16384 21.9 and 17.1; 16 sequences of
        // 16400 keys 14.6 and 19.2, of 65000 43 and 36; 64 of 16400 16.2 and 18.4, of 65000 56 and 36.
        pl.list = ceil_div(blocks, splits) * (items * splits > slots ? items * splits : slots) > 10 * slots;
        pl.p.own.splits = (int)splits;
        pl.p.own.cluster = true;
        if (pl.list) pl.parts = paged_list_q8_workspace(batch, kv_heads, head_dim, pl.rows, pl.tiles);
        return pl;
    } else {
        const int64_t width = ceil_div(ctx, 128);
        pl.width = width > 0x7fffffff ? 0x7fffffff : (int)width;
        const int64_t copy = width * kv_heads * 128 * head_dim * (int64_t)sizeof(__half);  // of a sequence's K
        const int64_t meta = width * kv_heads * 8 * (int64_t)sizeof(float2), ids = (width + 1) * (int64_t)sizeof(int32_t);
        int64_t most = kQ8Copy / (2 * copy + meta + ids);
        if (most < 1) most = 1;
        const int64_t groups = ceil_div(batch, most);
        pl.seqs = (int)ceil_div(batch, groups);
        pl.pages = (size_t)(pl.seqs * copy);
        pl.scales = ((size_t)(pl.seqs * meta) + 255) / 256 * 256;
        pl.tables = ((size_t)(pl.seqs * ids) + 255) / 256 * 256;
        // a group has its share of the rows, but its partials are numbered through all of them
        pl.p.own = tile_phase((int)ceil_div(total, groups), pl.seqs, heads, kv_heads, max_new, ctx, num_sms(), part_us, false);
    }
    pl.parts = (plan_bytes(pl.p, total, heads, head_dim) + 255) / 256 * 256;
    return pl;
}

int run_plan_q8(const PlanQ8& pl, PackedArgs& a, const float* ks, const float* vs, void* workspace, size_t workspace_bytes,
                cudaStream_t st) {
    if (a.batch > 65535 || a.kv_heads > 65535) return NPUB_ERR_UNSUPPORTED;
    if (pl.bytes()) {
        if (!workspace || workspace_bytes < pl.bytes()) return NPUB_ERR_WORKSPACE;
        NPUB_CHECK_ARG(npub_aligned(workspace, 256));
    }
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    if (!pl.p.few) {
        if ((int64_t)pl.seqs * pl.width > 0x7fffffff) return NPUB_ERR_UNSUPPORTED;
        uint8_t *k = ws + pl.parts, *v = k + pl.pages;
        float2* key_scale = reinterpret_cast<float2*>(v + pl.pages);
        int32_t* table = reinterpret_cast<int32_t*>(v + pl.pages + pl.scales);
        int32_t* lens = table + (int64_t)pl.seqs * pl.width;
        for (int b0 = 0; b0 < a.batch; b0 += pl.seqs) {
            PackedArgs g = a;  // sequences b0 .. : rows outside of their offsets are left as they are
            g.batch = a.batch - b0 < pl.seqs ? a.batch - b0 : pl.seqs;
            g.cu = a.cu + b0;
            g.lens = a.lens + b0;
            g.kv.table = a.kv.table + b0 * a.kv.ldt;
            int rc = expand_q8(g, ks, vs, pl.width, k, v, table, lens, key_scale, st);
            if (rc) return rc;
            g.key_scale = key_scale;
            g.scale = 0.6931472f;  // of exponents of 2, where partials are joined
            g.kv.k = k;
            g.kv.v = v;
            g.kv.table = table;
            g.kv.ldt = g.kv.max_pages = pl.width;
            g.kv.n_pages = g.batch * pl.width;
            g.kv.page_size = 128;
            g.lens = lens;
            rc = run_plan(pl.p, g, workspace, pl.parts, st);
            if (rc) return rc;
        }
        return NPUB_OK;
    }
    if (pl.list) return paged_list_q8(a, ks, vs, pl.rows, pl.tiles, workspace, st);
    a.splits = pl.p.own.splits;
    return paged_decode_q8(a, ks, vs, pl.rows, pl.tiles, st);
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

extern "C" int npub_attention_paged_q8(const void* q, int64_t ldq, const int8_t* k_pages, const int8_t* v_pages,
                                       const float* k_scales, const float* v_scales, int n_pages, int page_size,
                                       const int32_t* page_table, int64_t ldt, int max_pages, const int32_t* lens,
                                       const int32_t* cu_seqlens, int batch, int total, int max_new, int ctx_len,
                                       void* out, int64_t ldo, int heads, int kv_heads, int head_dim, float scale,
                                       int causal, void* workspace, size_t workspace_bytes, void* stream) {
    using namespace npub;
    NPUB_CHECK_ARG(batch >= 0 && total >= 0 && max_new >= 0 && ctx_len >= 0 &&
                   dims_ok(heads, kv_heads, head_dim, scale));
    if (batch == 0 || total == 0) return NPUB_OK;
    NPUB_CHECK_ARG(q && out && lens && cu_seqlens &&
                   pool_ok(k_pages, v_pages, n_pages, page_size, page_table, ldt, max_pages));
    NPUB_CHECK_ARG(k_scales && v_scales && npub_aligned(k_scales, 4) && npub_aligned(v_scales, 4));
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
    const PlanQ8 pl = make_plan_q8(batch, total, max_new, ctx_len > 0 && ctx_len < cap ? ctx_len : cap, heads, kv_heads,
                                   head_dim);
    return run_plan_q8(pl, a, k_scales, v_scales, workspace, workspace_bytes, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" size_t npub_attention_paged_q8_workspace(int batch, int total, int max_new, int64_t ctx_len, int heads,
                                                    int kv_heads, int head_dim) {
    using namespace npub;
    if (batch <= 0 || total <= 0 || max_new < 0 || ctx_len < 0 || !dims_ok(heads, kv_heads, head_dim, 1.0f) ||
        !dims_supported(heads, kv_heads, head_dim))
        return 0;
    return make_plan_q8(batch, total, max_new, ctx_len, heads, kv_heads, head_dim).bytes();
}

extern "C" int npub_attention_paged_decode_q8(const void* q, int64_t ldq, const int8_t* k_pages, const int8_t* v_pages,
                                              const float* k_scales, const float* v_scales, int n_pages, int page_size,
                                              const int32_t* page_table, int64_t ldt, int max_pages, const int32_t* lens,
                                              int batch, int ctx_len, void* out, int64_t ldo, int heads, int kv_heads,
                                              int head_dim, float scale, void* workspace, size_t workspace_bytes,
                                              void* stream) {
    using namespace npub;
    NPUB_CHECK_ARG(batch >= 0 && ctx_len >= 0 && dims_ok(heads, kv_heads, head_dim, scale));
    if (batch == 0) return NPUB_OK;
    NPUB_CHECK_ARG(q && out && lens && pool_ok(k_pages, v_pages, n_pages, page_size, page_table, ldt, max_pages));
    NPUB_CHECK_ARG(k_scales && v_scales && npub_aligned(k_scales, 4) && npub_aligned(v_scales, 4));
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
    a.lens = lens;
    a.total_q = batch;
    a.batch = batch;
    a.heads = heads;
    a.kv_heads = kv_heads;
    a.head_dim = head_dim;
    a.scale = scale;
    a.causal = 1;
    const int64_t cap = (int64_t)max_pages * page_size;
    const PlanQ8 pl = make_plan_q8(batch, batch, 1, ctx_len > 0 && ctx_len < cap ? ctx_len : cap, heads, kv_heads, head_dim);
    return run_plan_q8(pl, a, k_scales, v_scales, workspace, workspace_bytes, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" size_t npub_attention_paged_decode_q8_workspace(int batch, int64_t ctx_len, int heads, int kv_heads,
                                                           int head_dim) {
    using namespace npub;
    if (batch <= 0 || ctx_len < 0 || !dims_ok(heads, kv_heads, head_dim, 1.0f) || !dims_supported(heads, kv_heads, head_dim))
        return 0;
    return make_plan_q8(batch, batch, 1, ctx_len, heads, kv_heads, head_dim).bytes();
}
