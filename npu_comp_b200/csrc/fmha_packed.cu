// Attention of packed (ragged) query rows over packed K/V rows or a paged KV
// cache, grouped heads, head_dim <= 128, on sm_100a.
//
// O = softmax(scale Q K^T + mask) V per sequence and head, the attention of
// b_program_examples/llama_layer.py:114-137 in the max-subtracted form of
// d_compiler/npu_compiler/model.py:145-150.  Query row i of a sequence with n
// new rows and m keys sees keys 0 .. m - n + i (all m without the causal
// mask); a row that sees no key gives zeros.
//
// A tile is 128 rows of one kv head: row r = (token r / G, head r % G) of its
// G query heads, so that the group shares every K/V load and a prompt of few
// tokens still fills rows.  A CTA takes two tiles, which share K and V:
//   S_q(j) = Q_q K_j^T          tcgen05.mma, fp32 in TMEM
//   P_q(j) = exp2(S c - m c)    one thread per row; fp16, over S_q's own TMEM columns (both operands of a kind::f16
//                               MMA are fp16, as V is: half a step, 2^-11 of each weight; sums, S and O are fp32)
//   O_q   += P_q(j) V_j         tcgen05.mma with A = P from TMEM, V read MN-major
// O stays in TMEM over the whole key loop.  A row's reference maximum m moves
// (and its O and sum are rescaled) only when the row maximum has grown by more
// than 2^8: P then stays below 2^8, far inside fp16, and the rescale, which
// reads and writes the O tile, is rare.  The tensor core works on one tile
// while the other is in its softmax; P is handed over in two halves of 64 keys.
//
// What bounds it (clock64 stamps in one CTA, 8192 causal tokens, 32/8 heads):
// at head_dim 128 a pair of tiles takes 2820 cycles per key block, of which
// the tensor core runs 2048 (0.73; over the whole kernel, with its start, item
// changes and end, 0.62); a tile's chain is its softmax (1850: 160 to read
// S, 440 for the maximum and the rescale test, 1250 for the exponentials) and
// then the second half of P V and the next S.  One call after the other it takes
// 507-514 us, 1080 TFLOP/s: 0.65 of the burst rate, 0.76 of the sustained one,
// with the clock at 1.57 GHz under the power limit.  At head_dim 64 (414 us,
// 660 TFLOP/s) the products are half as long and the
// exponentials bound it (16 per cycle and SM), so a quarter of them runs as a
// polynomial on the FMA pipe there.  The pairs of times from here on compare
// two builds of their day in short runs at a higher clock: the polynomial 437
// against 469 us; at head_dim 128 it only costs issue slots and power (462 / 458
// us).  Tried and left out: P beside S at head_dim 64, so that the next S is formed during the
// softmax (8192 tokens 207 -> 204 us, twelve ragged prompts 48 -> 51); two
// threads per row, 16 softmax warps (454 -> 495-553 us, 48 -> 56: the pairs'
// exchange and the second read of S, which 104 registers force); the
// exponentials formed with the old maximum while the new one is found (458 ->
// 487 us: spills); P handed over as 96 + 32 keys (no difference); the output
// through shared memory.
// The MMA thread is one elected thread for the whole loop: issuing from
// "lane 0" branches of a warp cost 90-130 cycles per MMA (606 us) where the
// tensor core needs 64.
//
// Keys past a sequence's end inside its last 128-key block are whatever lies
// behind them (the next sequence's rows, a page's stale slots): their scores
// are masked by a select, and their V rows are zeroed in shared memory before
// the product, since 0 * NaN and 0 * inf are NaN.
//
// Roles (384 threads): warps 0-3 and 4-7 softmax and output of tile 0 and 1,
// warp 8 TMA, warp 9 tensor-memory allocation and MMA issue (one thread), warp
// 10 the scheduler of this CTA's items (persistent grid), warp 11 the zeroing
// of V rows behind the last key.
#include "common.cuh"
#include "f32x2.cuh"
#include "fmha_packed.h"
#include "gemm_tc.h"

#include <cmath>

namespace npub {
namespace fpk {

constexpr int kThreads = 384;
constexpr int kBlk = 128;  // keys per block
constexpr int kRows = 128;

template <int HD>
struct Smem {
    static constexpr int kChunks = HD / 64;
    static constexpr int kChunk = 128 * 128;           // 128 rows of one swizzled 128-byte row each
    static constexpr int kTile = kChunks * kChunk;     // one K, V or Q tile
    static constexpr int kStages = HD == 128 ? 5 : 10;  // ring of K and V tiles
    static constexpr int kOffQ = 0;
    static constexpr int kOffRing = 2 * kTile;
    static constexpr int kOffBar = kOffRing + kStages * kTile;
    static constexpr int kOffItem = kOffBar + 384;
    static constexpr int kTotal = kOffItem + 256;
    static_assert(kTotal <= 232448, "shared memory budget");
};

struct Params {
    CUtensorMap tmQ, tmK, tmV;
    const int32_t *cu, *lens, *table;
    int64_t ldt;
    int max_keys, page_shift, box_rows, n_pages;
    int total_q, batch, heads, kv_heads, group, tpt, head_dim;
    uint32_t span_inv;  // ceil(2^32 / (tiles * tpt)), 2^32 - 1 for 1
    int tiles, n_items, sorted, splits, first, split0, shared, causal;
    float c;  // scale * log2(e)
    const float2* key_scale;  // SCALED (PackedArgs)
    __half* out;
    int64_t ldo;
    int out32;  // output rows are 32-byte aligned
    float* part_o;
    float2* part_ml;
    int* err;
};

struct Item {
    int q_row0;      // first row of the sequence
    int ntok, tok0;  // rows of the sequence, first row of tile 0
    int kv_row0;     // packed K/V: first row of the sequence
    int seq, kvh, split;
    int off;         // row i sees keys <= off + i
    int kb[2];       // first key of each tile's range
    int ke[2];       // its end
    int n[2];        // key blocks of each tile
    int steps[2];    // 16-key steps of its last block
    int vfix;        // keys of the last block when V rows behind them need zeroing, else 0
    int vfix_q;      // its tile (two ranges)
    int state;       // 1: an item, 0: the last one is behind
};
constexpr int kItemSlots = 2;  // the scheduler works one item ahead

__device__ __forceinline__ void set_err(int* err, int code) {
    if (err) atomicCAS(err, 0, code);
}

// Rows of a sequence, [r0, r1), and its keys.
struct SeqRows {
    int r0, r1, klen;
};
// Those of sequence b (none past the batch).  Reads cu and lens as they are:
// whatever they hold, rows stay inside [0, total_q) and keys inside the table.
template <bool PAGED>
__device__ __forceinline__ SeqRows seq_rows(const Params& p, int b) {
    SeqRows r = {0, 0, 0};
    if (b < p.batch) {
        r.r0 = p.cu ? max(0, min(p.total_q, __ldg(p.cu + b))) : b;
        r.r1 = p.cu ? max(r.r0, min(p.total_q, __ldg(p.cu + b + 1))) : r.r0 + 1;
        r.klen = PAGED ? max(0, min(p.max_keys, __ldg(p.lens + b))) : r.r1 - r.r0;
    }
    return r;
}

// Tiles of a sequence that reach into key block `level` or behind it: tile t
// ends at key off + (t + 1) * span (a causal tile's cost; others all cost the
// same and count as level 0).
__device__ __forceinline__ int tiles_from(const Params& p, int ntok, int klen, int level, int span) {
    const int nt = (ntok + span - 1) / span;
    if (level <= 0) return nt;
    if (!p.causal) return 0;
    const int64_t first = (int64_t)level * kBlk - (klen - ntok);  // rows behind this one reach the level
    if (first <= 0) return nt;
    if (first >= ntok) return 0;
    uint32_t t = __umulhi((uint32_t)first, p.span_inv);  // first / span, at most one off
    if (t * (uint32_t)span > (uint32_t)first) --t;
    else if ((uint32_t)first - t * (uint32_t)span >= (uint32_t)span) ++t;
    return nt - (int)t;
}

// Key blocks of the item's keys [k0, kend): the same for both tiles, or (DUAL)
// one half for each, and what the last ones need.  lim[q]: keys that some row
// of tile q may see end here; used[q]: the tile has rows.
template <bool DUAL>
__device__ __forceinline__ void cut_item(Item& it, int k0, int kend, const int (&lim)[2], const bool (&used)[2]) {
    const int mid = DUAL ? min(kend, k0 + ((kend - k0 + kBlk - 1) / kBlk + 1) / 2 * kBlk) : kend;
    it.vfix = it.vfix_q = 0;
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        it.kb[q] = DUAL && q ? mid : k0;
        it.ke[q] = DUAL && !q ? mid : kend;
        const int end = min(lim[q], it.ke[q]);
        it.n[q] = used[q] && end > it.kb[q] ? (end - it.kb[q] + kBlk - 1) / kBlk : 0;
        it.steps[q] = min(kBlk / 16, (end - it.kb[q] - (it.n[q] - 1) * kBlk + 15) >> 4);
    }
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        const int nb = DUAL ? it.n[q] : max(it.n[0], it.n[1]);
        const int vb = it.ke[q] - it.kb[q] - (nb - 1) * kBlk;  // > 128: the causal limit ends the range earlier
        if (nb > 0 && vb < kBlk && (vb & 15)) {
            it.vfix = vb;
            it.vfix_q = q;
        }
    }
}

// Tiles of the whole batch that reach into `level` or behind it, by a warp;
// near: the lane's own of the first 32 sequences.
template <bool PAGED>
__device__ __forceinline__ int batch_tiles_from(const Params& p, const SeqRows& near, int level, int span) {
    int sum = tiles_from(p, near.r1 - near.r0, near.klen, level, span);
#pragma unroll 1
    for (int b = 32 + (threadIdx.x & 31); b - (int)(threadIdx.x & 31) < p.batch; b += 32) {
        const SeqRows r = seq_rows<PAGED>(p, b);
        sum += tiles_from(p, r.r1 - r.r0, r.klen, level, span);
    }
    return __reduce_add_sync(0xffffffffu, sum);
}

// Where the scheduler stands.  A CTA's item numbers only ascend, so each search
// goes on from the last one: 1000 prompts of 100 rows, 32 / 8 heads of 64, in
// 490 us (11.9 ms with a search of the whole batch for every item, 86 us each).
// In shared memory: its warp's 56 registers do not hold it without spills.
struct Place {
    int level;       // tiles of this level are handed out (sorted; else all tiles are one level)
    int above;       // tiles of the levels above
    int here;        // tiles of this level
    int s0, before;  // the 32 sequences that the last tile was found in, and the tiles of this level ahead of them
};
template <bool PAGED>
__device__ __forceinline__ Place first_place(const Params& p, const SeqRows& near) {
    if (!p.sorted) return Place{0, 0, 0x7fffffff, 0, 0};
    int keys = near.klen;
#pragma unroll 1
    for (int b = 32 + (threadIdx.x & 31); b - (int)(threadIdx.x & 31) < p.batch; b += 32)
        keys = max(keys, seq_rows<PAGED>(p, b).klen);
    return Place{(int)(__reduce_max_sync(0xffffffffu, (unsigned)keys) / kBlk) + 1, 0, 0, 0, 0};  // no tile reaches it
}

// Item number -> rows and keys, by the scheduler warp.  Tiles are numbered
// from the most expensive down (p.sorted), so that the CTAs, which take items
// round by round in alternating direction, end together: the tiles of a key
// level, then those of the next level that has any, found from the last one
// down in doubling steps and a bisection, each step a sum over the sequences
// (32 per warp step); within a level a scan for the sequence.  Without p.sorted
// (no CTA has a second item, or the order is given) the scan alone.
template <bool PAGED, bool DUAL>
__device__ __forceinline__ bool get_item(const Params& p, const SeqRows& near, Place& at, int idx, Item& it) {
    const int lane = threadIdx.x & 31;
    it.split = idx % p.splits;
    idx /= p.splits;
    it.kvh = idx % p.kv_heads;
    int tile = idx / p.kv_heads;
    const int span = p.tiles * p.tpt;
    if (PAGED && p.shared > 0) {
        it.seq = 0;
        it.q_row0 = 0;
        it.ntok = p.total_q;
        it.tok0 = tile * span;
        it.kv_row0 = 0;
        it.off = p.shared;  // no causal limit; each row has its own
        const int per = ((p.shared + kBlk - 1) / kBlk + p.splits - 1) / p.splits * kBlk;
        const int k0 = min(p.shared, it.split * per);
        if (it.tok0 >= it.ntok) return false;
        cut_item<DUAL>(it, k0, min(p.shared, k0 + per), {p.shared, p.shared},
                       {true, DUAL || (p.tiles == 2 && it.tok0 + p.tpt < it.ntok)});
        return true;
    }
    if (tile - at.above >= at.here) {  // (sorted) the next level: tiles from `lo` on > tile >= tiles from `hi` on
        int hi = at.level, nhi = at.above + at.here, lo = hi, nlo = nhi;
        for (int step = 1; nlo <= tile; step *= 2) {
            if (lo == 0) return false;  // behind the last tile
            hi = lo;
            nhi = nlo;
            lo = max(0, lo - step);
            nlo = batch_tiles_from<PAGED>(p, near, lo, span);
        }
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1, n = batch_tiles_from<PAGED>(p, near, mid, span);
            if (n > tile) {
                lo = mid;
                nlo = n;
            } else {
                hi = mid;
                nhi = n;
            }
        }
        __syncwarp();
        at = Place{lo, nhi, nlo - nhi, 0, 0};
        __syncwarp();
    }
    tile -= at.above + at.before;
    int b = -1, r0 = 0, r1 = 0, klen = 0;
    int s0 = at.s0;
    for (; s0 < p.batch; s0 += 32) {
        const SeqRows r = s0 == 0 ? near : seq_rows<PAGED>(p, s0 + lane);
        const int n = r.r1 - r.r0, all = (n + span - 1) / span;
        const int over = p.sorted ? tiles_from(p, n, r.klen, at.level + 1, span) : 0;
        const int cnt = (p.sorted ? tiles_from(p, n, r.klen, at.level, span) : all) - over;
        int sum = cnt;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, sum, d);
            if (lane >= d) sum += v;
        }
        const uint32_t vote = __ballot_sync(0xffffffffu, sum > tile);
        if (vote) {
            const int l = __ffs(vote) - 1;
            tile -= __shfl_sync(0xffffffffu, sum - cnt, l);
            r0 = __shfl_sync(0xffffffffu, r.r0, l);
            r1 = __shfl_sync(0xffffffffu, r.r1, l);
            klen = __shfl_sync(0xffffffffu, r.klen, l);
            tile = __shfl_sync(0xffffffffu, all - 1 - over, l) - tile;  // longest causal rows first
            b = s0 + l;
            break;
        }
        sum = __shfl_sync(0xffffffffu, sum, 31);
        tile -= sum;
        __syncwarp();
        if (lane == 0) at.before += sum;
    }
    if (lane == 0) at.s0 = s0;
    __syncwarp();
    if (b < 0) return false;
    it.seq = b;
    it.q_row0 = r0;
    it.kv_row0 = r0;
    it.ntok = r1 - r0;
    it.tok0 = tile * span;
    it.off = p.causal ? klen - it.ntok : klen;
    // every sequence's own keys in p.splits equal ranges of whole blocks
    const int per = ((max(0, klen - p.first) + kBlk - 1) / kBlk + p.splits - 1) / p.splits * kBlk;
    const int k0 = min(klen, p.first + it.split * per);
    const int t0 = it.tok0 + (DUAL ? 0 : p.tpt), t1 = min(it.ntok, it.tok0 + p.tpt), t2 = min(it.ntok, t0 + p.tpt);
    cut_item<DUAL>(it, k0, it.split == p.splits - 1 ? klen : min(klen, k0 + per),
                   {p.causal ? it.off + t1 : klen, p.causal ? it.off + t2 : klen},
                   {true, DUAL || (p.tiles == 2 && t0 < it.ntok)});
    return true;
}

__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&r)[32]) {
    __syncwarp();
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
        "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr)
        : "memory");
}

__device__ __forceinline__ void st_global_v8(void* p, const uint32_t* v) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]),
                 "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
                 : "memory");
}

// A row's 128 scores, one wait.
__device__ __forceinline__ void tmem_ld128(uint32_t taddr, float (&x)[128]) {
    uint32_t r[4][32];
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint32_t(&v)[32] = r[i];
        asm volatile(
            "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,"
            "%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
            : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
              "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]),
              "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]),
              "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
            : "r"(taddr + 32u * i)
            : "memory");
    }
    // the wait takes every destination as an operand, so that no use (or copy) of one is moved before it
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint32_t(&v)[32] = r[i];
        asm volatile("tcgen05.wait::ld.sync.aligned;"
                     : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]),
                       "+r"(v[8]), "+r"(v[9]), "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]),
                       "+r"(v[15]), "+r"(v[16]), "+r"(v[17]), "+r"(v[18]), "+r"(v[19]), "+r"(v[20]), "+r"(v[21]),
                       "+r"(v[22]), "+r"(v[23]), "+r"(v[24]), "+r"(v[25]), "+r"(v[26]), "+r"(v[27]), "+r"(v[28]),
                       "+r"(v[29]), "+r"(v[30]), "+r"(v[31])
                     :
                     : "memory");
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < 32; ++e) x[i * 32 + e] = __uint_as_float(r[i][e]);
}

// An exponent is x c - m c in one FMA.  From |m c| = 1024 on the rounding of m c
// (2^-14 there) would weigh blocks and key ranges with other references
// differently by more than a quarter of P's rounding, and from 2^28 on overflow
// P: the warp's rows then subtract their reference from the scores first.  (The
// branch costs twelve ragged prompts at head_dim 64 47.7 -> 48.5 us and drafted
// rows 1 %, long prompts nothing; subtracting always 49.3 and 1 % everywhere, a
// copy of the exponentials for it 48.9.)
__device__ __forceinline__ bool far_off(float m, float c) {
    return __any_sync(0xffffffffu, m != -INFINITY && !(fabsf(m) * c <= 1024.0f));
}

// The largest of three, NaN when one is.
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

__device__ __forceinline__ uint64_t exp2_hw2(uint64_t y) {
    float a, b;
    unpack2(y, a, b);
    return pack2(ex2_approx(a), ex2_approx(b));
}
// 2^y on the FMA pipe, y <= 8: y = n + f with n the nearest integer (by adding
// 1.5 * 2^23, which leaves n in the low bits of the sum) and |f| <= 1/2, the
// degree-4 interpolation of 2^f at the Chebyshev points of [-1/2, 1/2] (largest
// relative error 4e-6, a hundredth of half a step of fp16), and n added to the
// exponent field.  y is held at -126, below which P is zero in fp16 anyway; so is
// a NaN, which the row's end puts right.
__device__ __forceinline__ uint64_t exp2_poly2(uint64_t y) {
    float a, b;
    unpack2(y, a, b);
    y = pack2(fmaxf(a, -126.0f), fmaxf(b, -126.0f));
    const uint64_t big = pack2(12582912.0f, 12582912.0f), nbig = pack2(-12582912.0f, -12582912.0f);
    const uint64_t t = add2(y, big);
    const uint64_t f = fma2(add2(t, nbig), pack2(-1.0f, -1.0f), y);
    uint64_t r = pack2(0.00966636852f, 0.00966636852f);
    r = fma2(r, f, pack2(0.0559219758f, 0.0559219758f));
    r = fma2(r, f, pack2(0.24022349f, 0.24022349f));
    r = fma2(r, f, pack2(0.693121045f, 0.693121045f));
    r = fma2(r, f, pack2(1.0f, 1.0f));
    float r0, r1, t0, t1;
    unpack2(r, r0, r1);
    unpack2(t, t0, t1);
    return pack2(__uint_as_float(__float_as_uint(r0) + (__float_as_uint(t0) << 23)),
                 __uint_as_float(__float_as_uint(r1) + (__float_as_uint(t1) << 23)));
}

// One lane of a converged warp, by elect.sync: the compiler then knows that a
// single thread runs the branch and keeps descriptors in uniform registers.
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}

__device__ __forceinline__ float row_max(const float (&x)[128]) {
    float m4[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) m4[i] = max3_nan(x[i], x[4 + i], x[8 + i]);
#pragma unroll
    for (int e = 12; e < 124; e += 8) {
#pragma unroll
        for (int i = 0; i < 4; ++i) m4[i] = max3_nan(m4[i], x[e + i], x[e + 4 + i]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) m4[i] = max3_nan(m4[i], x[124 + i], x[124 + i]);
    return max3_nan(max3_nan(m4[0], m4[1], m4[2]), m4[3], m4[3]);
}
// The next item of this CTA, published by the scheduler warp; false at the end
// or when a wait ran out (ok = false).  A whole warp.
__device__ __forceinline__ bool next_item(const Item* slots, uint64_t* full, uint64_t* empty, uint32_t& k, Item& it,
                                          volatile int* abort, bool& ok) {
    const uint32_t s = k % kItemSlots;
    ok = mbar_wait_warp(&full[s], (k / kItemSlots) & 1u, abort);
    if (!ok) return false;
    it = slots[s];
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(&empty[s]);
    ++k;
    return it.state != 0;
}

// DUAL (partials only): the two tiles are the same rows on the two halves of the
// item's keys, for items whose rows fill one tile: two chains of products and
// softmax keep a CTA's loads going where one would wait for itself.
// SCALED (pages): K and V hold whole numbers, and 16 keys each have a scale of K
// and one of V (PackedArgs::key_scale).  The scores become exponents that weigh
// a key times its scale of V, so that P V needs no scales, and the sum of the
// weights takes them out again: 64 packed products more for a row of 128 scores,
// but no rounding of K and V to fp16 (error against 64 bits 0.00048 -> 0.00029
// where the output's rounding alone is 0.00021).
template <int HD, bool PAGED, bool PART, bool DUAL, bool SCALED>
__global__ void __launch_bounds__(kThreads, 1) fmha_packed_kernel(const __grid_constant__ Params p) {
    using L = Smem<HD>;
    // The successor may start once every CTA holds its tensor memory (it may want some itself and then wait for this
    // kernel).  Behind a shared-prefix phase it may start only after this kernel's own wait: paged_decode on the
    // sequences' own keys then needs no wait before its loads and runs beside this kernel.
    const bool late = PART && p.shared > 0;
    extern __shared__ __align__(1024) uint8_t smem[];
    if (smem_u32(smem) & 1023u) {  // the swizzled tiles need 1024-byte alignment
        if (threadIdx.x == 0) set_err(p.err, 0x500);
        pdl_wait();
        return;
    }
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::kOffBar);
    uint64_t* q_full = bars;       // 1
    uint64_t* q_empty = bars + 1;  // 1
    uint64_t* s_full = bars + 2;   // [2]
    uint64_t* p_full = bars + 4;   // [2 tiles][2 halves of the keys]
    uint64_t* o_full = bars + 8;   // [2]
    uint64_t* mma_done = bars + 10;
    uint64_t* v_seen = bars + 11;
    uint64_t* v_fixed = bars + 12;
    uint64_t* kv_full = bars + 13;  // [kStages]
    uint64_t* kv_empty = kv_full + L::kStages;
    uint64_t* it_full = kv_empty + L::kStages;  // [kItemSlots]
    uint64_t* it_empty = it_full + kItemSlots;  // [kItemSlots]
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(it_empty + kItemSlots);
    volatile uint32_t* vfix_stage = tmem_slot + 2;
    Item* slots = reinterpret_cast<Item*>(smem + L::kOffItem);
    Place* place = reinterpret_cast<Place*>(slots + kItemSlots);
    static_assert(kItemSlots * sizeof(Item) + sizeof(Place) <= 256 && (13 + 2 * L::kStages + 2 * kItemSlots) * 8 + 12 <= 384, "layout");
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        mbar_init(q_full, 1);
        mbar_init(q_empty, 1);
        for (int i = 0; i < 2; ++i) {
            mbar_init(&s_full[i], 1);
            mbar_init(&p_full[2 * i], 4);
            mbar_init(&p_full[2 * i + 1], 4);
            mbar_init(&o_full[i], 1);
        }
        mbar_init(mma_done, 1);
        mbar_init(v_seen, 1);
        mbar_init(v_fixed, 1);
        for (int i = 0; i < L::kStages; ++i) {
            mbar_init(&kv_full[i], 1);
            mbar_init(&kv_empty[i], 1);
        }
        for (int i = 0; i < kItemSlots; ++i) {
            mbar_init(&it_full[i], 1);
            mbar_init(&it_empty[i], 11);
        }
        *abort_flag = 0;
        fence_barrier_init();
    }
    if (warp == 8 && lane == 0) {
        prefetch_tmap(&p.tmQ);
        prefetch_tmap(&p.tmK);
        prefetch_tmap(&p.tmV);
    }
    if (warp == 9) {
        tmem_alloc(tmem_slot, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    cta_sync_divergent();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    int never = 0;
    volatile int* no_abort = &never;
    if (!late) pdl_trigger();
    pdl_wait();
    if (late) pdl_trigger();

    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
        if (warp == 8) {
            // ------------------------------------------------------------ TMA producer
            uint32_t n = 0, nz = 0, ni = 0;  // ring tiles, non-empty items, items so far
            bool ok = true;
            const int nbox = PAGED ? kBlk / p.box_rows : 1;
            Item it;
            while (ok && next_item(slots, it_full, it_empty, ni, it, abort_flag, ok)) {
                const int nblk = max(it.n[0], it.n[1]);
                if (nblk == 0) continue;
                ok = mbar_wait_warp(q_empty, (nz & 1u) ^ 1u, abort_flag);
                if (!ok) break;
                const int nq = !DUAL && it.n[1] > 0 ? 2 : 1;
                if (lane == 0) {
                    const uint32_t bytes = (uint32_t)(p.group * p.tpt) * 128u * L::kChunks;
                    mbar_arrive_expect_tx(q_full, bytes * nq);
                    for (int q = 0; q < nq; ++q)
                        for (int ch = 0; ch < L::kChunks; ++ch)
                            tma_load_3d(smem + L::kOffQ + q * L::kTile + ch * L::kChunk, &p.tmQ, q_full, ch * 64,
                                        it.kvh * p.group, it.q_row0 + it.tok0 + q * p.tpt);
                }
                ++nz;
                // in the order of their use: V of block j - 1, K of block j (of both ranges in turn)
                const int box = lane / L::kChunks, ch = lane % L::kChunks;
                for (int j = 0; j <= nblk && ok; ++j) {
#pragma unroll
                    for (int u = 0; u < (DUAL ? 4 : 2); ++u) {
                        const int q = u >> 1, kv = 1 - (u & 1), jb = j - kv;
                        if (jb < 0 || jb >= (DUAL ? it.n[q] : nblk)) continue;
                        const int key = it.kb[q] + jb * kBlk;
                        int c2 = 0, c3 = 0;
                        if (PAGED) {
                            // lane -> (page piece, 64-column chunk); past the keys: a page outside the pool, which
                            // the copy fills with zeros
                            const int kk = key + box * p.box_rows;
                            c3 = p.n_pages;
                            if (box < nbox && kk < it.ke[q]) {
                                const int id = __ldg(p.table + (int64_t)it.seq * p.ldt + (kk >> p.page_shift));
                                if (id >= 0 && id < p.n_pages) c3 = id;
                            }
                            c2 = kk & ((1 << p.page_shift) - 1);
                        }
                        const uint32_t s = n % L::kStages, ph = (n / L::kStages) & 1u;
                        ok = mbar_wait_warp(&kv_empty[s], ph ^ 1u, abort_flag);
                        if (!ok) break;
                        uint8_t* dst = smem + L::kOffRing + s * L::kTile + ch * L::kChunk;
                        if (lane == 0) mbar_arrive_expect_tx(&kv_full[s], (uint32_t)L::kTile);
                        __syncwarp();
                        if (box < nbox) {
                            if (PAGED)
                                tma_load_4d(dst + box * p.box_rows * 128, kv ? &p.tmV : &p.tmK, &kv_full[s], ch * 64,
                                            c2, it.kvh, c3);
                            else
                                tma_load_3d(dst, kv ? &p.tmV : &p.tmK, &kv_full[s], ch * 64, it.kvh,
                                            it.kv_row0 + key);
                        }
                        ++n;
                    }
                }
            }
            if (!ok) {  // copies in flight land before the CTA leaves
                if (lane == 0) {
                    *abort_flag = 1;
                    set_err(p.err, 0x501);
                    if (nz) mbar_wait_bounded(q_full, (nz - 1) & 1u, no_abort, 200000000ull);
                    for (uint32_t i = n > L::kStages ? n - L::kStages : 0; i < n; ++i)
                        mbar_wait_bounded(&kv_full[i % L::kStages], (i / L::kStages) & 1u, no_abort, 200000000ull);
                }
            }
        } else if (warp == 9) {
            // ------------------------------------------------------------ MMA issuer: one thread
            if (elect_one()) {
                constexpr uint32_t idesc_s = umma_idesc_f16(kRows, kBlk);
                constexpr uint32_t idesc_o = umma_idesc_f16_bmn(kRows, HD);
                // descriptors step by 16-byte units in their low 14 bits: no carry below 256 KB
                const uint64_t qd0 = umma_desc_sw128(smem_u32(smem + L::kOffQ));
                const uint64_t kd0 = umma_desc_sw128(smem_u32(smem + L::kOffRing));
                const uint64_t vd0 = umma_desc_sw128_mn(smem_u32(smem + L::kOffRing), (uint32_t)L::kChunk, 1024u);
                uint32_t st = 0, ph = 0, nz = 0, ni = 0, np[2] = {0, 0}, nv = 0;
                bool ok = true;
                while (ok) {
                    const uint32_t slot = ni % kItemSlots;
                    ok = mbar_wait_quick(&it_full[slot], (ni / kItemSlots) & 1u, abort_flag);
                    if (!ok) break;
                    const Item& it = slots[slot];
                    const int n0 = it.n[0], n1 = it.n[1], state = it.state;
                    const int last0 = it.steps[0], last1 = it.steps[1], vfix = it.vfix, vfix_q = it.vfix_q;
                    mbar_arrive(&it_empty[slot]);
                    ++ni;
                    if (!state) break;
                    const int nblk = max(n0, n1);
                    if (nblk == 0) continue;
                    ok = mbar_wait_quick(q_full, nz & 1u, abort_flag);
                    ++nz;
                    for (int j = 0; ok && j <= nblk; ++j) {
                        uint32_t vs = 0, ks = 0;
#pragma unroll
                        for (int q = 0; q < 2; ++q) {
                            const int n = q ? n1 : n0, nkv = DUAL ? n : nblk;
                            const uint32_t sq = tmem + (uint32_t)(q * 128), oq = tmem + 256u + (uint32_t)(q * 128);
                            const bool mine = DUAL || q == 0;  // this tile takes the next K and V off the ring
                            if (mine && j >= 1 && j <= nkv) {  // V_{j-1}
                                vs = st;
                                ok = mbar_wait_quick(&kv_full[st], ph, abort_flag);
                                if (++st == L::kStages) st = 0, ph ^= 1u;
                                if (ok && vfix && j == nkv && (!DUAL || q == vfix_q)) {  // warp 11's turn; P takes longer
                                    *vfix_stage = vs;
                                    mbar_arrive(v_seen);
                                    ok = mbar_wait_quick(v_fixed, nv++ & 1u, abort_flag);
                                }
                                if (!ok) break;
                            }
                            if (j >= 1 && j <= n) {  // O_q += P_q(j-1) V_{j-1}
                                const uint64_t vd = vd0 + (uint64_t)(vs * (L::kTile >> 4));
                                const int steps = j < n ? kBlk / 16 : (q ? last1 : last0);
#pragma unroll
                                for (int hf = 0; hf < 2; ++hf) {  // the first 64 keys' P is ready ahead of the rest
                                    ok = mbar_wait_quick(&p_full[2 * q + hf], np[q] & 1u, abort_flag);
                                    if (!ok) break;
                                    tc_fence_after();
                                    if (steps == kBlk / 16) {
#pragma unroll
                                        for (int kk = hf * 4; kk < hf * 4 + 4; ++kk)
                                            tc_mma_f16_ts(oq, sq + (uint32_t)kk * 8u, vd + (uint64_t)(kk * 128),
                                                          idesc_o, (j > 1 || kk > 0) ? 1u : 0u);
                                    } else {
#pragma unroll 1
                                        for (int kk = hf * 4; kk < min(steps, hf * 4 + 4); ++kk)
                                            tc_mma_f16_ts(oq, sq + (uint32_t)kk * 8u, vd + (uint64_t)(kk * 128),
                                                          idesc_o, (j > 1 || kk > 0) ? 1u : 0u);
                                    }
                                }
                                if (!ok) break;
                                ++np[q];
                                if (j == n) tc_commit(&o_full[q]);
                                if (DUAL) tc_commit(&kv_empty[vs]);
                            }
                            if (mine && j < nkv) {  // K_j
                                ks = st;
                                ok = mbar_wait_quick(&kv_full[st], ph, abort_flag);
                                if (++st == L::kStages) st = 0, ph ^= 1u;
                                if (!ok) break;
                            }
                            if (j < n) {  // S_q(j) = Q_q K_j^T
                                const uint64_t kd = kd0 + (uint64_t)(ks * (L::kTile >> 4));
                                const uint64_t qd = qd0 + (uint64_t)((DUAL ? 0 : q) * (L::kTile >> 4));
#pragma unroll
                                for (int kk = 0; kk < HD / 16; ++kk) {
                                    const uint64_t o = (uint64_t)(((kk >> 2) * L::kChunk + (kk & 3) * 32) >> 4);
                                    tc_mma_f16(sq, qd + o, kd + o, idesc_s, kk > 0 ? 1u : 0u);
                                }
                                tc_commit(&s_full[q]);
                                if (DUAL) tc_commit(&kv_empty[ks]);
                            }
                        }
                        if (!ok) break;
                        if (!DUAL) {
                            if (j >= 1) tc_commit(&kv_empty[vs]);
                            if (j < nblk) tc_commit(&kv_empty[ks]);
                        }
                        if (j == nblk - 1) tc_commit(q_empty);
                    }
                }
                if (!ok) {
                    *abort_flag = 1;
                    set_err(p.err, 0x502);
                }
                tc_commit(mma_done);  // every MMA issued above completes before TMEM is freed
                if (!mbar_wait_bounded(mma_done, 0, no_abort, 200000000ull)) set_err(p.err, 0x503);
            }
            __syncwarp();
        } else if (warp == 11) {
            // ------------------------------------------------------------ V rows behind the last key
            uint32_t ni = 0, nv = 0;
            bool ok = true;
            Item it;
            while (ok && next_item(slots, it_full, it_empty, ni, it, abort_flag, ok)) {
                if (!it.vfix) continue;
                ok = mbar_wait_warp(v_seen, nv++ & 1u, abort_flag);  // the MMA thread has seen the tile land
                if (!ok) break;
                uint8_t* v = smem + L::kOffRing + *vfix_stage * L::kTile;
                const int vb = it.vfix, n16 = (16 - (vb & 15)) * 8;  // zeroed up to the end of the last 16-key step
                for (int i = lane; i < n16 * L::kChunks; i += 32) {
                    const int ch = i / n16, e = i - ch * n16;
                    *reinterpret_cast<uint4*>(v + ch * L::kChunk + vb * 128 + e * 16) = make_uint4(0, 0, 0, 0);
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(v_fixed);
            }
        } else if (warp == 10) {
            // ------------------------------------------------------------ scheduler
            uint32_t k = 0;
            bool ok = true;
            SeqRows near = {0, 0, 0};  // of the first 32 sequences, loaded once
            if (!(PAGED && p.shared > 0)) near = seq_rows<PAGED>(p, lane);
            Place& at = *place;
            at = first_place<PAGED>(p, near);
            __syncwarp();
            for (uint32_t round = 0; ok; ++round) {
                const uint32_t idx = round * gridDim.x + ((round & 1) ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
                Item it;
                // no item with this number: none with the later ones either
                it.state = idx < (uint32_t)p.n_items && get_item<PAGED, DUAL>(p, near, at, (int)idx, it) ? 1 : 0;
                const uint32_t s = k % kItemSlots;
                ok = mbar_wait_warp(&it_empty[s], ((k / kItemSlots) & 1u) ^ 1u, abort_flag);
                if (!ok) {
                    if (lane == 0) {
                        *abort_flag = 1;
                        set_err(p.err, 0x505);
                    }
                    break;
                }
                if (lane == 0) {
                    slots[s] = it;
                    mbar_arrive(&it_full[s]);
                }
                ++k;
                if (!it.state) break;
            }
        }
    } else {
        // ---------------------------------------------------------------- softmax / output
        asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
        const int q = warp >> 2;
        const int r = threadIdx.x & 127;  // row of the tile == TMEM lane
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t sq = tmem + lanes + (uint32_t)(q * 128), oq = tmem + lanes + 256u + (uint32_t)(q * 128);
        const int tl = r / p.group, g = r - tl * p.group;
        const float c = SCALED ? 1.0f : p.c;
        uint32_t ns = 0, no = 0, ni = 0;
        bool ok = true;
        Item it;
        while (ok && next_item(slots, it_full, it_empty, ni, it, abort_flag, ok)) {
            const int tok = it.tok0 + (DUAL ? 0 : q * p.tpt) + tl;
            const bool valid = (DUAL || q < p.tiles) && tl < p.tpt && tok < it.ntok;
            const int kb = q ? it.kb[1] : it.kb[0];
            int lim = q ? it.ke[1] : it.ke[0];  // this row's keys end here
            if (valid) {
                if (PAGED && p.shared > 0) lim = min(lim, __ldg(p.lens + tok));
                else if (p.causal) lim = min(lim, it.off + tok + 1);
            }
            float m = -INFINITY, l = 0.0f;
            bool far = false;  // some row's reference is, in this warp
            const int nb = q ? it.n[1] : it.n[0];
            for (int j = 0; j < nb; ++j) {
                float2 ks[8];
                if (SCALED) {
                    const int64_t at = ((int64_t)it.seq * p.kv_heads + it.kvh) * (p.max_keys / 16) + (kb + j * kBlk) / 16;
#pragma unroll
                    for (int e = 0; e < 8; ++e) ks[e] = __ldg(p.key_scale + at + e);
                }
                ok = mbar_wait_warp(&s_full[q], ns & 1u, abort_flag);
                if (!ok) break;
                ++ns;
                tc_fence_after();
                float x[128];
                tmem_ld128(sq, x);
                if (SCALED) {
#pragma unroll
                    for (int e = 0; e < 64; ++e)
                        unpack2(fma2(pack2(x[2 * e], x[2 * e + 1]), pack2(ks[e / 8].x, ks[e / 8].x), pack2(ks[e / 8].y, ks[e / 8].y)),
                                x[2 * e], x[2 * e + 1]);
                }
                const int left = lim - (kb + j * kBlk);
                if (__any_sync(0xffffffffu, left < kBlk)) {
#pragma unroll
                    for (int e = 0; e < 128; ++e) x[e] = e < left ? x[e] : -INFINITY;
                }
                const float mx = max3_nan(m, row_max(x), m);
                if (j == 0) {
                    m = mx;
                    far = far_off(m, c);
                } else {
                    const bool need = mx != -INFINITY && !((mx - m) * c <= 8.0f);  // also when the maximum is NaN
                    if (__any_sync(0xffffffffu, need)) {  // P_q(j-1) V_{j-1} is complete: S_q(j) was issued behind it
                        const float corr = need ? ex2_approx((m - mx) * c) : 1.0f;
                        if (need) m = mx;
                        far |= far_off(m, c);
                        l *= corr;
#pragma unroll 1
                        for (int e0 = 0; e0 < HD; e0 += 32) {
                            uint32_t o[32];
                            tmem_ld32(oq + (uint32_t)e0, o);
#pragma unroll
                            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * corr);
                            tmem_st32(oq + (uint32_t)e0, o);
                        }
                    }
                }
                const float ref = m == -INFINITY ? 0.0f : m;  // 0: every exponential of the row is 2^-inf
                float mc = -ref * c;
                if (far) {
                    mc = 0.0f;
#pragma unroll
                    for (int e = 0; e < 128; ++e) x[e] -= ref;
                }
                const uint64_t c2 = pack2(c, c), mc2 = pack2(mc, mc);
                uint64_t sum2[2] = {0, 0}, all2 = 0;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    uint32_t pk[32];
#pragma unroll
                    for (int e = 0; e < 32; ++e) {
                        const uint64_t y = fma2(pack2(x[h * 64 + 2 * e], x[h * 64 + 2 * e + 1]), c2, mc2);
                        const uint64_t pp = (HD == 64 && (e & 3) == 0) ? exp2_poly2(y) : exp2_hw2(y);
                        sum2[e & 1] = add2(sum2[e & 1], pp);
                        if (SCALED && (e & 7) == 7) {
                            const float sv = ex2_approx(-ks[h * 4 + e / 8].y);
                            all2 = fma2(add2(sum2[0], sum2[1]), pack2(sv, sv), all2);
                            sum2[0] = sum2[1] = 0;
                        }
                        float p0, p1;
                        unpack2(pp, p0, p1);
                        __half2 hh = __floats2half2_rn(p0, p1);
                        pk[e] = *reinterpret_cast<uint32_t*>(&hh);
                    }
                    tmem_st32(sq + (uint32_t)(h * 32), pk);
                    tmem_wait_st();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&p_full[2 * q + h]);
                }
                float s0, s1;
                unpack2(SCALED ? all2 : add2(sum2[0], sum2[1]), s0, s1);
                l += s0 + s1;
            }
            if (!ok) break;
            if (nb > 0) {
                ok = mbar_wait_warp(&o_full[q], no & 1u, abort_flag);
                if (!ok) break;
                ++no;
                tc_fence_after();
            }
            // Output straight from a lane's registers, whole 32-byte sectors where the row allows it.  (Through shared
            // memory, for 128-byte lines, it took as long: the staging competes with the operand reads of the other
            // tile's MMAs, which use all of the shared-memory bandwidth.)
            const int64_t row = (int64_t)it.q_row0 + tok;
            const int head = it.kvh * p.group + g;
            const bool none = lim <= kb;  // no key in the range: zeros (no partial)
            // A score of +inf or NaN: the row is NaN, as x - m is in the formula.  Its weights need not be: exp2_poly2
            // holds a NaN at 2^-126, and the sum and O would then be zeros.
            if (!(m < INFINITY)) l = NAN;
            // Keys, but all scores -inf: 0 / 0 in the formula.  A partial (m = -inf, l = 1) weighs 2^-inf beside others
            // that have a maximum, and NaN where none has.
            const bool flat = m == -INFINITY;
            if (flat) l = none ? 0.0f : PART ? 1.0f : NAN;
            const int sp = p.split0 + (DUAL ? 2 * it.split + q : it.split);
            const int64_t at = PART ? ((int64_t)sp * p.total_q + row) * p.heads + head : 0;
            if (PART && valid) p.part_ml[at] = make_float2(m, l);
            const bool put = valid && !(PART && flat);
            const float inv = none ? 0.0f : 1.0f / l;
            float* dstf = p.part_o + at * p.head_dim;
            __half* dsth = p.out + row * p.ldo + (int64_t)head * p.head_dim;
            if (__any_sync(0xffffffffu, put)) {
#pragma unroll 1
                for (int e0 = 0; e0 < p.head_dim; e0 += 32) {
                    uint32_t o[32];
                    if (nb > 0) tmem_ld32(oq + (uint32_t)e0, o);
                    if (!put) continue;
                    if (PART) {
                        const int n = p.head_dim - e0 < 32 ? p.head_dim - e0 : 32;  // a multiple of 16
#pragma unroll
                        for (int e = 0; e < 32; e += 8)
                            if (e < n) st_global_v8(dstf + e0 + e, &o[e]);
                    } else {
                        uint32_t pk[16];
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            __half2 hh = __floats2half2_rn(__uint_as_float(o[2 * i]) * inv,
                                                           __uint_as_float(o[2 * i + 1]) * inv);
                            pk[i] = none ? 0u : *reinterpret_cast<uint32_t*>(&hh);
                        }
                        if (p.out32) {
                            st_global_v8(dsth + e0, pk);
                            if (e0 + 16 < p.head_dim) st_global_v8(dsth + e0 + 16, pk + 8);
                        } else {
#pragma unroll
                            for (int i = 0; i < 4; ++i)
                                if (e0 + i * 8 < p.head_dim)
                                    *reinterpret_cast<uint4*>(dsth + e0 + i * 8) =
                                        make_uint4(pk[4 * i], pk[4 * i + 1], pk[4 * i + 2], pk[4 * i + 3]);
                        }
                    }
                }
            }
            tc_fence_before();  // the O reads above, before the next item's first P lets its product overwrite them
        }
        if (!ok) {
            *abort_flag = 1;
            set_err(p.err, 0x504);
        }
    }

    tc_fence_before();
    cta_sync_divergent();
    if (warp == 9) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

template <int HD, bool PAGED, bool PART, bool DUAL = false, bool SCALED = false>
int launch(const Params& p, int grid, cudaStream_t st) {
    auto kern = fmha_packed_kernel<HD, PAGED, PART, DUAL, SCALED>;
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Smem<HD>::kTotal);
    if (e != cudaSuccess) {
        npub_internal_set_cuda_error(e);
        return NPUB_ERR_CUDA;
    }
    return launch_pdl(kern, dim3(grid), dim3(kThreads), Smem<HD>::kTotal, st, p);
}

}  // namespace fpk

int64_t fmha_packed_items(int total_q, int batch, int heads, int kv_heads, int max_new, int tiles) {
    const int64_t span = (int64_t)tiles * (128 / (heads / kv_heads));
    int64_t n = total_q / span + batch;  // sum of ceil(rows / span) over the sequences is at most this
    if (batch == 1) n = (total_q + span - 1) / span;
    if (n > total_q) n = total_q;
    if (max_new > 0 && n > batch * ((max_new + span - 1) / span)) n = batch * ((max_new + span - 1) / span);
    return n;
}

int fmha_packed(const PackedArgs& a, cudaStream_t st) {
    using namespace fpk;
    const int group = a.heads / a.kv_heads;
    const bool paged = a.kv.table != nullptr;
    Params p;
    memset(&p, 0, sizeof(p));
    p.group = group;
    p.tpt = kRows / group;
    int rc = make_tmap_3d(&p.tmQ, false, a.q, (uint64_t)a.head_dim, (uint64_t)a.heads, (uint64_t)a.total_q,
                          (uint64_t)a.head_dim, (uint64_t)a.ldq, (uint32_t)group, (uint32_t)p.tpt, true);
    if (rc) return rc;
    if (paged) {
        p.box_rows = a.kv.page_size < kBlk ? a.kv.page_size : kBlk;
        rc = make_tmap_pages(&p.tmK, a.kv.k, a.kv.n_pages, a.kv_heads, a.kv.page_size, a.head_dim, p.box_rows);
        if (rc) return rc;
        rc = make_tmap_pages(&p.tmV, a.kv.v, a.kv.n_pages, a.kv_heads, a.kv.page_size, a.head_dim, p.box_rows);
        if (rc) return rc;
        while ((1 << p.page_shift) < a.kv.page_size) ++p.page_shift;
        const int64_t mk = (int64_t)a.kv.max_pages << p.page_shift;
        p.max_keys = mk > 0x7ff00000 ? 0x7ff00000 : (int)mk;
        p.n_pages = a.kv.n_pages;
        p.table = a.kv.table;
        p.ldt = a.kv.ldt;
        p.lens = a.lens;
    } else {
        rc = make_tmap_3d(&p.tmK, false, a.kv.k, (uint64_t)a.head_dim, (uint64_t)a.kv_heads, (uint64_t)a.total_q,
                          (uint64_t)a.head_dim, (uint64_t)a.kv.ldk, 1, kBlk, true);
        if (rc) return rc;
        rc = make_tmap_3d(&p.tmV, false, a.kv.v, (uint64_t)a.head_dim, (uint64_t)a.kv_heads, (uint64_t)a.total_q,
                          (uint64_t)a.head_dim, (uint64_t)a.kv.ldv, 1, kBlk, true);
        if (rc) return rc;
    }
    p.cu = a.cu;
    p.total_q = a.total_q;
    p.batch = a.batch;
    p.heads = a.heads;
    p.kv_heads = a.kv_heads;
    p.head_dim = a.head_dim;
    p.shared = a.shared;
    p.causal = a.causal ? 1 : 0;
    p.c = a.scale * 1.4426950408889634f;
    p.key_scale = a.key_scale;
    p.out = reinterpret_cast<__half*>(a.out);
    p.ldo = a.ldo;
    p.out32 = npub_aligned(a.out, 32) && a.ldo % 16 == 0;
    p.part_o = a.part_o;
    p.part_ml = a.part_ml;
    p.err = npub_internal_device_error_word();
    const bool part = a.part_o != nullptr;
    p.splits = part ? a.splits : 1;
    p.first = a.first;
    p.split0 = a.split0;
    const int batch = a.shared > 0 ? 1 : a.batch;
    p.tiles = a.tiles;
    if (p.tiles == 0) {  // one tile per CTA while that still leaves SMs free
        const int64_t one = fmha_packed_items(a.total_q, batch, a.heads, a.kv_heads, 0, 1);
        p.tiles = one * a.kv_heads <= num_sms() ? 1 : 2;
    }
    // a bound that no value of the offsets exceeds while they ascend
    const int64_t items = fmha_packed_items(a.total_q, batch, a.heads, a.kv_heads, 0, p.tiles) * a.kv_heads * p.splits;
    if (items > 0x7fffffff) return NPUB_ERR_UNSUPPORTED;
    p.n_items = (int)items;
    const int grid = p.n_items < num_sms() ? p.n_items : num_sms();
    // One sequence's tiles come from the most expensive down anyway, and without the causal limit they cost the same;
    // the search takes the first item 2 us (2048 tokens of one prompt 36.6 against 34.5 us, twelve ragged ones 48.4
    // against 50.8).
    p.sorted = p.n_items > grid && a.shared == 0 && a.batch > 1 && a.causal;
    p.span_inv = (uint32_t)((0x100000000ull + p.tiles * p.tpt - 1) / (p.tiles * p.tpt) - (p.tiles * p.tpt == 1));
    const bool small = a.head_dim <= 64;
    if (a.key_scale) {
        if (!paged || a.shared > 0) return NPUB_ERR_UNSUPPORTED;
        if (part && a.dual)
            return small ? launch<64, true, true, true, true>(p, grid, st) : launch<128, true, true, true, true>(p, grid, st);
        if (part) return small ? launch<64, true, true, false, true>(p, grid, st) : launch<128, true, true, false, true>(p, grid, st);
        return small ? launch<64, true, false, false, true>(p, grid, st) : launch<128, true, false, false, true>(p, grid, st);
    }
    if (part) {
        if (!paged) return NPUB_ERR_UNSUPPORTED;
        if (a.dual) return small ? launch<64, true, true, true>(p, grid, st) : launch<128, true, true, true>(p, grid, st);
        return small ? launch<64, true, true>(p, grid, st) : launch<128, true, true>(p, grid, st);
    }
    if (paged) return small ? launch<64, true, false>(p, grid, st) : launch<128, true, false>(p, grid, st);
    return small ? launch<64, false, false>(p, grid, st) : launch<128, false, false>(p, grid, st);
}

}  // namespace npub
