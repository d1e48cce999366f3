"""The paged cache in 8 bits on the GPU against 64-bit forms.

Bounds.  Append: y is the row behind norm and rotation in 64 bits, e = 2^-20 of
its head's largest |column| the fp32 arithmetic's error (as in paged_cases);
  scale      max(s, max|y| / 127), off by e / 127 and two roundings, 2^-23
  new rows   |q s' - y| <= s' / 2 + e + 2^-22 |y| (the step's rounding, e, and the
             product with 1 / s' and that quotient's roundings)
  old rows   |q' s' - q s| <= s' / 2 + 2^-22 |q s| where the scale grew, else untouched
Attention over the 8-bit keys, with V = s q: as attention_exact's bound, but
  - a weight that falls below fp16's normal range is off by 2^-25 of the largest
    weight times scale, against integers: 2^-25 * max s_v * sum |q_v| in place
    of 2^-25 sum |v| / L;
  - a score is a sum of products with integers q_k + 128 <= 255, from which 128
    sum(q) is taken: its fp32 roundings are relative to 255 sum |q|, at most
    2^-22 of scale * s_k * 255 sum |q| together, and a weight is off by that
    many e-folds against the row's other weights: twice that of sum w |v|.
Calls of few rows read the pages, others an fp16 copy of their integers."""
import math

import pytest
import torch

import npu_comp_b200 as nb
from npu_comp_b200 import npu
from paged_cases import append64, table_for
from paged_exact import attention_exact, same

pytestmark = pytest.mark.gpu


def i32(v, dev="cuda"):
    return torch.tensor(v, dtype=torch.int32, device=dev)


def offsets(n):
    cu = [0]
    for x in n:
        cu.append(cu[-1] + x)
    return i32(cu)


# ------------------------------------------------------------------- append

def check_append(new, start, H, KV, hd, rot, inter, norm, ps, packed, *, spread=1.0, scale_spread=1.0, extra=0, seed=0):
    dev, g = "cuda", torch.Generator().manual_seed(sum(new) + hd + seed)
    T, keys = sum(new), [s + n for s, n in zip(start, new)]
    first = [s // ps for s in start]
    W = max((k + ps - 1) // ps for k in keys) + 1
    need = [(k + ps - 1) // ps - f for k, f in zip(keys, first)]
    n_pages = sum(need) + 2
    ids = torch.randperm(n_pages, generator=g).int()
    table = torch.full((len(new), W + 3), -5, dtype=torch.int32)
    at = 0
    for b in range(len(new)):
        table[b, first[b]:first[b] + need[b]] = ids[at:at + need[b]]
        at += need[b]
    x = (spread * torch.randn((T + extra, (H + 2 * KV) * hd + 8), generator=g)).half().to(dev)[:, :(H + 2 * KV) * hd]
    pos = i32([s + i for s, n in zip(start, new) for i in range(n)] + [0] * extra)
    f = nb.rope_freqs(rot, 500000.0, device=dev)
    gam = [(1 + 0.3 * torch.randn(hd, generator=g)).half().to(dev) if norm else None for _ in range(2)]
    pool = [torch.randint(-127, 128, (n_pages, KV, ps, hd), generator=g, dtype=torch.int8) for _ in range(2)]
    sc = [(0.01 + 0.04 * torch.rand((n_pages, KV), generator=g)) * scale_spread for _ in range(2)]
    for s in sc:
        s[ids[-2:].long()] = float("nan")  # pages of nobody
    kp, vp, ks, vs = (t.to(dev) for t in (*pool, *sc))
    out = torch.full((T + extra, H * hd + 16), 3.0, dtype=torch.float16, device=dev)[:, :H * hd]
    q = nb.rope_paged_append_q8(x, H, KV, hd, pos, f, kp, vp, ks, vs, table.to(dev)[:, :W],
                                cu_seqlens=offsets(new) if packed else None, rot_dim=rot, interleaved=inter,
                                q_gamma=gam[0], k_gamma=gam[1], eps=1e-6, out=out)
    assert q.data_ptr() == out.data_ptr() and (q[T:] == 3.0).all()
    x3 = x[:T].reshape(T, H + 2 * KV, hd)
    (qe, qb), (ke, _) = append64(x3, H, KV, pos[:T], f, rot, inter, gam[0], gam[1], 1e-6)
    err = (q[:T].double() - qe.reshape(T, -1)).abs()
    assert (err <= qb.reshape(T, -1)).all()
    for what, y, pages, scales, p0, s0 in (("k", ke.cpu(), kp.cpu(), ks.cpu(), pool[0], sc[0]),
                                           ("v", x3[:, H + KV:].double().cpu(), vp.cpu(), vs.cpu(), pool[1], sc[1])):
        e = 2.0 ** -20 * y.abs().amax(-1, keepdim=True) if what == "k" else torch.zeros(T, KV, 1, dtype=torch.float64)
        touched = torch.zeros(n_pages, dtype=torch.bool)
        t = 0
        for b, n in enumerate(new):
            p = start[b]
            while p < keys[b]:
                m, page, slot = min(ps - p % ps, keys[b] - p), int(table[b, p // ps]), p % ps
                touched[page] = True
                r = y[t:t + m].transpose(0, 1)                       # [KV, m, hd]
                er = e[t:t + m].transpose(0, 1)
                was = s0[page].double() if slot else torch.zeros(KV, dtype=torch.float64)
                want = torch.maximum(was, r.abs().amax((1, 2)) / 127)
                got = scales[page].double()
                assert ((got - want).abs() <= er.amax((1, 2)) / 127 + 2.0 ** -23 * want).all(), (what, page)
                now = got[:, None, None]
                v = pages[page].double() * now
                d = (v[:, slot:slot + m] - r).abs() - (now / 2 + er + 2.0 ** -22 * r.abs())
                assert (d <= 0).all(), (what, page, d.max())
                old, before = pages[page, :, :slot], p0[page, :, :slot]
                grew = scales[page] > s0[page]
                assert torch.equal(old[~grew], before[~grew])
                d = (v[:, :slot] - before.double() * was[:, None, None]).abs() - (
                    now / 2 + 2.0 ** -22 * (before.double() * was[:, None, None]).abs())
                assert (d[grew] <= 0).all()
                assert torch.equal(pages[page, :, slot + m:], p0[page, :, slot + m:])  # slots behind
                p, t = p + m, t + m
        assert torch.equal(pages[~touched], p0[~touched]) and torch.equal(scales[~touched].nan_to_num(9), s0[~touched].nan_to_num(9))


@pytest.mark.parametrize("new,start,H,KV,hd,rot,inter,norm,ps", [
    ([1], [0], 1, 1, 16, 16, False, False, 16),
    ([1], [1499], 32, 8, 128, 128, False, True, 16),
    ([1] * 37, [0, 130000] + [5000 + 7 * i for i in range(35)], 4, 4, 128, 64, True, True, 64),
    ([5, 0, 1, 70], [3, 9, 100001, 0], 6, 2, 64, 32, False, False, 32),
    ([33, 31], [0, 15], 8, 2, 80, 48, True, True, 128),
    ([3, 300, 17], [255, 2, 250], 2, 1, 112, 112, False, True, 256),
    ([700] * 2, [0, 64], 16, 16, 128, 128, False, False, 32),
    ([1] * 40 + [2] * 9 + [0, 0, 33], [16 * i + i % 16 for i in range(52)], 2, 2, 64, 64, True, False, 16),
    ([257], [1], 1, 1, 32, 16, False, True, 16),
])
@pytest.mark.parametrize("packed", [True, False])
@pytest.mark.parametrize("scale_spread", [1.0, 1e-3, 100.0])
def test_append(cuda_device, new, start, H, KV, hd, rot, inter, norm, ps, packed, scale_spread):
    """Scales like the rows' (some pages grow), far smaller (all grow) and far larger (none does)."""
    if not packed and any(n != 1 for n in new):
        pytest.skip("a decode step has one row per sequence")
    check_append(new, start, H, KV, hd, rot, inter, norm, ps, packed, scale_spread=scale_spread, extra=2 if packed else 0)


@pytest.mark.parametrize("eps", [0.0, 1e-5])
def test_append_norm_of_few_rows(cuda_device, eps):
    """Rows that do not fill a page's threads, with eps 0 too."""
    g = torch.Generator().manual_seed(2)
    H, KV, hd, ps = 2, 1, 80, 64
    x = torch.randn((3, (H + 2 * KV) * hd), generator=g).half().cuda()
    kp = torch.zeros((1, KV, ps, hd), dtype=torch.int8, device="cuda")
    vp, ks, vs = kp.clone(), torch.ones(1, KV, device="cuda"), torch.ones(1, KV, device="cuda")
    f, gam = nb.rope_freqs(hd, device="cuda"), torch.ones(hd, device="cuda").half()
    pos = i32([0, 1, 2])
    nb.rope_paged_append_q8(x, H, KV, hd, pos, f, kp, vp, ks, vs, i32([[0]]), cu_seqlens=i32([0, 3]), q_gamma=gam, k_gamma=gam,
                            eps=eps)
    _, (ke, _) = append64(x.view(3, -1, hd), H, KV, pos, f, hd, False, gam, gam, eps)
    assert torch.isfinite(ks).all()
    assert ((kp[0, 0, :3].double() * ks.item() - ke[:, 0]).abs() <= 0.501 * ks.item()).all()


def test_append_wide_values(cuda_device):
    check_append([40], [8], 2, 2, 64, 64, False, False, 32, True, spread=300.0)
    check_append([40], [8], 2, 2, 64, 64, False, False, 32, True, spread=1e-6, scale_spread=1e-8)


def one_page(rows, ps=16, hd=64, KV=1):
    kp = torch.full((1, KV, ps, hd), 7, dtype=torch.int8, device="cuda")
    s = torch.full((1, KV), 0.5, device="cuda")
    return kp, kp.clone(), s, s.clone()


def append_at(rows, pos, pool, packed=False):
    """rows [n, hd] as k = v of one head at pos.., angles 0 (position 0 is stored separately below)."""
    n, hd = rows.shape
    x = torch.cat([rows, rows, rows], 1).half().cuda()
    f = torch.zeros(hd // 2, device="cuda")  # no rotation
    t = torch.zeros((1 if packed else n, 4), dtype=torch.int32, device="cuda")
    return nb.rope_paged_append_q8(x, 1, 1, hd, i32([pos + i for i in range(n)]), f, *pool[:2], *pool[2:], t,
                                   cu_seqlens=i32([0, n]) if packed else None)


@pytest.mark.parametrize("packed", [False, True])
def test_append_zeros_and_values_that_are_not_finite(cuda_device, packed):
    z = torch.zeros(1, 64)
    pool = one_page(1)
    append_at(z, 0, pool, packed)
    assert pool[2].item() == 0 and not pool[0][0, 0, 0].any() and (pool[0][0, 0, 1:] == 7).all()
    append_at(torch.linspace(-1, 1, 64)[None], 1, pool, packed)
    assert not pool[0][0, 0, 0].any() and abs(pool[2].item() - 1 / 127) < 1e-9 and pool[0][0, 0, 1, 0] == -127
    for bad in (math.nan, math.inf, -math.inf):
        r = torch.ones(1, 64)
        r[0, 3] = bad
        pool = one_page(1)
        append_at(r, 2, pool, packed)
        assert torch.isnan(pool[2]).all() and (pool[0][0, 0, :2] == 7).all()
        append_at(torch.ones(1, 64), 3, pool, packed)
        assert torch.isnan(pool[2]).all()  # until the page begins anew
        append_at(torch.ones(1, 64), 0, pool, packed)
        assert abs(pool[2].item() - 1 / 127) < 1e-9 and (pool[0][0, 0, 0] == 127).all()


def test_append_unstored_rows_and_in_place(cuda_device):
    """Positions outside the table and page ids outside the pool: q is rotated, nothing is stored; out may be qkv's q columns."""
    g = torch.Generator().manual_seed(5)
    H, KV, hd, ps, T = 4, 2, 128, 16, 6
    x = torch.randn((T, (H + 2 * KV) * hd), generator=g).half().cuda()
    pos = i32([-1, 32, 31, 5, 2 ** 31 - 1, -2 ** 31])
    table = i32([[0, 1]] * 2 + [[0, 99], [-7, 1]] + [[0, 1]] * 2)
    kp = torch.zeros((3, KV, ps, hd), dtype=torch.int8, device="cuda")
    sc = torch.ones((3, KV), device="cuda")
    vp, vs = kp.clone(), sc.clone()
    f = nb.rope_freqs(hd, device="cuda")
    q = nb.rope_paged_append_q8(x, H, KV, hd, pos, f, kp, vp, sc, vs, table)
    assert not kp.any() and not vp.any() and (sc == 1).all() and (vs == 1).all()
    (qe, qb), _ = append64(x.view(T, H + 2 * KV, hd), H, KV, pos, f, hd, False, None, None, 0.0)
    assert ((q[:4].double() - qe.reshape(T, -1)[:4]).abs() <= qb.reshape(T, -1)[:4]).all()
    y = x.clone()
    r = nb.rope_paged_append_q8(y, H, KV, hd, pos, f, kp, vp, sc, vs, table, out=y[:, :H * hd])
    assert torch.equal(r, q) and torch.equal(y[:, H * hd:], x[:, H * hd:])
    # packed: the first row's position decides; one that lies outside leaves the sequence's rows up to the table unstored
    one = i32([[0, 1]])
    nb.rope_paged_append_q8(x, H, KV, hd, i32([30, 31, 32, 33, 34, 35]), f, kp, vp, sc, vs, one, cu_seqlens=i32([0, 6]))
    assert kp[1, :, 14:].any() and not kp[0].any() and not kp[2].any() and not kp[1, :, :14].any()


# ---------------------------------------------------------------- attention

class Cache:
    def __init__(self, keys, KV, hd, ps, *, seed, lo=0.01, hi=0.03):
        g = torch.Generator().manual_seed(seed)
        table, n = table_for(keys, ps, gen=g)
        self.ps, self.keys, self.table = ps, keys, table.cuda()
        q = lambda: torch.randint(-127, 128, (n, KV, ps, hd), generator=g, dtype=torch.int8).cuda()  # noqa: E731
        s = lambda: torch.exp(torch.empty(n, KV).uniform_(math.log(lo), math.log(hi), generator=g)).cuda()  # noqa: E731
        self.kp, self.vp, self.ks, self.vs = q(), q(), s(), s()
        used = torch.zeros(n, dtype=torch.bool)
        for b, m in enumerate(keys):
            used[table[b, :(m + ps - 1) // ps].long()] = True
        self.ks[~used.cuda()], self.vs[~used.cuda()] = float("nan"), float("inf")
        self.args = (self.kp, self.vp, self.ks, self.vs, self.table)
        self.lens = i32(keys)

    def seq(self, b):
        """(k, v, integers of v, scales of v) of sequence b in 64 bits"""
        at = torch.arange(self.keys[b], device="cuda")
        page, slot = self.table[b].long()[at // self.ps], at % self.ps
        kq, vq = self.kp[page, :, slot].double(), self.vp[page, :, slot].double()
        ks, vs = self.ks[page].double()[..., None], self.vs[page].double()[..., None]
        return kq * ks, vq * vs, vq, vs


def expected(cache, b, q, scale, causal):
    k, v, vq, vs = cache.seq(b)
    o, _ = attention_exact(q, k, v, scale, causal)
    n, H, d = q.shape
    m, KV = k.shape[:2]
    if m == 0:
        return o, torch.zeros_like(o)
    rep = lambda t: t.repeat_interleave(H // KV, 1)  # noqa: E731
    s = torch.einsum("nhd,mhd->hnm", q.double(), rep(k)) * scale
    seen = torch.ones((n, m), dtype=torch.bool, device="cuda")
    if causal:
        seen = torch.arange(m, device="cuda")[None, :] <= (m - n + torch.arange(n, device="cuda"))[:, None]
    w = torch.nan_to_num(torch.softmax(s.masked_fill(~seen, -math.inf), -1))
    a = torch.einsum("hnm,mhd->nhd", w, rep(v.abs())).reshape(n, -1)
    low = 2.0 ** -25 * torch.einsum("nm,mhd->nhd", seen.double(), rep(vq.abs())) * rep(vs.amax(0, keepdim=True))
    ks = cache.ks[cache.table[b].long()[:(m + cache.ps - 1) // cache.ps]].double().amax(0).repeat_interleave(H // KV)
    off = 2 * 2.0 ** -22 * scale * 255 * ks * q.double().abs().sum(-1)  # [n, H]
    bound = 2.0 ** -11 * o.abs() + 2.0 ** -25 + 1.25 * 2.0 ** -11 * a + low.reshape(n, -1)
    bound = bound + off.repeat_interleave(d, 1) * a
    bound[~seen.any(-1)] = 0.0
    return o, bound


def check_chunks(new, keys, H, KV, hd, ps, *, causal=True, max_new=None, ctx=0, scale=None, seed=0, qs=1.0, **kw):
    c = Cache(keys, KV, hd, ps, seed=seed + sum(keys), **kw)
    g = torch.Generator().manual_seed(seed)
    T = sum(new)
    q = (qs * torch.randn((T + 2, H * hd + 8), generator=g)).half().cuda()[:, :H * hd]
    q[T:] = float("nan")
    out = torch.full((T + 2, H * hd), 3.0, dtype=torch.float16, device="cuda")
    mn = max(new) if max_new is None else max_new
    nb.attention_paged_q8(q, *c.args, c.lens, offsets(new), heads=H, max_new=mn, ctx_len=ctx, causal=causal, scale=scale,
                          out=out)
    assert npu.device_error() == 0
    assert (out[T:] == 3.0).all()
    at = 0
    for b, n in enumerate(new):
        if n == 0:
            continue
        o, bound = expected(c, b, q[at:at + n].reshape(n, H, hd), scale or 1 / math.sqrt(hd), causal)
        same(out[at:at + n], o, bound)
        at += n


@pytest.mark.parametrize("H,KV,hd", [(1, 1, 16), (4, 4, 64), (8, 2, 128), (6, 2, 80), (32, 8, 128), (16, 1, 128), (10, 2, 48),
                                     (7, 1, 112)])
@pytest.mark.parametrize("ps", [16, 32, 64, 256])
def test_few_rows(cuda_device, H, KV, hd, ps):
    check_chunks([1, 2, 0, 3, 1], [1, 2, 5, 130, 1000], H, KV, hd, ps)


@pytest.mark.parametrize("H,KV,new", [(4, 4, 33), (4, 4, 128), (8, 2, 16), (32, 8, 5), (16, 1, 4), (6, 2, 17), (5, 1, 25), (128, 1, 1),
                                      (24, 1, 5), (34, 2, 3)])
@pytest.mark.parametrize("causal", [True, False])
def test_row_tiles(cuda_device, H, KV, new, causal):
    """Several tiles of 16 rows, the last of them partly filled, sequences shorter than their rows among them."""
    check_chunks([new, max(1, new - 7), new, 1], [700, new, max(0, new - 3), 65], H, KV, 64, 32, causal=causal)
    check_chunks([new], [5000], H, KV, 128, 64, causal=causal)


@pytest.mark.parametrize("H,KV,hd,ps", [(8, 2, 128, 16), (4, 4, 64, 64), (6, 2, 80, 32), (64, 2, 128, 128), (32, 1, 16, 256)])
@pytest.mark.parametrize("causal", [True, False])
def test_many_rows(cuda_device, H, KV, hd, ps, causal):
    check_chunks([100, 0, 1, 300], [100, 50, 400, 513], H, KV, hd, ps, causal=causal)
    check_chunks([3, 1], [2000, 1], H, KV, hd, ps, causal=causal, max_new=0)
    check_chunks([90, 20], [91, 0], H, KV, hd, ps, causal=causal)  # rows beyond their keys, and no keys at all


@pytest.mark.parametrize("H,KV,hd,ps", [(32, 8, 128, 16), (8, 8, 128, 64), (4, 1, 64, 128), (16, 1, 96, 32), (40, 2, 128, 16)])
@pytest.mark.parametrize("keys", [[1], [777], [0, 1, 15, 16, 17], [64, 65, 127, 128, 129, 5000], [20000]])
def test_decode(cuda_device, H, KV, hd, ps, keys):
    c = Cache(keys, KV, hd, ps, seed=sum(keys) + H)
    B = len(keys)
    q = torch.randn((B, H * hd), generator=torch.Generator().manual_seed(1)).half().cuda()
    for ctx in (0, max(keys + [1])):
        o = nb.attention_paged_decode_q8(q, *c.args, c.lens, heads=H, ctx_len=ctx)
        assert npu.device_error() == 0
        for b in range(B):
            want, bound = expected(c, b, q[b:b + 1].reshape(1, H, hd), 1 / math.sqrt(hd), True)
            same(o[b:b + 1], want, bound)


@pytest.mark.parametrize("H,KV,hd,ps", [(8, 8, 128, 16), (32, 8, 64, 64), (16, 1, 80, 32), (6, 3, 128, 128)])
@pytest.mark.parametrize("seqs,most", [(1, 30000), (70, 3000), (200, 400)])
def test_long_and_many_sequences(cuda_device, H, KV, hd, ps, seqs, most):
    """Ragged contexts, empty ones among them, with no rows, one, or several tiles: cut over the GPU wherever it falls."""
    g = torch.Generator().manual_seed(seqs + H)
    keys = [int(most * x) for x in torch.rand(seqs, generator=g).square().tolist()]
    keys[0] = most
    if seqs > 1:
        keys[1::7] = [0] * len(keys[1::7])
    new = torch.randint(0, 3 * 16 * KV // H + 1, (seqs,), generator=g).clamp(max=12).tolist()
    new[0] = max(new[0], 1)
    check_chunks(new, keys, H, KV, hd, ps, ctx=most)
    c = Cache(keys, KV, hd, ps, seed=seqs)
    q = torch.randn((seqs, H * hd), generator=g).half().cuda()
    o = nb.attention_paged_decode_q8(q, *c.args, c.lens, heads=H, ctx_len=most)
    for b in range(0, seqs, 9):
        want, bound = expected(c, b, q[b:b + 1].reshape(1, H, hd), 1 / math.sqrt(hd), True)
        same(o[b:b + 1], want, bound)


def planted_cache(m, KV, hd, ps, every, gen):
    """m keys of which one at a random place of every `every` scores alike and stands out in v, the others low: a stretch
    that is lost or weighed wrongly shows."""
    n = (m + ps - 1) // ps
    kq = torch.randint(-20, 21, (n, KV, ps, hd), generator=gen, dtype=torch.int8)
    vq = torch.randint(-1, 2, (n, KV, ps, hd), generator=gen, dtype=torch.int8)
    sign = torch.randint(0, 2, (KV, hd), generator=gen) * 2 - 1
    first = torch.arange(0, m, every)
    at = first + (torch.rand(len(first), generator=gen) * torch.clamp(m - first, max=every)).long()
    kq[at // ps, :, at % ps] = (sign * 100).to(torch.int8)
    vq[at // ps, :, at % ps] = 0
    vq[at // ps, :, at % ps, torch.arange(len(at)) % hd] = 120
    return kq, vq, sign.half()


@pytest.mark.parametrize("H,KV,n", [(8, 2, 1), (16, 1, 1), (8, 2, 14)])
def test_planted_keys_over_a_long_context(cuda_device, H, KV, n):
    g = torch.Generator().manual_seed(H + n)
    m, hd, ps = 100003, 128, 32
    kq, vq, sign = planted_cache(m, KV, hd, ps, 61, g)
    pages = kq.shape[0]
    c = Cache.__new__(Cache)
    c.ps, c.keys, c.kp, c.vp = ps, [m], kq.cuda(), vq.cuda()
    c.table = torch.arange(pages, dtype=torch.int32, device="cuda")[None]
    c.ks, c.vs = torch.full((pages, KV), 0.008, device="cuda"), torch.full((pages, KV), 0.02, device="cuda")
    q = sign.repeat_interleave(H // KV, 0).reshape(1, H * hd).repeat(n, 1).cuda()
    o = nb.attention_paged_q8(q, c.kp, c.vp, c.ks, c.vs, c.table, i32([m]), i32([0, n]), heads=H, max_new=n)
    want, bound = expected(c, 0, q.reshape(n, H, hd), 1 / math.sqrt(hd), True)
    same(o, want, bound)


@pytest.mark.parametrize("lo,hi", [(1e-6, 10.0), (1e-12, 1e-10), (1e-38, 1.0), (5.0, 400.0)])
def test_scales_far_apart(cuda_device, lo, hi):
    """Pages of one sequence with scales orders apart, the keys of the last far larger than fp16 holds too."""
    qs = 1.0 if hi < 5 else 1e-3
    check_chunks([2, 1], [300, 1000], 8, 2, 128, 16, lo=lo, hi=hi, qs=qs)
    check_chunks([100], [300], 8, 2, 128, 16, lo=lo, hi=hi, qs=qs)
    check_chunks([70, 90], [300, 1000], 4, 1, 64, 32, lo=lo, hi=hi, qs=qs)


@pytest.mark.parametrize("scale", [1e-38, 1e-3, 3.0])
def test_scale_argument(cuda_device, scale):
    check_chunks([2, 1], [300, 1000], 8, 2, 128, 16, scale=scale, qs=0.3)
    check_chunks([100], [300], 8, 2, 128, 16, scale=scale, qs=0.3)


@pytest.mark.parametrize("n", [1, 100])
def test_scales_of_zero_and_nan(cuda_device, n):
    keys, KV, hd, ps, H = [200, 200, 200], 2, 64, 32, 4
    c = Cache(keys, KV, hd, ps, seed=3)
    new = [n] * 3
    q = torch.randn((3 * n, H * hd), generator=torch.Generator().manual_seed(1)).half().cuda()
    c.ks[c.table[0, 1].long()] = 0.0
    c.vs[c.table[0, 2].long()] = 0.0
    c.vs[c.table[1, :7].long(), 1] = 0.0  # one head's values are all zero
    c.ks[c.table[2, 0].long(), 0] = float("nan")
    c.vs[c.table[2, 1].long(), 1] = float("inf")
    o = nb.attention_paged_q8(q, *c.args, c.lens, offsets(new), heads=H, max_new=n)
    for b in range(2):
        want, bound = expected(c, b, q[b * n:b * n + n].reshape(n, H, hd), 1 / 8, True)
        same(o[b * n:b * n + n], want, bound)
    assert (o[n:2 * n].view(n, H, hd)[:, 2:] == 0).all()
    assert torch.isnan(o[2 * n:].view(n, H, hd)).all()


def test_rows_past_max_new_and_keys_past_ctx_len(cuda_device):
    """max_new too small: zeros past the tiles that it gives, the rows before them as they are; ctx_len too small for a
    call of many rows: zeros for the sequence, the others as they are."""
    H, KV, hd, ps = 8, 2, 64, 16
    c = Cache([300, 40], KV, hd, ps, seed=8)
    q = torch.randn((12, H * hd), generator=torch.Generator().manual_seed(1)).half().cuda()
    o = nb.attention_paged_q8(q, *c.args, c.lens, i32([0, 10, 12]), heads=H, max_new=4)
    want, bound = expected(c, 0, q[:10].reshape(10, H, hd), 1 / 8, True)
    same(o[:4], want[:4], bound[:4])
    assert not o[4:10].any()
    want, bound = expected(c, 1, q[10:].reshape(2, H, hd), 1 / 8, True)
    same(o[10:], want, bound)
    q = torch.randn((120, H * hd), generator=torch.Generator().manual_seed(1)).half().cuda()
    o = nb.attention_paged_q8(q, *c.args, c.lens, i32([0, 90, 120]), heads=H, max_new=90, ctx_len=100)
    assert not o[:90].any()
    want, bound = expected(c, 1, q[90:].reshape(30, H, hd), 1 / 8, True)
    same(o[90:], want, bound)


def test_page_ids_outside_the_pool(cuda_device):
    """Their keys count as zeros, here with the weight exp(0)."""
    H, KV, hd, ps = 4, 2, 64, 16
    c = Cache([64], KV, hd, ps, seed=2)
    c.table[0, 1], c.table[0, 3] = -1, 1 << 30
    for n in (1, 80):
        q = torch.randn((n, H * hd), generator=torch.Generator().manual_seed(1)).half().cuda()
        o = nb.attention_paged_q8(q, *c.args, c.lens, i32([0, n]), heads=H, max_new=n)
        t = c.table.clone()
        t[0, 1] = t[0, 3] = 0
        at = torch.arange(64, device="cuda")
        page, ok = t[0].long()[at // ps], ((at // ps) % 2 == 0)[:, None, None]
        k = torch.where(ok, c.kp[page, :, at % ps].double() * c.ks[page].double()[..., None], 0.0)
        v = torch.where(ok, c.vp[page, :, at % ps].double() * c.vs[page].double()[..., None], 0.0)
        want, bound = attention_exact(q.reshape(n, H, hd), k, v, 1 / 8)
        same(o, want, bound + 2.0 ** -25 * 64 * 127 * 0.03)


def test_append_then_attend(cuda_device):
    """A prompt in chunks, then decode steps: the cache read back by the attention is what the appends stored, and
    within the steps of its scales of the rows themselves."""
    g = torch.Generator().manual_seed(11)
    H, KV, hd, ps, B = 8, 2, 128, 32, 3
    f = nb.rope_freqs(hd, device="cuda")
    W = 12
    table = torch.randperm(B * W, generator=g).int().view(B, W).cuda()
    kp = torch.randint(-127, 128, (B * W, KV, ps, hd), generator=g, dtype=torch.int8).cuda()
    vp = kp.flip(0).contiguous()
    ks, vs = torch.full((B * W, KV), 77.0, device="cuda"), torch.full((B * W, KV), float("nan"), device="cuda")
    held, lens = [[] for _ in range(B)], [0] * B
    for new in ([50, 1, 7], [100, 33, 64], [1, 1, 1], [1, 1, 1], [5, 70, 1], [1, 1, 1]):
        T = sum(new)
        x = torch.randn((T, (H + 2 * KV) * hd), generator=g).half().cuda()
        pos = i32([l + i for l, n in zip(lens, new) for i in range(n)])
        packed = max(new) > 1
        q = nb.rope_paged_append_q8(x, H, KV, hd, pos, f, kp, vp, ks, vs, table, cu_seqlens=offsets(new) if packed else None)
        (_, _), (ke, _) = append64(x.view(T, -1, hd), H, KV, pos, f, hd, False, None, None, 0.0)
        ve = x.view(T, -1, hd)[:, H + KV:].double()
        lens = [a + n for a, n in zip(lens, new)]
        at = 0
        for b, n in enumerate(new):
            held[b].append((ke[at:at + n], ve[at:at + n]))
            at += n
        ln = i32(lens)
        o = (nb.attention_paged_q8(q, kp, vp, ks, vs, table, ln, offsets(new), heads=H, max_new=max(new)) if packed
             else nb.attention_paged_decode_q8(q, kp, vp, ks, vs, table, ln, heads=H))
        at = 0
        for b, n in enumerate(new):
            c = Cache.__new__(Cache)
            c.ps, c.keys, c.table, c.kp, c.vp, c.ks, c.vs = ps, lens, table, kp, vp, ks, vs
            want, bound = expected(c, b, q[at:at + n].reshape(n, H, hd), 1 / math.sqrt(hd), True)
            same(o[at:at + n], want, bound)
            k, v, _, _ = c.seq(b)
            page = table[b].long()[torch.arange(lens[b], device="cuda") // ps]
            for got, s, rows in ((k, ks, 0), (v, vs, 1)):
                true = torch.cat([h[rows] for h in held[b]])
                # half a step at its own append and half at each later one of its page (here at most six)
                assert ((got - true).abs() <= 3.6 * s[page].double()[..., None]).all()
                assert ((got - true).square().mean() <= (0.6 * s[page].double()).square().mean())
            at += n


def test_the_same_bits_and_a_graph(cuda_device):
    keys, H, KV, hd, ps = [3000, 10, 700, 0], 8, 2, 128, 16
    c = Cache(keys, KV, hd, ps, seed=4)
    q = torch.randn((4, H * hd), generator=torch.Generator().manual_seed(2)).half().cuda()
    qm = torch.randn((400, H * hd), generator=torch.Generator().manual_seed(2)).half().cuda()
    cu = i32([0, 300, 310, 400, 400])

    def step():
        return (nb.attention_paged_decode_q8(q, *c.args, c.lens, heads=H, ctx_len=3000),
                nb.attention_paged_q8(qm, *c.args, c.lens, cu, heads=H, max_new=300, ctx_len=3000))
    want = step()
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(want, step()))
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        other = step()
    st.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, other))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    c.lens[0] = 1234
    q.mul_(0.5)
    want = step()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, held))


def test_refusals(cuda_device):
    H, KV, hd, ps = 4, 2, 64, 16
    c = Cache([40, 3], KV, hd, ps, seed=1)
    q = torch.randn(2, H * hd, device="cuda").half()
    d = lambda **kw: nb.attention_paged_decode_q8(kw.pop("q", q), kw.pop("kp", c.kp), c.vp, kw.pop("ks", c.ks), c.vs,  # noqa: E731
                                                  c.table, kw.pop("lens", c.lens), heads=kw.pop("heads", H), **kw)
    for kw in (dict(q=q.float()), dict(q=q[:1]), dict(kp=c.kp.half()), dict(kp=c.kp[:, :1]), dict(ks=c.ks.half()),
               dict(ks=c.ks[:1]), dict(ks=c.ks.t()), dict(lens=c.lens.long()), dict(heads=3), dict(scale=0.0),
               dict(scale=math.inf), dict(ks=c.ks.cpu())):
        with pytest.raises(ValueError):
            d(**kw)
    x = torch.randn(2, (H + 2 * KV) * hd, device="cuda").half()
    f = nb.rope_freqs(hd, device="cuda")
    a = lambda **kw: nb.rope_paged_append_q8(kw.pop("x", x), H, KV, kw.pop("hd", hd), kw.pop("pos", c.lens), kw.pop("f", f),  # noqa: E731
                                             c.kp, c.vp, c.ks, kw.pop("vs", c.vs), c.table, **kw)
    for kw in (dict(x=x[:, 8:]), dict(hd=32), dict(pos=c.lens[:1]), dict(f=f[1:]), dict(vs=c.vs.double()), dict(rot_dim=24),
               dict(q_gamma=f), dict(cu_seqlens=c.lens), dict(x=x[:1])):
        with pytest.raises(ValueError):
            a(**kw)
