"""64-bit forms of attention over packed rows and pages that keep what a score
of inf or NaN does, with bounds that divide by the row's own softmax sum, and
keys planted so that every stretch of a long context shows in the result.

Bound per element (half a step of fp16 is 2^-11 relative, 2^-25 absolute below
the normal range), w the weights, s the scores, L = sum_j exp(s_j - max s):
  2^-11 |o| + 2^-25            the output's rounding
  1.25 * 2^-11 sum w |v|       each weight's rounding to fp16 before the
                               product, and a quarter of it for fp32 scores
                               (sums of up to 128 products of magnitude ~10,
                               each off by 2^-24), exp2 and sums
  2^-25 sum |v| / L            weights below fp16's normal range: 2^-25 each
                               against the reference maximum of their range of
                               keys, which is never above max s, so the sum of
                               weights they are divided by is at least L
"""
import math

import torch


def attention_exact(q, k, v, scale, causal=True):
    """(o, bound): q [n, H, d] the last n of the m keys k, v [m, KV, d].  A row
    that sees no key is zero (bound 0); a row with a score of NaN or +inf, or
    whose visible scores are all -inf, is NaN."""
    n, H, d = q.shape
    m, KV = k.shape[:2]
    if m == 0:
        z = torch.zeros(n, H * d, dtype=torch.float64, device=q.device)
        return z, z.clone()
    k = k.double().repeat_interleave(H // KV, 1)
    v = v.double().repeat_interleave(H // KV, 1)
    s = torch.einsum("nhd,mhd->hnm", q.double(), k) * scale
    seen = torch.ones((n, m), dtype=torch.bool, device=q.device)
    if causal:
        j, i = torch.arange(m, device=q.device), torch.arange(n, device=q.device)
        seen = j[None, :] <= (m - n + i)[:, None]
    s = s.masked_fill(~seen, -math.inf)
    e = torch.exp(s - s.amax(-1, keepdim=True))  # NaN for +inf - +inf and -inf - -inf, as in the formula
    e = e.masked_fill(~seen, 0.0)
    L = e.sum(-1, keepdim=True)
    blind = ~seen.any(-1)  # rows without keys
    w = (e / L).masked_fill(blind[None, :, None], 0.0)
    o = torch.einsum("hnm,mhd->nhd", w, v)
    a = torch.einsum("hnm,mhd->nhd", w, v.abs())
    below = torch.einsum("nm,mhd->nhd", seen.double(), v.abs()) / L[..., 0].T[:, :, None]
    bound = 2.0 ** -11 * o.abs() + 2.0 ** -25 + 1.25 * 2.0 ** -11 * a + 2.0 ** -25 * below
    bound[blind] = 0.0
    return o.reshape(n, -1), bound.reshape(n, -1)


def same(got, want, bound):
    """NaN exactly where the formula has it, all else within the bound."""
    bad = torch.isnan(got) != torch.isnan(want)
    assert not bad.any(), f"{int(bad.sum())} elements differ in being NaN, first at {bad.nonzero()[0].tolist()}"
    err = (got.double() - want).abs()
    ok = torch.isnan(want) | (err <= bound)
    assert ok.all(), f"worst excess {(err - bound)[~ok].max().item():.3g} at {(~ok).nonzero()[0].tolist()}"


def to_pages(k, v, ps, *, shared=0, seed=0):
    """Lists of k, v [m, KV, d] of the sequences -> (k_pages, v_pages, table,
    lens): shuffled pages, NaN in every slot that no key uses, ids outside the
    pool past a sequence's keys; the first `shared` keys of all in the pages of
    sequence 0."""
    dev, (_, KV, d) = k[0].device, k[0].shape
    sp, need = shared // ps, [(x.shape[0] + ps - 1) // ps for x in k]
    n = sp + sum(max(0, x - sp) for x in need) + 2
    ids = torch.randperm(n, generator=torch.Generator().manual_seed(seed)).tolist()
    table = torch.full((len(k), max(need + [sp]) + 1), 1 << 30, dtype=torch.int32)
    pools = [torch.full((n, KV, ps, d), float("nan"), dtype=torch.float16, device=dev) for _ in range(2)]
    at = sp
    for b, m in enumerate(need):
        own = max(0, m - sp)
        row = ids[:sp] + ids[at:at + own]
        at += own
        table[b, :len(row)] = torch.tensor(row, dtype=torch.int32)
        p = torch.arange(k[b].shape[0], device=dev)
        page = torch.tensor(row or [0], device=dev)[p // ps]
        if b == 0 or shared == 0 or own:
            pools[0][page, :, p % ps], pools[1][page, :, p % ps] = k[b], v[b]
    lens = torch.tensor([x.shape[0] for x in k], dtype=torch.int32, device=dev)
    return pools[0], pools[1], table.to(dev), lens


def planted(m, KV, hd, *, every, gen, dev="cpu"):
    """(u, k, v): m keys of which one at a random place of every `every` has the
    score sqrt(hd) against the query u [KV, hd] of +-1 (an exact sum) and v one
    at column (its number mod hd); the others have scores ~ N(0, 1) and small v.
    The planted keys carry the result alike, so losing a stretch of keys, or
    weighing it wrongly, shows in the columns that it plants."""
    u = torch.randint(0, 2, (KV, hd), generator=gen).mul(2).sub(1).half()
    k = torch.randn((m, KV, hd), generator=gen).half()
    v = (0.01 * torch.randn((m, KV, hd), generator=gen)).half()
    first = torch.arange(0, m, every)
    at = first + (torch.rand(len(first), generator=gen) * torch.clamp(m - first, max=every)).long()
    k[at] = u
    v[at] = 0.0
    v[at, :, torch.arange(len(at)) % hd] = 1.0
    return u.to(dev), k.to(dev), v.to(dev)
