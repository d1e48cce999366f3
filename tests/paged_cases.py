"""Plain 64-bit forms and error bounds of the paged-cache operators, shared by
their GPU tests.

Bounds, per element (half a step of fp16 is 2^-11 relative, 2^-25 absolute
below the normal range):
  append     one rounding of an fp32 value: 2^-11 |y|, plus the fp32 arithmetic
             of the norm and of a cos - b sin, within 2^-20 of the largest
             |column| of the head.
  attention  the output's rounding 2^-11 |o|; each weight's rounding to fp16
             before the product, 2^-11 of its share of sum w |v|, with a
             quarter of that again for the fp32 scores (sums of up to 128
             products of magnitude ~10), exp2 and sums; weights below fp16's
             normal range, 2^-25 each at a sum of at least 1.
"""
import math

import torch


def table_for(keys, ps, *, gen, n_extra=3, shared=0, width=None):
    """A shuffled page table int32 [B, W] for `keys` keys per sequence, the
    first `shared` keys of all in the same pages, and the pool's page count.
    Entries past a sequence's keys are ids outside the pool."""
    sp = shared // ps
    need = [max(0, (k + ps - 1) // ps - sp) for k in keys]
    n = sp + sum(need) + n_extra
    ids = torch.randperm(n, generator=gen).tolist()
    W = width or max(1, max((k + ps - 1) // ps for k in keys), sp) + 1
    t = torch.full((len(keys), W), 1 << 30, dtype=torch.int32)
    at = sp
    for b, m in enumerate(need):
        t[b, :sp] = torch.tensor(ids[:sp], dtype=torch.int32)
        t[b, sp:sp + m] = torch.tensor(ids[at:at + m], dtype=torch.int32)
        at += m
    return t, n


def poison(kp, vp, table, keys, ps):
    """NaN and inf in every slot that no key of the batch uses."""
    used = torch.zeros(kp.shape[0], ps, dtype=torch.bool)
    for b, n in enumerate(keys):
        for w in range((n + ps - 1) // ps):
            used[int(table[b, w]), :min(ps, n - w * ps)] = True
    free = (~used).nonzero()
    kp[free[:, 0], :, free[:, 1]] = float("nan")
    vp[free[:, 0], :, free[:, 1]] = float("inf")
    vp[free[::2, 0], :, free[::2, 1]] = float("nan")


def attention64(q, k, v, scale, causal=True):
    """(o, bound) in 64 bits: q [n, H, d] the last n of the m keys k, v [m, KV, d]."""
    n, H, d = q.shape
    m, KV = k.shape[:2]
    if m == 0:
        z = torch.zeros(n, H * d, dtype=torch.float64, device=q.device)
        return z, z.clone()
    k = k.double().repeat_interleave(H // KV, 1)
    v = v.double().repeat_interleave(H // KV, 1)
    s = torch.einsum("nhd,mhd->hnm", q.double(), k) * scale
    if causal:
        j, i = torch.arange(m, device=q.device), torch.arange(n, device=q.device)
        s = s.masked_fill(j[None, :] > (m - n + i)[:, None], -math.inf)
    w = torch.nan_to_num(torch.softmax(s, -1), nan=0.0)  # a row without keys
    o = torch.einsum("hnm,mhd->nhd", w, v).reshape(n, -1)
    a = torch.einsum("hnm,mhd->nhd", w, v.abs()).reshape(n, -1)
    bound = 2.0 ** -11 * o.abs() + 1.25 * 2.0 ** -11 * a + (m * v.abs().max().item() + 1) * 2.0 ** -25
    return o, bound * (w.sum(-1).amax(0) > 0)[:, None]  # rows without keys: exactly zero


def gather(pages, row, n, ps):
    at = torch.arange(n, device=pages.device)
    return pages[row.to(pages.device).long()[at // ps], :, at % ps]


def append64(x, H, KV, positions, inv_freq, rot, interleaved, gq, gk, eps):
    """x [T, (H + 2 KV), hd] -> (q, k) in 64 bits with their bounds."""
    x = x.double()
    out = []
    for y, g in ((x[:, :H], gq), (x[:, H:H + KV], gk)):
        if g is not None:
            y = y / torch.sqrt(y.square().mean(-1, keepdim=True) + eps) * g.double()
        a = (positions.double()[:, None] * inv_freq.double())[:, None]
        c, s = a.cos(), a.sin()
        z = y.clone()
        i0 = slice(0, rot, 2) if interleaved else slice(0, rot // 2)
        i1 = slice(1, rot, 2) if interleaved else slice(rot // 2, rot)
        z[..., i0] = y[..., i0] * c - y[..., i1] * s
        z[..., i1] = y[..., i1] * c + y[..., i0] * s
        out.append((z, 2.0 ** -11 * z.abs() + 2.0 ** -20 * y.abs().amax(-1, keepdim=True) + 2.0 ** -25))
    return out
