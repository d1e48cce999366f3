"""Scales that are not finite in a long 8-bit paged cache: rows that see such a
page are NaN in that head, wherever the keys are cut, and all others are as the
64-bit form has them (bounds of test_gpu_paged_q8)."""
import math

import pytest
import torch

import npu_comp_b200 as nb
from npu_comp_b200 import _lib, npu
from paged_exact import same
from test_gpu_paged_q8 import Cache, expected, i32, offsets

pytestmark = pytest.mark.gpu


def spoil(c, b, lo, hi, head, which, value):
    """The scale of every page of sequence b that holds one of its keys lo .. hi - 1."""
    pages = c.table[b, lo // c.ps:(hi - 1) // c.ps + 1].long()
    (c.ks if which == "k" else c.vs)[pages, head] = value


def attend(c, q, new, H, **kw):
    o = (nb.attention_paged_decode_q8(q, *c.args, c.lens, heads=H) if kw.pop("decode", False)
         else nb.attention_paged_q8(q, *c.args, c.lens, offsets(new), heads=H, **kw))
    assert npu.device_error() == 0
    return o


def is_list(B, total, max_new, keys, H, KV, hd, ps):
    """The call takes the list of all sequences' steps: the only few-row kernel with a workspace."""
    ctx = ((max(keys) + ps - 1) // ps + 1) * ps  # the table's width
    return _lib.query("npub_attention_paged_q8_workspace", B, total, max_new, ctx, H, KV, hd) > 0


@pytest.mark.parametrize("which,value", [("k", math.nan), ("v", math.nan), ("k", math.inf), ("v", -math.inf)])
@pytest.mark.parametrize("ps", [16, 128, 256])
@pytest.mark.parametrize("where", ["first", "middle", "last", "one page"])
@pytest.mark.parametrize("n", [1, 6])
def test_one_long_sequence(cuda_device, which, value, ps, where, n):
    """16384 keys of 8 heads are 1024 parts of 128 keys: whole parts have no finite score (few rows: the combination by
    blocks)."""
    H, KV, hd, m = 32, 8, 128, 16384
    assert is_list(1, n, n, [m], H, KV, hd, ps)
    c = Cache([m], KV, hd, ps, seed=ps + n)
    lo, hi = {"first": (0, 512), "middle": (7936, 8448), "last": (m - 512, m), "one page": (5120, 5121)}[where]
    spoil(c, 0, lo, hi, 3, which, value)
    q = torch.randn((n, H * hd), generator=torch.Generator().manual_seed(n)).half().cuda()
    o = attend(c, q, [n], H, decode=n == 1, **({} if n == 1 else {"max_new": n}))
    nan = torch.isnan(o.view(n, KV, -1))
    assert nan[:, 3].all() and not nan[:, :3].any() and not nan[:, 4:].any()
    want, bound = expected(c, 0, q.view(n, H, hd), 1 / math.sqrt(hd), True)
    same(o, want, bound)


@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("ps", [32, 256])
@pytest.mark.parametrize("n", [1, 2])
def test_many_long_sequences(cuda_device, which, ps, n):
    """24 sequences, the combination by warps: parts of several hundred keys, of which some sequences' are all spoilt."""
    H, KV, hd, B = 32, 8, 128, 24
    keys = [6000 + 100 * b for b in range(B)]
    assert is_list(B, B * n, n, keys, H, KV, hd, ps)
    c = Cache(keys, KV, hd, ps, seed=ps + n)
    at = {b: 0 if b % 2 else keys[b] - 2600 for b in range(0, B, 3)}
    for b, lo in at.items():
        spoil(c, b, lo, lo + 2500, b % KV, which, math.nan)
    q = torch.randn((B * n, H * hd), generator=torch.Generator().manual_seed(n)).half().cuda()
    o = attend(c, q, [n] * B, H, max_new=n).view(B, n, KV, -1)
    nan = torch.isnan(o)
    for b in range(B):
        for h in range(KV):
            assert nan[b, :, h].all() if b in at and h == b % KV else not nan[b, :, h].any(), (b, h)
    for b in (0, 1, 9, B - 1):
        want, bound = expected(c, b, q[b * n:b * n + n].view(n, H, hd), 1 / math.sqrt(hd), True)
        same(o[b].reshape(n, -1), want, bound)


def test_nan_beside_scores_far_above(cuda_device):
    """A part with a NaN and finite scores more than 126 powers of two below the others'."""
    H, KV, hd, ps, m = 8, 8, 128, 16, 32768
    assert is_list(1, 1, 1, [m], H, KV, hd, ps)
    c = Cache([m], KV, hd, ps, seed=5)
    q = torch.ones((1, H * hd)).half().cuda()
    c.kp[:] = 1
    c.ks[:] = 1.0
    c.ks[c.table[0, :128].long()] = 30.0  # the first 2048 keys score 30 * 128 / sqrt(128), the others a thirtieth of it
    spoil(c, 0, 20000, 20001, 2, "k", math.nan)
    o = attend(c, q, [1], H, decode=True)
    nan = torch.isnan(o.view(KV, -1))
    assert nan[2].all() and not nan[:2].any() and not nan[3:].any()


@pytest.mark.parametrize("which,value", [("k", math.nan), ("v", math.nan), ("v", math.inf)])
@pytest.mark.parametrize("m,n,max_new,hd", [
    (208, 32, 32, 128),     # one CTA
    (1010, 24, 24, 64),     # ranges of a cluster
    (16400, 24, 24, 128),   # the list
    (300, 100, 100, 128),   # tiles
    (5005, 30, 0, 64),      # tiles, keys in parts
    (36000, 200, 200, 128),
])
def test_pages_behind_a_row(cuda_device, which, value, m, n, max_new, hd):
    """Rows that the causal mask keeps from a page whose scale is not finite do not see it; the rows behind them do."""
    H, KV, ps = 4, 4, 16
    c = Cache([m, 40], KV, hd, ps, seed=m)
    from_key = (m - 1) // ps * ps  # of the last page
    clean = n - (m - from_key)     # rows that end ahead of it
    assert 0 < clean < n
    q = torch.randn((n + 1, H * hd), generator=torch.Generator().manual_seed(n)).half().cuda()
    want, bound = expected(c, 0, q[:n].view(n, H, hd), 1 / math.sqrt(hd), True)
    alone, alone_bound = expected(c, 1, q[n:].view(1, H, hd), 1 / math.sqrt(hd), True)
    spoil(c, 0, from_key, m, 1, which, value)
    o = attend(c, q, [n, 1], H, max_new=max_new)
    nan = torch.isnan(o[:n].view(n, H, hd))
    assert nan[clean:, 1].all()
    assert not nan[clean:, 0].any() and not nan[clean:, 2:].any() and not nan[:clean].any()
    want.view(n, H, hd)[clean:, 1] = math.nan
    same(o[:n], want, bound)
    same(o[n:], alone, alone_bound)


@pytest.mark.parametrize("scale,spread", [(1e30, 100.0), (1e-3, 1e36), (1e34, 1e-3)])
@pytest.mark.parametrize("m,n,hd", [(500, 1, 128), (1000, 9, 64), (16400, 2, 128), (600, 80, 128)])
def test_scores_of_any_size(cuda_device, scale, spread, m, n, hd):
    """Finite scores of 1e30 and more: the largest takes all of the weight."""
    H, KV, ps = 8, 2, 16
    c = Cache([m], KV, hd, ps, seed=m + n)
    c.ks[c.table[0, :(m + ps - 1) // ps].long()] = spread
    q = (torch.randn((n, H * hd), generator=torch.Generator().manual_seed(n)) / 8).half().cuda()
    k, v, _, _ = c.seq(0)
    x = torch.einsum("nhd,mhd->hnm", q.view(n, H, hd).double(), k.repeat_interleave(H // KV, 1) / spread)
    seen = torch.arange(m, device="cuda")[None] <= (m - n + torch.arange(n, device="cuda"))[:, None]
    best = x.masked_fill(~seen, -math.inf).topk(2, -1)
    # fp32 roundings of 255 sum |q| (two for a bit each at every one of hd terms), and exp(-scale * spread * gap) is 0 beyond
    off = hd * 2.0 ** -22 * 255 * q.view(n, H, hd).double().abs().sum(-1).T
    clear = best.values[..., 0] - best.values[..., 1] > off
    assert clear.double().mean() > 0.9 and (best.values[..., 0] * scale * spread * 1.45 < 3e38).all()
    o = attend(c, q, [n], H, max_new=n, scale=scale)
    assert torch.isfinite(o).all()
    want = v.repeat_interleave(H // KV, 1)[best.indices[..., 0], torch.arange(H, device="cuda")[:, None]].transpose(0, 1)
    err = (o.view(n, H, hd).double() - want).abs()
    assert (err[clear.T] <= 1.25 * 2.0 ** -11 * want.abs()[clear.T] + 2.0 ** -24).all()
