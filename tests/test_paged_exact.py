"""The planted contexts of paged_exact.py (CPU): a stretch of keys that is lost
or weighed wrongly leaves the bound, at every size that the GPU tests use."""
import math

import pytest
import torch

from paged_exact import attention_exact, planted, to_pages


@pytest.mark.parametrize("m,hd,every", [(70001, 128, 64), (66000, 64, 64), (20000, 128, 64), (4096 + 300, 128, 64)])
def test_a_lost_stretch_leaves_the_bound(m, hd, every):
    u, k, v = planted(m, 1, hd, every=every, gen=torch.Generator().manual_seed(m))
    scale = 1 / math.sqrt(hd)
    o, bound = attention_exact(u[None], k, v, scale)
    s = (k[:, 0].double() @ u[0].double()) * scale
    w = torch.exp(s - s.max())
    vd = v[:, 0].double()
    num, den = w @ vd, w.sum()
    assert ((num / den - o[0]).abs() <= 1e-12).all()
    for k0 in range(0, m, every):
        part = slice(k0, min(m, k0 + every))
        n, d = w[part] @ vd[part], w[part].sum()
        for f in (-1.0, 1.0, 0.1):  # lost, taken twice, a tenth too heavy
            wrong = (num + f * n) / (den + f * d)
            assert ((wrong - o[0]).abs() > bound[0]).any(), (k0, f)


def test_nonfinite_scores_and_blind_rows():
    g = torch.Generator().manual_seed(1)
    q = torch.randn((3, 1, 16), generator=g).abs().half()
    k, v = torch.randn((4, 1, 16), generator=g).half(), torch.randn((4, 1, 16), generator=g).half()
    k[2, 0, 0] = math.inf  # seen by rows 1 and 2 of the last three
    o, b = attention_exact(q, k, v, 0.25)
    assert torch.isnan(o).all(1).tolist() == [False, True, True] and torch.isfinite(b[0]).all()
    k[:2, 0, 0], k[2, 0, 0] = -math.inf, 1.0
    o, _ = attention_exact(q, k, v, 0.25)
    assert torch.isnan(o).all(1).tolist() == [True, False, False]
    o, b = attention_exact(q, k[2:3], v[2:3], 0.25)  # more rows than keys
    assert not o[:2].any() and not b[:2].any() and torch.isfinite(o).all() and o[2].any()


def test_pages_hold_the_keys():
    g = torch.Generator().manual_seed(2)
    k = [torch.randn((n, 2, 16), generator=g).half() for n in (70, 48, 33)]
    for x in k[1:]:
        x[:32] = k[0][:32]
    kp, _, table, lens = to_pages(k, k, 16, shared=32)
    assert lens.tolist() == [70, 48, 33] and (table[:, :2] == table[0, :2]).all()
    for b, x in enumerate(k):
        p = torch.arange(len(x))
        assert torch.equal(kp[table[b].long()[p // 16], :, p % 16], x)
    assert int(torch.isfinite(kp).all(-1).all(1).sum()) == 32 + 38 + 16 + 1
