"""Sampling on the GPU against the definition, walked token by token in 64 bits
(weights from math.exp, sums from math.fsum).

The tokens have to be equal: the kernel's sums are fp64, off by at most 1e-13 of
the sum, so a random number would have to fall within 1e-13 of a border; where a
test puts numbers on a border its weights are exact in fp64."""
import math

import pytest
import torch

import npu_comp_b200 as nb

pytestmark = pytest.mark.gpu


def order_of(l):
    """Indices by descending logit, ties by index; -inf and NaN left out."""
    l = l.double().cpu()
    idx = torch.argsort(torch.nan_to_num(l, nan=-math.inf, posinf=math.inf, neginf=-math.inf), descending=True, stable=True)
    return [i for i in idx.tolist() if l[i] > -math.inf]


def draw(l, u, t, k, p, m):
    order = order_of(l)
    if not order:
        return -1
    l = l.double().tolist()
    if not t > 0:
        return order[0]
    top = l[order[0]]
    w = [1.0 if l[i] == top else 0.0 if top == math.inf else math.exp((l[i] - top) / t) for i in order]
    n = min(k, len(w)) if k > 0 else len(w)
    goal, run, kept = p * math.fsum(w[:n]), 0.0, 0
    for x in w[:n]:
        if kept and ((p < 1.0 and run >= goal) or x < m):
            break
        run, kept = run + x, kept + 1
    goal, run = u * math.fsum(w[:kept]), 0.0
    for i in range(kept):
        run += w[i]
        if run > goal:
            return order[i]
    return order[kept - 1]


def f32(*v):
    return torch.tensor(v, dtype=torch.float32)


def check(x, u, t, k, p, m):
    rows = x.shape[0]
    spread = lambda v, d: v.to(d).expand(rows).contiguous() if isinstance(v, torch.Tensor) else torch.full((rows,), v, dtype=d)  # noqa: E731
    t, k, p, m = spread(t, torch.float32), spread(k, torch.int32), spread(p, torch.float32), spread(m, torch.float32)
    got = nb.sample(x, u.cuda(), temperature=t.cuda(), top_k=k.cuda(), top_p=p.cuda(), min_p=m.cuda()).tolist()
    xs = x.cpu()
    want = [draw(xs[r], u[r].item(), t[r].item(), k[r].item(), p[r].item(), m[r].item()) for r in range(rows)]
    assert got == want, [(r, a, b) for r, (a, b) in enumerate(zip(got, want)) if a != b][:5]
    return got


@pytest.mark.parametrize("vocab", [1, 2, 7, 300, 1003, 32000, 40960, 40961, 81920, 81929, 128256, 200003, 524224])
def test_sizes_and_settings(cuda_device, vocab):
    g = torch.Generator().manual_seed(vocab)
    rows = 12 if vocab < 30000 else 4 if vocab < 100000 else 2
    x = (2.5 * torch.randn((rows, vocab), generator=g)).half().cuda()
    pick = lambda *v: torch.tensor(v)[torch.randint(0, len(v), (rows,), generator=g)]  # noqa: E731
    check(x, torch.rand(rows, generator=g), pick(0.0, 0.7, 1.0, 1.5), pick(0, 1, 5, 50, vocab, vocab + 9),
          pick(1.0, 0.99, 0.9, 0.3, 0.0), pick(0.0, 0.0, 0.05, 1.0))
    check(x, torch.rand(rows, generator=g), 1.0, 0, 1.0, 0.0)
    check(x, torch.rand(rows, generator=g), 1.3, 0, 0.95, 0.0)


@pytest.mark.parametrize("rows,vocab", [(1, 40000), (30, 40000), (37, 60000), (70, 60000), (148, 50000), (149, 65000), (300, 1500),
                                        (70, 128256), (19, 300000)])
def test_many_rows(cuda_device, rows, vocab):
    """Every number of CTAs for a row, against the definition in whole-row fp64 operations (whose sums run in another order)."""
    g = torch.Generator(device="cuda").manual_seed(rows)
    x = (3.0 * torch.randn((rows, vocab), generator=g, device="cuda")).half()
    x[:, ::5] = -math.inf
    u = torch.rand(rows, generator=g, device="cuda")
    pick = lambda *v: torch.tensor(v, device="cuda")[torch.randint(0, len(v), (rows,), generator=g, device="cuda")]  # noqa: E731
    t, k = pick(0.5, 1.0, 1.7).float(), pick(0, 0, 3, 77, 1000).int()
    p, m = pick(1.0, 0.97, 0.8, 0.2).float(), pick(0.0, 0.0, 0.003, 0.2).float()
    l, index = torch.sort(x.double(), dim=-1, descending=True, stable=True)
    w = torch.exp((l - l[:, :1]) / t.double()[:, None])
    cum = torch.cumsum(w, -1)
    n = torch.where(k > 0, k, vocab).long()[:, None]
    kept = (torch.arange(vocab, device="cuda") < n) & (w >= m.double()[:, None])
    goal = p.double()[:, None] * cum.gather(-1, n - 1)
    kept &= (p >= 1.0)[:, None] | (cum - w < goal)
    n = kept.sum(-1, keepdim=True).clamp(min=1)
    at = torch.minimum((cum <= u.double()[:, None] * cum.gather(-1, n - 1)).sum(-1, keepdim=True), n - 1)
    want = index.gather(-1, at)[:, 0].int()
    assert torch.equal(nb.sample(x, u, temperature=t, top_k=k, top_p=p, min_p=m), want)


@pytest.mark.parametrize("spread", [0.0, 1e-3, 0.05, 30.0, 20000.0])
@pytest.mark.parametrize("t", [1e-3, 0.5, 1.0, 100.0, 1e6, math.inf])
def test_distributions(cuda_device, spread, t):
    """Flat, nearly flat and peaked rows; +-0, subnormals and the largest values among them."""
    g = torch.Generator().manual_seed(7)
    x = (spread * torch.randn((4, 5000), generator=g)).clamp(-65504, 65504).half()
    x[1, ::3] = -0.0
    x[2, 100:110] = torch.tensor([2.0 ** -24, -2.0 ** -24, 0.0, -0.0, 65504, 65472, -65504, 65440, 64000, 63500]).half()
    u = torch.tensor([0.0, 0.3, 0.6, 0.999999])
    check(x.cuda(), u, t, 0, 1.0, 0.0)
    check(x.cuda(), u, t, 40, 0.9, 0.01)


def test_borders_are_exact(cuda_device):
    """Equal logits: the weights are 1, the sums whole numbers; u, top_p and top_k on the borders."""
    x = torch.full((1, 64), 3.0).half()
    for i in range(64):
        assert check(x.cuda(), f32(i / 64), 1.0, 0, 1.0, 0.0) == [i]
        assert check(x.cuda(), f32(i / 64 - 2.0 ** -24 if i else 0.0), 1.0, 0, 1.0, 0.0) == [max(0, i - 1)]
    for n in (1, 2, 31, 32, 64):
        assert check(x.cuda(), f32(1 - 2.0 ** -24), 1.0, n, 1.0, 0.0) == [n - 1]
        assert check(x.cuda(), f32(1 - 2.0 ** -24), 1.0, 0, n / 64, 0.0) == [n - 1]
        assert check(x.cuda(), f32(1 - 2.0 ** -24), 1.0, 48, n / 64, 0.0) == [math.ceil(48 * n / 64) - 1]
    assert check(x.cuda(), f32(1 - 2.0 ** -24), 1.0, 0, 1.0, 1.0) == [63]  # w == min_p is kept
    assert check(x.cuda(), f32(0.5), 1.0, 0, 1.0, 2.0) == [0]              # the first always


def test_ties_go_by_index_over_the_whole_row(cuda_device):
    """Thousands of equal logits over all CTAs of a row: every rank of the tie is found."""
    for vocab in (5000, 100000, 300000):
        x = torch.full((1, vocab), -4.0).half()
        at = torch.arange(3, vocab, 7)
        x[0, at] = 2.0
        u = torch.rand(24, generator=torch.Generator().manual_seed(vocab))
        got = nb.sample(x.expand(24, vocab).contiguous().cuda(), u.cuda(), top_k=len(at)).tolist()
        assert got == [int(at[int(math.floor(v * len(at)))]) for v in u.double().tolist()]


def test_masks(cuda_device):
    """-inf and NaN are never drawn, the lowest finite value only by its weight; +inf takes all; rows of nothing give -1."""
    g = torch.Generator().manual_seed(9)
    x = torch.randn((8, 50000), generator=g).half()
    x[0, :] = -math.inf
    x[1, :] = math.nan
    x[2, :] = -math.inf
    x[2, 49999] = -65504.0
    x[3, 1:] = -65504.0
    x[4, ::2] = math.nan
    x[4, 1::4] = -math.inf
    x[5, 777] = math.inf
    x[5, 40000] = math.inf
    x[6, :] = -65504.0
    x[7, 100:] = -math.inf
    u = torch.rand(8, generator=g)
    got = check(x.cuda(), u, 1.0, 0, 1.0, 0.0)
    assert got[0] == got[1] == -1 and got[2] == 49999 and got[3] == 0 and got[5] in (777, 40000)
    check(x.cuda(), u, 0.0, 0, 1.0, 0.0)
    check(x.cuda(), u, math.inf, 10, 0.5, 0.0)


def test_numbers_outside_the_range(cuda_device):
    x = torch.tensor([[1.0, 3.0, 2.0, 3.0]]).half().cuda()
    s = lambda u, **kw: nb.sample(x, f32(u).cuda(), **kw).item()  # noqa: E731
    assert s(1.0) == 0 and s(7.0) == 0 and s(-1.0) == 1 and s(math.nan) == 1
    assert s(1.0, top_k=2) == 3 and s(0.9, temperature=-1.0) == 1 and s(0.9, temperature=math.nan) == 1
    assert s(0.9, top_k=-3) == s(0.9) and s(0.9, top_p=math.nan) == s(0.9) and s(0.9, top_p=-1.0) == 1


def test_strides_rows_and_argmax(cuda_device):
    g = torch.Generator().manual_seed(4)
    buf = torch.randn((700, 1001), generator=g).half().cuda()
    x = buf[:, 1:1000]  # odd stride, base not 16-byte aligned
    u = torch.rand(700, generator=g)
    got = nb.sample(x, u.cuda(), temperature=0.8, top_k=30, top_p=0.9, min_p=0.01)
    t, p, m = (f32(v).item() for v in (0.8, 0.9, 0.01))
    xs = x.cpu()
    assert got.tolist() == [draw(xs[r], u[r].item(), t, 30, p, m) for r in range(700)]
    ids = torch.full((702,), 9, dtype=torch.int32, device="cuda")
    assert nb.sample(x, u.cuda(), temperature=0.0, ids=ids[1:701]).data_ptr() == ids[1:].data_ptr()
    assert torch.equal(ids[1:701], nb.argmax(x)[0]) and ids[0] == 9 and ids[701] == 9
    assert nb.sample(x[:0], u[:0].cuda()).shape == (0,)


def test_shares(cuda_device):
    """Drawn shares of 20000 rows against the softmax: 5 sigma of a binomial."""
    l = torch.tensor([0.5, -1.0, 2.0, 0.0, 1.0, -3.0]).half()
    n = 20000
    u = torch.rand(n, generator=torch.Generator().manual_seed(1)).cuda()
    got = torch.bincount(nb.sample(l.expand(n, 6).contiguous().cuda(), u).long(), minlength=6).cpu().double() / n
    p = torch.softmax(l.double(), 0)
    assert ((got - p).abs() <= 5 * torch.sqrt(p * (1 - p) / n)).all()


def test_stream_and_graph(cuda_device):
    x = torch.randn(16, 128256, device="cuda").half()
    u = torch.rand(16, device="cuda")
    want = nb.sample(x, u, top_p=0.9)
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        assert torch.equal(nb.sample(x, u, top_p=0.9), want)
    st.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = nb.sample(x, u, top_p=0.9)
    u.uniform_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(held, nb.sample(x, u, top_p=0.9))


def test_refusals(cuda_device):
    x, u = torch.randn(4, 100, device="cuda").half(), torch.rand(4, device="cuda")
    for bad in (dict(logits=x.float()), dict(logits=x[0]), dict(logits=x.cpu()), dict(u=u[:3]), dict(u=u.double()), dict(u=u.cpu()),
                dict(temperature=u.double()), dict(top_k=u), dict(top_p=u[:2]), dict(min_p=u.cpu()),
                dict(ids=torch.zeros(4, dtype=torch.int64, device="cuda")), dict(logits=x[:, :0])):
        kw = dict(logits=x, u=u, **{}) | bad
        with pytest.raises(ValueError):
            nb.sample(kw.pop("logits"), kw.pop("u"), **kw)
    with pytest.raises(nb.NpubError):
        nb.sample(torch.zeros(1, 524232, device="cuda").half(), u[:1])
