"""Products in 8-bit integers on the GPU against 64-bit forms.

Bounds per element (half a step of fp16 is 2^-11 relative, 2^-25 absolute below
the normal range, half a step of fp32 2^-24 relative):
  q            exact: q = round(127 t / max|t|), halves to even, of t exact in fp32
  scale        without gamma one division of an exact value, 2^-24; with gamma
               the fp32 sum of squares (d additions of positive terms in a tree
               of at most 32 + 16 + 10 sequential steps), the root, a division,
               a product and a division: within 64 * 2^-24
  product      the integer sum is exact; its conversion, the product of the
               scales and their product, 3 * 2^-24 of |z|, the residual's
               addition 2^-24 of the result, one rounding to fp16: 2^-11 |C| +
               2^-25 + 2^-21 |z|
  SwiGLU       gate and up within 2^-21 each; silu's slope is at most 1.1, so
               the product is within 2.1 * 2^-21 |up| (|gate| + 1); the fast exp
               and divide add a few 2^-22 of the result (their argument's
               rounding in exp(-g) is |g| 2^-24 more): 2^-11 |C| + 2^-25 +
               2^-18 |up| (|gate| + 1)
"""
import pytest
import torch

import npu_comp_b200 as nb
from npu_comp_b200 import npu

pytestmark = pytest.mark.gpu


def rows64(x, gamma=None, eps=1e-5, residual=None):
    """(q, scale, h) of the definition in 64 bits."""
    h = x if residual is None else (x.float() + residual.float()).half()  # one addition in fp32 of two fp16, then fp16
    t = h.double() if gamma is None else h.double() * gamma.double()
    top = t.abs().amax(-1, keepdim=True)
    q = torch.nan_to_num(127.0 * t / top).round()
    s = top / 127.0
    if gamma is not None:
        s = s / torch.sqrt(h.double().square().mean(-1, keepdim=True) + eps)
    return q, s[:, 0], h


@pytest.mark.parametrize("rows,d", [(1, 8), (3, 16), (5, 264), (32, 4096), (2, 2056), (7, 8200), (2, 16384), (3, 40008),
                                    (300, 1024), (1, 70000)])
@pytest.mark.parametrize("norm,add", [(False, False), (True, False), (True, True), (False, True)])
def test_quantize_rows(cuda_device, rows, d, norm, add):
    g = torch.Generator(device="cuda").manual_seed(rows * 7 + d)
    x = torch.randn((rows, d + 8), generator=g, device="cuda").half()[:, :d]
    r = torch.randn((rows, d), generator=g, device="cuda").half() if add else None
    gam = (1 + 0.3 * torch.randn(d, generator=g, device="cuda")).half() if norm else None
    if rows > 2:
        x[1] = 0  # a row of zeros
        if add:
            r[1] = 0
    q, s, h = rows64(x, gam, 1e-5, r)
    out = torch.full((rows, d + 16), 5, dtype=torch.int8, device="cuda")
    got = nb.quantize_rows(x, gamma=gam, eps=1e-5, residual=r, out=out[:, :d])
    assert got[0].data_ptr() == out.data_ptr() and (out[:, d:] == 5).all()
    assert torch.equal(got[0].double(), q)
    assert ((got[1].double() - s).abs() <= 2.0 ** -24 * s * (64 if norm else 1)).all()
    if add:
        assert torch.equal(got[2], h)


def test_quantize_rows_halves_extremes_and_values_that_are_not_finite(cuda_device):
    """Every fp16 value beside every one of some row maxima: exact, halves to
    even; rows with an infinity or NaN have scale NaN and q 0."""
    v = torch.arange(0, 0x7c00, dtype=torch.int32).to(torch.int16).view(torch.float16).cuda()
    v = torch.cat([v, -v])
    for top in (65504.0, 1.0, 127.0, 254.0, 0.1, 2.0 ** -14, 2.0 ** -24, 3 * 2.0 ** -24, 33.0):
        x = v[v.abs() <= top]
        n = (x.numel() + 1 + 7) // 8 * 8
        row = torch.zeros(1, n, dtype=torch.float16, device="cuda")
        row[0, :x.numel()] = x
        row[0, -1] = top
        q, s = nb.quantize_rows(row)
        assert torch.equal(q.double(), rows64(row)[0]), top
    x = torch.randn(4, 64, device="cuda").half()
    x[0, 5], x[1, 63], x[2, 0] = float("inf"), float("nan"), float("-inf")
    q, s = nb.quantize_rows(x)
    assert torch.isnan(s[:3]).all() and torch.isfinite(s[3]) and not q[:3].any()
    z = nb.matmul_w8a8(q, s, torch.ones(3, 64, dtype=torch.int8, device="cuda"), torch.ones(3, device="cuda").half())
    assert torch.isnan(z[:3]).all() and torch.isfinite(z[3]).all()


def test_quantize_rows_of_zeros(cuda_device):
    x = torch.zeros((3, 64), device="cuda", dtype=torch.float16)
    x[1, 7] = 2.0
    for gamma in (None, torch.ones(64, device="cuda").half()):
        for eps in (1e-5, 0.0):
            q, s = nb.quantize_rows(x, gamma=gamma, eps=eps)
            assert s[0] == 0 and s[2] == 0 and not q[0].any() and not q[2].any()
            assert q[1, 7] == 127 and q[1].count_nonzero() == 1


def product64(q, s, w, ws, res=None, swiglu=False):
    z = (q.double() @ w.double().T) * s.double()[:, None] * ws.double()
    if swiglu:
        gate, up = z[:, 0::2], z[:, 1::2]
        c = gate * torch.sigmoid(gate) * up
        return c, 2.0 ** -11 * c.abs() + 2.0 ** -25 + 2.0 ** -18 * up.abs() * (gate.abs() + 1)
    c = z if res is None else z + res.double()
    return c, 2.0 ** -11 * c.abs() + 2.0 ** -25 + 2.0 ** -21 * z.abs()


def check(M, N, K, *, res=False, swiglu=False, lda=0, ldc=0, odd=0, extremes=False):
    g = torch.Generator(device="cuda").manual_seed(M * 31 + N * 7 + K)
    i8 = lambda *s: torch.randint(-127, 128, s, generator=g, device="cuda", dtype=torch.int8)  # noqa: E731
    a, w = i8(M, K + lda)[:, :K], i8(N, K + lda)[:, :K]
    if extremes:
        a[0], w[0] = -128, -128
        a[-1], w[-1] = 127, -128
    s = torch.rand(M, generator=g, device="cuda") * 1e-2
    ws = (torch.rand(N + odd, generator=g, device="cuda") * 1e-2).half()[odd:]
    r = torch.randn((M, N + ldc), generator=g, device="cuda").half()[:, :N] if res else None
    cols = N // 2 if swiglu else N
    buf = torch.full((M + 1, cols + ldc + odd), 3.0, device="cuda", dtype=torch.float16)
    out = buf[:M, odd:odd + cols]
    c = nb.matmul_w8a8(a, s, w, ws, residual=r, swiglu=swiglu, out=out)
    assert npu.device_error() == 0
    want, bound = product64(a, s, w, ws, r, swiglu)
    err = (c.double() - want).abs()
    assert torch.isfinite(c).all() and (err <= bound).all(), f"worst excess {(err - bound).max().item():.3g}"
    buf[:M, odd:odd + cols] = 3.0
    assert (buf == 3.0).all()  # nothing else was written


@pytest.mark.parametrize("M,N,K", [
    (1, 1, 16), (1, 128, 128), (2, 7, 16), (16, 256, 4096), (17, 130, 144), (32, 12288, 4096), (33, 1000, 2064),
    (64, 4096, 11008), (65, 512, 512), (100, 22016, 4096), (128, 128, 131056), (129, 640, 1024), (255, 257, 272),
    (300, 3, 64), (777, 1003, 2064), (2048, 4096, 1024), (1024, 12288, 4096), (5000, 130, 128), (1, 32000, 4096),
    (3, 5, 131056),
])
def test_matmul_sizes(cuda_device, M, N, K):
    check(M, N, K)


@pytest.mark.parametrize("M", [1, 24, 64, 100, 200, 600, 1500])
@pytest.mark.parametrize("kw", [dict(res=True), dict(swiglu=True), dict(res=True, ldc=8), dict(ldc=8, lda=16),
                                dict(ldc=5, res=True), dict(odd=1), dict(odd=1, swiglu=True), dict(swiglu=True, ldc=3)])
def test_matmul_forms(cuda_device, M, kw):
    for N in (1024, 2050, 70, 2):
        check(M, N, 528, **kw)


@pytest.mark.parametrize("M,N,K", [(1200, 11200, 64), (1024, 18688, 4096), (2100, 9000, 2304), (4000, 2500, 4096)])
@pytest.mark.parametrize("kw", [{}, dict(res=True), dict(swiglu=True), dict(res=True, ldc=3)])
def test_matmul_several_tiles_of_a_cta(cuda_device, M, N, K, kw):
    check(M, N, K, **kw)


def test_many_calls_in_flight(cuda_device):
    """Rows quantised and multiplied again and again: every call ends, with the same bits."""
    g = torch.Generator(device="cuda").manual_seed(5)
    for M, N, K in ((4096, 11008, 2048), (2048, 18688, 4096), (64, 4096, 4096)):
        x = torch.randn((M, K), generator=g, device="cuda").half()
        gamma = torch.ones(K, device="cuda", dtype=torch.float16)
        w = torch.randint(-127, 128, (N, K), generator=g, device="cuda", dtype=torch.int8)
        ws = torch.full((N,), 1e-3, device="cuda", dtype=torch.float16)
        first = None
        for i in range(400):
            q, s = nb.quantize_rows(x, gamma=gamma)
            c = nb.matmul_w8a8(q, s, w, ws, swiglu=True)
            if i % 100 == 0:
                first = c if first is None else first
                assert torch.equal(c, first)
        assert torch.equal(c, first) and npu.device_error() == 0


def test_matmul_largest_sums(cuda_device):
    """-128 * -128 over the longest K: 2^31 - 2^18 exactly, and its negative side."""
    for M in (2, 300):
        check(M, 300, 131056, extremes=True)


def test_matmul_residual_in_place_and_empty(cuda_device):
    q, s = nb.quantize_rows(torch.randn(5, 64, device="cuda").half())
    w, ws = nb.quantize_w8(torch.randn(64, 48, device="cuda"))
    r = torch.randn(5, 48, device="cuda").half()
    want = nb.matmul_w8a8(q, s, w, ws, residual=r)
    assert nb.matmul_w8a8(q, s, w, ws, residual=r, out=r) is r and torch.equal(r, want)
    e = torch.zeros(0, 64, device="cuda").half()
    qe, se = nb.quantize_rows(e)
    assert nb.matmul_w8a8(qe, se, w, ws).shape == (0, 48)
    assert nb.matmul_w8a8(q, s, w[:0], ws[:0]).shape == (5, 0)


def test_against_matmul(cuda_device):
    """A projection of the W8A16 path and its 8-bit form on the same weights:
    the difference is the activations' rounding, at most half a step each,
    scale / 2 * sum |w| per element."""
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn((40, 512), generator=g, device="cuda").half()
    w, ws = nb.quantize_w8(torch.randn((512, 256), generator=g, device="cuda") * 0.05)
    q, s = nb.quantize_rows(x)
    a, b = nb.matmul(x, w, ws).double(), nb.matmul_w8a8(q, s, w, ws).double()
    bound = 0.5 * s.double()[:, None] * (w.double().abs().sum(1) * ws.double()) + 2.0 ** -10 * b.abs() + 2.0 ** -20
    assert ((a - b).abs() <= bound).all()


def test_streams_and_graph(cuda_device):
    """The same call on another stream and replayed from a graph gives the same bits."""
    x = torch.randn(48, 1024, device="cuda").half()
    gam = torch.randn(1024, device="cuda").half()
    w, ws = nb.quantize_w8(torch.randn(1024, 640, device="cuda"))

    def step():
        q, s = nb.quantize_rows(x, gamma=gam)
        return nb.matmul_w8a8(q, s, w, ws)
    want = step()
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        other = step()
    st.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    x.mul_(2.0)
    want2 = step()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(want, other) and torch.equal(held, want2)
