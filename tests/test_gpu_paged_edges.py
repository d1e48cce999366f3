"""The paged-cache operators on the GPU where calls go wrong most easily
(paged_exact.py derives the bounds)."""
import math

import pytest
import torch

import npu_comp_b200 as nb
from npu_comp_b200 import _lib, npu
from paged_exact import attention_exact, planted, same, to_pages

pytestmark = pytest.mark.gpu


def offsets(lens, dev):
    return torch.tensor([0] + list(torch.tensor(lens).cumsum(0)), dtype=torch.int32, device=dev)


# How a call reaches each kernel: new rows and keys per sequence, heads, the keys that take turns in the test.
#   packed / tiles: tile kernel, keys whole; ranges: the tile kernel's partials; few: up to 16 rows per kv head, keys
#   whole, in a cluster, or as partials; decode, prefix, prefix_phase: one row, without a shared prefix, with one that
#   every sequence reads, and with one that has a phase of its own
PATHS = {
    "packed": ([200, 70, 1], [200, 70, 1], 4, 2),
    "tiles": ([150, 3, 9], [300, 77, 4], 4, 2),
    "ranges": ([40, 2], [9000, 300], 8, 2),
    "few": ([3, 1, 4], [100, 70, 2], 4, 2),
    "few_long": ([3, 1, 4], [6000, 70, 700], 4, 2),
    "decode": ([1] * 4, [300, 0, 65, 2000], 8, 2),
    "prefix": ([1] * 4, [700, 520, 600, 513], 8, 2),
    "prefix_phase": ([1] * 20, [2500, 2049, 2048] + [2100 + 7 * i for i in range(17)], 32, 8),
}


class Call:
    """One call of PATHS with random inputs; x.run() compares every row with the 64-bit form."""

    def __init__(self, dev, path, hd, causal=True, ps=16):
        self.path, self.hd, self.causal, self.ps, self.dev = path, hd, causal, ps, dev
        self.new, self.keys, self.H, self.KV = PATHS[path]
        self.decode = path in ("decode", "prefix", "prefix_phase")
        g = torch.Generator(device=dev).manual_seed(hd + sum(self.keys))
        rnd = lambda *s: torch.randn(s, generator=g, device=dev).half()  # noqa: E731
        self.q = [rnd(n, self.H, hd) for n in self.new]
        self.k = [rnd(n, self.KV, hd) for n in self.keys]
        self.v = [rnd(n, self.KV, hd) for n in self.keys]
        self.shared = {"prefix": 512, "prefix_phase": 2048}.get(path, 0)
        for x in (self.k, self.v):
            for y in x[1:]:
                y[:self.shared] = x[0][:self.shared]

    def run(self, scale=None):
        dev, H, KV, hd = self.dev, self.H, self.KV, self.hd
        q, cu = torch.cat(self.q).reshape(-1, H * hd), offsets(self.new, dev)
        if self.path == "packed":
            o = nb.attention_packed(q, torch.cat(self.k).reshape(-1, KV * hd), torch.cat(self.v).reshape(-1, KV * hd),
                                    cu, H, KV, head_dim=hd, causal=self.causal, scale=scale)
        else:
            kp, vp, table, lens = to_pages(self.k, self.v, self.ps, shared=self.shared)
            if self.decode:
                o = nb.attention_paged_decode(q, kp, vp, table, lens, heads=H, shared_len=self.shared, scale=scale)
            else:
                o = nb.attention_paged(q, kp, vp, table, lens, cu, heads=H, causal=self.causal, scale=scale,
                                       max_new=max(self.new) if "few" in self.path else 0)
        assert npu.device_error() == 0
        scale = scale or 1 / math.sqrt(hd)
        want = [attention_exact(a, b, c, scale, self.causal) for a, b, c in zip(self.q, self.k, self.v)]
        same(o, torch.cat([w[0] for w in want]), torch.cat([w[1] for w in want]))
        return o


@pytest.mark.parametrize("hd", [16, 64, 96, 128])
@pytest.mark.parametrize("path", PATHS)
def test_infinite_and_nan_scores(cuda_device, path, hd):
    """A key whose score is +inf or NaN makes the rows that see it NaN, and no
    other row: at every place of a group of eight keys, in the first, a middle
    and the last block of a row's keys."""
    for causal in (True, False):
        c = Call(cuda_device, path, hd, causal)
        if c.decode and not causal:
            continue
        m = c.keys[0]
        for j in sorted({*range(8), 64, 65, min(129, m - 1), m // 2, *range(m - 9, m)}):
            for value in (math.inf, math.nan):
                if value != value and j % 8 != 1:
                    continue
                k = c.k[0].clone()
                c.q[0][..., 3] = c.q[0][..., 3].abs() + 0.125
                c.k[0][j, 0, 3] = value
                if c.shared:
                    held = [y[:c.shared].clone() for y in c.k]
                    for y in c.k[1:]:
                        y[:c.shared] = c.k[0][:c.shared]
                    if j < c.shared:  # all of them see it
                        for y in c.q[1:]:
                            y[..., 3] = y[..., 3].abs() + 0.125
                o = c.run()
                assert torch.isnan(o).any()
                c.k[0] = k
                if c.shared:
                    for y, h in zip(c.k[1:], held[1:]):
                        y[:c.shared] = h

@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("path", PATHS)
def test_scores_of_minus_infinity(cuda_device, path, hd):
    """Scores of -inf weigh nothing beside finite ones, in whole blocks and key
    ranges too; a row all of whose scores are -inf is NaN (0 / 0), unlike a row
    that sees no key, which is zero."""
    c = Call(cuda_device, path, hd)
    m = c.keys[0]
    for n in sorted({1, 2, 64, 130, m // 2, m - 1, m}):  # the first n keys
        k = c.k[0].clone()
        c.q[0][..., 3] = c.q[0][..., 3].abs() + 0.125
        c.k[0][:n, 0, 3] = -math.inf
        if c.shared:
            for y, x in zip(c.k[1:], c.q[1:]):
                y[:c.shared] = c.k[0][:c.shared]
                x[..., 3] = x[..., 3].abs() + 0.125
        o = c.run()
        # the first sequence's first row sees nothing else, or another sequence whose keys end with the prefix
        assert torch.isnan(o).any() == (n > m - c.new[0] or 0 < min(c.keys) <= min(n, c.shared))
        c.k[0] = k

@pytest.mark.parametrize("keys", [[40, 9, 30, 7], [900, 9, 30, 1200], [30000, 9, 30, 20000]])  # whole, cluster, partials
@pytest.mark.parametrize("H,KV", [(8, 2), (16, 1), (3, 3)])
@pytest.mark.parametrize("causal", [True, False])
def test_more_rows_than_max_new(cuda_device, keys, H, KV, causal):
    """max_new below a sequence's rows: the rows up to 16 * kv_heads / heads see
    the keys they should, the others are zero; where max_new takes the call to
    the tile kernel, all rows are computed."""
    dev, hd, ps, new = cuda_device, 128, 16, [7, 1, 23, 7]
    g = torch.Generator(device=dev).manual_seed(sum(keys) + H)
    q = [torch.randn((n, H, hd), generator=g, device=dev).half() for n in new]
    k, v = ([torch.randn((n, KV, hd), generator=g, device=dev).half() for n in keys] for _ in range(2))
    kp, vp, table, lens = to_pages(k, v, ps)
    cu, T = offsets(new, dev) + 2, sum(new)
    x = torch.cat([torch.zeros_like(q[0][:2]), *q, torch.zeros_like(q[0][:2])]).reshape(T + 4, H * hd)
    want = [attention_exact(a, b, c, 1 / math.sqrt(hd), causal) for a, b, c in zip(q, k, v)]
    for max_new in (1, 4, 17):
        few = max_new * (H // KV) <= 16
        kept = [min(n, 16 // (H // KV)) if few else n for n in new]
        o, b = ([w[i].clone() for w in want] for i in (0, 1))
        for i, n in enumerate(kept):
            o[i][n:], b[i][n:] = 0.0, 0.0
        out = torch.full_like(x, 3.0)
        npu._paged_query.cache_clear()
        held = torch.full((64 << 20,), float("nan"), device=dev)  # scratch that is used unwritten shows as NaN
        del held
        nb.attention_paged(x, kp, vp, table, lens, cu, heads=H, max_new=max_new, causal=causal, out=out)
        assert npu.device_error() == 0
        same(out[2:T + 2], torch.cat(o), torch.cat(b))
        assert (out[:2] == 3.0).all() and (out[T + 2:] == 3.0).all()

@pytest.mark.parametrize("pages", [2 ** 23, 2 ** 23 + 1, 2 ** 24 + 4])
def test_tables_past_32_bits_of_keys(cuda_device, pages):
    """A table wider than 2^31 keys (pages * 256) is no reason to refuse a call,
    nor to plan it for another number of keys than its workspace."""
    dev, H, KV, hd, ps = cuda_device, 4, 2, 64, 256
    g = torch.Generator(device=dev).manual_seed(3)
    k, v = ([torch.randn((900, KV, hd), generator=g, device=dev).half()] for _ in range(2))
    q = torch.randn((1, H, hd), generator=g, device=dev).half()
    kp, vp, narrow, lens = to_pages(k, v, ps)
    table = torch.zeros((1, pages), dtype=torch.int32, device=dev)
    table[:, :narrow.shape[1]] = narrow
    o, b = attention_exact(q, k[0], v[0], 1 / math.sqrt(hd))
    x = q.reshape(1, H * hd)
    for ctx in (0, 900, 2 ** 31, 2 ** 33):
        same(nb.attention_paged_decode(x, kp, vp, table, lens, heads=H, ctx_len=ctx), o, b)
        for max_new in (0, 1):
            same(nb.attention_paged(x, kp, vp, table, lens, offsets([1], dev), heads=H, ctx_len=ctx, max_new=max_new),
                 o, b)
    assert npu.device_error() == 0


def test_hints_past_32_bits(cuda_device):
    """A max_new or shared_len past an int is not taken for its low 32 bits."""
    dev, H, KV, hd, ps, new = cuda_device, 4, 2, 64, 16, [20, 3]
    g = torch.Generator(device=dev).manual_seed(5)
    k, v = ([torch.randn((n, KV, hd), generator=g, device=dev).half() for n in (90, 40)] for _ in range(2))
    q = [torch.randn((n, H, hd), generator=g, device=dev).half() for n in new]
    kp, vp, table, lens = to_pages(k, v, ps)
    want = [attention_exact(a, b, c, 1 / math.sqrt(hd)) for a, b, c in zip(q, k, v)]
    x = torch.cat(q).reshape(-1, H * hd)
    o = nb.attention_paged(x, kp, vp, table, lens, offsets(new, dev), heads=H, max_new=2 ** 32 + 1)
    same(o, torch.cat([w[0] for w in want]), torch.cat([w[1] for w in want]))
    for n in (2 ** 32, 2 ** 32 + 16, -2 ** 32):
        with pytest.raises(ValueError):
            nb.attention_paged_decode(x[:2], kp, vp, table, lens, heads=H, shared_len=n)

def test_rows_of_one_slot(cuda_device):
    """Rows at the same position of the same pages: every run of eight columns of
    the slot comes from one of them, and no other slot changes."""
    dev, H, KV, hd, ps, n = cuda_device, 4, 2, 128, 16, 6
    g = torch.Generator(device=dev).manual_seed(1)
    x = torch.randn((n, (H + 2 * KV) * hd), generator=g, device=dev).half()
    f, table = nb.rope_freqs(hd, device=dev), torch.tensor([[1, 0, 2]] * n, dtype=torch.int32, device=dev)
    pos = torch.full((n,), 19, dtype=torch.int32, device=dev)
    kp = torch.full((3, KV, ps, hd), 3.0, dtype=torch.float16, device=dev)
    vp = kp.clone()
    q = nb.rope_paged_append(x, H, KV, hd, pos, f, kp, vp, table)
    one = [torch.full((n + 2, KV, ps, hd), 3.0, dtype=torch.float16, device=dev) for _ in range(2)]
    own = torch.arange(n, device=dev)[:, None] + torch.tensor([2, 0, 2], device=dev)  # the rows in pages of their own
    assert torch.equal(q, nb.rope_paged_append(x, H, KV, hd, pos, f, *one, own.int()))
    for got, rows in zip((kp, vp), one):
        cand = rows[:n, :, 3].reshape(n, KV, hd // 8, 8)
        slot = got[0, :, 3].reshape(1, KV, hd // 8, 8)
        assert (cand == slot).all(-1).any(0).all()
        got[0, :, 3] = 3.0
        assert (got == 3.0).all()

# ------------------------------------------------- long contexts, planted keys

@pytest.mark.parametrize("H,KV,hd", [(8, 8, 128), (16, 1, 64), (64, 1, 128)])
def test_long_planted_contexts(cuda_device, H, KV, hd):
    """Contexts of up to 70001 keys over the largest numbers of key ranges: every
    64 keys hold one that the result cannot do without (test_paged_exact.py),
    by one row, a chunk of rows, and behind a shared prefix."""
    dev, ps, keys, shared = cuda_device, 64, [70001, 300, 66000], 0
    sc = 1 / math.sqrt(hd)
    plant = [planted(m, KV, hd, every=64, gen=torch.Generator().manual_seed(m), dev=dev) for m in keys]
    q = torch.stack([u.repeat_interleave(H // KV, 0) for u, _, _ in plant])
    k, v = [p[1] for p in plant], [p[2] for p in plant]
    kp, vp, table, lens = to_pages(k, v, ps)
    want = [attention_exact(q[b:b + 1], k[b], v[b], sc) for b in range(3)]
    o, bound = torch.cat([w[0] for w in want]), torch.cat([w[1] for w in want])
    x = q.reshape(3, H * hd)
    for kw in (dict(), dict(ctx_len=70001), dict(ctx_len=500)):
        same(nb.attention_paged_decode(x, kp, vp, table, lens, heads=H, **kw), o, bound)
        same(nb.attention_paged(x, kp, vp, table, lens, offsets([1] * 3, dev), heads=H, **kw), o, bound)
    same(nb.attention_paged_decode(x[:1], kp, vp, table[:1], lens[:1], heads=H), o[:1], bound[:1])
    n = 20  # a chunk of the longest: partials of the tile kernel
    rows = q[:1].expand(n, H, hd).contiguous()
    e, b = attention_exact(rows, k[0], v[0], sc)
    y = rows.reshape(n, H * hd)
    assert _lib.query("npub_attention_paged_workspace", 1, n, 0, 70001, H, KV, hd) > 0
    same(nb.attention_paged(y, kp, vp, table[:1], lens[:1], offsets([n], dev), heads=H, ctx_len=70001), e, b)
    assert npu.device_error() == 0


@pytest.mark.parametrize("H,KV,hd,B", [(8, 2, 128, 5), (4, 4, 64, 3), (32, 1, 128, 2)])
def test_long_planted_prefix(cuda_device, H, KV, hd, B):
    """A shared prefix of 20032 keys with own keys behind it, one sequence inside
    the prefix: every 64 keys of both phases hold one that shows."""
    dev, ps, shared, sc = cuda_device, 64, 20032, 1 / math.sqrt(hd)
    gen = torch.Generator().manual_seed(B)
    u, k0, v0 = planted(shared, KV, hd, every=64, gen=gen, dev=dev)
    k, v = [], []
    for b in range(B):
        m = [4368, 700, 64, 1, 9000][b]
        _, kb, vb = planted(m, KV, hd, every=64, gen=gen, dev=dev)
        flat = (kb.abs() == 1).all(-1)  # the planted ones, against the prefix's query
        kb[flat] = u.expand_as(kb)[flat]
        k.append(torch.cat([k0, kb]))
        v.append(torch.cat([v0, vb]))
    kp, vp, table, lens = to_pages(k, v, ps, shared=shared)
    lens[-1] = 15001  # ends inside the prefix
    keys = lens.tolist()
    q = u.repeat_interleave(H // KV, 0).expand(B, H, hd).contiguous()
    want = [attention_exact(q[b:b + 1], k[b][:keys[b]], v[b][:keys[b]], sc) for b in range(B)]
    o, bound = torch.cat([w[0] for w in want]), torch.cat([w[1] for w in want])
    for kw in (dict(shared_len=shared), dict(shared_len=shared, ctx_len=max(keys)), dict()):
        same(nb.attention_paged_decode(q.reshape(B, H * hd), kp, vp, table, lens, heads=H, **kw), o, bound)
    assert npu.device_error() == 0

# ------------------------------------------------------------ calls in flight

def serving_inputs(dev, seed, B=4, H=8, KV=2, hd=128, m=6000):
    """q, its pages, and the 64-bit result of a decode batch and of chunks whose
    calls use scratch: other values for every seed."""
    g = torch.Generator(device=dev).manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=g, device=dev).half()  # noqa: E731
    keys, new = [m - 701 * b - 13 * seed for b in range(B)], [9, 2, 30, 5]
    k, v = [r(n, KV, hd) for n in keys], [r(n, KV, hd) for n in keys]
    for x in (k, v):
        for y in x[1:]:
            y[:512] = x[0][:512]
    q1, qn = r(B, H, hd), r(sum(new), H, hd)
    sc = 1 / math.sqrt(hd)
    w1 = [attention_exact(q1[b:b + 1], k[b], v[b], sc) for b in range(B)]
    wn = [attention_exact(a, k[b], v[b], sc) for b, a in enumerate(qn.split(new))]
    cat = lambda w: tuple(torch.cat([y[i] for y in w]) for i in (0, 1))  # noqa: E731
    pages = to_pages(k, v, 16, shared=512, seed=seed)
    # both calls leave partials in scratch
    W = pages[2].shape[1] * 16
    assert _lib.query("npub_attention_paged_decode_workspace", B, W, 512, H, KV, hd) > 0
    assert _lib.query("npub_attention_paged_workspace", B, sum(new), 0, W, H, KV, hd) > 0
    cu = offsets(new, dev)

    def step():
        kp, vp, table, lens = pages
        return (nb.attention_paged_decode(q1.reshape(B, -1), kp, vp, table, lens, heads=H, shared_len=512),
                nb.attention_paged(qn.reshape(-1, H * hd), kp, vp, table, lens, cu, heads=H))

    def check(outs):
        for got, (o, b) in zip(outs, (cat(w1), cat(wn))):
            same(got, o, b)

    return step, check


def captured(step):
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    return graph, outs


def test_two_graphs_in_flight(cuda_device):
    """Two captured steps of different inputs, replayed on two streams with
    nothing between them: neither writes the other's scratch or outputs."""
    calls = [serving_inputs(cuda_device, s) for s in (1, 2)]
    graphs = [captured(step) for step, _ in calls]
    streams = [torch.cuda.Stream(device=cuda_device) for _ in graphs]
    for _ in range(5):
        for _, outs in graphs:
            for o in outs:
                o.fill_(float("nan"))
        torch.cuda.synchronize()
        for _ in range(20):
            for (graph, _), st in zip(graphs, streams):
                with torch.cuda.stream(st):
                    graph.replay()
        torch.cuda.synchronize()
        for (_, outs), (_, check) in zip(graphs, calls):
            check(outs)
    assert npu.device_error() == 0
    del graph
    graphs.clear()


def test_graph_beside_eager_calls(cuda_device):
    """A captured step replayed on a stream of its own while another stream runs
    the same operators on other inputs, with no wait between the two."""
    dev = cuda_device
    (step1, check1), (step2, check2) = serving_inputs(dev, 3), serving_inputs(dev, 4)
    graph, outs = captured(step1)
    sides = [torch.cuda.Stream(device=dev) for _ in range(2)]
    for _ in range(5):
        for o in outs:
            o.fill_(float("nan"))
        torch.cuda.synchronize()
        eager = []
        for _ in range(10):
            with torch.cuda.stream(sides[0]):
                graph.replay()
            with torch.cuda.stream(sides[1]):
                eager.append(step2())
        torch.cuda.synchronize()
        check1(outs)
        for x in eager:
            check2(x)
    assert npu.device_error() == 0
    del graph


@pytest.mark.parametrize("path", PATHS)
@pytest.mark.parametrize("hd", [64, 128])
def test_same_bits_every_time(cuda_device, path, hd):
    c = Call(cuda_device, path, hd)
    first = c.run()
    for _ in range(3):
        assert torch.equal(c.run(), first)

# --------------------------------------------------------------- many prompts

@pytest.mark.parametrize("H,KV,hd", [(8, 2, 64), (4, 4, 128)])
@pytest.mark.parametrize("causal", [True, False])
def test_hundreds_of_prompts(cuda_device, H, KV, hd, causal):
    """Ragged prompts past what one step of the scheduler looks at, empty ones
    and long ones among them, packed and over pages."""
    dev = cuda_device
    new = [(i * 37) % 91 if i % 11 else 0 for i in range(1100)] + [0] * 70 + [700, 1, 2, 300]
    g = torch.Generator(device=dev).manual_seed(hd)
    x = torch.randn((sum(new), H + 2 * KV, hd), generator=g, device=dev).half()
    q, k, v = x[:, :H], x[:, H:H + KV], x[:, H + KV:]
    o = nb.attention_packed(q.reshape(-1, H * hd), k.reshape(-1, KV * hd), v.reshape(-1, KV * hd), offsets(new, dev), H,
                            KV, head_dim=hd, causal=causal)
    cut = lambda t: t.split(new)  # noqa: E731
    want = [attention_exact(a, b, c, 1 / math.sqrt(hd), causal) for a, b, c in zip(cut(q), cut(k), cut(v))]
    same(o, torch.cat([w[0] for w in want]), torch.cat([w[1] for w in want]))
    # the last rows of each, the first ones cached already
    late = [n // 2 for n in new]
    rows = torch.cat([t[n - m:] for t, n, m in zip(cut(q), new, late)]).reshape(-1, H * hd)
    kp, vp, table, lens = to_pages(cut(k), cut(v), 16)
    want = [(w[0][n - m:], w[1][n - m:]) for w, n, m in zip(want, new, late)]
    o = nb.attention_paged(rows, kp, vp, table, lens, offsets(late, dev), heads=H, causal=causal)
    same(o, torch.cat([w[0] for w in want]), torch.cat([w[1] for w in want]))
    assert npu.device_error() == 0


def test_more_sequences_than_a_grid_row(cuda_device):
    """70000 sequences, most of one row that sees its own key alone (its v)."""
    dev, H, KV, hd, B = cuda_device, 4, 2, 64, 70000
    g = torch.Generator(device=dev).manual_seed(7)
    x = torch.randn((B, (H + 2 * KV) * hd), generator=g, device=dev).half()
    q, k, v = x[:, :H * hd], x[:, H * hd:(H + KV) * hd], x[:, (H + KV) * hd:]
    cu = torch.arange(B + 1, dtype=torch.int32, device=dev)
    cu[500:900] = 500  # 400 empty ones, then one of 400 rows
    o = nb.attention_packed(q, k, v, cu, H, KV, head_dim=hd).view(B, H, hd)
    own = v.reshape(B, KV, hd).repeat_interleave(H // KV, 1)
    alone = torch.ones(B, dtype=torch.bool, device=dev)
    alone[500:900] = False
    assert torch.equal(o[alone], own[alone])
    r = slice(500, 900)
    e, b = attention_exact(q[r].reshape(-1, H, hd), k[r].reshape(-1, KV, hd), v[r].reshape(-1, KV, hd), 1 / math.sqrt(hd))
    same(o[r].reshape(400, -1), e, b)
    kp, vp = torch.zeros((B, KV, 16, hd), dtype=torch.float16, device=dev), torch.zeros((B, KV, 16, hd), dtype=torch.float16, device=dev)
    kp[:, :, 0], vp[:, :, 0] = k.reshape(B, KV, hd), v.reshape(B, KV, hd)
    table = torch.arange(B, dtype=torch.int32, device=dev)[:, None]
    ones, cu = torch.ones(B, dtype=torch.int32, device=dev), torch.arange(B + 1, dtype=torch.int32, device=dev)
    for max_new in (0, 1):
        o = nb.attention_paged(q.contiguous(), kp, vp, table, ones, cu, heads=H, max_new=max_new)
        assert torch.equal(o.view(B, H, hd), own)
    assert npu.device_error() == 0


def test_many_short_prompts_take_no_longer_than_equal_ones(cuda_device):
    """1000 prompts of 100 rows: the packed kernel, which looks up whose rows it
    takes, against attention() on the same rows, which is told (a ninth of its
    time; with a search of all sequences for every item it took three times it)."""
    dev, B, T, H, KV, hd = cuda_device, 1000, 100, 32, 8, 64
    x = torch.randn((B * T, (H + 2 * KV) * hd), generator=torch.Generator(device=dev).manual_seed(1), device=dev).half()
    q, k, v = x[:, :H * hd], x[:, H * hd:(H + KV) * hd], x[:, (H + KV) * hd:]
    cu = offsets([T] * B, dev)
    took = []
    for call in (lambda: nb.attention_packed(q, k, v, cu, H, KV, head_dim=hd),
                 lambda: nb.attention(q, k, v, H, KV, head_dim=hd, batch=B)):
        call()
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        for _ in range(5):
            call()
        b.record()
        b.synchronize()
        took.append(a.elapsed_time(b))
    assert took[0] < took[1], took


def test_append_to_many_sequences(cuda_device):
    """20000 sequences, packed, against the decode form of the same call: the same
    bits, in not much more time; then with empty sequences between them."""
    dev, B, H, KV, hd, ps = cuda_device, 20000, 32, 8, 128, 16
    g = torch.Generator(device=dev).manual_seed(2)
    x = torch.randn((B, (H + 2 * KV) * hd), generator=g, device=dev).half()
    f, table = nb.rope_freqs(hd, device=dev), torch.randperm(B, generator=g, device=dev).int()[:, None]
    pos = torch.randint(0, ps, (B,), generator=g, device=dev, dtype=torch.int32)
    cu = torch.arange(B + 1, dtype=torch.int32, device=dev)
    outs, took = [], []
    for c in (None, cu):
        kp, vp = (torch.zeros((B, KV, ps, hd), dtype=torch.float16, device=dev) for _ in range(2))
        run = lambda: nb.rope_paged_append(x, H, KV, hd, pos, f, kp, vp, table, cu_seqlens=c)  # noqa: E731
        outs.append((run(), kp, vp))
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        for _ in range(10):
            run()
        b.record()
        b.synchronize()
        took.append(a.elapsed_time(b))
    for a, b in zip(*outs):
        assert torch.equal(a, b)
    assert took[1] < 2 * took[0], took  # eight times it when every block looked through all sequences
    # sequence 3 b + 2 holds row b, rows 0 and 1 belong to none
    wide = torch.full((3 * B, 1), 1 << 30, dtype=torch.int32, device=dev)
    wide[2::3] = table
    cu3 = 2 + torch.arange(3 * B + 1, device=dev).div(3, rounding_mode="floor").int()
    q = torch.full((B + 2, H * hd), 3.0, dtype=torch.float16, device=dev)
    two = torch.zeros((2,), dtype=torch.int32, device=dev)
    kp, vp = (torch.zeros((B, KV, ps, hd), dtype=torch.float16, device=dev) for _ in range(2))
    nb.rope_paged_append(torch.cat([x[:2], x]), H, KV, hd, torch.cat([two, pos]), f, kp, vp, wide, cu_seqlens=cu3, out=q)
    assert (q[:2] == 3.0).all() and torch.equal(q[2:], outs[0][0])
    assert torch.equal(kp, outs[0][1]) and torch.equal(vp, outs[0][2])

# ------------------------------------------------------ the shared prefix's plan

def launches(call):
    n = _lib.launch_count()
    call()
    return _lib.launch_count() - n


@pytest.mark.parametrize("keys,shared,H,KV,hd,ps", [
    ([4100 + i for i in range(40)], 4096, 16, 2, 128, 16),                       # several row tiles
    ([9000, 10, 0, 8192, 8191, 8193] + [8300] * 20, 8192, 6, 2, 128, 64),         # sequences inside the prefix
    ([4096] * 33, 4096, 8, 8, 64, 256),                                          # nothing but the prefix
    ([16700, 16900] * 12, 16384, 32, 1, 128, 16),                                # groups of 32: tiles on the own keys
    ([900, 1100, 640], 640, 32, 1, 64, 16),                                      # which keep the phase in any case
    ([6200, 6512, 5000, 600], 512, 32, 1, 128, 64),
    ([4500, 4097, 4100, 5003] * 8, 4096, 40, 8, 96, 32),
    ([40000 + i for i in range(20)], 39936, 32, 8, 128, 64),                     # the prefix on most SMs
])
def test_prefix_phase(cuda_device, keys, shared, H, KV, hd, ps):
    """Batches whose prefix has a phase of its own (three launches), with other
    lengths than the plan was made for too."""
    dev, B = cuda_device, len(keys)
    g = torch.Generator(device=dev).manual_seed(B + shared)
    rnd = lambda *s: torch.randn(s, generator=g, device=dev).half()  # noqa: E731
    full = [max(n, shared) for n in keys]  # every sequence holds the prefix's pages, used or not
    k, v = ([rnd(n, KV, hd) for n in full] for _ in range(2))
    for x in (k, v):
        for y in x[1:]:
            y[:shared] = x[0][:shared]
    kp, vp, table, lens = to_pages(k, v, ps, shared=shared)
    table[1:, :shared // ps] = 1 << 30  # the prefix is looked up in row 0
    q = rnd(B, H, hd)
    for lengths in (keys, [max(0, n - 700 - 13 * b) for b, n in enumerate(keys)]):
        lens.copy_(torch.tensor(lengths))
        out = torch.empty((B, H * hd), dtype=torch.float16, device=dev)
        n = launches(lambda: nb.attention_paged_decode(q.reshape(B, -1), kp, vp, table, lens, heads=H, shared_len=shared,
                                                       ctx_len=max(keys), out=out))
        assert n == 3 and npu.device_error() == 0
        want = [attention_exact(q[b:b + 1], k[b][:m], v[b][:m], 1 / math.sqrt(hd)) for b, m in enumerate(lengths)]
        same(out, torch.cat([w[0] for w in want]), torch.cat([w[1] for w in want]))


@pytest.mark.parametrize("B,shared,own", [(2, 64, 100), (2, 512, 100), (4, 512, 100), (64, 131072, 100)])
def test_a_prefix_costs_nothing(cuda_device, B, shared, own):
    """Telling of a shared prefix takes no longer than not telling of it (short
    ones took up to 1.6 times as long, through a phase of their own)."""
    dev, H, KV, hd, ps = cuda_device, 32, 8, 128, 64
    g = torch.Generator(device=dev).manual_seed(B)
    pages = shared // ps + B * -(-own // ps)
    kp, vp = (torch.randn((pages, KV, ps, hd), generator=g, device=dev).half() for _ in range(2))
    at = shared // ps
    table = torch.arange(pages, dtype=torch.int32, device=dev)
    table = torch.cat([table[:at].expand(B, at), table[at:].view(B, -1)], 1).contiguous()
    lens = torch.full((B,), shared + own, dtype=torch.int32, device=dev)
    q = torch.randn((B, H * hd), generator=g, device=dev).half()
    took = []
    for sl in (shared, 0):
        graph = torch.cuda.CUDAGraph()
        run = lambda: nb.attention_paged_decode(q, kp, vp, table, lens, heads=H, shared_len=sl)  # noqa: E731
        run()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            for _ in range(20):
                run()
        graph.replay()
        best = math.inf
        for _ in range(5):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            graph.replay()
            b.record()
            b.synchronize()
            best = min(best, a.elapsed_time(b))
        took.append(best)
        del graph
    assert took[0] < 1.2 * took[1], took


@pytest.mark.parametrize("keys,shared,H,KV,hd,ps", [
    ([700, 300, 0, 512, 511, 513], 512, 8, 2, 128, 16),   # few rows, in a cluster or whole
    ([12000, 4200], 4096, 8, 2, 128, 64),                  # as partials
    ([9000], 8192, 4, 2, 128, 128),
])
def test_prefix_without_a_phase(cuda_device, keys, shared, H, KV, hd, ps):
    """Batches that are quicker without a phase for the prefix find it in row 0
    of the table all the same."""
    dev, B = cuda_device, len(keys)
    g = torch.Generator(device=dev).manual_seed(shared)
    rnd = lambda *s: torch.randn(s, generator=g, device=dev).half()  # noqa: E731
    k, v = ([rnd(max(n, shared), KV, hd) for n in keys] for _ in range(2))
    for x in (k, v):
        for y in x[1:]:
            y[:shared] = x[0][:shared]
    kp, vp, table, lens = to_pages(k, v, ps, shared=shared)
    lens.copy_(torch.tensor(keys))
    table[1:, :shared // ps] = 1 << 30
    q = rnd(B, H, hd)
    out = torch.empty((B, H * hd), dtype=torch.float16, device=dev)
    n = launches(lambda: nb.attention_paged_decode(q.reshape(B, -1), kp, vp, table, lens, heads=H, shared_len=shared,
                                                   ctx_len=max(keys), out=out))
    assert n < 3 and npu.device_error() == 0
    want = [attention_exact(q[b:b + 1], k[b][:m], v[b][:m], 1 / math.sqrt(hd)) for b, m in enumerate(keys)]
    same(out, torch.cat([w[0] for w in want]), torch.cat([w[1] for w in want]))

# ----------------------------------------------------------------- large scores

@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("path", PATHS)
@pytest.mark.parametrize("at", [0.0, 2.0 ** 12, 1e6, -1e6])
def test_scores_far_from_zero(cuda_device, path, hd, at):
    """Scores of `at` + u, exact in fp32 (u a multiple of 1/8, rising over the
    keys so that every block and key range has another maximum): the weights
    depend on u alone."""
    c = Call(cuda_device, path, hd)
    root = math.sqrt(abs(at))  # 0, 64 or 1000
    for b, m in enumerate(c.keys):
        u = torch.arange(m, device=cuda_device) * (30.0 / max(m, 1)) + 4 * torch.rand(m, device=cuda_device)
        if c.shared and b:
            u[:c.shared] = first[:c.shared]
        elif b == 0:
            first = u
        c.q[b].zero_()
        c.q[b][..., 0], c.q[b][..., 1] = root, 1.0
        c.k[b].zero_()
        c.k[b][..., 0], c.k[b][..., 1] = math.copysign(root, at), ((u * 8).round() / 8)[:, None]
    c.run(scale=1.0)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("path", PATHS)
def test_the_largest_finite_scores(cuda_device, path, hd):
    """q and k at +-60000 in every column: equal scores give the mean of v, and
    one key ahead of the others its v."""
    c = Call(cuda_device, path, hd)
    for sign in (1, -1):
        for b in range(len(c.keys)):
            c.q[b].fill_(60000.0)
            c.k[b].fill_(sign * 60000.0)
        c.run()
    for b, m in enumerate(c.keys):
        if m > max(1, c.shared):  # (the prefix's keys stay alike)
            c.k[b][max(m - 2, c.shared)] = 30000.0
    c.run()


# ------------------------------------------------------- lengths and padding

@pytest.mark.parametrize("H,KV,hd", [(4, 2, 128), (32, 1, 64)])
def test_lengths_outside_the_table(cuda_device, H, KV, hd):
    """lens past the table's width count as the width, negative ones as none, by
    rows, chunks and behind a prefix."""
    dev, ps, n = cuda_device, 16, 320
    g = torch.Generator(device=dev).manual_seed(H)
    rnd = lambda *s: torch.randn(s, generator=g, device=dev).half()  # noqa: E731
    lengths, new = [2 ** 31 - 1, -5, n + 1, -2 ** 31, 100], [1, 1, 3, 2, 2]
    k, v = ([rnd(n, KV, hd) for _ in lengths] for _ in range(2))
    for x in (k, v):
        for y in x[1:]:
            y[:64] = x[0][:64]
    kp, vp, table, lens = to_pages(k, v, ps, shared=64)
    table = table[:, :n // ps]
    lens.copy_(torch.tensor(lengths))
    sc, keys = 1 / math.sqrt(hd), [max(0, min(n, m)) for m in lengths]
    q = rnd(sum(new), H, hd)
    want = [attention_exact(a, k[b][:keys[b]], v[b][:keys[b]], sc) for b, a in enumerate(q.split(new))]
    for max_new in (0, 3):
        o = nb.attention_paged(q.reshape(-1, H * hd), kp, vp, table, lens, offsets(new, dev), heads=H, max_new=max_new)
        same(o, torch.cat([w[0] for w in want]), torch.cat([w[1] for w in want]))
    q = rnd(len(lengths), H, hd)
    want = [attention_exact(q[b:b + 1], k[b][:keys[b]], v[b][:keys[b]], sc) for b in range(len(lengths))]
    for shared in (0, 64):
        o = nb.attention_paged_decode(q.reshape(-1, H * hd), kp, vp, table, lens, heads=H, shared_len=shared)
        same(o, torch.cat([w[0] for w in want]), torch.cat([w[1] for w in want]))
    assert npu.device_error() == 0


def test_a_mostly_empty_batch(cuda_device):
    """A batch padded for a graph: 20000 rows of which 40 are in use, 300 sequences
    of which three hold them; then none."""
    dev, T, B, H, KV, hd, ps = cuda_device, 20000, 300, 8, 2, 128, 16
    g = torch.Generator(device=dev).manual_seed(1)
    x = torch.randn((T, (H + 2 * KV) * hd), generator=g, device=dev).half()
    x[40:] = float("nan")
    q, k, v = x[:, :H * hd], x[:, H * hd:(H + KV) * hd], x[:, (H + KV) * hd:]
    cu = torch.full((B + 1,), 40, dtype=torch.int32, device=dev)
    cu[:101], cu[101:201] = 0, 3  # sequence 100: 3 rows, 200: 37
    f, pos = nb.rope_freqs(hd, device=dev), torch.zeros(T, dtype=torch.int32, device=dev)
    pos[:40] = torch.tensor([0, 1, 2] + list(range(37)))
    kp, vp = (torch.full((8, KV, ps, hd), 3.0, dtype=torch.float16, device=dev) for _ in range(2))
    table = torch.full((B, 3), 1 << 30, dtype=torch.int32, device=dev)
    table[100, 0], table[200] = 6, torch.tensor([1, 5, 0])
    lens = torch.zeros(B, dtype=torch.int32, device=dev)
    lens[100], lens[200] = 3, 37
    parts = [slice(0, 3), slice(3, 40)]
    o = torch.full((T, H * hd), 3.0, dtype=torch.float16, device=dev)
    for _ in range(2):
        nb.attention_packed(q, k, v, cu, H, KV, head_dim=hd, out=o)
        rot = torch.full((T, H * hd), 3.0, dtype=torch.float16, device=dev)
        nb.rope_paged_append(x, H, KV, hd, pos, f, kp, vp, table, cu_seqlens=cu, out=rot)
        for r in parts:
            n = r.stop - r.start
            e, b = attention_exact(q[r].reshape(n, H, hd), k[r].reshape(n, KV, hd), v[r].reshape(n, KV, hd),
                                   1 / math.sqrt(hd))
            same(o[r], e, b)
        assert (o[40:] == 3.0).all() and (rot[40:] == 3.0).all()
        for max_new in (0, 2):  # sequences of 3 and 37 rows: max_new is not one of this batch's
            out = torch.full((T, H * hd), 3.0, dtype=torch.float16, device=dev)
            nb.attention_paged(rot, kp, vp, table, lens, cu, heads=H, max_new=max_new, out=out)
            for r, ids in zip(parts, ([6], [1, 5, 0])):
                n = r.stop - r.start
                kk, vv = (p[ids].transpose(1, 2).reshape(-1, KV, hd)[:n] for p in (kp, vp))
                m = n if max_new == 0 else min(n, 4)
                e, b = attention_exact(rot[r].reshape(n, H, hd), kk, vv, 1 / math.sqrt(hd))
                same(out[r][:m], e[:m], b[:m])
                assert not out[r][m:].any()
            assert (out[40:] == 3.0).all()
    cu.zero_()
    for run in (lambda y: nb.attention_packed(q, k, v, cu, H, KV, head_dim=hd, out=y),
                lambda y: nb.attention_paged(rot, kp, vp, table, lens, cu, heads=H, out=y),
                lambda y: nb.attention_paged(rot, kp, vp, table, lens, cu, heads=H, max_new=1, out=y),
                lambda y: nb.rope_paged_append(x, H, KV, hd, pos, f, kp, vp, table, cu_seqlens=cu, out=y)):
        y = torch.full((T, H * hd), 3.0, dtype=torch.float16, device=dev)
        run(y)
        assert (y == 3.0).all()
    assert npu.device_error() == 0
