"""Decoder steps with everything in 8 bits, as a server would run them: row
quantisation behind the residual add and norm, products in 8-bit integers, the
8-bit paged cache and its attention, and sampling, against a plain model on the
values that the quantised tensors stand for.

The plain model quantises rows at the same places and keeps K and V unquantised.
What is left on a step's way to the logits are two dozen roundings to fp16
(2^-11 each), and the cache's: half a step is 1 / 254 of a page's largest value
(about 3 sigma of its elements), so a key's score is off by some 0.7 percent of
|q| |k| / sqrt(head_dim) and the values likewise, averaged over the keys: within
2 percent of an attention output, of which two layers add to the stream.  The
tolerance, 5 percent of the largest logit, is that with a factor of two."""
import math

import pytest
import torch

import npu_comp_b200 as nb
from npu_comp_b200 import npu

pytestmark = pytest.mark.gpu

D, H, KV, HD, F, VOCAB, PS, LAYERS, EPS = 256, 8, 2, 64, 384, 1000, 16, 2, 1e-5


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


class Model:
    def __init__(self, seed, seqs, pages):
        g = torch.Generator(device="cuda").manual_seed(seed)
        rnd = lambda *s, std=0.05: torch.randn(s, generator=g, device="cuda") * std  # noqa: E731
        self.embed = rnd(VOCAB, D, std=0.5).half()
        self.layers = []
        for _ in range(LAYERS):
            gate, up = nb.quantize_w8(rnd(D, F)), nb.quantize_w8(rnd(D, F))
            gu = npu.interleave_gate_up(torch.cat([gate[0], up[0]]), torch.cat([gate[1], up[1]]))
            self.layers.append(dict(
                qkv=nb.quantize_w8(rnd(D, (H + 2 * KV) * HD)), o=nb.quantize_w8(rnd(H * HD, D)), gu=gu, down=nb.quantize_w8(rnd(F, D)),
                g1=(1 + rnd(D, std=0.1)).half(), g2=(1 + rnd(D, std=0.1)).half(),
                kp=torch.zeros(pages, KV, PS, HD, dtype=torch.int8, device="cuda"),
                vp=torch.zeros(pages, KV, PS, HD, dtype=torch.int8, device="cuda"),
                ks=torch.zeros(pages, KV, device="cuda"), vs=torch.zeros(pages, KV, device="cuda"),
                held=[[] for _ in range(seqs)]))
        self.gf = (1 + rnd(D, std=0.1)).half()
        self.head = nb.quantize_w8(rnd(D, VOCAB))
        self.freqs = nb.rope_freqs(HD, 10000.0, device="cuda")


def step(m, ids, positions, table, lens, cu, new, u):
    """(logits of the last rows, tokens)"""
    x, h = nb.embed(ids, m.embed), None
    for w in m.layers:
        if h is None:
            h = x
            q, s = nb.quantize_rows(x, gamma=w["g1"], eps=EPS)
        else:
            q, s, h = nb.quantize_rows(x, gamma=w["g1"], eps=EPS, residual=h)
        qkv = nb.matmul_w8a8(q, s, *w["qkv"])
        cache = (w["kp"], w["vp"], w["ks"], w["vs"], table)
        a = nb.rope_paged_append_q8(qkv, H, KV, HD, positions, m.freqs, *cache, cu_seqlens=cu)
        if cu is None:
            a = nb.attention_paged_decode_q8(a, *cache, lens, heads=H)
        else:
            a = nb.attention_paged_q8(a, *cache, lens, cu, heads=H, max_new=new, ctx_len=table.shape[1] * PS)
        x = nb.matmul_w8a8(*nb.quantize_rows(a), *w["o"])
        q, s, h = nb.quantize_rows(x, gamma=w["g2"], eps=EPS, residual=h)
        x = nb.matmul_w8a8(*nb.quantize_rows(nb.matmul_w8a8(q, s, *w["gu"], swiglu=True)), *w["down"])
    if cu is not None:
        last = (cu[1:] - 1).long()
        x, h = x[last].contiguous(), h[last].contiguous()
    q, s, _ = nb.quantize_rows(x, gamma=m.gf, eps=EPS, residual=h)
    logits = nb.matmul_w8a8(q, s, *m.head)
    return logits, nb.sample(logits, u, temperature=0.8, top_k=50, top_p=0.95, min_p=0.01)


def rows8(x):
    top = x.abs().amax(-1, keepdim=True)
    return torch.nan_to_num(127 * x / top).round() * top / 127


def norm(x, g):
    return x / torch.sqrt(x.square().mean(-1, keepdim=True) + EPS) * g.double()


def plain_step(m, ids, positions, seq):
    """The same in 64 bits, K and V unquantised (held as rows): logits of each sequence's last row."""
    x = m.embed[ids.long()].double()
    T = x.shape[0]
    val = lambda w: w[0].double() * w[1].double()[:, None]  # noqa: E731
    turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), positions.double()[:, None] * m.freqs.double())
    rot = lambda y: torch.view_as_real(torch.complex(y[..., :HD // 2], y[..., HD // 2:]) * turn[:, None])  # noqa: E731
    for w in m.layers:
        y = (rows8(norm(x, w["g1"])) @ val(w["qkv"]).T).view(T, H + 2 * KV, HD)
        qk = rot(y[:, :H + KV])
        qk = torch.cat([qk[..., 0], qk[..., 1]], -1)
        a = torch.empty(T, H * HD, dtype=torch.float64, device="cuda")
        for t in range(T):
            b = seq[t]
            w["held"][b].append((qk[t, H:], y[t, H + KV:]))
            k, v = (torch.stack([r[i] for r in w["held"][b]]).repeat_interleave(H // KV, 1) for i in (0, 1))
            p = torch.softmax(torch.einsum("hd,mhd->hm", qk[t, :H], k) / math.sqrt(HD), -1)
            a[t] = torch.einsum("hm,mhd->hd", p, v).reshape(-1)
        x = x + rows8(a) @ val(w["o"]).T
        z = rows8(norm(x, w["g2"])) @ val(w["gu"]).T
        x = x + rows8(torch.nn.functional.silu(z[:, 0::2]) * z[:, 1::2]) @ val(w["down"]).T
    last = [max(t for t in range(T) if seq[t] == b) for b in sorted(set(seq))]
    return rows8(norm(x[last], m.gf)) @ val(m.head).T


def test_prompts_then_decode(cuda_device):
    seqs, width = 3, 6
    m = Model(5, seqs, seqs * width + 1)
    g = torch.Generator().manual_seed(1)
    table = (torch.randperm(seqs * width, generator=g) + 1).int().view(seqs, width).cuda()
    lens = [0] * seqs
    new = [37, 5, 20]
    ids = torch.randint(0, VOCAB, (sum(new),), generator=g).int().cuda()
    for turn in range(5):
        T = sum(new)
        pos = i32([l + i for l, n in zip(lens, new) for i in range(n)])
        seq = [b for b, n in enumerate(new) for _ in range(n)]
        lens = [l + n for l, n in zip(lens, new)]
        cu = i32([sum(new[:b]) for b in range(seqs + 1)]) if turn == 0 else None
        u = torch.rand(seqs, generator=g).cuda()
        logits, tokens = step(m, ids, pos, table, i32(lens), cu, max(new), u)
        assert npu.device_error() == 0 and logits.shape == (seqs, VOCAB)
        want = plain_step(m, ids, pos, seq)
        err = (logits.double() - want).abs().max() / want.abs().max()
        assert err < 0.05, float(err)
        # the tokens are the definition's on the logits
        order = torch.sort(logits.double(), dim=-1, descending=True, stable=True)
        p, mp = (torch.tensor(v, dtype=torch.float32).item() for v in (0.95, 0.01))
        t32 = torch.tensor(0.8, dtype=torch.float32).item()
        w = torch.exp((order.values - order.values[:, :1]) / t32)[:, :50]
        cum = torch.cumsum(w, -1)
        n = ((cum - w < p * cum[:, -1:]) & (w >= mp)).sum(-1, keepdim=True).clamp(min=1)
        at = torch.minimum((cum <= u.double()[:, None] * cum.gather(-1, n - 1)).sum(-1, keepdim=True), n - 1)
        assert torch.equal(tokens, order.indices.gather(-1, at)[:, 0].int())
        ids, new = tokens, [1] * seqs
    assert T == seqs


def test_captured_decode_step(cuda_device):
    """A decode step as a CUDA graph, replayed beside another graph that holds workspaces of its own, gives the bits of the
    calls; both caches advance as they do by calls."""
    seqs, width = 4, 3
    ms = [Model(7, seqs, seqs * width) for _ in range(3)]
    table = torch.arange(seqs * width, dtype=torch.int32, device="cuda").view(seqs, width)
    ids, pos, lens = i32([1, 2, 3, 4]), i32([0, 0, 0, 0]), i32([1, 1, 1, 1])
    u = torch.rand(seqs, generator=torch.Generator().manual_seed(3)).cuda()
    state = [[t.clone() for t in (ids, pos, lens)] for _ in ms]

    def run(i):
        a = state[i]
        return step(ms[i], a[0], a[1], table, a[2], None, 1, u)
    run(0)
    for w in ms[0].layers:
        for t in ("kp", "vp", "ks", "vs"):
            w[t].zero_()
    torch.cuda.synchronize()
    graphs = []
    for i in (1, 2):
        st = torch.cuda.Stream()
        st.wait_stream(torch.cuda.current_stream())
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=st):
            out = run(i)
        graphs.append((gr, out, torch.cuda.Stream()))
    for i in (1, 2):
        for w in ms[i].layers:
            for t in ("kp", "vp", "ks", "vs"):
                w[t].zero_()
    torch.cuda.synchronize()
    for n in range(20):
        logits, tokens = run(0)
        for gr, _, st in graphs:  # at once, on streams of their own
            with torch.cuda.stream(st):
                gr.replay()
        torch.cuda.synchronize()
        for _, (l, t), _ in graphs:
            assert torch.equal(l, logits) and torch.equal(t, tokens), n
        for a in state:
            a[0].copy_(tokens)
            a[1].add_(1)
            a[2].add_(1)
    for i in (1, 2):
        for w, v in zip(ms[0].layers, ms[i].layers):
            assert all(torch.equal(w[t], v[t]) for t in ("kp", "vp", "ks", "vs"))
