"""The 8-bit serving operators as workloads: projections in 8-bit integers with
a scale for each token and channel, a paged KV cache in 8 bits with a scale for
each page and head (its append and its attention), and sampling from given
random numbers.

Every operator has a plain form in elementary torch operations (fp32; fp64 for
angles and for the sums that sampling compares) beside the framework's calls;
`exact` restates each definition in fp64.  What the cache holds in 8 bits is
returned as the values it stands for, in fp16."""
import math
import random

import torch

own = False

EPS = 1e-5
THETA = 500000.0


# ------------------------------------------------------------------ cases

def listed():
    return [
        # the QKV projection of a decode step of 32 sequences, behind the residual add and its RMSNorm
        dict(name="proj_decode", op="proj", rows=32, n=12288, k=4096, norm=True, add=True, swiglu=False, res=False),
        # sizes that fill no tile: a draft head on a ragged prompt
        dict(name="proj_odd", op="proj", rows=777, n=1003, k=2064, norm=False, add=False, swiglu=False, res=False),
        # the down projection of a prompt chunk, the residual stream added in its epilogue
        dict(name="proj_down", op="proj", rows=2048, n=4096, k=11008, norm=False, add=False, swiglu=False, res=True),
        # gate and up projections of eight long prompts
        dict(name="proj_gate_up", op="proj", rows=8192, n=22016, k=4096, norm=True, add=False, swiglu=True, res=False),
        # a full decode batch: one row into the last page of every sequence
        dict(name="append_batch", op="append", rows=250, seqs=250, heads=32, kv_heads=8, head_dim=128, rot=128,
             interleaved=False, norm=False, page=16, start=3000, prompt=False),
        # packed prompts of one scheduler step, some continuing a cached prefix
        dict(name="append_prompts", op="append", rows=4096, seqs=6, heads=32, kv_heads=8, head_dim=128, rot=128,
             interleaved=False, norm=True, page=64, start=700, prompt=True),
        # one user's decode step: latency
        dict(name="decode_1", op="decode", seqs=1, heads=32, kv_heads=8, head_dim=128, page=16, keys=777),
        # a decode batch with contexts of its own, ungrouped heads of the 7B layer
        dict(name="decode_ragged", op="decode", seqs=32, heads=32, kv_heads=32, head_dim=128, page=16, keys=65000),
        # a few drafted tokens per request verified against long contexts
        dict(name="chunk_drafts", op="chunk", rows=96, seqs=24, heads=32, kv_heads=8, head_dim=128, page=64,
             keys=70001),
        # prompt chunks of several requests against what their pages already hold
        dict(name="chunk_mixed", op="chunk", rows=2000, seqs=6, heads=32, kv_heads=8, head_dim=128, page=16,
             keys=36000),
        # one user's next token
        dict(name="sample_1", op="sample", rows=1, vocab=32000, spread=3.0),
        # the next tokens of a batch over a large vocabulary, every row with settings of its own
        dict(name="sample_batch", op="sample", rows=64, vocab=128256, spread=2.5),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["proj", "append", "decode", "chunk", "sample"])
    if op == "proj":
        swiglu = rng.random() < 0.3
        norm = rng.random() < 0.5
        n = _log(rng, 64, 20000)
        k = 16 * _log(rng, 8, min(700, 5700000 // n))
        return dict(op=op, rows=_log(rng, 1, 8000), n=n + n % 2 if swiglu else n, k=k, norm=norm,
                    add=norm and rng.random() < 0.5, swiglu=swiglu, res=not swiglu and rng.random() < 0.4)
    if op == "sample":
        return dict(op=op, rows=_log(rng, 1, 64), vocab=_log(rng, 300, 128256), spread=rng.choice([0.5, 2.0, 4.0]))
    kv = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 2, 4, 8])
    hd = rng.choice([64, 128, 128])
    page = rng.choice([16, 32, 64, 128])
    if op == "append":
        prompt = rng.random() < 0.5
        rows = _log(rng, 1, 6000) if prompt else _log(rng, 1, 400)
        return dict(op=op, rows=rows, seqs=rng.randint(1, min(rows, 40)) if prompt else rows, heads=kv * group,
                    kv_heads=kv, head_dim=hd, rot=rng.choice([hd, hd, hd // 2]), interleaved=rng.random() < 0.4,
                    norm=rng.random() < 0.5, page=page, start=_log(rng, 1, 100000) if rng.random() < 0.7 else 0,
                    prompt=prompt)
    if op == "chunk":
        seqs = rng.randint(1, 16)
        rows = seqs * _log(rng, 1, 400) + rng.randint(0, 3)
        return dict(op=op, rows=rows, seqs=seqs, heads=kv * group, kv_heads=kv, head_dim=hd, page=page,
                    keys=rows + _log(rng, 1, 30000))
    seqs = _log(rng, 1, 80)
    return dict(op=op, seqs=seqs, heads=kv * group, kv_heads=kv, head_dim=hd, page=page,
                keys=seqs * _log(rng, 1, 1500) + rng.randint(0, 5))


def _split(total, n, least, spread=0.7):
    """`total` in n ragged parts of at least `least`: a function of its arguments alone."""
    r = random.Random(total * 1009 + n)
    w = [r.lognormvariate(0.0, spread) for _ in range(n)]
    free = total - n * least
    parts = [least + int(free * x / sum(w)) for x in w]
    parts[r.randrange(n)] += total - sum(parts)
    return parts


def _lengths(c):
    """(new rows of each sequence, keys of each sequence)"""
    n = c["seqs"]
    if c["op"] == "append":
        rows = _split(c["rows"], n, 1) if c["prompt"] else [1] * n
        r = random.Random(c["start"] * 7 + n)
        return rows, [x + (r.randint(c["start"] // 2, c["start"]) if c["start"] else 0) for x in rows]
    if c["op"] == "chunk":
        rows = _split(c["rows"], n, 1, 0.3)
        return rows, [x + y for x, y in zip(rows, _split(c["keys"] - c["rows"], n, 0))]
    return [1] * n, _split(c["keys"], n, 1)


# ----------------------------------------------------------------- inputs

def prepare(case, seed):
    c = case
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731

    def normal(*shape, scale=1.0):
        return torch.randn(shape, generator=g, device=dev, dtype=torch.float16).mul_(scale)

    def uniform(lo, hi, *shape):
        return torch.rand(shape, generator=g, device=dev).mul_(hi - lo).add_(lo)

    s = dict(case=c)
    if c["op"] == "proj":
        M, N, K = c["rows"], c["n"], c["k"]
        # activations with a few large channels; weights as they are held: 8 bits and a scale for each channel
        s["x"] = normal(M, K) * (1.0 + 9.0 * (uniform(0.0, 1.0, K) < 0.01)).half()
        s["gamma"] = 1.0 + normal(K, scale=0.2) if c["norm"] else None
        s["stream"] = normal(M, K) if c["add"] else None
        s["w"] = torch.randint(-127, 128, (N, K), generator=g, device=dev, dtype=torch.int8)
        s["ws"] = uniform(0.5e-4, 3e-4, N).half()
        s["res"] = normal(M, N) if c["res"] else None
        return s
    if c["op"] == "sample":
        R, V = c["rows"], c["vocab"]
        s["logits"] = normal(R, V, scale=c["spread"])
        s["u"] = uniform(0.0, 1.0, R)
        pick = lambda *v: torch.tensor(v, device=dev)[torch.randint(0, len(v), (R,), generator=g, device=dev)]  # noqa: E731
        s["temperature"] = pick(0.0, 0.6, 0.8, 1.0, 1.0, 1.3).float()
        s["top_k"] = pick(0, 0, 1, 20, 50, 1000).int()
        s["top_p"] = pick(1.0, 1.0, 0.95, 0.9, 0.5).float()
        s["min_p"] = pick(0.0, 0.0, 0.02, 0.1).float()
        return s
    r = random.Random(seed)
    new, keys = _lengths(c)
    H, KV, hd, B, ps = c["heads"], c["kv_heads"], c["head_dim"], c["seqs"], c["page"]
    T = sum(new)
    cu = [0]
    for x in new:
        cu.append(cu[-1] + x)
    s.update(cu=i32(cu), heads=H, kv_heads=KV, head_dim=hd)
    width = max((x + ps - 1) // ps for x in keys)
    # the pages that this step touches: an append's last ones, all of an attention's
    first = [(y - x) // ps if c["op"] == "append" else 0 for x, y in zip(new, keys)]
    n_pages = sum((y + ps - 1) // ps - f for y, f in zip(keys, first)) + 2
    ids = list(range(n_pages))
    r.shuffle(ids)
    table = torch.randint(0, n_pages, (B, width), generator=torch.Generator().manual_seed(seed), dtype=torch.int32)
    at = 0
    for b in range(B):
        n = (keys[b] + ps - 1) // ps - first[b]
        table[b, first[b]:first[b] + n] = torch.tensor(ids[at:at + n], dtype=torch.int32)
        at += n
    s["table"] = table.to(dev)
    s["lens"] = i32(keys)
    for name in ("k", "v"):  # as appends left it: the largest of a page's values, within a few percent, at 127
        q = torch.randn((n_pages, KV, ps, hd), generator=g, device=dev).mul_(36.0).round_().clamp_(-127, 127)
        s[name + "_pages"], s[name + "_scales"] = q.to(torch.int8), uniform(0.02, 0.035, n_pages, KV)
    if c["op"] == "append":
        s["qkv"] = normal(T, (H + 2 * KV) * hd)
        s["positions"] = i32([p for x, y in zip(new, keys) for p in range(y - x, y)])
        i = torch.arange(0, c["rot"], 2, dtype=torch.float64, device=dev)
        s["inv_freq"] = (THETA ** (-i / c["rot"])).float()
        s["q_gamma"] = (1.0 + normal(hd, scale=0.2)) if c["norm"] else None
        s["k_gamma"] = (1.0 + normal(hd, scale=0.2)) if c["norm"] else None
    else:
        s["q"] = normal(T, H * hd, scale=1.2)
        s["ctx"], s["max_new"] = max(keys), max(new)  # what the scheduler of a batch knows
    return s


# ------------------------------------------------------------ plain forms

def _plain_proj(s):
    c = s["case"]
    y = s["x"].float()
    out = []
    if s["stream"] is not None:  # the residual stream goes on in fp16
        h = (y + s["stream"].float()).half()
        out.append(h)
        y = h.float()
    if s["gamma"] is not None:
        y = y / torch.sqrt(y.square().mean(-1, keepdim=True) + EPS) * s["gamma"].float()
    a = y.abs().amax(-1, keepdim=True)
    q = torch.round(torch.where(a > 0, 127.0 * y / a, 0.0))
    z = torch.matmul(q, s["w"].float().T) * (a / 127.0) * s["ws"].float()
    if c["swiglu"]:  # rows of the weight: gate 0, up 0, gate 1, ...
        gate, up = z[:, 0::2], z[:, 1::2]
        z = gate / (1.0 + torch.exp(-gate)) * up
    if s["res"] is not None:
        z = z + s["res"].float()
    return out + [z.half()]


def _seq_of_rows(cu, rows):
    return torch.searchsorted(cu, torch.arange(rows, device=cu.device, dtype=torch.int32), right=True) - 1


def _rotated(x, cos, sin, rot, interleaved):
    y = x.clone()
    if interleaved:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        y[..., 0:rot:2], y[..., 1:rot:2] = a * cos - b * sin, b * cos + a * sin
    else:
        h = rot // 2
        a, b = x[..., :h], x[..., h:rot]
        y[..., :h], y[..., h:rot] = a * cos - b * sin, b * cos + a * sin
    return y


def _values(pages, scales):
    """What 8-bit pages stand for, in fp16."""
    return torch.mul(pages, scales[:, :, None, None], out=torch.empty(pages.shape, dtype=torch.float16, device=pages.device))


def _plain_write(pages, scales, rows, page, slot):
    """rows [T, KV, hd] (fp32) into 8-bit pages; the pages' scales grow with them."""
    n, KV, ps, hd = pages.shape
    T = rows.shape[0]
    one = torch.ones((), dtype=torch.int64, device=page.device)
    first = torch.full((n,), ps, dtype=torch.int64, device=page.device).scatter_reduce(0, page, slot, "amin")
    most = torch.zeros((n, KV), device=page.device).scatter_reduce(
        0, (page[:, None] * one).expand(T, KV), rows.abs().amax(-1), "amax")
    touched = (first < ps)[:, None]
    before = torch.where((first == 0)[:, None], 0.0, scales)  # a page written from its start begins anew
    after = torch.where(touched, torch.maximum(before, most / 127.0), scales)
    grown = touched & (after > before)
    kept = torch.where(grown, before / after, 1.0)
    old = torch.arange(ps, device=page.device) < first[:, None]  # rows ahead of the new ones
    old = (old & touched)[:, None, :, None]
    pages.copy_(torch.where(old, torch.round(pages.float() * kept[:, :, None, None]), pages.float()).to(torch.int8))
    scales.copy_(after)
    at = after[page][:, :, None]
    q = torch.round(torch.where(at > 0, rows / at, 0.0)).clamp(-127, 127)
    pages[page, :, slot] = q.to(torch.int8)


def _plain_append(s):
    c, H, KV, hd = s["case"], s["heads"], s["kv_heads"], s["head_dim"]
    T = s["qkv"].shape[0]
    x = s["qkv"].view(T, H + 2 * KV, hd).float()
    q, k, v = x[:, :H], x[:, H:H + KV], x[:, H + KV:]
    if s["q_gamma"] is not None:
        q = q / torch.sqrt(q.square().mean(-1, keepdim=True) + EPS) * s["q_gamma"].float()
        k = k / torch.sqrt(k.square().mean(-1, keepdim=True) + EPS) * s["k_gamma"].float()
    angle = s["positions"].double()[:, None] * s["inv_freq"].double()
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    q = _rotated(q, cos, sin, c["rot"], c["interleaved"]).half().view(T, H * hd)
    k = _rotated(k, cos, sin, c["rot"], c["interleaved"])
    pos = s["positions"].long()
    page = s["table"][_seq_of_rows(s["cu"], T), pos // c["page"]].long()
    _plain_write(s["k_pages"], s["k_scales"], k, page, pos % c["page"])
    _plain_write(s["v_pages"], s["v_scales"], v, page, pos % c["page"])
    return q


def _plain_paged(s):
    H, KV, hd = s["heads"], s["kv_heads"], s["head_dim"]
    G = H // KV
    T, B = s["q"].shape[0], s["table"].shape[0]
    cu, lens = s["cu"].long(), s["lens"].long()
    seq = _seq_of_rows(s["cu"], T)
    at = torch.arange(T, device=seq.device) - cu[seq]  # row within its sequence
    M = s["max_new"]
    q = torch.zeros((B, M, H, hd), device=seq.device)
    q[seq, at] = s["q"].view(T, H, hd).float()
    q = q.view(B, M, KV, G, hd).permute(0, 2, 3, 1, 4).reshape(B, KV, G * M, hd)
    table = s["table"].long()
    L = table.shape[1] * s["k_pages"].shape[2]
    k = s["k_pages"][table].float() * s["k_scales"][table][..., None, None]
    k = k.permute(0, 2, 4, 1, 3).reshape(B, KV, hd, L)
    p = torch.matmul(q, k).mul_(1.0 / math.sqrt(hd))
    new = cu[1:] - cu[:-1]
    last = (lens - new)[:, None] + torch.arange(M, device=seq.device)  # the last key that a row sees
    hidden = torch.arange(L, device=seq.device) > last[:, :, None]
    p.view(B, KV, G, M, L).masked_fill_(hidden[:, None, None], -math.inf)
    p.sub_(p.amax(-1, keepdim=True)).exp_()
    v = s["v_pages"][table].float() * s["v_scales"][table][..., None, None]
    v = v.permute(0, 2, 1, 3, 4).reshape(B, KV, L, hd)
    o = torch.matmul(p, v) / p.sum(-1, keepdim=True)
    o = o.view(B, KV, G, M, hd).permute(0, 3, 1, 2, 4).reshape(B, M, H * hd)
    return o[seq, at].half()


def _plain_sample(s):
    V = s["logits"].shape[1]
    rank = torch.arange(V, device=s["u"].device)
    l, index = torch.sort(s["logits"].double(), dim=-1, descending=True, stable=True)
    t = s["temperature"].double()[:, None]
    w = torch.exp((l - l[:, :1]) / torch.where(t > 0, t, 1.0))
    k = torch.where(s["top_k"] > 0, s["top_k"], V).clamp(max=V).long()[:, None]
    k = torch.where(t > 0, k, 1)
    cum = torch.cumsum(w, -1)
    p = s["top_p"].double()[:, None]
    kept = (rank < k) & ((p >= 1.0) | (cum - w < p * cum.gather(-1, k - 1))) & (w >= s["min_p"].double()[:, None])
    n = kept.sum(-1, keepdim=True).clamp(min=1)  # a prefix; the first always
    mass = cum.gather(-1, n - 1)
    at = torch.minimum((cum <= s["u"].double()[:, None] * mass).sum(-1, keepdim=True), n - 1)
    return index.gather(-1, at)[:, 0].int()


def run(state):
    s, c = state, state["case"]
    op = c["op"]
    if not own:
        if op == "append":
            q = _plain_append(s)
        else:
            return {"proj": _plain_proj, "sample": _plain_sample}.get(op, _plain_paged)(s)
    else:
        from npu_comp_b200 import npu
        if op == "proj":
            a = npu.quantize_rows(s["x"], gamma=s["gamma"], eps=EPS, residual=s["stream"])
            z = npu.matmul_w8a8(a[0], a[1], s["w"], s["ws"], residual=s["res"], swiglu=c["swiglu"])
            return [*a[2:], z]
        if op == "sample":
            return npu.sample(s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"],
                              min_p=s["min_p"])
        H, KV, hd = s["heads"], s["kv_heads"], s["head_dim"]
        cache = (s["k_pages"], s["v_pages"], s["k_scales"], s["v_scales"], s["table"])
        if op == "chunk":
            return npu.attention_paged_q8(s["q"], *cache, s["lens"], s["cu"], heads=H, ctx_len=s["ctx"],
                                          max_new=s["max_new"])
        if op == "decode":
            return npu.attention_paged_decode_q8(s["q"], *cache, s["lens"], heads=H, ctx_len=s["ctx"])
        q = npu.rope_paged_append_q8(s["qkv"], H, KV, hd, s["positions"], s["inv_freq"], *cache,
                                     cu_seqlens=s["cu"] if c["prompt"] else None, rot_dim=c["rot"],
                                     interleaved=c["interleaved"], q_gamma=s["q_gamma"], k_gamma=s["k_gamma"], eps=EPS)
    return [q, _values(s["k_pages"], s["k_scales"]), _values(s["v_pages"], s["v_scales"]), s["k_scales"], s["v_scales"]]


# -------------------------------------------------------- work and oracle

def work(case):
    c = case
    if c["op"] == "proj":
        M, N, K = c["rows"], c["n"], c["k"]
        moved = M * K * (2 + 4 * c["add"]) + N * K + 2 * N + M * N * (1 if c["swiglu"] else 2) + 2 * M * N * c["res"]
        return {"bytes": moved + 2 * K * c["norm"], "flops": 2 * M * N * K}
    if c["op"] == "sample":
        return {"bytes": c["rows"] * (2 * c["vocab"] + 24), "flops": 0}
    new, keys = _lengths(c)
    T, H, KV, hd = sum(new), c["heads"], c["kv_heads"], c["head_dim"]
    if c["op"] == "append":
        moved = T * (H + 2 * KV) * hd * 2 + T * H * hd * 2 + T * 2 * KV * hd
        return {"bytes": moved + T * 8 + c["rot"] * 2, "flops": T * (H + KV) * (3 * c["rot"] + 4 * hd * c["norm"])}
    pairs = sum(n * (y - n) + n * (n + 1) // 2 for n, y in zip(new, keys))
    held = sum((y + c["page"] - 1) // c["page"] for y in keys)
    return {"bytes": 2 * T * H * hd * 2 + 2 * sum(keys) * KV * hd + 2 * held * KV * 4, "flops": 4 * H * hd * pairs}


def _exact_attention(q, k, v, scale):
    """q [n, H, d], k and v [m, KV, d] in fp64; the last query sees all m keys, each before it one less."""
    n, H, d = q.shape
    m, KV = k.shape[0], k.shape[1]
    out = torch.empty((n, H, d), dtype=torch.float64, device=q.device)
    j = torch.arange(m, device=q.device)
    for h in range(H):
        kh, vh = k[:, h // (H // KV)], v[:, h // (H // KV)]
        w = q[:, h].double() @ kh.T * scale
        w = w.masked_fill(j[None, :] > (m - n + torch.arange(n, device=q.device))[:, None], -math.inf)
        out[:, h] = torch.softmax(w, -1) @ vh
    return out.reshape(n, H * d)


def _exact_proj(s, c):
    x, out = s["x"].double(), []
    if s["stream"] is not None:
        out.append(x + s["stream"].double())
        x = out[0].half().double()  # the definition normalises the rounded stream
    if s["gamma"] is not None:
        x = x / x.square().mean(-1, keepdim=True).add(EPS).sqrt() * s["gamma"].double()
    top = x.abs().max(-1, keepdim=True).values
    q = torch.nan_to_num(127.0 * x / top).round()  # exact halves go to the even step
    z = torch.empty((x.shape[0], c["n"]), dtype=torch.float64, device=x.device)
    for n0 in range(0, c["n"], 4096):
        z[:, n0:n0 + 4096] = q @ s["w"][n0:n0 + 4096].double().T
    z *= top / 127.0
    z *= s["ws"].double()
    if c["swiglu"]:
        z = z[:, 0::2] * torch.sigmoid(z[:, 0::2]) * z[:, 1::2]
    if s["res"] is not None:
        z += s["res"].double()
    return out + [z]


def _exact_sample(s):
    got = []
    for r in range(s["u"].shape[0]):
        l = s["logits"][r].double().cpu()
        t, k, p, m = (s[x][r].item() for x in ("temperature", "top_k", "top_p", "min_p"))
        if t == 0:
            got.append(int((l == l.max()).nonzero()[0]))
            continue
        order = torch.argsort(l, descending=True, stable=True)  # ties by index
        order = order[:k] if k > 0 else order
        w = torch.exp((l[order] - l.max()) / t).tolist()
        goal, run_, n = p * math.fsum(w), 0.0, 0
        for x in w:
            if n and not ((p >= 1.0 or run_ < goal) and x >= m):
                break
            run_, n = run_ + x, n + 1
        goal, run_, at = s["u"][r].item() * math.fsum(w[:n]), 0.0, 0
        while at < n - 1 and run_ + w[at] <= goal:
            run_, at = run_ + w[at], at + 1
        got.append(int(order[at]))
    return torch.tensor(got, dtype=torch.int32)


def exact(case, seed):
    s = prepare(case, seed)
    c = case
    if c["op"] == "proj":
        return _exact_proj(s, c)
    if c["op"] == "sample":
        return _exact_sample(s)
    H, KV, hd, ps = s["heads"], s["kv_heads"], s["head_dim"], c["page"]
    new, keys = _lengths(c)
    if c["op"] != "append":
        out = []
        for b, q in enumerate(s["q"].view(-1, H, hd).split(new)):
            at = torch.arange(keys[b], device=q.device)
            page, slot = s["table"][b].long()[at // ps], at % ps
            k, v = (s[x + "_pages"][page, :, slot].double() * s[x + "_scales"][page].double()[..., None] for x in "kv")
            out.append(_exact_attention(q, k, v, 1.0 / math.sqrt(hd)))
        return torch.cat(out)
    # append: pairs as complex numbers, multiplied by exp(i angle)
    x = s["qkv"].view(-1, H + 2 * KV, hd).double()
    if s["q_gamma"] is not None:
        rms = x.square().mean(-1, keepdim=True).add(EPS).sqrt()
        x[:, :H] = x[:, :H] / rms[:, :H] * s["q_gamma"].double()
        x[:, H:H + KV] = x[:, H:H + KV] / rms[:, H:H + KV] * s["k_gamma"].double()
    R = c["rot"]
    turn = torch.polar(torch.ones((), dtype=torch.float64, device=x.device),
                       s["positions"].double()[:, None] * s["inv_freq"].double())[:, None]
    qk = x[:, :H + KV]
    if c["interleaved"]:
        z = torch.view_as_complex(qk[..., :R].reshape(*qk.shape[:2], R // 2, 2).contiguous()) * turn
        qk[..., :R] = torch.view_as_real(z).reshape(*qk.shape[:2], R)
    else:
        z = torch.complex(qk[..., :R // 2], qk[..., R // 2:R]) * turn
        qk[..., :R] = torch.cat([z.real, z.imag], -1)
    values, scales = [], []
    for name, rows in (("k", x[:, H:H + KV]), ("v", x[:, H + KV:])):
        q, sc = s[name + "_pages"].double(), s[name + "_scales"].double()
        t = 0
        for b in range(c["seqs"]):  # page by page of each sequence
            p = keys[b] - new[b]
            while p < keys[b]:
                n = min(ps - p % ps, keys[b] - p)
                page, at = int(s["table"][b, p // ps]), p % ps
                y = rows[t:t + n].transpose(0, 1)  # [KV, n, hd]
                was = sc[page] if at else torch.zeros_like(sc[page])
                now = torch.maximum(was, y.abs().amax((1, 2)) / 127.0)
                step = now[:, None, None]
                q[page, :, :at] = torch.where((now > was)[:, None, None], (q[page, :, :at] * was[:, None, None] / step).round(),
                                              q[page, :, :at])
                q[page, :, at:at + n] = torch.nan_to_num(y / step).round()
                sc[page] = now
                p, t = p + n, t + n
        values.append(q * sc[:, :, None, None])
        scales.append(sc)
    return [x[:, :H].reshape(-1, H * hd), *values, *scales]
