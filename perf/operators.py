"""The paged-cache serving operators as workloads: appending rotated keys to a
paged KV cache, attention over packed prompts, attention of new tokens over
the pages, and decode attention with a shared prefix.

Every operator has a plain form in elementary torch operations (fp32, angles
in fp64) beside the framework's call; `exact` restates each definition in
fp64, sequence by sequence."""
import math
import random

import torch

own = False

EPS = 1e-5
THETA = 500000.0


# ------------------------------------------------------------------ cases

def listed():
    return [
        # one user's decode step: launch latency is all there is
        dict(name="append_1", op="append", rows=1, seqs=1, heads=32, kv_heads=8, head_dim=128, rot=128,
             interleaved=False, norm=False, page=16, start=1500, prompt=False),
        # a full decode batch of a model with per-head norms, far into its contexts
        dict(name="append_batch", op="append", rows=250, seqs=250, heads=32, kv_heads=32, head_dim=128, rot=128,
             interleaved=False, norm=True, page=64, start=130000, prompt=False),
        # packed prompts of one scheduler step (8 of them), some continuing a cached prefix
        dict(name="append_prompts", op="append", rows=8192, seqs=8, heads=32, kv_heads=8, head_dim=128, rot=128,
             interleaved=False, norm=True, page=64, start=700, prompt=True),
        # interleaved pairs on half of a narrow head, odd row count
        dict(name="append_partial", op="append", rows=1001, seqs=5, heads=16, kv_heads=4, head_dim=64, rot=32,
             interleaved=True, norm=False, page=32, start=0, prompt=True),
        # three short prompts of a tensor-parallel shard: latency
        dict(name="packed_short", op="packed", rows=75, seqs=3, heads=8, kv_heads=2, head_dim=128),
        # an ordinary scheduler step: a dozen ragged prompts, 64-wide heads
        dict(name="packed_ragged", op="packed", rows=6001, seqs=12, heads=32, kv_heads=8, head_dim=64),
        # long prompts at the width of a 7B layer's grouped variant
        dict(name="packed_long", op="packed", rows=16384, seqs=4, heads=32, kv_heads=8, head_dim=128),
        # prompt chunks of several requests against what their pages already hold
        dict(name="chunk_mixed", op="chunk", rows=2000, seqs=6, heads=32, kv_heads=8, head_dim=128, page=16,
             keys=36000),
        # a few drafted tokens per request verified against long contexts
        dict(name="chunk_drafts", op="chunk", rows=96, seqs=24, heads=32, kv_heads=8, head_dim=128, page=64,
             keys=70001),
        # one user's decode step
        dict(name="decode_1", op="decode", seqs=1, heads=32, kv_heads=8, head_dim=128, page=16, shared=0, keys=777),
        # a decode batch with contexts of its own, ungrouped heads of the 7B layer
        dict(name="decode_ragged", op="decode", seqs=32, heads=32, kv_heads=32, head_dim=128, page=16, shared=0,
             keys=65000),
        # many users behind one long system prompt
        dict(name="decode_shared", op="decode", seqs=64, heads=32, kv_heads=8, head_dim=128, page=64, shared=8192,
             keys=17001),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "packed", "chunk", "decode"])
    kv = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 2, 4, 8])
    hd = rng.choice([64, 128, 128])
    page = rng.choice([16, 32, 64, 128])
    if op == "append":
        prompt = rng.random() < 0.5
        rows = _log(rng, 1, 8000) if prompt else _log(rng, 1, 500)
        return dict(op=op, rows=rows, seqs=rng.randint(1, min(rows, 40)) if prompt else rows, heads=kv * group,
                    kv_heads=kv, head_dim=hd, rot=rng.choice([hd, hd, hd // 2]), interleaved=rng.random() < 0.4,
                    norm=rng.random() < 0.5, page=page, start=_log(rng, 1, 100000) if rng.random() < 0.7 else 0,
                    prompt=prompt)
    if op == "packed":
        rows = _log(rng, 1, 9000)
        return dict(op=op, rows=rows, seqs=rng.randint(1, min(rows, 24)), heads=kv * group, kv_heads=kv, head_dim=hd)
    if op == "chunk":
        seqs = rng.randint(1, 16)
        rows = seqs * _log(rng, 1, 400) + rng.randint(0, 3)
        return dict(op=op, rows=rows, seqs=seqs, heads=kv * group, kv_heads=kv, head_dim=hd, page=page,
                    keys=rows + _log(rng, 1, 40000))
    seqs = _log(rng, 1, 80)
    return dict(op=op, seqs=seqs, heads=kv * group, kv_heads=kv, head_dim=hd, page=page,
                shared=page * rng.randint(1, 4096 // page) if rng.random() < 0.6 else 0,
                keys=seqs * _log(rng, 1, 800) + rng.randint(0, 5))


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
    if c["op"] == "packed":
        rows = _split(c["rows"], n, 1)
        return rows, rows
    if c["op"] == "chunk":
        rows = _split(c["rows"], n, 1, 0.3)
        return rows, [x + y for x, y in zip(rows, _split(c["keys"] - c["rows"], n, 0))]
    # a decode step: shared keys, then at least one of its own
    return [1] * n, [c["shared"] + x for x in _split(c["keys"], n, 1)]


# ----------------------------------------------------------------- inputs

def prepare(case, seed):
    c = case
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    r = random.Random(seed)
    new, keys = _lengths(c)
    H, KV, hd, B = c["heads"], c["kv_heads"], c["head_dim"], c["seqs"]
    T = sum(new)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731

    def normal(*shape, scale=1.0):
        return torch.randn(shape, generator=g, device=dev, dtype=torch.float16).mul_(scale)

    cu = [0]
    for x in new:
        cu.append(cu[-1] + x)
    s = dict(case=c, cu=i32(cu), heads=H, kv_heads=KV, head_dim=hd)
    if c["op"] == "packed":  # the rows of a fused, rotated QKV projection
        s["qkv"] = normal(T, (H + 2 * KV) * hd, scale=1.2)
        return s
    ps = c["page"]
    width = max((x + ps - 1) // ps for x in keys)
    if c["op"] == "append":
        first = [(y - x) // ps for x, y in zip(new, keys)]  # pages that this step writes to
        shared = 0
    else:
        shared = c.get("shared", 0) // ps  # leading pages that all sequences hold
        first = [shared] * B
    need = shared + sum((y + ps - 1) // ps - f for y, f in zip(keys, first))
    ids = list(range(need + 2))
    r.shuffle(ids)
    table = torch.zeros((B, width), dtype=torch.int32)
    table[:, :] = torch.randint(0, need + 2, (B, width), generator=torch.Generator().manual_seed(seed),
                                dtype=torch.int32)
    at = shared
    for b in range(B):
        n = (keys[b] + ps - 1) // ps - first[b]
        table[b, :shared] = torch.tensor(ids[:shared], dtype=torch.int32)
        table[b, first[b]:first[b] + n] = torch.tensor(ids[at:at + n], dtype=torch.int32)
        at += n
    s["table"] = table.to(dev)
    s["k_pages"] = normal(need + 2, KV, ps, hd)
    s["v_pages"] = normal(need + 2, KV, ps, hd)
    s["lens"] = i32(keys)
    if c["op"] == "append":
        s["qkv"] = normal(T, (H + 2 * KV) * hd, scale=1.5)
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


def _plain_append(s):
    c, H, KV, hd = s["case"], s["heads"], s["kv_heads"], s["head_dim"]
    T = s["qkv"].shape[0]
    x = s["qkv"].view(T, H + 2 * KV, hd)
    q, k, v = x[:, :H].float(), x[:, H:H + KV].float(), x[:, H + KV:]
    if s["q_gamma"] is not None:
        q = q / torch.sqrt(q.square().mean(-1, keepdim=True) + EPS) * s["q_gamma"].float()
        k = k / torch.sqrt(k.square().mean(-1, keepdim=True) + EPS) * s["k_gamma"].float()
    angle = s["positions"].double()[:, None] * s["inv_freq"].double()
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    q = _rotated(q, cos, sin, c["rot"], c["interleaved"]).half().view(T, H * hd)
    k = _rotated(k, cos, sin, c["rot"], c["interleaved"]).half()
    pos = s["positions"].long()
    page = s["table"][_seq_of_rows(s["cu"], T), pos // c["page"]].long()
    s["k_pages"][page, :, pos % c["page"]] = k
    s["v_pages"][page, :, pos % c["page"]] = v
    return [q, s["k_pages"], s["v_pages"]]


def _plain_packed(s):
    H, KV, hd = s["heads"], s["kv_heads"], s["head_dim"]
    G = H // KV
    N = s["qkv"].shape[0]
    x = s["qkv"].view(N, H + 2 * KV, hd)
    q = x[:, :H].permute(1, 0, 2).float().reshape(KV, G * N, hd)
    k = x[:, H:H + KV].permute(1, 2, 0).float()
    v = x[:, H + KV:].permute(1, 0, 2).float()
    seq = _seq_of_rows(s["cu"], N)
    i = torch.arange(N, device=seq.device)
    hidden = (seq[:, None] != seq[None, :]) | (i[None, :] > i[:, None])
    p = torch.matmul(q, k).mul_(1.0 / math.sqrt(hd))
    p.view(KV, G, N, N).masked_fill_(hidden, -math.inf)
    p.sub_(p.amax(-1, keepdim=True)).exp_()
    o = torch.matmul(p, v) / p.sum(-1, keepdim=True)
    return o.view(H, N, hd).permute(1, 0, 2).reshape(N, H * hd).half()


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
    k = s["k_pages"][table].permute(0, 2, 4, 1, 3).reshape(B, KV, hd, L).float()
    p = torch.matmul(q, k).mul_(1.0 / math.sqrt(hd))
    new = cu[1:] - cu[:-1]
    last = (lens - new)[:, None] + torch.arange(M, device=seq.device)  # the last key that a row sees
    hidden = torch.arange(L, device=seq.device) > last[:, :, None]
    p.view(B, KV, G, M, L).masked_fill_(hidden[:, None, None], -math.inf)
    p.sub_(p.amax(-1, keepdim=True)).exp_()
    v = s["v_pages"][table].permute(0, 2, 1, 3, 4).reshape(B, KV, L, hd).float()
    o = torch.matmul(p, v) / p.sum(-1, keepdim=True)
    o = o.view(B, KV, G, M, hd).permute(0, 3, 1, 2, 4).reshape(B, M, H * hd)
    return o[seq, at].half()


def run(state):
    s, op = state, state["case"]["op"]
    if not own:
        return {"append": _plain_append, "packed": _plain_packed}.get(op, _plain_paged)(s)
    from npu_comp_b200 import npu
    H, KV, hd = s["heads"], s["kv_heads"], s["head_dim"]
    if op == "append":
        c = s["case"]
        q = npu.rope_paged_append(s["qkv"], H, KV, hd, s["positions"], s["inv_freq"], s["k_pages"], s["v_pages"],
                                  s["table"], cu_seqlens=s["cu"] if c["prompt"] else None, rot_dim=c["rot"],
                                  interleaved=c["interleaved"], q_gamma=s["q_gamma"], k_gamma=s["k_gamma"], eps=EPS)
        return [q, s["k_pages"], s["v_pages"]]
    if op == "packed":
        x = s["qkv"]
        return npu.attention_packed(x[:, :H * hd], x[:, H * hd:(H + KV) * hd], x[:, (H + KV) * hd:], s["cu"], H, KV,
                                    head_dim=hd)
    if op == "chunk":
        return npu.attention_paged(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lens"], s["cu"], heads=H,
                                   ctx_len=s["ctx"], max_new=s["max_new"])
    return npu.attention_paged_decode(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lens"], heads=H,
                                      shared_len=s["case"]["shared"], ctx_len=s["ctx"])


# -------------------------------------------------------- work and oracle

def work(case):
    c = case
    new, keys = _lengths(c)
    T, H, KV, hd = sum(new), c["heads"], c["kv_heads"], c["head_dim"]
    if c["op"] == "append":
        moved = T * (H + 2 * KV) * hd * 2
        return {"bytes": 2 * moved + T * 8 + c["rot"] * 2, "flops": T * (H + KV) * (3 * c["rot"] + 4 * hd * c["norm"])}
    pairs = sum(n * (y - n) + n * (n + 1) // 2 for n, y in zip(new, keys))
    shared = c.get("shared", 0)
    held = sum(keys) - shared * (c["seqs"] - 1)  # keys that have to be read, the shared ones once
    return {"bytes": 2 * T * H * hd * 2 + 2 * held * KV * hd * 2, "flops": 4 * H * hd * pairs}


def _exact_attention(q, k, v, scale):
    """q [n, H, d], k and v [m, KV, d]; the last query sees all m keys, each before it one less."""
    n, H, d = q.shape
    m, KV = k.shape[0], k.shape[1]
    out = torch.empty((n, H, d), dtype=torch.float64, device=q.device)
    j = torch.arange(m, device=q.device)
    for h in range(H):
        kh, vh = k[:, h // (H // KV)].double(), v[:, h // (H // KV)].double()
        for r0 in range(0, n, 4096):
            rows = torch.arange(r0, min(n, r0 + 4096), device=q.device)
            w = q[rows, h].double() @ kh.T * scale
            w = w.masked_fill(j[None, :] > (m - n + rows)[:, None], -math.inf)
            out[rows, h] = torch.softmax(w, -1) @ vh
    return out.reshape(n, H * d)


def exact(case, seed):
    s = prepare(case, seed)
    c, H, KV, hd = case, s["heads"], s["kv_heads"], s["head_dim"]
    new, keys = _lengths(c)
    scale = 1.0 / math.sqrt(hd)
    if c["op"] == "packed":
        x = s["qkv"].view(-1, H + 2 * KV, hd).split(new)
        return torch.cat([_exact_attention(y[:, :H], y[:, H:H + KV], y[:, H + KV:], scale) for y in x])
    if c["op"] != "append":
        out = []
        for b, q in enumerate(s["q"].view(-1, H, hd).split(new)):
            at = torch.arange(keys[b], device=q.device)
            page, slot = s["table"][b].long()[at // c["page"]], at % c["page"]
            out.append(_exact_attention(q, s["k_pages"][page, :, slot], s["v_pages"][page, :, slot], scale))
        return torch.cat(out)
    # append: pairs as complex numbers, multiplied by exp(i angle)
    kp, vp = s["k_pages"].double(), s["v_pages"].double()
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
    b = torch.repeat_interleave(torch.arange(c["seqs"], device=x.device), torch.tensor(new, device=x.device))
    pos = s["positions"].long()
    page = s["table"][b, pos // c["page"]].long()
    kp[page, :, pos % c["page"]] = x[:, H:H + KV]
    vp[page, :, pos % c["page"]] = x[:, H + KV:]
    return [x[:, :H].reshape(-1, H * hd), kp, vp]
