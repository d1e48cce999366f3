"""The paged-cache operators on the GPU against plain 64-bit forms
(paged_cases.py derives the bounds)."""
import math

import pytest
import torch

import npu_comp_b200 as nb
from npu_comp_b200 import npu
from paged_cases import append64, attention64, gather, poison, table_for

pytestmark = pytest.mark.gpu


def offsets(lens, dev):
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    return torch.tensor(cu, dtype=torch.int32, device=dev)


def within(got, want, bound):
    err = (got.double() - want).abs()
    assert torch.isfinite(got).all()
    assert (err <= bound).all(), f"worst excess {(err - bound).max().item():.3g}"


# ------------------------------------------------------------------- append

@pytest.mark.parametrize("new,start,H,KV,hd,rot,inter,norm,ps", [
    ([1], [0], 1, 1, 16, 16, False, False, 16),
    ([1], [1499], 32, 8, 128, 128, False, True, 16),
    ([1] * 37, [0, 130000] + [5000] * 35, 4, 4, 128, 64, True, True, 64),   # decode rows, far positions
    ([5, 0, 1, 70], [3, 9, 100001, 0], 6, 2, 64, 32, False, False, 1),       # packed, an empty one, pages of one slot
    ([33, 31], [0, 15], 8, 2, 80, 48, True, True, 128),                      # units that fill no power of two
    ([3, 300], [1, 2], 2, 1, 256, 256, False, True, 256),
    ([2], [2], 1, 1, 512, 512, True, True, 16),
    ([700] * 2, [0, 64], 16, 16, 128, 128, False, False, 32),
])
@pytest.mark.parametrize("packed", [True, False])
def test_append(cuda_device, new, start, H, KV, hd, rot, inter, norm, ps, packed):
    if not packed and any(n != 1 for n in new):
        pytest.skip("a decode step has one row per sequence")
    dev, g = cuda_device, torch.Generator().manual_seed(sum(new) + hd)
    T, keys = sum(new), [s + n for s, n in zip(start, new)]
    first = [s // ps for s in start]
    W = max((k + ps - 1) // ps for k in keys) + 1
    need = [(k + ps - 1) // ps - f for k, f in zip(keys, first)]
    n_pages = sum(need) + 2
    ids = torch.randperm(n_pages, generator=g).int()
    table = torch.full((len(new), W + 3), -5, dtype=torch.int32)
    at = 0
    for b in range(len(new)):
        table[b, first[b]:first[b] + need[b]] = ids[at:at + need[b]]
        at += need[b]
    table = table.to(dev)[:, :W]  # a strided table
    extra = 2 if packed else 0  # rows behind the last sequence
    x = torch.randn((T + extra, (H + 2 * KV) * hd + 8), generator=g).half().to(dev)[:, :(H + 2 * KV) * hd]
    pos = torch.tensor([s + i for s, n in zip(start, new) for i in range(n)] + [0] * extra, dtype=torch.int32, device=dev)
    f = nb.rope_freqs(rot, 500000.0, device=dev)
    gam = [(1 + 0.3 * torch.randn(hd, generator=g)).half().to(dev) if norm else None for _ in range(2)]
    kp = torch.randn((n_pages, KV, ps, hd), generator=g).half().to(dev)
    vp = torch.randn((n_pages, KV, ps, hd), generator=g).half().to(dev)
    kw, vw = kp.clone(), vp.clone()
    out = torch.full((T + extra, H * hd + 16), 3.0, dtype=torch.float16, device=dev)[:, :H * hd]
    q = nb.rope_paged_append(x, H, KV, hd, pos, f, kp, vp, table, cu_seqlens=offsets(new, dev) if packed else None,
                             rot_dim=rot, interleaved=inter, q_gamma=gam[0], k_gamma=gam[1], eps=1e-6, out=out)
    assert q.data_ptr() == out.data_ptr()
    x3 = x[:T].reshape(T, H + 2 * KV, hd)
    (qe, qb), (ke, kb) = append64(x3, H, KV, pos[:T], f, rot, inter, gam[0], gam[1], 1e-6)
    within(q[:T], qe.reshape(T, -1), qb.reshape(T, -1))
    assert (q[T:] == 3.0).all()
    seq = torch.repeat_interleave(torch.arange(len(new)), torch.tensor(new)).to(dev)
    page, slot = table[seq, pos[:T].long() // ps].long(), pos[:T].long() % ps
    within(kp[page, :, slot], ke, kb)
    assert torch.equal(vp[page, :, slot], x3[:, H + KV:])
    kp[page, :, slot], vp[page, :, slot] = kw[page, :, slot], vw[page, :, slot]
    assert torch.equal(kp, kw) and torch.equal(vp, vw)  # nothing else was written


def test_append_unstored_rows_and_in_place(cuda_device):
    """Positions outside the table and page ids outside the pool: q is rotated,
    nothing is stored; out may be the q columns of qkv, with the same bits."""
    dev, g = cuda_device, torch.Generator().manual_seed(5)
    H, KV, hd, ps, T = 4, 2, 128, 16, 6
    x = torch.randn((T, (H + 2 * KV) * hd), generator=g).half().to(dev)
    pos = torch.tensor([-1, 32, 31, 5, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32, device=dev)
    table = torch.tensor([[0, 1]] * 2 + [[0, 99], [-7, 1]] + [[0, 1]] * 2, dtype=torch.int32, device=dev)
    kp = torch.zeros((3, KV, ps, hd), dtype=torch.float16, device=dev)
    vp = torch.zeros_like(kp)
    f = nb.rope_freqs(hd, device=dev)
    q = nb.rope_paged_append(x, H, KV, hd, pos, f, kp, vp, table)
    assert not kp.any() and not vp.any()
    (qe, qb), _ = append64(x.view(T, H + 2 * KV, hd), H, KV, pos, f, hd, False, None, None, 0.0)
    within(q[:4], qe.reshape(T, -1)[:4], qb.reshape(T, -1)[:4])
    y = x.clone()
    r = nb.rope_paged_append(y, H, KV, hd, pos, f, kp, vp, table, out=y[:, :H * hd])
    assert torch.equal(r, q) and torch.equal(y[:, H * hd:], x[:, H * hd:])


# ------------------------------------------------------------------- packed

def run_packed(dev, lens, H, KV, hd, causal=True, behind=3, bad=(), scale=None, spread=1.0):
    g = torch.Generator(device=dev).manual_seed(sum(lens) * 7 + H)
    T = sum(lens)
    x = spread * torch.randn((T + behind, (H + 2 * KV) * hd), generator=g, device=dev)
    x = x.half()
    cu = offsets(lens, dev)
    for b in bad:  # a sequence full of NaN
        x[int(cu[b]):int(cu[b + 1])] = float("nan")
    x[T:] = float("nan")
    q, k, v = x[:, :H * hd], x[:, H * hd:(H + KV) * hd], x[:, (H + KV) * hd:]
    out = torch.full((T + behind, H * hd), 3.0, dtype=torch.float16, device=dev)
    o = nb.attention_packed(q, k, v, cu, H, KV, head_dim=hd, causal=causal, scale=scale, out=out)
    assert npu.device_error() == 0
    assert (o[T:] == 3.0).all()
    sc = scale or 1 / math.sqrt(hd)
    for b, n in enumerate(lens):
        r = slice(int(cu[b]), int(cu[b]) + n)
        if n == 0 or b in bad:
            continue
        e, bound = attention64(q[r].reshape(n, H, hd), k[r].reshape(n, KV, hd), v[r].reshape(n, KV, hd), sc, causal)
        within(o[r], e, bound)
    return o


@pytest.mark.parametrize("lens,H,KV,hd", [
    ([1], 1, 1, 128), ([2, 1, 1], 2, 1, 64), ([128], 2, 2, 128), ([127, 129], 4, 4, 128), ([1, 0, 7, 57, 0], 8, 2, 128),
    ([300], 3, 1, 128), ([700, 129], 10, 2, 64), ([33, 95], 7, 1, 96), ([40, 8], 4, 2, 16), ([513, 1], 16, 1, 80),
    ([20, 300], 64, 1, 128), ([5, 17], 128, 1, 64), ([64] * 50, 8, 4, 128), ([1] * 333, 4, 2, 64),
    ([2000, 1, 1500, 0, 0, 900], 8, 2, 128), ([3000], 4, 4, 64),
])
@pytest.mark.parametrize("causal", [True, False])
def test_packed(cuda_device, lens, H, KV, hd, causal):
    run_packed(cuda_device, lens, H, KV, hd, causal)


def test_packed_neighbours_do_not_leak(cuda_device):
    """NaN rows of one sequence, and behind the last one, reach no other."""
    run_packed(cuda_device, [70, 40, 5, 130], 4, 2, 128, bad=(1, 3))
    run_packed(cuda_device, [70, 40, 5, 130], 4, 2, 64, bad=(1, 3), causal=False)


def test_packed_peaked_scores(cuda_device):
    """Scores of a few hundred: the running maximum moves many times."""
    run_packed(cuda_device, [900, 33], 4, 2, 128, scale=0.5, spread=2.0)
    run_packed(cuda_device, [1], 4, 2, 128, scale=40.0, spread=2.0)


def test_packed_rising_maximum(cuda_device):
    """Keys sorted so that every block's maximum is far above the last one's,
    and so that it only falls."""
    dev, n, hd = cuda_device, 1024, 128
    for rising in (True, False):
        q = torch.zeros((n, hd), device=dev)
        q[:, 0] = 1.0
        k = torch.zeros((n, hd), device=dev)
        k[:, 0] = torch.linspace(-300, 300, n, device=dev) * (1 if rising else -1)
        v = torch.randn((n, hd), generator=torch.Generator(device=dev).manual_seed(1), device=dev)
        q, k, v = q.half(), k.half(), v.half()
        o = nb.attention_packed(q, k, v, offsets([n], dev), 1, 1, scale=1.0)
        e, b = attention64(q.view(n, 1, hd), k.view(n, 1, hd), v.view(n, 1, hd), 1.0)
        within(o, e, b)


def test_packed_equals_attention_on_equal_lengths(cuda_device):
    dev, T, H, KV, hd = cuda_device, 320, 8, 2, 128
    x = torch.randn((2 * T, (H + 2 * KV) * hd), generator=torch.Generator(device=dev).manual_seed(3), device=dev).half()
    q, k, v = x[:, :H * hd], x[:, H * hd:(H + KV) * hd], x[:, (H + KV) * hd:]
    a = nb.attention(q, k, v, H, KV, head_dim=hd, batch=2).double()
    b = nb.attention_packed(q, k, v, offsets([T, T], dev), H, KV, head_dim=hd).double()
    e = torch.cat([attention64(q[r].reshape(T, H, hd), k[r].reshape(T, KV, hd), v[r].reshape(T, KV, hd),
                               1 / math.sqrt(hd))[1] for r in (slice(0, T), slice(T, 2 * T))])
    assert ((a - b).abs() <= 2 * e).all()


# -------------------------------------------------------------------- paged

def make_cache(dev, keys, KV, hd, ps, shared=0, seed=0, extra=3):
    gen = torch.Generator().manual_seed(seed + sum(keys))
    g = torch.Generator(device=dev).manual_seed(seed + sum(keys))
    table, n = table_for(keys, ps, gen=gen, shared=shared, n_extra=extra)
    kp = torch.randn((n, KV, ps, hd), generator=g, device=dev).half()
    vp = torch.randn((n, KV, ps, hd), generator=g, device=dev).half()
    kh, vh = kp.cpu(), vp.cpu()
    poison(kh, vh, table, keys, ps)
    kp.copy_(kh)
    vp.copy_(vh)
    return kp, vp, table.to(dev), torch.tensor(keys, dtype=torch.int32, device=dev)


def check_rows(o, q, kp, vp, table, new, keys, H, ps, causal=True, scale=None):
    hd, at = kp.shape[3], 0
    for b, n in enumerate(new):
        if n:
            k, v = gather(kp, table[b], keys[b], ps), gather(vp, table[b], keys[b], ps)
            e, bound = attention64(q[at:at + n].reshape(n, H, hd), k, v, scale or 1 / math.sqrt(hd), causal)
            within(o[at:at + n], e, bound)
        at += n


@pytest.mark.parametrize("new,keys,H,KV,hd,ps", [
    ([1], [1], 1, 1, 128, 16),
    ([5, 128, 1], [5, 200, 999], 8, 2, 128, 16),
    ([5, 0, 1, 3], [5, 200, 999, 0], 8, 2, 64, 64),          # a sequence without rows, one without keys
    ([5, 300, 1, 3], [3, 200, 999, 1], 4, 4, 64, 32),        # more rows than keys: rows that see nothing
    ([256, 300], [3000, 4001], 32, 8, 128, 128),
    ([17, 30], [3000, 4001], 3, 1, 96, 256),
    ([2, 2, 2], [129, 4000, 65], 5, 1, 128, 16),             # few rows, key splits
    ([4] * 24, [100 + 97 * i for i in range(24)], 32, 8, 128, 64),
    ([8, 3, 1], [1000, 3, 1], 2, 1, 16, 16),
    ([1, 1], [6000, 17], 32, 1, 128, 16),                    # 32 query heads on one kv head
    ([16, 2], [16, 333], 1, 1, 80, 32),
    ([40], [20000], 16, 2, 128, 16),                         # one chunk, long context: splits of the tile kernel
])
@pytest.mark.parametrize("known", [True, False])
@pytest.mark.parametrize("causal", [True, False])
def test_paged(cuda_device, new, keys, H, KV, hd, ps, known, causal):
    dev = cuda_device
    kp, vp, table, lens = make_cache(dev, keys, KV, hd, ps)
    T = sum(new)
    q = torch.randn((T + 2, H * hd), generator=torch.Generator(device=dev).manual_seed(T), device=dev).half()
    out = torch.full((T + 2, H * hd), 3.0, dtype=torch.float16, device=dev)
    o = nb.attention_paged(q, kp, vp, table, lens, offsets(new, dev), heads=H, max_new=max(new) if known else 0,
                           ctx_len=max(keys) if known else 0, causal=causal, out=out)
    assert npu.device_error() == 0
    assert (o[T:] == 3.0).all()
    check_rows(o, q, kp, vp, table, new, keys, H, ps, causal)


def test_paged_context_hint_is_only_a_hint(cuda_device):
    """Keys past ctx_len count all the same."""
    dev, new, keys, H, KV, hd, ps = cuda_device, [2, 1], [5000, 700], 4, 2, 128, 16
    kp, vp, table, lens = make_cache(dev, keys, KV, hd, ps)
    q = torch.randn((3, H * hd), device=dev).half()
    for kw in (dict(max_new=2), dict()):
        check_rows(nb.attention_paged(q, kp, vp, table, lens, offsets(new, dev), heads=H, ctx_len=600, **kw), q, kp,
                   vp, table, new, keys, H, ps)
    check_rows(nb.attention_paged_decode(q[:2], kp, vp, table, lens, heads=H, ctx_len=600), q, kp, vp, table, [1, 1],
               keys, H, ps)


def test_paged_bad_pages_read_as_zeros(cuda_device):
    """Ids outside the pool inside a sequence's keys: zero keys and values."""
    dev, H, KV, hd, ps, keys = cuda_device, 4, 2, 128, 16, [100, 60]
    kp, vp, table, lens = make_cache(dev, keys, KV, hd, ps)
    table[0, 2], table[0, 4], table[1, 0] = -1, kp.shape[0], 2 ** 31 - 1
    kz, vz = torch.cat([kp, torch.zeros_like(kp[:1])]), torch.cat([vp, torch.zeros_like(vp[:1])])
    tz = torch.where((table < 0) | (table >= kp.shape[0]), kp.shape[0], table)
    q = torch.randn((6, H * hd), device=dev).half()
    o = nb.attention_paged(q, kp, vp, table, lens, offsets([4, 2], dev), heads=H)
    check_rows(o, q, kz, vz, tz, [4, 2], keys, H, ps)
    o = nb.attention_paged(q, kp, vp, table, lens, offsets([4, 2], dev), heads=H, max_new=4)
    check_rows(o, q, kz, vz, tz, [4, 2], keys, H, ps)


# ------------------------------------------------------------------- decode

@pytest.mark.parametrize("keys,shared,H,KV,hd,ps", [
    ([1], 0, 1, 1, 128, 16), ([777], 0, 32, 8, 128, 16), ([0], 0, 4, 2, 128, 16), ([5000], 0, 8, 1, 64, 128),
    ([300, 0, 64, 65, 1, 4000], 0, 8, 2, 128, 16),
    ([100 + 31 * i for i in range(64)], 0, 4, 4, 128, 32),
    ([1000] * 3, 512, 32, 8, 128, 64),
    ([2048 + i for i in range(40)], 2048, 16, 2, 128, 16),   # 320 rows per kv head: two pairs of tiles
    ([2049, 10, 0, 2048, 2047, 3000], 2048, 6, 2, 128, 64),  # sequences inside the prefix
    ([256] * 5, 256, 8, 8, 64, 256),                         # nothing but the prefix
    ([700, 900], 640, 32, 1, 128, 16),                       # groups of 32: the tile kernel on the own keys
    ([4500, 4097, 4100], 4096, 40, 8, 96, 32),
    ([130] * 300, 128, 2, 2, 128, 16),
])
def test_decode(cuda_device, keys, shared, H, KV, hd, ps):
    dev, B = cuda_device, len(keys)
    full = [max(k, shared) for k in keys]  # every sequence holds the prefix's pages, used or not
    kp, vp, table, _ = make_cache(dev, full, KV, hd, ps, shared=shared)
    if not shared:
        kp, vp, table, _ = make_cache(dev, keys, KV, hd, ps)
    lens = torch.tensor(keys, dtype=torch.int32, device=dev)
    q = torch.randn((B, H * hd + 8), generator=torch.Generator(device=dev).manual_seed(B), device=dev).half()[:, :H * hd]
    for sl in {0, shared}:
        o = nb.attention_paged_decode(q, kp, vp, table, lens, heads=H, shared_len=sl, ctx_len=max(keys))
        assert npu.device_error() == 0
        check_rows(o, q, kp, vp, table, [1] * B, keys, H, ps)
        assert torch.equal(o, nb.attention_paged_decode(q, kp, vp, table, lens, heads=H, shared_len=sl,
                                                        ctx_len=max(keys)))


def test_offsets_past_32_bits(cuda_device):
    """Pages behind 2^31 elements of the pool."""
    dev, H, KV, hd, ps = cuda_device, 8, 8, 128, 64
    n = 2 ** 31 // (KV * ps * hd) + 40
    kp = torch.empty((n, KV, ps, hd), dtype=torch.float16, device=dev)
    vp = torch.empty_like(kp)
    ids = torch.tensor([[n - 1, n - 7, 3, n - 20]], dtype=torch.int32, device=dev)
    kp[ids[0].long()] = torch.randn((4, KV, ps, hd), device=dev).half()
    vp[ids[0].long()] = torch.randn((4, KV, ps, hd), device=dev).half()
    x = torch.randn((3, (H + 2 * KV) * hd), device=dev).half()
    pos = torch.tensor([190, 191, 192], dtype=torch.int32, device=dev)
    f = nb.rope_freqs(hd, device=dev)
    cu, lens = offsets([3], dev), torch.tensor([193], dtype=torch.int32, device=dev)
    q = nb.rope_paged_append(x, H, KV, hd, pos, f, kp, vp, ids, cu_seqlens=cu)
    (qe, qb), (ke, kb) = append64(x.view(3, -1, hd), H, KV, pos, f, hd, False, None, None, 0.0)
    within(q, qe.reshape(3, -1), qb.reshape(3, -1))
    within(gather(kp, ids[0], 193, ps)[190:], ke, kb)
    for kw in (dict(), dict(max_new=3)):
        check_rows(nb.attention_paged(q, kp, vp, ids, lens, cu, heads=H, **kw), q, kp, vp, ids, [3], [193], H, ps)
    check_rows(nb.attention_paged_decode(q[2:], kp, vp, ids, lens, heads=H), q[2:], kp, vp, ids, [1], [193], H, ps)


# ----------------------------------------------------------------- together

def test_serving_run(cuda_device):
    """Prompts in two chunks behind a common prefix, then decode steps, all
    through the pages, against attention over the plain rows in 64 bits."""
    dev, H, KV, hd, ps, B = cuda_device, 8, 2, 128, 16, 3
    g = torch.Generator(device=dev).manual_seed(9)
    prefix, chunks, steps = 64, ([40, 7, 130], [1, 60, 3]), 3
    width, n_pages = 32, 100
    table = torch.zeros((B, width), dtype=torch.int32)
    ids = torch.randperm(n_pages, generator=torch.Generator().manual_seed(2)).int()
    table[:, :4] = ids[:4]
    table[:, 4:] = ids[4:4 + B * 28].view(B, 28)
    table = table.to(dev)
    kp = torch.full((n_pages, KV, ps, hd), float("nan"), dtype=torch.float16, device=dev)
    vp = kp.clone()
    f = nb.rope_freqs(hd, 500000.0, llama3_scaling=True, device=dev)
    gam = (1 + 0.2 * torch.randn(hd, generator=g, device=dev)).half()
    hist = [[] for _ in range(B)]  # the fused rows of each sequence so far
    rows = lambda n: torch.randn((n, (H + 2 * KV) * hd), generator=g, device=dev).half()  # noqa: E731

    def want(b, n):
        x = torch.cat(hist[b]).view(-1, H + 2 * KV, hd)
        pos = torch.arange(x.shape[0], device=dev)
        (qe, _), (ke, _) = append64(x, H, KV, pos, f, hd, False, gam, gam, 1e-5)
        # the operators' own q and k are fp16: so are the formula's
        return attention64(qe[-n:].half(), ke.half(), x[:, H + KV:], 1 / math.sqrt(hd))

    def check(o, new):
        at = 0
        for b, n in enumerate(new):
            if n:
                e, bound = want(b, n)
                # q and k may round to the neighbouring fp16 value where the fp32 and the 64-bit results straddle a
                # border: one step of 2^-10 in a few of the 128 products of a score
                err = (o[at:at + n].double() - e).abs()
                assert (err <= 4 * bound).all()
            at += n

    x = rows(prefix)  # the prefix, once, for sequence 0's pages (all hold them)
    for b in range(B):
        hist[b].append(x)
    pos = torch.arange(prefix, dtype=torch.int32, device=dev)
    q = nb.rope_paged_append(x, H, KV, hd, pos, f, kp, vp, table[:1], cu_seqlens=offsets([prefix], dev), q_gamma=gam,
                             k_gamma=gam)
    o = nb.attention_paged(q, kp, vp, table[:1], torch.tensor([prefix], dtype=torch.int32, device=dev),
                           offsets([prefix], dev), heads=H)
    e, bound = want(0, prefix)
    assert ((o.double() - e).abs() <= 4 * bound).all()
    lens = [prefix] * B
    for new in chunks:
        x = rows(sum(new))
        for b, part in enumerate(x.split(new)):
            hist[b].append(part)
        pos = torch.tensor([lens[b] + i for b in range(B) for i in range(new[b])], dtype=torch.int32, device=dev)
        lens = [a + n for a, n in zip(lens, new)]
        cu = offsets(new, dev)
        q = nb.rope_paged_append(x, H, KV, hd, pos, f, kp, vp, table, cu_seqlens=cu, q_gamma=gam, k_gamma=gam)
        o = nb.attention_paged(q, kp, vp, table, torch.tensor(lens, dtype=torch.int32, device=dev), cu, heads=H,
                               max_new=max(new))
        check(o, new)
    for _ in range(steps):
        x = rows(B)
        for b in range(B):
            hist[b].append(x[b:b + 1])
        pos = torch.tensor(lens, dtype=torch.int32, device=dev)
        lens = [n + 1 for n in lens]
        q = nb.rope_paged_append(x, H, KV, hd, pos, f, kp, vp, table, q_gamma=gam, k_gamma=gam)
        o = nb.attention_paged_decode(q, kp, vp, table, pos + 1, heads=H, shared_len=prefix)
        check(o, [1] * B)
    assert npu.device_error() == 0


def test_graph_replay_and_streams(cuda_device):
    """A decode step captured once and replayed with other lengths, positions
    and pages, on a stream of its own while another runs the same ops."""
    dev, H, KV, hd, ps, B, W = cuda_device, 8, 2, 128, 16, 4, 40
    g = torch.Generator(device=dev).manual_seed(4)
    kp = torch.randn((B * W, KV, ps, hd), generator=g, device=dev).half()
    vp = torch.randn((B * W, KV, ps, hd), generator=g, device=dev).half()
    table = torch.randperm(B * W, generator=g, device=dev).int().view(B, W)
    table[:, :8] = table[0, :8]
    x = torch.randn((B, (H + 2 * KV) * hd), generator=g, device=dev).half()
    pos = torch.zeros(B, dtype=torch.int32, device=dev)
    f = nb.rope_freqs(hd, device=dev)

    def step():
        lens = pos + 1
        q = nb.rope_paged_append(x, H, KV, hd, pos, f, kp, vp, table)
        return q, nb.attention_paged_decode(q, kp, vp, table, lens, heads=H, shared_len=128, ctx_len=W * ps)

    pos.copy_(torch.tensor([200, 300, 130, 128]))
    side = torch.cuda.Stream(device=dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream(dev).wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q, o = step()
    for p in ([200, 300, 130, 128], [500, 129, 400, 639]):
        pos.copy_(torch.tensor(p))
        x.copy_(torch.randn(x.shape, generator=g, device=dev).half())
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graph.replay()
        other = torch.randn((B, H * hd), generator=g, device=dev).half()
        lens2 = torch.tensor([150, 140, 129, 640], dtype=torch.int32, device=dev)
        torch.cuda.synchronize()
        o2 = nb.attention_paged_decode(other, kp, vp, table, lens2, heads=H, shared_len=128)
        torch.cuda.synchronize()
        keys = [n + 1 for n in p]
        check_rows(o, q, kp, vp, table, [1] * B, keys, H, ps)
        check_rows(o2, other, kp, vp, table, [1] * B, lens2.tolist(), H, ps)
    del graph


def test_rows_outside_the_offsets_stay(cuda_device):
    """Offsets that start behind row 0 and end ahead of the last row, and
    outputs whose rows are only 16-byte aligned."""
    dev, H, KV, hd, ps = cuda_device, 4, 2, 80, 16
    g = torch.Generator(device=dev).manual_seed(8)
    T, cu = 60, torch.tensor([5, 5, 40, 57], dtype=torch.int32, device=dev)
    x = torch.randn((T, (H + 2 * KV) * hd), generator=g, device=dev).half()
    q, k, v = x[:, :H * hd], x[:, H * hd:(H + KV) * hd], x[:, (H + KV) * hd:]
    kp, vp, table, lens = make_cache(dev, [7, 200, 90], KV, hd, ps)
    f = nb.rope_freqs(hd, device=dev)
    for run in (lambda o: nb.attention_packed(q, k, v, cu, H, KV, head_dim=hd, out=o),
                lambda o: nb.attention_paged(q.contiguous(), kp, vp, table, lens, cu, heads=H, out=o),
                lambda o: nb.attention_paged(q.contiguous(), kp, vp, table, lens, cu, heads=H, ctx_len=64, out=o),
                lambda o: nb.rope_paged_append(x, H, KV, hd, torch.zeros(T, dtype=torch.int32, device=dev), f,
                                               kp.clone(), vp.clone(), table, cu_seqlens=cu, out=o)):
        outs = []
        for off, pad in ((0, 0), (8, 24)):
            base = torch.full((T, off + H * hd + pad), 3.0, dtype=torch.float16, device=dev)
            o = run(base[:, off:off + H * hd])
            assert (o[:5] == 3.0).all() and (o[57:] == 3.0).all() and (o[5:57] != 3.0).any(dim=1).all()
            assert (base[:, :off] == 3.0).all() and (base[:, off + H * hd:] == 3.0).all()
            outs.append(o.clone())
        assert torch.equal(*outs)
    o = nb.attention_packed(q, k, v, cu, H, KV, head_dim=hd)
    e, b = attention64(q[40:57].reshape(-1, H, hd), k[40:57].reshape(-1, KV, hd), v[40:57].reshape(-1, KV, hd),
                       1 / math.sqrt(hd))
    within(o[40:57], e, b)


def test_many_sequences(cuda_device):
    """More sequences than a warp holds, of 0 to 90 rows, and a long one."""
    lens = [(i * 37) % 91 for i in range(200)] + [900]
    run_packed(cuda_device, lens, 8, 2, 64)
    run_packed(cuda_device, lens, 16, 16, 128)
    dev, H, KV, hd, ps = cuda_device, 8, 2, 128, 16
    new = [(i * 5) % 7 for i in range(100)] + [70]
    keys = [n + (i * 53) % 300 for i, n in enumerate(new)]
    kp, vp, table, ln = make_cache(dev, keys, KV, hd, ps)
    q = torch.randn((sum(new), H * hd), device=dev).half()
    check_rows(nb.attention_paged(q, kp, vp, table, ln, offsets(new, dev), heads=H), q, kp, vp, table, new, keys, H, ps)


@pytest.mark.parametrize("H,KV,hd", [(8, 8, 128), (16, 1, 64), (64, 1, 128)])
def test_long_context(cuda_device, H, KV, hd):
    """Contexts past 2^16 keys: the largest numbers of key ranges."""
    dev, ps, keys = cuda_device, 64, [70001, 1, 66000]
    kp, vp, table, lens = make_cache(dev, keys, KV, hd, ps)
    q = torch.randn((3, H * hd), device=dev).half()
    for kw in (dict(), dict(ctx_len=70001)):
        check_rows(nb.attention_paged_decode(q, kp, vp, table, lens, heads=H, **kw), q, kp, vp, table, [1] * 3, keys,
                   H, ps)
    check_rows(nb.attention_paged_decode(q[:1], kp, vp, table[:1], lens[:1], heads=H), q[:1], kp, vp, table[:1], [1],
               keys[:1], H, ps)


def test_prompt_graph_replay(cuda_device):
    """Packed prompts and chunks captured once, replayed with other offsets and
    lengths of the same totals; two graphs do not share scratch."""
    dev, H, KV, hd, ps, B, T = cuda_device, 8, 2, 128, 16, 3, 90
    keys = [400, 500, 300]
    kp, vp, table, lens = make_cache(dev, keys, KV, hd, ps)
    g = torch.Generator(device=dev).manual_seed(6)
    x = torch.randn((T, (H + 2 * KV) * hd), generator=g, device=dev).half()
    q, k, v = x[:, :H * hd], x[:, H * hd:(H + KV) * hd], x[:, (H + KV) * hd:]
    qc = q.contiguous()
    cu = offsets([30, 30, 30], dev)
    nb.attention_paged(qc, kp, vp, table, lens, cu, heads=H)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            a = nb.attention_packed(q, k, v, cu, H, KV, head_dim=hd)
            b = nb.attention_paged(qc, kp, vp, table, lens, cu, heads=H)
        graphs.append((graph, a, b))
    side = torch.cuda.Stream(device=dev)
    for new, left in (([1, 60, 29], [400, 77, 300]), ([0, 0, 90], [1, 500, 90])):
        cu.copy_(offsets(new, dev))
        lens.copy_(torch.tensor(left))
        torch.cuda.synchronize()
        graphs[0][0].replay()
        with torch.cuda.stream(side):
            graphs[1][0].replay()
        torch.cuda.synchronize()
        for _, a, b in graphs:
            at = 0
            for n in new:
                if n:
                    r = slice(at, at + n)
                    e, bound = attention64(q[r].reshape(n, H, hd), k[r].reshape(n, KV, hd), v[r].reshape(n, KV, hd),
                                           1 / math.sqrt(hd))
                    within(a[r], e, bound)
                at += n
            check_rows(b, qc, kp, vp, table, new, left, H, ps)
    graphs.clear()


def test_python_refusals(cuda_device):
    dev, H, KV, hd, ps = cuda_device, 4, 2, 128, 16
    z = lambda *s, t=torch.float16: torch.zeros(s, dtype=t, device=dev)  # noqa: E731
    i32 = lambda *s: z(*s, t=torch.int32)  # noqa: E731
    kp, table, lens, cu, q = z(4, KV, ps, hd), i32(2, 3), i32(2), i32(3), z(2, H * hd)
    x, f = z(2, (H + 2 * KV) * hd), z(64, t=torch.float32)
    ok = dict(heads=H)
    nb.attention_paged_decode(q, kp, kp, table, lens, **ok)
    bad = [
        lambda: nb.attention_paged_decode(q, kp, kp, table, lens, heads=3),
        lambda: nb.attention_paged_decode(q, kp, kp, table, lens, heads=H, shared_len=8),       # not whole pages
        lambda: nb.attention_paged_decode(q, kp, kp, table, lens, heads=H, shared_len=64),      # past the table
        lambda: nb.attention_paged_decode(q, kp, kp, table, lens, heads=H, shared_len=-16),
        lambda: nb.attention_paged_decode(q, kp, kp, table, lens, heads=H, scale=-1.0),
        lambda: nb.attention_paged_decode(q, kp, kp, table, lens, heads=H, scale=float("nan")),
        lambda: nb.attention_paged_decode(q, kp, kp, table.long(), lens, **ok),
        lambda: nb.attention_paged_decode(q, kp, kp, table, lens[:1], **ok),
        lambda: nb.attention_paged_decode(q, kp, kp.transpose(1, 2), table, lens, **ok),
        lambda: nb.attention_paged_decode(q.float(), kp, kp, table, lens, **ok),
        lambda: nb.attention_paged_decode(q.cpu(), kp, kp, table, lens, **ok),
        lambda: nb.attention_paged_decode(q, z(4, KV, 24, hd), z(4, KV, 24, hd), table, lens, **ok),
        lambda: nb.attention_paged_decode(q, z(4, KV, 8, hd), z(4, KV, 8, hd), table, lens, **ok),
        lambda: nb.attention_paged(q, kp, kp, table, lens, cu[:2], **ok),
        lambda: nb.attention_paged(q, kp, kp, table, lens, cu, heads=H, max_new=-1),
        lambda: nb.attention_packed(q, q, q, cu, 4, 3, head_dim=hd),
        lambda: nb.attention_packed(q, q[:1], q, cu, 4, 2, head_dim=hd),
        lambda: nb.attention_packed(q, q, q, cu.long(), 4, 2, head_dim=hd),
        lambda: nb.rope_paged_append(x, H, KV, hd, lens, f[:32], kp, kp, table),
        lambda: nb.rope_paged_append(x, H, KV, hd, lens, f[:4], kp, kp, table, rot_dim=8),
        lambda: nb.rope_paged_append(x[:1], H, KV, hd, lens[:1], f, kp, kp, table),
        lambda: nb.rope_paged_append(x, H, KV, hd, lens, f, kp, kp, table, q_gamma=z(64)),
        lambda: nb.rope_paged_append(x[:, 8:], H, KV, hd, lens, f, kp, kp, table),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was not refused")
    with pytest.raises(nb.NpubError):  # head_dim past 128
        nb.attention_packed(z(2, 144), z(2, 144), z(2, 144), cu, 1, 1, head_dim=144)
    assert nb.attention_packed(z(0, H * hd), z(0, KV * hd), z(0, KV * hd), i32(1), H, KV, head_dim=hd).shape == (0, H * hd)
