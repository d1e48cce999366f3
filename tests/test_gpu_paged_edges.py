"""The paged-cache operators on the GPU where calls go wrong most easily
(paged_exact.py derives the bounds)."""
import math

import pytest
import torch

import npu_comp_b200 as nb
from npu_comp_b200 import npu
from paged_exact import attention_exact, same, to_pages

pytestmark = pytest.mark.gpu


def offsets(lens, dev):
    return torch.tensor([0] + list(torch.tensor(lens).cumsum(0)), dtype=torch.int32, device=dev)


# How a call reaches each kernel: new rows and keys per sequence, heads, the keys that take turns in the test.
#   packed / tiles: tile kernel, keys whole; ranges: the tile kernel's partials; few: up to 16 rows per kv head, keys
#   whole, in a cluster, or as partials; decode, prefix: one row, with and without a shared prefix
PATHS = {
    "packed": ([200, 70, 1], [200, 70, 1], 4, 2),
    "tiles": ([150, 3, 9], [300, 77, 4], 4, 2),
    "ranges": ([40, 2], [9000, 300], 8, 2),
    "few": ([3, 1, 4], [100, 70, 2], 4, 2),
    "few_long": ([3, 1, 4], [6000, 70, 700], 4, 2),
    "decode": ([1] * 4, [300, 0, 65, 2000], 8, 2),
    "prefix": ([1] * 4, [700, 520, 600, 513], 8, 2),
}


class Call:
    """One call of PATHS with random inputs; x.run() compares every row with the 64-bit form."""

    def __init__(self, dev, path, hd, causal=True, ps=16):
        self.path, self.hd, self.causal, self.ps, self.dev = path, hd, causal, ps, dev
        self.new, self.keys, self.H, self.KV = PATHS[path]
        g = torch.Generator(device=dev).manual_seed(hd + sum(self.keys))
        rnd = lambda *s: torch.randn(s, generator=g, device=dev).half()  # noqa: E731
        self.q = [rnd(n, self.H, hd) for n in self.new]
        self.k = [rnd(n, self.KV, hd) for n in self.keys]
        self.v = [rnd(n, self.KV, hd) for n in self.keys]
        self.shared = 512 if path == "prefix" else 0
        for x in (self.k, self.v):
            for y in x[1:]:
                y[:self.shared] = x[0][:self.shared]

    def run(self):
        dev, H, KV, hd = self.dev, self.H, self.KV, self.hd
        q, cu = torch.cat(self.q).reshape(-1, H * hd), offsets(self.new, dev)
        if self.path == "packed":
            o = nb.attention_packed(q, torch.cat(self.k).reshape(-1, KV * hd), torch.cat(self.v).reshape(-1, KV * hd),
                                    cu, H, KV, head_dim=hd, causal=self.causal)
        else:
            kp, vp, table, lens = to_pages(self.k, self.v, self.ps, shared=self.shared)
            if self.path in ("decode", "prefix"):
                o = nb.attention_paged_decode(q, kp, vp, table, lens, heads=H, shared_len=self.shared)
            else:
                o = nb.attention_paged(q, kp, vp, table, lens, cu, heads=H, causal=self.causal,
                                       max_new=max(self.new) if "few" in self.path else 0)
        assert npu.device_error() == 0
        want = [attention_exact(a, b, c, 1 / math.sqrt(hd), self.causal) for a, b, c in zip(self.q, self.k, self.v)]
        same(o, torch.cat([w[0] for w in want]), torch.cat([w[1] for w in want]))
        return o


@pytest.mark.parametrize("hd", [16, 64, 96, 128])
@pytest.mark.parametrize("path", PATHS)
def test_infinite_and_nan_scores(cuda_device, path, hd):
    """A key whose score is +inf or NaN makes the rows that see it NaN, and no
    other row: at every place of a group of eight keys, in the first, a middle
    and the last block of a row's keys."""
    for causal in (True, False) if path not in ("decode", "prefix") else (True,):
        c = Call(cuda_device, path, hd, causal)
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
        assert torch.isnan(o).any() == (n > m - c.new[0])
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
