"""Long 8-bit paged contexts, whose attention keeps partial results in a
workspace, on several streams and in several graphs at once: every call has the
bits that it has alone."""
import pytest
import torch

import npu_comp_b200 as nb
from npu_comp_b200 import _lib, npu
from test_gpu_paged_q8 import Cache, offsets

pytestmark = pytest.mark.gpu
H, KV, HD, PS = 32, 8, 128, 32


class Work:
    """A decode step and a few drafted rows over one cache, both by the list kernel."""

    def __init__(self, keys, new, seed):
        g = torch.Generator().manual_seed(seed)
        self.c, self.new, self.cu = Cache(keys, KV, HD, PS, seed=seed), new, offsets(new)
        self.q = torch.randn((len(keys), H * HD), generator=g).half().cuda()
        self.qm = torch.randn((sum(new), H * HD), generator=g).half().cuda()
        width = self.c.table.shape[1] * PS
        assert _lib.query("npub_attention_paged_decode_q8_workspace", len(keys), width, H, KV, HD) > 0
        assert _lib.query("npub_attention_paged_q8_workspace", len(keys), sum(new), max(new), width, H, KV, HD) > 0

    def __call__(self):
        return (nb.attention_paged_decode_q8(self.q, *self.c.args, self.c.lens, heads=H),
                nb.attention_paged_q8(self.qm, *self.c.args, self.c.lens, self.cu, heads=H, max_new=max(self.new)))


def works():
    return [Work([40000], [8], 1), Work([9000 + 50 * b for b in range(20)], [1 + b % 5 for b in range(20)], 2),
            Work([3000, 0, 60000, 5, 17000], [4, 2, 0, 1, 6], 3)]


def same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


def test_calls_on_several_streams(cuda_device):
    ws = works()
    want = [w() for w in ws]
    streams = [torch.cuda.Stream() for _ in ws]
    torch.cuda.synchronize()
    got = []
    for _ in range(10):
        for w, st in zip(ws, streams):
            with torch.cuda.stream(st):
                got.append(w())
    torch.cuda.synchronize()
    assert npu.device_error() == 0
    assert all(same(want[i % len(ws)], g) for i, g in enumerate(got))


def test_graphs_beside_graphs_and_calls(cuda_device):
    ws = works()
    for w in ws:
        w()
    graphs = []
    for w in ws[:2]:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = w()
        graphs.append((gr, out, torch.cuda.Stream()))
    third = torch.cuda.Stream()
    for turn in range(10):
        # other inputs for the same graphs: shorter contexts, other rows
        for w in ws:
            w.c.lens.mul_(9).div_(10, rounding_mode="floor")
            w.q.neg_()
            w.qm.mul_(0.9)
        want = [w() for w in ws]
        torch.cuda.synchronize()
        for _, out, _ in graphs:
            for t in out:
                t.fill_(9.0)
        torch.cuda.synchronize()
        for gr, _, st in graphs:
            with torch.cuda.stream(st):
                gr.replay()
        with torch.cuda.stream(third):
            got = ws[2]()
        torch.cuda.synchronize()
        assert npu.device_error() == 0
        assert same(got, want[2]), turn
        for (_, out, _), w in zip(graphs, want):
            assert same(out, w), turn
