"""Many rows over 8-bit pages whose sequences take turns in the fp16 copy: a
page table far wider than what the sequences hold, 537 MB of copy for each of
its 131072-key rows of 8 heads, and rows, sequences without rows and without
keys as in one piece (bounds of test_gpu_paged_q8)."""
import math

import pytest
import torch

import npu_comp_b200 as nb
from npu_comp_b200 import npu
from paged_exact import same
from test_gpu_paged_q8 import Cache, expected, i32, offsets

pytestmark = pytest.mark.gpu
H, KV, HD, PS, WIDTH = 16, 8, 128, 64, 131072


def wide(keys, seed):
    c = Cache(keys, KV, HD, PS, seed=seed)
    t = torch.full((len(keys), WIDTH // PS + 8), 1 << 30, dtype=torch.int32, device="cuda")
    t[:, :c.table.shape[1]] = c.table
    c.table = t[:, :WIDTH // PS]
    c.args = (*c.args[:4], c.table)
    return c


def call(c, q, cu, **kw):
    return nb.attention_paged_q8(q, *c.args, c.lens, cu, heads=H, **kw)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("new,keys", [
    ([100, 0, 1, 300, 7, 64, 65, 2], [100, 50, 400, 513, 0, 5000, 64, 1]),  # three groups
    ([2, 1, 3, 1, 1], [20000, 1, 70000, 0, 300]),                           # two, keys in parts
    ([5] * 13, [17 * i for i in range(13)]),
])
def test_groups(cuda_device, new, keys, causal):
    c = wide(keys, sum(keys))
    T, first = sum(new), 3  # rows ahead of the first sequence and behind the last stay as they are
    q = torch.randn((first + T + 2, H * HD), generator=torch.Generator().manual_seed(T)).half().cuda()
    q[:first] = q[first + T:] = float("nan")
    out = torch.full((first + T + 2, H * HD), 3.0, dtype=torch.float16, device="cuda")
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    held = torch.cuda.memory_allocated()
    call(c, q, offsets(new) + first, causal=causal, out=out)
    assert npu.device_error() == 0
    assert torch.cuda.max_memory_allocated() - held < 2.1 * 2 ** 30
    assert (out[:first] == 3.0).all() and (out[first + T:] == 3.0).all()
    at = first
    for b, n in enumerate(new):
        if n:
            want, bound = expected(c, b, q[at:at + n].view(n, H, HD), 1 / math.sqrt(HD), causal)
            same(out[at:at + n], want, bound)
        at += n


def test_groups_in_graphs_on_two_streams(cuda_device):
    """Calls and replays of two graphs at once, every group in the workspace of its own call."""
    new, keys = [40, 3, 0, 90, 17, 33], [4000, 300, 20, 9000, 17, 6000]
    cs = [wide(keys, s) for s in (1, 2)]
    g = torch.Generator().manual_seed(3)
    qs = [torch.randn((sum(new), H * HD), generator=g).half().cuda() for _ in cs]
    cu = offsets(new)
    want = [call(c, q, cu) for c, q in zip(cs, qs)]
    graphs, held = [], []
    for c, q in zip(cs, qs):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            held.append(call(c, q, cu))
        graphs.append((gr, torch.cuda.Stream()))
    for _ in range(5):
        for gr, st in graphs:
            with torch.cuda.stream(st):
                gr.replay()
        again = call(cs[0], qs[0], cu)
        torch.cuda.synchronize()
        assert torch.equal(again, want[0]) and all(torch.equal(a, b) for a, b in zip(held, want))
