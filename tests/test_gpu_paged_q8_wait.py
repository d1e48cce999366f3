"""Few rows over 8-bit pages when a page's copy never comes: the wait for it
runs out (2 s), the error word says so, the sequences that need no key of the
part are right, and so is the next call."""
import ctypes
import math
import os
import shutil
import subprocess

import pytest
import torch

import npu_comp_b200 as nb
from npu_comp_b200 import _lib, build, npu
from test_gpu_paged_q8 import Cache

pytestmark = pytest.mark.gpu
HERE = os.path.dirname(os.path.abspath(__file__))
NAME = "npub_attention_paged_decode_q8"


@pytest.fixture(scope="module")
def broken(cuda_device, tmp_path_factory):
    if not (os.path.exists(build.NVCC) or shutil.which(build.NVCC)):
        pytest.skip("no nvcc")
    so = str(tmp_path_factory.mktemp("missing") / "missing_page.so")
    where = os.path.dirname(_lib.LIB_PATH)
    subprocess.run([build.NVCC, *build.CFLAGS, "-I" + build.CSRC, "-shared", "-o", so,
                    os.path.join(HERE, "native", "missing_page.cu"), "-L" + where, "-l:" + os.path.basename(_lib.LIB_PATH),
                    "-Xlinker", "-rpath=" + where, "-Xlinker", "-Bsymbolic", "-lcudart_static", "-ldl", "-lrt", "-lpthread"],
                   check=True)
    lib = ctypes.CDLL(so)
    for name in (NAME, NAME + "_workspace"):
        f = getattr(lib, name)
        f.restype, f.argtypes = _lib.SIGNATURES[name]
    yield lib
    npu.device_error(clear=True)


def decode(lib, c, q, H, out, ctx, ws):
    n_pages, KV, ps, hd = c.kp.shape
    st = getattr(lib, NAME)(q.data_ptr(), q.stride(0), c.kp.data_ptr(), c.vp.data_ptr(), c.ks.data_ptr(), c.vs.data_ptr(), n_pages,
                            ps, c.table.data_ptr(), c.table.stride(0), c.table.shape[1], c.lens.data_ptr(), len(c.keys), ctx,
                            out.data_ptr(), out.stride(0), H, KV, hd, 1 / math.sqrt(hd), ws.data_ptr() if ws is not None else None,
                            ws.numel() if ws is not None else 0, torch.cuda.current_stream().cuda_stream)
    assert st == 0
    torch.cuda.synchronize()


def check(lib, keys, H, KV, hd, ps, missing, codes, whole):
    """missing: (sequence, key, kv head) of the page piece; whole: the rows that need none of the part that waits for it."""
    c = Cache(keys, KV, hd, ps, seed=sum(keys))
    B, ctx = len(keys), c.table.shape[1] * ps
    q = torch.randn((B, H * hd), generator=torch.Generator().manual_seed(1)).half().cuda()
    want = nb.attention_paged_decode_q8(q, *c.args, c.lens, heads=H)
    n = getattr(lib, NAME + "_workspace")(B, ctx, H, KV, hd)
    # its first contents would be far outside of it, taken as places
    ws = torch.full((n,), 0x7f, dtype=torch.uint8, device="cuda") if n else None
    out = torch.full_like(want, 3.0)
    assert npu.device_error(clear=True) == 0
    decode(lib, c, q, H, out, ctx, ws)
    assert torch.equal(out, want)
    b, key, head = missing
    if ws is not None:
        ws.fill_(0x7f)
    out.fill_(3.0)
    assert lib.leave_out(0, head, int(c.table[b, key // ps])) == 0
    decode(lib, c, q, H, out, ctx, ws)
    assert lib.leave_out(-1, -1, -1) == 0
    assert npu.device_error(clear=True) in codes
    got, ok = out.clone().view(B, KV, -1), want.view(B, KV, -1)
    for i in range(B):
        for h in range(KV):
            if whole(i, h):
                assert torch.equal(got[i, h], ok[i, h]), (i, h)
    for _ in range(10):
        decode(lib, c, q, H, out, ctx, ws)
        assert torch.equal(out, want)
        assert torch.equal(nb.attention_paged_decode_q8(q, *c.args, c.lens, heads=H), want)
    assert npu.device_error() == 0
    return got


@pytest.mark.parametrize("H,KV", [(32, 8), (16, 1)])
@pytest.mark.parametrize("seqs,keys", [(1, 16384), (70, 3000)])
def test_list(broken, seqs, keys, H, KV):
    """The warp with the last step of an item, and the first ones of the next: that one's places are never written, and the
    combination does not follow what stands there."""
    ks = [keys + 40 * b for b in range(seqs)]
    b, h = seqs // 2, KV // 2
    assert getattr(broken, NAME + "_workspace")(seqs, ks[-1], H, KV, 128) > 0
    at = b * KV + h  # a warp's part is shorter than an item: of this one and the next
    got = check(broken, ks, H, KV, 128, 16, (b, ks[b] - 1, h), (0x731,), lambda i, j: i * KV + j not in (at, at + 1))
    if (seqs, KV) == (70, 8):
        nan = torch.isnan(got[(at + 1) // KV, (at + 1) % KV])
        assert bool(nan.all())


@pytest.mark.parametrize("H,KV,hd", [(32, 8, 128), (16, 1, 64), (4, 4, 64)])
@pytest.mark.parametrize("keys,key", [([100, 90], 16), ([700, 5000, 900], 4999), ([2000], 0)])
def test_ranges(broken, keys, key, H, KV, hd):
    """One CTA for an item, or a cluster: all its rows are NaN, whichever range waited in vain."""
    assert getattr(broken, NAME + "_workspace")(len(keys), max(keys), H, KV, hd) == 0
    b, h = len(keys) // 2, KV - 1
    got = check(broken, keys, H, KV, hd, 32, (b, key, h), (0x721, 0x722), lambda i, j: (i, j) != (b, h))
    assert torch.isnan(got[b, h]).all()
