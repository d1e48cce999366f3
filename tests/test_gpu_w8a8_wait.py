"""matmul_w8a8 when a copy never comes: the wait for it runs out (2 s), the error
word says so, what needs the copy is not stored and all else is right, and the
next product finds tensor memory and shared memory free."""
import ctypes
import os
import shutil
import subprocess

import pytest
import torch

import npu_comp_b200 as nb
from npu_comp_b200 import _lib, build, npu

pytestmark = pytest.mark.gpu
HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.fixture(scope="module")
def broken(cuda_device, tmp_path_factory):
    if not (os.path.exists(build.NVCC) or shutil.which(build.NVCC)):
        pytest.skip("no nvcc")
    so = str(tmp_path_factory.mktemp("missing") / "missing_copy.so")
    where = os.path.dirname(_lib.LIB_PATH)
    subprocess.run([build.NVCC, *build.CFLAGS, "-I" + build.CSRC, '-DSOURCE="gemm_w8a8.cu"', "-shared", "-o", so,
                    os.path.join(HERE, "native", "missing_copy.cu"), "-L" + where, "-l:" + os.path.basename(_lib.LIB_PATH),
                    "-Xlinker", "-rpath=" + where, "-Xlinker", "-Bsymbolic", "-lcudart_static", "-ldl", "-lrt", "-lpthread"],
                   check=True)
    lib = ctypes.CDLL(so)
    res, args = _lib.SIGNATURES["npub_w8a8_gemm"]
    lib.npub_w8a8_gemm.restype, lib.npub_w8a8_gemm.argtypes = res, args
    yield lib
    npu.device_error(clear=True)


def product(lib, a, sa, w, sw, out):
    st = lib.npub_w8a8_gemm(a.data_ptr(), a.stride(0), sa.data_ptr(), w.data_ptr(), w.stride(0), sw.data_ptr(), out.data_ptr(),
                            out.stride(0), None, 0, a.shape[0], w.shape[0], a.shape[1], 0,
                            torch.cuda.current_stream().cuda_stream)
    assert st == 0
    torch.cuda.synchronize()


@pytest.mark.parametrize("M,N,K,tokens,cluster", [
    (32, 1024, 4096, 32, True), (64, 12288, 4096, 64, True), (7, 16384, 4096, 32, False), (100, 12288, 8192, 128, True),
    (256, 12288, 4096, 1, False), (2048, 4096, 11008, 2, False),
])
@pytest.mark.parametrize("tile", ["first", "last"])
def test_copy_that_never_comes(broken, M, N, K, tokens, cluster, tile):
    """tokens: of the few-token kernel's tiles, or 1 and 2: the tile kernel with 128 and 256."""
    assert broken.w8a8_kernel_of(M, N, K) == tokens and (broken.w8a8_cluster_of(M, N, K) > 1) == cluster
    g = torch.Generator(device="cuda").manual_seed(M + N)
    r = lambda *s: torch.randint(-127, 128, s, generator=g, device="cuda", dtype=torch.int8)  # noqa: E731
    a, w = r(M, K), r(N, K)
    sa, sw = torch.rand(M, device="cuda", generator=g) / 100, (torch.rand(N, device="cuda", generator=g) / 100).half()
    want = nb.matmul_w8a8(a, sa, w, sw)
    out = torch.full_like(want, 3.0)
    assert npu.device_error(clear=True) == 0
    product(broken, a, sa, w, sw, out)
    assert torch.equal(out, want)
    width = 128 if tokens > 2 else 256
    n0 = 3 * 256  # (no tile of tokens starts at this row, but for the largest: its tokens' box is missing as well)
    k0 = 0 if tile == "first" else (K - 1) // 128 * 128
    assert broken.leave_out(k0, n0, 0) == 0
    out.fill_(3.0)
    product(broken, a, sa, w, sw, out)
    assert broken.leave_out(-1, -1, -1) == 0
    assert npu.device_error(clear=True) in (0x701, 0x702, 0x703, 0x704, 0x711, 0x712, 0x713)
    skipped = torch.zeros_like(out, dtype=torch.bool)
    skipped[:, n0:n0 + width] = True
    if M > n0:
        skipped[n0:n0 + 256] = True
    assert (out[skipped] == 3.0).all()
    assert torch.equal(out[~skipped], want[~skipped])
    for _ in range(20):  # every SM again
        product(broken, a, sa, w, sw, out)
        assert torch.equal(out, want)
        assert torch.equal(nb.matmul_w8a8(a, sa, w, sw), want)
    assert npu.device_error() == 0
