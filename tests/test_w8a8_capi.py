"""The entry points of the products in 8-bit integers (CPU): bad arguments are
refused before any device work, empty work is a no-op."""
import ctypes

from npu_comp_b200 import _lib

P = ctypes.c_void_p(4096)  # never dereferenced: validation fails first
ODD = ctypes.c_void_p(4100)


def quant(lib, x=P, ldx=64, r=None, ldr=0, h=None, ldh=0, g=None, rows=4, cols=64, q=P, ldq=64, s=P):
    return lib.npub_quantize_rows(x, ldx, r, ldr, h, ldh, g, 1e-5, rows, cols, q, ldq, s, None)


def test_quantize_refusals(libnpub_path):
    lib = _lib.load()
    assert quant(lib, rows=0, x=None) == 0
    for kw in (dict(x=None), dict(q=None), dict(s=None), dict(x=ODD), dict(q=ODD), dict(g=ODD), dict(rows=-1), dict(cols=0),
               dict(cols=60), dict(ldx=56), dict(ldx=68), dict(ldq=56), dict(ldq=68), dict(r=P, ldr=64),
               dict(r=P, ldr=56, h=P, ldh=64), dict(r=P, ldr=64, h=P, ldh=60), dict(r=ODD, ldr=64, h=P, ldh=64),
               dict(s=ctypes.c_void_p(4098))):
        assert quant(lib, **kw) == -1, kw


def gemm(lib, a=P, lda=64, sa=P, w=P, ldw=64, sw=P, c=P, ldc=32, r=None, ldr=0, M=4, N=32, K=64, swiglu=0):
    return lib.npub_w8a8_gemm(a, lda, sa, w, ldw, sw, c, ldc, r, ldr, M, N, K, swiglu, None)


def test_gemm_refusals(libnpub_path):
    lib = _lib.load()
    assert gemm(lib, M=0, a=None) == 0 and gemm(lib, N=0, a=None) == 0
    for kw in (dict(a=None), dict(sa=None), dict(w=None), dict(sw=None), dict(c=None), dict(a=ODD), dict(w=ODD),
               dict(lda=56), dict(lda=72), dict(ldw=48), dict(ldw=72), dict(ldc=31), dict(K=0), dict(K=72, lda=80, ldw=80),
               dict(M=-1), dict(N=-1), dict(r=P, ldr=31), dict(swiglu=1, r=P, ldr=32), dict(swiglu=1, N=31),
               dict(swiglu=1, ldc=15), dict(c=ctypes.c_void_p(4097)), dict(sa=ctypes.c_void_p(4098))):
        assert gemm(lib, **kw) == -1, kw
    assert gemm(lib, K=131072, lda=131072, ldw=131072) == -2
