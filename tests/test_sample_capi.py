"""npub_sample's argument checks (CPU): bad arguments are refused before any
device work, no rows are a no-op."""
import ctypes

from npu_comp_b200 import _lib

P = ctypes.c_void_p(4096)  # never dereferenced: validation fails first
ODD = ctypes.c_void_p(4097)


def sample(lib, x=P, ld=100, rows=2, vocab=100, u=P, t=None, k=None, p=None, m=None, ids=P):
    return lib.npub_sample(x, ld, rows, vocab, u, t, 1.0, k, 0, p, 1.0, m, 0.0, ids, None)


def test_refusals(libnpub_path):
    lib = _lib.load()
    assert sample(lib, rows=0, x=None) == 0
    for kw in (dict(x=None), dict(u=None), dict(ids=None), dict(ld=99), dict(rows=-1), dict(vocab=0), dict(vocab=-5), dict(x=ODD),
               dict(u=ODD), dict(t=ODD), dict(k=ODD), dict(p=ODD), dict(m=ODD), dict(ids=ODD)):
        assert sample(lib, **kw) == -1, kw
    assert sample(lib, vocab=524225, ld=600000) == -2
