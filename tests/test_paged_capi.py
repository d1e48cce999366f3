"""The paged-cache entry points of the C ABI (CPU): bad arguments are refused
before any device work, empty work is a no-op, workspace queries hold."""
import ctypes

from npu_comp_b200 import _lib

P = ctypes.c_void_p(4096)  # never dereferenced: validation fails first
ODD = ctypes.c_void_p(4104)


def append(lib, qkv=P, ldx=1024, q=P, ldq=512, tokens=4, hq=4, hk=2, hd=128, rot=128, pos=P, f=P, gq=None, kp=P,
           n_pages=8, ps=16, table=P, ldt=4, width=4, cu=None, batch=4):
    return lib.npub_rope_paged_append(qkv, ldx, q, ldq, tokens, hq, hk, hd, rot, 0, pos, f, gq, None, 1e-5, kp, P,
                                      n_pages, ps, table, ldt, width, cu, batch, None)


def test_append_refusals(libnpub_path):
    lib = _lib.load()
    assert append(lib, tokens=0, qkv=None, batch=0) == 0
    for kw in (dict(qkv=None), dict(q=None), dict(pos=None), dict(f=None), dict(kp=None), dict(table=None),
               dict(qkv=ODD), dict(q=ODD), dict(gq=ODD), dict(kp=ODD), dict(ldx=1023), dict(ldx=1016), dict(ldq=504),
               dict(hd=120), dict(hd=0), dict(hd=528, rot=16), dict(rot=0), dict(rot=8), dict(rot=144), dict(hq=0),
               dict(hk=0), dict(tokens=-1), dict(n_pages=0), dict(ps=0), dict(ps=24), dict(width=0), dict(ldt=3),
               dict(batch=3), dict(batch=0, cu=P)):
        assert append(lib, **kw) == -1, kw


def packed(lib, q=P, ldq=512, k=P, ldk=256, v=P, ldv=256, out=P, ldo=512, cu=P, batch=2, total=8, h=4, kv=2,
           hd=128, scale=0.1):
    return lib.npub_attention_packed(q, ldq, k, ldk, v, ldv, out, ldo, cu, batch, total, h, kv, hd, scale, 1,
                                     None)


def test_packed_refusals(libnpub_path):
    lib = _lib.load()
    assert packed(lib, total=0, q=None) == 0 and packed(lib, batch=0, q=None) == 0
    for kw in (dict(q=None), dict(k=None), dict(v=None), dict(out=None), dict(cu=None), dict(q=ODD), dict(k=ODD),
               dict(v=ODD), dict(out=ODD), dict(ldq=504), dict(ldk=248), dict(ldv=260), dict(ldo=511), dict(h=3),
               dict(kv=0), dict(hd=0), dict(hd=100), dict(scale=0.0), dict(scale=float("inf")),
               dict(scale=float("nan")), dict(total=-1), dict(batch=-1)):
        assert packed(lib, **kw) == -1, kw
    assert packed(lib, hd=144, ldq=1024, ldk=512, ldv=512, ldo=1024) == -2
    assert packed(lib, h=256, kv=1, hd=16, ldq=4096, ldo=4096) == -2


def paged(lib, q=P, ldq=512, kp=P, n_pages=8, ps=16, table=P, ldt=4, width=4, lens=P, cu=P, batch=2, total=8,
          max_new=0, ctx=0, out=P, ldo=512, h=4, kv=2, hd=128, scale=0.1, ws=None, wsb=0):
    return lib.npub_attention_paged(q, ldq, kp, P, n_pages, ps, table, ldt, width, lens, cu, batch, total, max_new,
                                    ctx, out, ldo, h, kv, hd, scale, 1, ws, wsb, None)


def decode(lib, q=P, ldq=512, kp=P, n_pages=8, ps=16, table=P, ldt=400, width=400, lens=P, batch=2, ctx=0, shared=0,
           out=P, ldo=512, h=4, kv=2, hd=128, scale=0.1, ws=None, wsb=0):
    return lib.npub_attention_paged_decode(q, ldq, kp, P, n_pages, ps, table, ldt, width, lens, batch, ctx, shared,
                                           out, ldo, h, kv, hd, scale, ws, wsb, None)


def test_paged_refusals(libnpub_path):
    lib = _lib.load()
    assert paged(lib, total=0, q=None) == 0 and paged(lib, batch=0, q=None) == 0 and decode(lib, batch=0, q=None) == 0
    both = (dict(q=None), dict(kp=None), dict(table=None), dict(lens=None), dict(out=None), dict(q=ODD), dict(kp=ODD),
            dict(out=ODD), dict(ldq=504), dict(ldo=500), dict(n_pages=0), dict(ps=8), dict(ps=48), dict(ps=512),
            dict(width=0), dict(ldt=3), dict(h=3), dict(hd=8), dict(scale=-1.0), dict(ctx=-1), dict(batch=-1))
    for kw in both:
        assert paged(lib, **kw) == -1, kw
        assert decode(lib, **kw) == -1, kw
    assert paged(lib, cu=None) == -1 and paged(lib, max_new=-1) == -1
    assert decode(lib, shared=8) == -1 and decode(lib, shared=6416) == -1 and decode(lib, shared=-16) == -1
    assert decode(lib, hd=256, ldq=1024, ldo=1024) == -2 and decode(lib, batch=65536) == -2
    # a call that is split needs its workspace, aligned
    n = lib.npub_attention_paged_decode_workspace(2, 6400, 0, 4, 2, 128)
    assert n > 0
    assert decode(lib) == -4 and decode(lib, ws=P, wsb=n - 1) == -4 and decode(lib, ws=ODD, wsb=n) == -1


def test_workspace_queries(libnpub_path):
    lib = _lib.load()
    d, p = lib.npub_attention_paged_decode_workspace, lib.npub_attention_paged_workspace
    assert d(0, 100, 0, 4, 2, 128) == 0 and d(4, 100, 0, 4, 3, 128) == 0 and d(1, 64, 0, 4, 2, 128) == 0
    assert d(1, 8192, 4096, 4, 2, 128) == d(1, 8192, 0, 4, 2, 128)  # nothing to share in a batch of one
    assert d(8, 8192, 4096, 4, 2, 128) > 0
    assert p(0, 8, 0, 100, 4, 2, 128) == 0 and p(2, 8, 0, 64, 4, 2, 128) == 0
    assert p(2, 100000, 0, 100000, 32, 8, 128) == 0  # enough tiles: no split
    # partials are (2 + head_dim) floats per row, head and split
    n = p(1, 4, 4, 65536, 4, 2, 128)
    assert n > 0 and n % (4 * 4 * 130 * 4) < 256
