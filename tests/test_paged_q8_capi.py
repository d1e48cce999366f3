"""The 8-bit paged cache's entry points (CPU): bad arguments are refused before
any device work, empty work is a no-op, workspace queries hold."""
import ctypes

from npu_comp_b200 import _lib

P = ctypes.c_void_p(4096)  # never dereferenced: validation fails first
ODD = ctypes.c_void_p(4104)
BYTE = ctypes.c_void_p(4097)


def append(lib, qkv=P, ldx=1024, q=P, ldq=512, tokens=4, hq=4, hk=2, hd=128, rot=128, pos=P, f=P, gq=None, kp=P, vp=P, ks=P,
           vs=P, n_pages=8, ps=16, table=P, ldt=4, width=4, cu=None, batch=4, ws=None, wsb=0):
    return lib.npub_rope_paged_append_q8(qkv, ldx, q, ldq, tokens, hq, hk, hd, rot, 0, pos, f, gq, None, 1e-5, kp, vp, ks, vs,
                                         n_pages, ps, table, ldt, width, cu, batch, ws, wsb, None)


def test_append_refusals(libnpub_path):
    lib = _lib.load()
    assert append(lib, tokens=0, qkv=None, batch=0) == 0
    for kw in (dict(qkv=None), dict(q=None), dict(pos=None), dict(f=None), dict(kp=None), dict(vp=None), dict(ks=None),
               dict(vs=None), dict(table=None), dict(qkv=ODD), dict(q=ODD), dict(gq=ODD), dict(kp=ODD), dict(vp=ODD),
               dict(ks=BYTE), dict(vs=BYTE), dict(ldx=1023), dict(ldx=1016), dict(ldq=504), dict(hd=120), dict(hd=0),
               dict(rot=0), dict(rot=8), dict(rot=144), dict(hq=0), dict(hk=0), dict(tokens=-1), dict(n_pages=0), dict(ps=8),
               dict(ps=24), dict(ps=512), dict(width=0), dict(ldt=3), dict(batch=3), dict(batch=0, cu=P)):
        assert append(lib, **kw) == -1, kw
    assert append(lib, hd=144, rot=16, ldx=2048, ldq=1024) == -2
    n = lib.npub_rope_paged_append_q8_workspace(4, 128, 1)
    assert n == 4 * 64 * 8 and lib.npub_rope_paged_append_q8_workspace(4, 128, 0) == 0
    assert append(lib, cu=P, batch=2) == -4 and append(lib, cu=P, batch=2, ws=P, wsb=n - 1) == -4
    assert append(lib, cu=P, batch=2, ws=ODD, wsb=n) == -1


def paged(lib, q=P, ldq=512, kp=P, ks=P, vs=P, n_pages=8, ps=16, table=P, ldt=4, width=4, lens=P, cu=P, batch=2, total=8,
          max_new=0, ctx=0, out=P, ldo=512, h=4, kv=2, hd=128, scale=0.1, ws=None, wsb=0):
    return lib.npub_attention_paged_q8(q, ldq, kp, P, ks, vs, n_pages, ps, table, ldt, width, lens, cu, batch, total, max_new,
                                       ctx, out, ldo, h, kv, hd, scale, 1, ws, wsb, None)


def decode(lib, q=P, ldq=512, kp=P, ks=P, vs=P, n_pages=8, ps=16, table=P, ldt=400, width=400, lens=P, batch=2, ctx=0, out=P,
           ldo=512, h=4, kv=2, hd=128, scale=0.1, ws=None, wsb=0):
    return lib.npub_attention_paged_decode_q8(q, ldq, kp, P, ks, vs, n_pages, ps, table, ldt, width, lens, batch, ctx, out,
                                              ldo, h, kv, hd, scale, ws, wsb, None)


def test_attention_refusals(libnpub_path):
    lib = _lib.load()
    assert paged(lib, total=0, q=None) == 0 and paged(lib, batch=0, q=None) == 0 and decode(lib, batch=0, q=None) == 0
    for kw in (dict(q=None), dict(kp=None), dict(ks=None), dict(vs=None), dict(table=None), dict(lens=None), dict(out=None),
               dict(q=ODD), dict(kp=ODD), dict(out=ODD), dict(ks=BYTE), dict(vs=BYTE), dict(ldq=504), dict(ldo=500),
               dict(n_pages=0), dict(ps=8), dict(ps=48), dict(ps=512), dict(width=0), dict(ldt=3), dict(h=3), dict(hd=8),
               dict(scale=-1.0), dict(scale=0.0), dict(ctx=-1), dict(batch=-1)):
        assert paged(lib, **kw) == -1, kw
        assert decode(lib, **kw) == -1, kw
    assert paged(lib, cu=None) == -1 and paged(lib, max_new=-1) == -1
    assert decode(lib, hd=256, ldq=1024, ldo=1024) == -2 and decode(lib, batch=65536) == -2
    # more rows than the few-row kernel takes need the workspace, aligned
    n = lib.npub_attention_paged_q8_workspace(2, 8, 0, 64, 4, 2, 128)
    assert paged(lib) == -4 and paged(lib, ws=P, wsb=n - 1) == -4 and paged(lib, ws=ODD, wsb=n) == -1


def test_workspace_queries(libnpub_path):
    lib = _lib.load()
    d, p = lib.npub_attention_paged_decode_q8_workspace, lib.npub_attention_paged_q8_workspace
    assert d(0, 100, 4, 2, 128) == 0 and d(4, 100, 4, 3, 128) == 0 and d(1, 64, 4, 2, 128) == 0
    # fp16 K and V of batch * ctx keys, in pages of 128
    n = p(3, 300, 100, 1000, 8, 2, 128)
    keys = 3 * 1024 * 2 * 128 * 2 * 2
    assert n >= keys + 3 * 9 * 4
    assert p(3, 300, 32, 1000, 8, 2, 128) != p(3, 300, 33, 1000, 8, 2, 128)  # at most 128 rows of a kv head: read as they are
    assert d(3, 1000, 128, 1, 128) < p(3, 3, 0, 1000, 128, 1, 128)
    assert p(0, 8, 0, 100, 4, 2, 128) == 0
