"""The 4-bit cache's and read-back's argument checks (they run on the host, before any launch)."""

import ctypes

import pytest

P = ctypes.c_void_p(1 << 20)     # an address no check reads through


def _read(**kw):
    from mlx_dspark import _hip
    a = dict(first=P, offset=0, B=1, n=4, nkv=2, hd=128, table=P, max_pages=2, page=64, kv=2, k=P, v=P, ks=P, vs=P, ko=P,
             vo=P, st=None)
    a.update(kw)
    return _hip.lib.dsk_kv_read(*a.values()), _hip.lib.dsk_last_error().decode()


@pytest.mark.parametrize("kw,word", [
    (dict(first=None), "null"), (dict(vo=None), "null"), (dict(kv=3), "kv_dtype"), (dict(hd=64), "head_dim"),
    (dict(hd=512), "head_dim"), (dict(n=0), "shape"), (dict(B=0), "shape"), (dict(page=48), "multiples of 32"),
    (dict(page=0), "page"), (dict(ks=None), "scale"), (dict(ko=ctypes.c_void_p((1 << 20) + 8)), "aligned"),
])
def test_read_refuses(kw, word):
    rc, msg = _read(**kw)
    assert rc == -1 and word in msg, msg


def _append(**kw):
    from mlx_dspark import _hip
    a = dict(qkv=P, splits=0, B=1, W=1, nq=4, nkv=2, hd=128, qn=P, kn=P, eps=1e-6, inv=P, sl=P, off=0, table=P,
             max_pages=2, page=64, kv=2, k=P, v=P, ks=P, vs=P, q=P, st=None)
    a.update(kw)
    return _hip.lib.dsk_qkv_rope_append(*a.values()), _hip.lib.dsk_last_error().decode()


@pytest.mark.parametrize("kw,word", [
    (dict(hd=512), "head_dim"), (dict(page=16), "multiple of 32"), (dict(vs=None), "scale"),
    (dict(kn=ctypes.c_void_p((1 << 20) + 2)), "aligned"), (dict(kv=3), "scale"), (dict(W=0), "shape"),
])
def test_append_refuses(kw, word):
    rc, msg = _append(**kw)
    assert rc == -1 and word in msg, msg


def test_cache_refuses():
    from mlx_dspark.kv import PagedKVCache

    for kw in (dict(kv_bits=5), dict(kv_bits=4, page=16), dict(kv_bits=4, page=48)):
        with pytest.raises(ValueError):
            PagedKVCache(1, 1, 2, 128, 64, device="cpu", **kw)
    with pytest.raises(ValueError):
        PagedKVCache(1, 1, 2, 512, 64, device="cpu", kv_bits=4)
