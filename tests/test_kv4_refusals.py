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


def _attend(**kw):
    from mlx_dspark import _hip
    a = dict(q=P, B=1, W=1, nq=4, nkv=2, hd=128, scale=0.1, causal=1, window=0, sinks=0, cap=0.0, terms=3, sl=P, max_ctx=100,
             table=P, max_pages=2, page=64, kv=2, k=P, v=P, ks=P, vs=P, out=P, packed=0, ws=None, wsb=0, st=None)
    a.update(kw)
    return _hip.lib.dsk_attention_sinks(*a.values()), _hip.lib.dsk_last_error().decode()


@pytest.mark.parametrize("kw,word", [
    (dict(q=None), "null"), (dict(hd=512), "head_dim"), (dict(nq=3), "shape"), (dict(W=0), "shape"),
    (dict(scale=0.0), "scale"), (dict(scale=float("nan")), "scale"), (dict(cap=-1.0), "softcap"), (dict(window=-1), "window"),
    (dict(sinks=-1), "sinks"), (dict(kv=3), "kv_dtype"), (dict(ks=None), "scale/bias"), (dict(kv=0, page=48), "multiples of 32"),
    (dict(page=16), "multiples of 32"), (dict(max_ctx=129), "max_ctx"), (dict(W=2, max_ctx=1), "max_ctx"),
    (dict(out=ctypes.c_void_p((1 << 20) + 8)), "aligned"), (dict(W=65, packed=1), "packed"),
    (dict(max_pages=1 << 24), "block table"), (dict(terms=2), "terms"), (dict(terms=1, W=90), "terms"),
])
def test_attention_refuses(kw, word):
    rc, msg = _attend(**kw)
    assert rc == -1 and word in msg, msg


def test_attention_workspace_too_small():
    from mlx_dspark import _hip

    need = _hip.lib.dsk_attention_sinks_ws_bytes(1, 1, 4, 2, 128, 1, 0, 0, 4096)
    assert need > 0
    for ws, n in ((None, 0), (P, need - 1)):
        rc, msg = _attend(max_ctx=4096, max_pages=64, ws=ws, wsb=n)
        assert rc == -4 and "workspace" in msg
    assert _hip.lib.dsk_attention_sinks_ws_bytes(1, 1, 4, 2, 64, 1, 0, 0, 4096) == 0


def test_python_refusals():
    """Host tensors, strided pools and lists of the wrong type, before anything is launched."""
    import torch
    from mlx_dspark import ops

    table, lens = torch.zeros((1, 2), dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    pool, sb = torch.zeros((2, 2, 64, 64), dtype=torch.uint8), torch.zeros((2, 2, 64, 2), dtype=torch.int32)
    q = torch.zeros((1, 512), dtype=torch.bfloat16)
    att = lambda **kw: ops.attention(q, 1, 1, 4, 2, 128, 0.1, lens, 64, table, 64, ops.DSK_KV_U4, pool, pool, sb, sb, **kw)
    for call in (att, lambda: ops.kv_read(lens, 3, 2, 128, table, 64, ops.DSK_KV_U4, pool, pool, sb, sb),
                 lambda: ops.qkv_rope_append(torch.zeros((1, 1024), dtype=torch.bfloat16), 1, 1, 4, 2, 128, None, None, 1e-6,
                                             torch.zeros(64), lens, table, 64, ops.DSK_KV_U4, pool, pool, sb, sb)):
        with pytest.raises(ValueError, match="device tensors"):
            call()
    with pytest.raises(ValueError, match="contiguous"):
        ops.kv_read(lens, 3, 2, 128, table, 64, ops.DSK_KV_U4, pool[:, :, ::2], pool, sb, sb)
    with pytest.raises(ValueError, match="int32"):
        ops.kv_read(lens.long(), 3, 2, 128, table, 64, ops.DSK_KV_U4, pool, pool, sb, sb)
    k, v = ops.kv_read(lens, 0, 2, 128, table, 64, ops.DSK_KV_U4, pool, pool, sb, sb)   # nothing to read
    assert k.shape == v.shape == (1, 0, 2, 128)
