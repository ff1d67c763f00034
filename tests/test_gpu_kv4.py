"""GPU parity of the 4-bit KV cache's write (q/k RMSNorm + RoPE + quantise) and of the read-back of every
cache type, against 64-bit references."""

import pytest
import torch

from _kv4 import decode, fill, quantise, words

pytestmark = pytest.mark.gpu

BF = 2.0 ** -8      # a bf16 rounding, relative
EPS = 1e-6


def _make(B, nkv, hd, max_pages, page, dev, seed, spare=3):
    g = torch.Generator().manual_seed(seed)
    n = B * max_pages + spare
    table = torch.randperm(n, generator=g)[:B * max_pages].view(B, max_pages).to(torch.int32)
    pool = lambda: torch.randint(0, 256, (n, nkv, page, hd // 2), generator=g, dtype=torch.uint8)
    sb = lambda: torch.full((n, nkv, page, hd // 64), 0x3F803F80, dtype=torch.int32)
    return table.to(dev), [t.to(dev) for t in (pool(), pool(), sb(), sb())]


def _rope64(x, pos, inv):
    h = x.shape[-1] // 2
    a = (pos.double()[:, None] * inv.double())[:, None]
    return torch.cat((x[..., :h] * a.cos() - x[..., h:] * a.sin(), x[..., h:] * a.cos() + x[..., :h] * a.sin()), -1)


def _norm64(x, w):
    return x / (x.square().mean(-1, keepdim=True) + EPS).sqrt() * w.double()


@pytest.mark.parametrize("nq,nkv,hd,page,B,W,lens,splits,opt", [
    (4, 2, 128, 64, 1, 1, [0], 0, ""), (16, 8, 128, 64, 1, 1, [311], 2, ""), (32, 8, 128, 64, 4, 9, [5, 60, 127, 333], 2, ""),
    (4, 2, 256, 32, 2, 7, [31, 90], 1, ""), (16, 8, 256, 128, 1, 33, [100], 0, ""), (4, 1, 128, 96, 3, 5, [0, 94, 190], 3, "rn"),
    (16, 8, 128, 64, 1, 300, [45], 0, ""), (4, 2, 256, 64, 1, 270, [3], 0, "vnorm"), (0, 2, 128, 64, 2, 6, [10, 20], 0, "offset"),
    (5, 5, 128, 32, 2, 3, [29, 31], 2, "nonorm"),
])
def test_append(dev, nq, nkv, hd, page, B, W, lens, splits, opt):
    from mlx_dspark import ops

    print(f"kv4 append {nq} {nkv} {hd} page={page} B={B} W={W} {lens} splits={splits} {opt}", flush=True)
    g = torch.Generator().manual_seed(nq * 7 + W)
    off = 3 if opt == "offset" else 0
    max_pages = -(-(max(lens) + W + off) // page) + 1
    table, (kp, vp, ks, vs) = _make(B, nkv, hd, max_pages, page, dev, W)
    before = [t.clone() for t in (kp, vp, ks, vs)]
    cols, M = (nq + 2 * nkv) * hd, B * W
    x = torch.randn((max(splits, 1), M, cols), generator=g)
    if not splits:
        x = x[0].to(torch.bfloat16)
    qn, kn, vn = ((1 + 0.2 * torch.randn(hd, generator=g)).to(torch.bfloat16) for _ in range(3))
    if opt == "nonorm":
        qn = kn = None
    vn = vn if opt == "vnorm" else None
    inv = ops.rope_inv_freq(hd, 1e6, "cpu")
    pk, scale = None, 1.0
    if opt == "rn":
        pk = ops.Packed.empty(M, 320, dev, normed_later=True, eps=1e-5)
        pk.ssq.copy_(torch.rand((M, 20), generator=g) * 40)
        scale = (pk.ssq.cpu().double().sum(1) / 320 + 1e-5).rsqrt()[:, None]
    sl = torch.tensor(lens, dtype=torch.int32, device=dev)
    to = lambda t: None if t is None else t.to(dev)
    q = ops.qkv_rope_append(x.to(dev), B, W, nq, nkv, hd, to(qn), to(kn), EPS, inv.to(dev), sl, table, page,
                            ops.DSK_KV_U4, kp, vp, ks, vs, pos_offset=off, v_norm=to(vn), x=pk)
    k_out, v_out = ops.kv_read(sl, W, nkv, hd, table, page, ops.DSK_KV_U4, kp, vp, ks, vs, offset=off)
    torch.cuda.synchronize()

    r = (x.double().sum(0) if splits else x.double()) * scale
    r = r.view(B, W, nq + 2 * nkv, hd)
    qr, kr, vr = r[:, :, :nq], r[:, :, nq:nq + nkv], r[:, :, nq + nkv:]
    if qn is not None:
        qr, kr = _norm64(qr, qn), _norm64(kr, kn)
    vr = _norm64(vr, vn) if vn is not None else vr
    kc, kv = decode(kp, ks, hd, "k")
    vc, vv = decode(vp, vs, hd, "v")
    mask = torch.zeros(kc.shape[:3], dtype=torch.bool)
    for b in range(B):
        pos = torch.arange(lens[b] + off, lens[b] + off + W)
        qb, kb, vb = _rope64(qr[b], pos, inv), _rope64(kr[b], pos, inv), vr[b]
        if nq:
            # one bf16 rounding of a float32 chain (sum, norm, rotation: a few 2^-24 of the row's size)
            err = (q.view(B, W, nq, hd)[b].cpu().double() - qb).abs()
            assert (err <= BF * qb.abs() + 2.0 ** -18 * qb.abs().amax(-1, keepdim=True)).all()
        pg, sl_ = table[b].cpu().long()[pos // page], pos % page
        mask[pg, :, sl_] = True
        for want, codes, vals, sb, out in ((kb, kc, kv, ks, k_out), (vb, vc, vv, vs, v_out)):
            got = vals[pg, :, sl_]
            assert torch.equal(out[b].cpu().double(), got)            # the read-back is the cache's values
            s, bias = (t[pg, :, sl_] for t in words(sb))
            c = codes[pg, :, sl_].view(W, nkv, -1, 64)
            w64 = want.view(W, nkv, -1, 64)
            lo, hi = w64.amin(-1), w64.amax(-1)
            tiny = 2.0 ** -18 * w64.abs().amax(-1)
            assert ((s - (hi - lo) / 15).abs() <= BF * s + tiny).all() and ((bias - lo).abs() <= BF * lo.abs() + tiny).all()
            # a code is the nearest one: off by half a step and what float32 moves the value by
            step = s[..., None]
            near = (w64 - bias[..., None]) / step
            assert ((c - near.clamp(0, 15)).abs() <= 0.5 + (tiny[..., None] / step)).all()
    # nothing else of the pools changed
    for now, was, which in ((kp, before[0], "k"), (vp, before[1], "v")):
        a, z = decode(now, ks, hd, which)[0], decode(was, before[2], hd, which)[0]
        assert torch.equal(a[~mask], z[~mask])
    for now, was in ((ks, before[2]), (vs, before[3])):
        assert torch.equal(now.cpu()[~mask], was.cpu()[~mask])


@pytest.mark.parametrize("hd,splits,start", [(128, 0, 0), (256, 0, 70001), (128, 3, 130000)])
def test_append_codes_are_the_nearest(dev, hd, splits, start):
    """Keys formed in 64 bits: scales, offsets and codes are those of the 64-bit reference, which leaves out values
    within 1e-7 of a step of the middle between two codes (a 64-bit chain is off by less than 1e-10 of one)."""
    from mlx_dspark import ops

    nq, nkv, W, page = 2, 2, 300, 64
    g = torch.Generator().manual_seed(hd + splits)
    max_pages = -(-(start + W) // page)
    table = (torch.arange(max_pages, dtype=torch.int32) % 7)[None].to(dev)
    kp, vp = (torch.zeros((7, nkv, page, hd // 2), dtype=torch.uint8, device=dev) for _ in range(2))
    ks, vs = (torch.zeros((7, nkv, page, hd // 64), dtype=torch.int32, device=dev) for _ in range(2))
    x = torch.randn((max(splits, 1), W, (nq + 2 * nkv) * hd), generator=g)
    x = x if splits else x[0].to(torch.bfloat16)
    kn = (1 + 0.2 * torch.randn(hd, generator=g)).to(torch.bfloat16)
    inv = ops.rope_inv_freq(hd, 1e6, "cpu")
    ops.qkv_rope_append(x.to(dev), 1, W, nq, nkv, hd, kn.to(dev), kn.to(dev), EPS, inv.to(dev),
                        torch.tensor([start], dtype=torch.int32, device=dev), table, page, ops.DSK_KV_U4, kp, vp, ks, vs)
    r = (x.double().sum(0) if splits else x.double()).view(W, nq + 2 * nkv, hd)
    pos = torch.arange(start, start + W)
    pg, sl = table[0].cpu().long()[pos // page], pos % page
    for which, pool, sb, want in (("k", kp, ks, _rope64(_norm64(r[:, nq:nq + nkv], kn), pos, inv)), ("v", vp, vs, r[:, nq + nkv:])):
        if which == "v" and not splits:
            continue    # bf16 values: float32, as test_append_bf16_values_exact has them
        w = want.view(W, nkv, -1, 64)
        lo, hi = w.amin(-1), w.amax(-1)
        s, b = ((t.float().to(torch.bfloat16)).double() for t in ((hi - lo) / 15, lo))
        got_s, got_b = (t[pg, :, sl].double() for t in words(sb))
        assert torch.equal(got_s, s) and torch.equal(got_b, b)
        near = (w - b[..., None]) / s[..., None]
        c = decode(pool, sb, hd, which)[0][pg, :, sl].view(W, nkv, -1, 64)
        sure = ((near - near.floor()) - 0.5).abs() > 1e-7
        assert torch.equal(c[sure].double(), near.round().clamp(0, 15)[sure])


@pytest.mark.parametrize("hd", [128, 256])
def test_append_bf16_values_exact(dev, hd):
    """V rows of a bf16 projection take no arithmetic before their codes: the float32 rule's own bits, constant
    and zero groups and groups far from zero among them."""
    from mlx_dspark import ops

    B, W, nkv, page = 1, 40, 3, 64
    g = torch.Generator().manual_seed(5)
    table, (kp, vp, ks, vs) = _make(B, nkv, hd, 2, page, dev, 1)
    x = torch.randn((W, 2 * nkv, hd), generator=g).to(torch.bfloat16)
    x[3] = 0.0
    x[4] = -7.25
    x[5] = x[5] * 1e-3 + 300
    x[6] = x[6] * 1e20
    x[7] = x[7] * 1e-20
    sl = torch.zeros(B, dtype=torch.int32, device=dev)
    ops.qkv_rope_append(x.view(W, -1).to(dev), B, W, 0, nkv, hd, None, None, EPS, ops.rope_inv_freq(hd, 1e6, dev), sl,
                        table, page, ops.DSK_KV_U4, kp, vp, ks, vs)
    codes = decode(vp, vs, hd, "v")[0]
    s, b = words(vs)
    pg = table[0].cpu().long()[0]
    c, s_, b_ = quantise(x[:, nkv:].float())
    at = lambda t: t[pg].transpose(0, 1)[:W]
    assert torch.equal(at(codes), c) and torch.equal(at(s), s_.double()) and torch.equal(at(b), b_.double())
    k, v = ops.kv_read(sl, W, nkv, hd, table, page, ops.DSK_KV_U4, kp, vp, ks, vs)
    want = (c.double().view(W, nkv, -1, 64) * s_[..., None].double() + b_[..., None].double()).to(torch.bfloat16)
    assert torch.equal(v[0].cpu(), want.view(W, nkv, hd))


def test_append_far_positions_and_table_end(dev):
    """Angles at positions past 2^17, and tokens past the block table dropped."""
    from mlx_dspark import ops

    nq, nkv, hd, page, W = 4, 2, 128, 64, 5
    inv = ops.rope_inv_freq(hd, 1e4, "cpu")
    pages = 4000
    table = torch.arange(pages, dtype=torch.int32, device=dev)[None] % 7
    kp, vp = (torch.zeros((7, nkv, page, hd // 2), dtype=torch.uint8, device=dev) for _ in range(2))
    ks, vs = (torch.zeros((7, nkv, page, hd // 64), dtype=torch.int32, device=dev) for _ in range(2))
    x = torch.randn((W, (nq + 2 * nkv) * hd), generator=torch.Generator().manual_seed(2)).to(torch.bfloat16)
    first = pages * page - 3
    sl = torch.tensor([first], dtype=torch.int32, device=dev)
    q = ops.qkv_rope_append(x.to(dev), 1, W, nq, nkv, hd, None, None, EPS, inv.to(dev), sl, table, page,
                            ops.DSK_KV_U4, kp, vp, ks, vs)
    pos = torch.arange(first, first + W)
    want = _rope64(x.double().view(W, -1, hd)[:, :nq], pos, inv)
    err = (q.view(W, nq, hd).cpu().double() - want).abs()[:3]
    assert (err <= BF * want.abs()[:3] + 2.0 ** -18 * want.abs().amax()).all()
    pg = (pages - 1) % 7
    assert int((ks.cpu() != 0).sum()) == 3 * nkv * 2 and bool((ks[pg, :, -3:] != 0).all())   # three tokens stored
    out = torch.full((1, W, nkv, hd), 7.0, dtype=torch.bfloat16, device=dev)
    k, v = ops.kv_read(sl, W, nkv, hd, table, page, ops.DSK_KV_U4, kp, vp, ks, vs, k_out=out, v_out=out.clone())
    assert bool((k[:, 3:] == 7).all()) and bool((v[:, 3:] == 7).all()) and not bool((v[:, :3] == 7).any())


@pytest.mark.parametrize("hd,nkv,page,bits", [(128, 8, 64, 4), (256, 2, 32, 4), (128, 1, 96, 4), (128, 2, 16, 8),
                                              (256, 8, 64, 8), (512, 1, 64, 8), (128, 3, 48, 0), (512, 2, 64, 0)])
@pytest.mark.parametrize("n,starts", [(1, [0, 33]), (31, [1, 0]), (100, [17, 64])])
def test_read(dev, hd, nkv, page, bits, n, starts):
    from mlx_dspark import ops

    print(f"kv read hd={hd} nkv={nkv} page={page} bits={bits} n={n} {starts}", flush=True)
    B, g = 2, torch.Generator().manual_seed(n + hd)
    max_pages = -(-(max(starts) + n) // page)
    pages = B * max_pages + 2
    table = torch.randperm(pages, generator=g)[:B * max_pages].view(B, max_pages).to(torch.int32)
    pools, sbs, vals = [], [], []
    for which in ("k", "v"):
        x = torch.randn((pages, nkv, page, hd), generator=g)
        sb = torch.zeros((pages, nkv, page, hd // 64), dtype=torch.int32) if bits else None
        if bits == 4:
            pool = torch.zeros((pages, nkv, page, hd // 2), dtype=torch.uint8)
            v = fill(pool, sb, hd, which, x)
        elif bits == 8:
            pool = torch.randint(0, 256, x.shape, generator=g, dtype=torch.uint8)
            s, b = (torch.rand((pages, nkv, page, hd // 64), generator=g).to(torch.bfloat16) for _ in range(2))
            sb.copy_((s.view(torch.int16).int() & 0xFFFF) | (b.view(torch.int16).int() << 16))
            v = (pool.double().view(*sb.shape, 64) * s[..., None].double() + b[..., None].double())
            v = v.float().to(torch.bfloat16).view(x.shape)
        else:
            pool = v = x.to(torch.bfloat16)
        pools.append(pool.to(dev))
        sbs.append(None if sb is None else sb.to(dev))
        vals.append(v.to(torch.bfloat16))
    kv = {0: ops.DSK_KV_BF16, 8: ops.DSK_KV_U8, 4: ops.DSK_KV_U4}[bits]
    first = torch.tensor([s - 5 for s in starts], dtype=torch.int32, device=dev)
    out = ops.kv_read(first, n, nkv, hd, table.to(dev), page, kv, *pools, *sbs, offset=5)
    for got, v in zip(out, vals):
        for b in range(B):
            pos = torch.arange(starts[b], starts[b] + n)
            assert torch.equal(got[b].cpu(), v[table[b].long()[pos // page], :, pos % page])


def test_cache_object(dev):
    from mlx_dspark import ops
    from mlx_dspark.kv import PagedKVCache

    c = PagedKVCache(2, 1, 2, 128, 130, kv_bits=4, device=dev)
    assert c.nbytes == 2 * 2 * 3 * 2 * 64 * (64 + 8)
    x = torch.randn((70, 4 * 128), generator=torch.Generator().manual_seed(0)).to(torch.bfloat16).to(dev)
    ops.qkv_rope_append(x, 1, 70, 0, 2, 128, None, None, EPS, ops.rope_inv_freq(128, 1e4, dev), c.seq_lens,
                        c.block_table, c.page, c.kv_dtype, *c.layer_args(1))
    c.set_lengths([70])
    k, v = c.read(1)
    assert tuple(k.shape) == (1, 70, 2, 128) == tuple(v.shape)
    k2, v2 = c.read(1, 40, 20)
    assert torch.equal(k[:, 40:60], k2) and torch.equal(v[:, 40:60], v2)
    assert tuple(c.read(0, 3, 0)[0].shape) == (1, 0, 2, 128)
    with pytest.raises(ValueError):
        c.read(0, 100, 200)
