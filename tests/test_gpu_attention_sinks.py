"""GPU parity of attention over 4-bit caches, and of sliding windows with sink tokens over every cache type,
against a 64-bit reference; masked places hold infinities and NaN."""

import math

import pytest
import torch

from _kv4 import fill

pytestmark = pytest.mark.gpu

BF = 2.0 ** -8
NAN_WORD = 0x7FC07F80   # bias NaN, scale +inf


class Cache:
    """A paged cache of seeded rows on the CPU, with its values, and its device copy."""

    def __init__(self, bits, B, nkv, hd, max_pages, page, seed):
        from mlx_dspark import ops

        self.bits, self.hd, self.page = bits, hd, page
        self.kv = {0: ops.DSK_KV_BF16, 8: ops.DSK_KV_U8, 4: ops.DSK_KV_U4}[bits]
        g = torch.Generator().manual_seed(seed)
        n = B * max_pages + 2
        self.table = torch.randperm(n, generator=g)[:B * max_pages].view(B, max_pages).to(torch.int32)
        self.pools, self.sbs, self.vals = [], [], []
        for which in ("k", "v"):
            x = torch.randn((n, nkv, page, hd), generator=g)
            sb = torch.zeros((n, nkv, page, hd // 64), dtype=torch.int32) if bits else None
            if bits == 4:
                pool = torch.zeros((n, nkv, page, hd // 2), dtype=torch.uint8)
                v = fill(pool, sb, hd, which, x)
            elif bits == 8:
                gr = x.view(n, nkv, page, hd // 64, 64)
                lo, hi = gr.amin(-1), gr.amax(-1)
                s, b = ((hi - lo) / 255).to(torch.bfloat16), lo.to(torch.bfloat16)
                q = ((gr - b.float()[..., None]) / s.float()[..., None]).round().clamp(0, 255)
                pool = q.view(x.shape).to(torch.uint8)
                sb.copy_((s.view(torch.int16).int() & 0xFFFF) | (b.view(torch.int16).int() << 16))
                v = (q.double() * s.double()[..., None] + b.double()[..., None]).float().to(torch.bfloat16).view(x.shape)
            else:
                pool = x.to(torch.bfloat16)
                v = pool
            self.pools.append(pool)
            self.sbs.append(sb)
            self.vals.append(v.double())

    def poison(self, b, positions):
        """Infinities and NaN at positions of row b (garbage codes, NaN words in quantised caches)."""
        pg, sl = self.table[b].long()[positions // self.page], positions % self.page
        for pool, sb, v in zip(self.pools, self.sbs, self.vals):
            if self.bits == 0:
                pool[pg, :, sl] = float("nan")
                pool[pg, :, sl, ::2] = float("inf")
            else:
                sb[pg, :, sl] = NAN_WORD
            v[pg, :, sl] = float("nan")

    def rows(self, b, n):
        pos = torch.arange(n)
        pg, sl = self.table[b].long()[pos // self.page], pos % self.page
        return tuple(v[pg, :, sl].transpose(0, 1) for v in self.vals)     # [nkv, n, hd]

    def args(self, dev):
        to = lambda t: None if t is None else t.to(dev)
        return (to(self.table), self.page, self.kv, *(to(p) for p in self.pools), *(to(s) for s in self.sbs))


def visible(n, W, total, causal, window, sinks):
    i, j = torch.arange(n, n + W)[:, None], torch.arange(total)[None]
    if not causal:
        return torch.ones((W, total), dtype=torch.bool)
    m = j <= i
    if window:
        m &= (j > i - window) | (j < sinks)
    return m


def reference(cache, q, lens, W, nq, nkv, causal, window, sinks, scale, softcap=0.0):
    """(out, tolerance) float64 [B, W, nq, hd]. A probability is off by its bf16 terms (two: 2^-17), by the
    float32 error of its score (each of hd products and sums 2^-24 of the sum of magnitudes, twice: in the
    score and in the maximum) and by its sum's (n additions); the result by one bf16 rounding."""
    B, hd, G = len(lens), cache.hd, nq // nkv
    jmax = cache.table.shape[1] * cache.page
    q = q.double().view(B, W, nq, hd)
    out, tol = torch.zeros((B, W, nq, hd), dtype=torch.float64), torch.zeros((B, W, nq, hd), dtype=torch.float64)
    for b, n in enumerate(lens):
        total = min(n + W, jmax)
        k, v = cache.rows(b, total)
        see = visible(n, W, total, causal, window, sinks)
        for h in range(nq):
            kk, vv = k[h // G], v[h // G]
            s = q[b, :, h] @ kk.T * scale
            if softcap:
                s = torch.tanh(s / softcap) * softcap
            s = s.masked_fill(~see, -math.inf)
            mag = (q[b, :, h].abs() @ kk.abs().T * scale).masked_fill(~see, 0.0).amax(-1, keepdim=True)
            p = torch.softmax(s, -1)
            # masked places count for nothing, whatever stands there
            vz = torch.where(see.any(0)[:, None], vv, torch.zeros_like(vv))
            o = torch.stack([(p[i][see[i]] @ vz[see[i]]) for i in range(W)])
            m = torch.stack([(p[i][see[i]] @ vz[see[i]].abs()) for i in range(W)])
            out[b, :, h] = o
            tol[b, :, h] = BF * o.abs() + (2.0 ** -16 + 4 * (hd + 4) * 2.0 ** -24 * mag + total * 2.0 ** -23) * m
    return out, tol


def run(dev, cache, q, lens, W, nq, nkv, causal=True, window=0, sinks=0, scale=None, softcap=0.0, packed=False,
        max_ctx=None, rows=False):
    from mlx_dspark import ops

    B, hd = len(lens), cache.hd
    fn = ops.attention_rows if rows else ops.attention
    kw = {} if rows else dict(softcap=softcap, packed=packed)
    sl = torch.tensor(lens, dtype=torch.int32, device=dev)
    out = fn(q.to(dev), B, W, nq, nkv, hd, scale or hd ** -0.5, sl, max_ctx or cache.table.shape[1] * cache.page,
             *cache.args(dev), causal=causal, window=window, sinks=sinks, **kw)
    torch.cuda.synchronize()
    return (out.unpack() if packed else out).cpu().double().view(B, W, nq, hd)


def queries(B, W, nq, hd, seed, std=1.5):
    return (torch.randn((B * W, nq * hd), generator=torch.Generator().manual_seed(seed)) * std).to(torch.bfloat16)


def check(got, want, tol):
    assert torch.equal(got.isnan(), want.isnan())
    ok = ((got - want).abs() <= tol) | want.isnan()
    assert ok.all(), f"{int((~ok).sum())} of {ok.numel()} outside, worst {float(((got - want).abs() / tol.clamp_min(1e-30))[~ok].max()):.3g}x"


CASES = [
    # hd, nq, nkv, page, W, lens, causal, window, sinks
    (128, 4, 2, 64, 1, [0], True, 0, 0),                     # the first token of all
    (128, 4, 2, 64, 1, [1, 31, 32, 63, 64, 65], True, 0, 0),
    (128, 16, 8, 64, 1, [311], True, 0, 0),
    (128, 32, 8, 64, 16, [700], True, 0, 0),                 # 64 query rows
    (128, 32, 8, 64, 9, [5, 900, 260], True, 0, 0),          # 36 rows, ragged batch
    (128, 8, 1, 96, 3, [250, 10], True, 0, 0),               # 24 rows, pages of 96
    (256, 16, 8, 64, 9, [333], True, 0, 0),
    (256, 4, 4, 32, 1, [40, 1000, 3], True, 0, 0),
    (128, 5, 5, 128, 13, [77], True, 0, 0),                  # no sharing of heads
    (128, 24, 2, 64, 30, [200], True, 0, 0),                 # 360 rows
    (128, 4, 2, 64, 7, [100], False, 0, 0),                  # bidirectional
    (256, 4, 2, 64, 20, [0], False, 0, 0),
    (128, 32, 8, 64, 150, [0], True, 0, 0),                  # prompts
    (128, 4, 2, 64, 203, [130], True, 0, 0),
    (256, 8, 2, 64, 100, [33], True, 0, 0),
    # windows and sinks
    (128, 4, 2, 64, 1, [500, 3, 64], True, 48, 4),
    (128, 32, 8, 64, 16, [700], True, 100, 1),
    (128, 16, 8, 32, 5, [1000, 90], True, 33, 70),
    (256, 16, 8, 64, 9, [850], True, 128, 4),
    (256, 4, 2, 64, 1, [333], True, 1, 2),
    (128, 4, 2, 64, 1, [2000], True, 40, 300),
    (128, 4, 4, 64, 2, [100, 30], True, 500, 4),             # the window covers all
    (128, 4, 2, 64, 4, [300], True, 64, 1000),               # the sinks do
    (128, 4, 2, 64, 180, [150], True, 40, 4),
    (128, 16, 4, 64, 100, [0], True, 17, 20),
    (256, 4, 2, 64, 90, [700], True, 64, 33),
]


# without sinks the other cache types run kernels of their own
@pytest.mark.parametrize("case,bits", [(c, bits) for c in CASES for bits in (4, 8, 0) if bits == 4 or c[-1]], ids=str)
def test_attention(dev, case, bits):
    hd, nq, nkv, page, W, lens, causal, window, sinks = case
    print(f"attention bits={bits} {case}", flush=True)
    max_pages = -(-(max(lens) + W) // page) + 1
    c = Cache(bits, len(lens), nkv, hd, max_pages, page, seed=W + hd)
    for b, n in enumerate(lens):   # what no query sees: behind the last key, and expired keys
        total = n + W
        see = visible(n, W, total, causal, window, sinks).any(0)
        dead = torch.cat((torch.nonzero(~see).view(-1), torch.arange(total, max_pages * page)))
        c.poison(b, dead)
    q = queries(len(lens), W, nq, hd, W)
    want, tol = reference(c, q, lens, W, nq, nkv, causal, window, sinks, hd ** -0.5)
    check(run(dev, c, q, lens, W, nq, nkv, causal, window, sinks, rows=W > 64), want, tol)


@pytest.mark.parametrize("bits,hd,nq,nkv,W,n,window,sinks", [
    (4, 128, 4, 2, 5, 70, 0, 0), (4, 128, 32, 8, 12, 300, 40, 4), (4, 256, 4, 2, 80, 30, 0, 0), (0, 128, 4, 2, 3, 100, 20, 4),
    (0, 128, 16, 4, 90, 64, 33, 8), (8, 256, 8, 4, 9, 200, 64, 2)])
def test_values_only_some_rows_see(dev, bits, hd, nq, nkv, W, n, window, sinks):
    """An infinity or NaN in one new token, and in a key that leaves the window while the rows advance: the
    rows that see it become NaN, the others are untouched."""
    print(f"guarded bits={bits} hd={hd} W={W} n={n} window={window}", flush=True)
    c = Cache(bits, 1, nkv, hd, -(-(n + W) // 64), 64, seed=9)
    c.poison(0, torch.tensor([n + W - 1]))
    if window:
        c.poison(0, torch.tensor([n - window + 1]))   # the first row's last windowed key
    q = queries(1, W, nq, hd, 1)
    want, tol = reference(c, q, [n], W, nq, nkv, True, window, sinks, hd ** -0.5)
    assert want.isnan().any() and not want.isnan().all()
    check(run(dev, c, q, [n], W, nq, nkv, True, window, sinks, rows=W > 64), want, tol)


@pytest.mark.parametrize("hd,nq,nkv,W", [(128, 4, 2, 5), (256, 4, 2, 9), (128, 8, 2, 70), (128, 2, 2, 5)])
def test_values_past_the_range_of_four_bits(dev, hd, nq, nkv, W):
    """A scale and offset that are finite, whose values are not (15 * 2^125 + 2^125), in the newest token: the
    rows before do not see it, the last one does (all its values are 2^125 or more)."""
    print(f"wide hd={hd} W={W}", flush=True)
    n = 70
    c = Cache(4, 1, nkv, hd, -(-(n + W) // 64), 64, seed=3)
    q = queries(1, W, nq, hd, 2)
    pg, sl = int(c.table[0][(n + W - 1) // 64]), (n + W - 1) % 64
    c.sbs[1][pg, :, sl] = 0x7E007E00
    c.vals[1][pg, :, sl] = 0.0
    want, tol = reference(c, q, [n], W, nq, nkv, True, 0, 0, hd ** -0.5)
    got = run(dev, c, q, [n], W, nq, nkv, rows=W > 64)
    check(got[:, :-1], want[:, :-1], tol[:, :-1])
    assert (~got[:, -1].isfinite() | (got[:, -1].abs() > 2.0 ** 90)).all()


@pytest.mark.parametrize("W,nq,nkv,hd", [(1, 4, 2, 128), (9, 16, 8, 256), (70, 8, 2, 128)])
def test_softcap_scale_and_sharp_scores(dev, W, nq, nkv, hd):
    """Soft-capped scores, another scale, and scores so large that the maximum moves block after block."""
    c = Cache(4, 1, nkv, hd, 12, 64, seed=3)
    q = queries(1, W, nq, hd, 2, std=8.0)
    # past 64 new tokens ops.attention takes the form with two terms of a probability
    for scale, cap in ((1.0, 30.0), (0.37, 0.0)):
        want, tol = reference(c, q, [600], W, nq, nkv, True, 0, 0, scale, cap)
        # tanh's argument and value: a few float32 roundings of a score of up to `cap`
        tol = tol + (cap and cap * 2.0 ** -20) * want.abs().amax()
        check(run(dev, c, q, [600], W, nq, nkv, scale=scale, softcap=cap), want, tol)


def test_packed_output_and_strided_use(dev):
    c = Cache(4, 3, 8, 128, 8, 64, seed=4)
    q = queries(3, 4, 32, 128, 5)
    plain = run(dev, c, q, [300, 0, 77], 4, 32, 8)
    assert torch.equal(run(dev, c, q, [300, 0, 77], 4, 32, 8, packed=True), plain)


def test_table_end(dev):
    """Rows whose positions pass the block table see the keys there are."""
    c = Cache(4, 1, 2, 128, 3, 64, seed=6)
    q = queries(1, 8, 4, 128, 5)
    want, tol = reference(c, q, [188], 8, 4, 2, True, 0, 0, 128 ** -0.5)
    check(run(dev, c, q, [188], 8, 4, 2), want, tol)


@pytest.mark.parametrize("nq,W", [(16, 1), (32, 9)])
def test_long_cache_many_splits(dev, nq, W):
    """More blocks per wave than one load of page ids covers, rows of very different lengths."""
    lens = [40000, 17, 9000]
    c = Cache(4, 3, 2, 128, -(-(40000 + W) // 64), 64, seed=8)
    q = queries(3, W, nq, 128, 5)
    want, tol = reference(c, q, lens, W, nq, 2, True, 0, 0, 128 ** -0.5)
    check(run(dev, c, q, lens, W, nq, 2), want, tol)


def test_many_rows_batch(dev):
    """More rows than a workgroup reads lengths of (no balancing), several splits each."""
    lens = [(37 * b) % 600 for b in range(70)]
    c = Cache(4, 70, 1, 128, 10, 64, seed=11)
    q = queries(70, 1, 2, 128, 5)
    want, tol = reference(c, q, lens, 1, 2, 1, True, 0, 0, 128 ** -0.5)
    check(run(dev, c, q, lens, 1, 2, 1), want, tol)


@pytest.mark.parametrize("B,W,hd,bits,window,sinks", [(40, 1, 128, 4, 0, 0), (33, 2, 128, 8, 600, 4), (12, 1, 256, 4, 0, 0),
                                                   (12, 1, 256, 0, 900, 8), (64, 1, 128, 4, 0, 0), (65, 1, 128, 4, 0, 0),
                                                   (3, 33, 128, 4, 0, 0), (5, 20, 128, 8, 300, 40), (2, 61, 256, 4, 0, 0)])
def test_one_long_row_among_short_ones(dev, B, W, hd, bits, window, sinks):
    """Splits are placed by the rows' lengths: one row gets most of them, empty rows one each."""
    print(f"placement B={B} W={W} hd={hd} bits={bits}", flush=True)
    lens = [(7 * b) % 40 for b in range(B)]
    lens[B // 2] = 1500
    c = Cache(bits, B, 8, hd, 24, 64, seed=B)
    q = queries(B, W, 8, hd, 5)
    want, tol = reference(c, q, lens, W, 8, 8, True, window, sinks, hd ** -0.5)
    check(run(dev, c, q, lens, W, 8, 8, True, window, sinks), want, tol)


@pytest.mark.parametrize("bits,nq,nkv,W,lens,window,sinks,rows", [
    (4, 8, 2, 64, [4100], 0, 0, False), (4, 8, 2, 70, [33], 0, 0, True), (4, 16, 2, 40, [4000, 7], 0, 0, False),
    (8, 8, 2, 90, [4060], 4060, 40, True), (0, 6, 1, 101, [4000], 4050, 3, True), (0, 8, 2, 64, [0, 4096], 4096, 1, False)])
def test_many_rows_long_context(dev, bits, nq, nkv, W, lens, window, sinks, rows):
    """Workgroups of 256 rows: contexts that may be 4096 long."""
    print(f"long bits={bits} W={W} lens={lens} window={window}", flush=True)
    c = Cache(bits, len(lens), nkv, 128, 68, 64, seed=W)
    for b, n in enumerate(lens):
        see = visible(n, W, n + W, True, window, sinks).any(0)
        c.poison(b, torch.cat((torch.nonzero(~see).view(-1), torch.arange(n + W, 68 * 64))))
    q = queries(len(lens), W, nq, 128, 5)
    want, tol = reference(c, q, lens, W, nq, nkv, True, window, sinks, 128 ** -0.5)
    check(run(dev, c, q, lens, W, nq, nkv, True, window, sinks, rows=rows), want, tol)


@pytest.mark.parametrize("bits,window,sinks,W", [(4, 0, 0, 1), (4, 64, 4, 9), (8, 64, 4, 1)])
def test_graph_replay_follows_lengths(dev, bits, window, sinks, W):
    """A captured append + attention replayed while the device lengths advance, against the eager calls; a
    second graph of the same shape replayed on another stream at the same time."""
    from mlx_dspark import ops

    nq, nkv, hd, B = 8, 2, 128, 2
    inv = ops.rope_inv_freq(hd, 1e6, dev)
    g = torch.Generator().manual_seed(0)
    xs = torch.randn((6, B * W, (nq + 2 * nkv) * hd), generator=g).to(torch.bfloat16).to(dev)
    caches = [Cache(bits, B, nkv, hd, 8, 64, seed=s).args(dev) for s in (1, 1, 2)]

    def step(x, sl, cache):
        q = ops.qkv_rope_append(x, B, W, nq, nkv, hd, None, None, 1e-6, inv, sl, *cache)
        o = ops.attention(q, B, W, nq, nkv, hd, hd ** -0.5, sl, 512, *cache, window=window, sinks=sinks)
        ops.lens_add(sl, None, W)
        return o

    lens = lambda: torch.tensor([130, 40], dtype=torch.int32, device=dev)
    graphs = []
    for cache in caches[1:]:
        x, sl = xs[0].clone(), lens()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(x, sl, cache)
        torch.cuda.current_stream().wait_stream(side)
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = step(x, sl, cache)
        sl.copy_(lens())
        graphs.append((gr, x, sl, out))
    torch.cuda.synchronize()
    sl = lens()
    other = torch.cuda.Stream()
    for i in range(6):
        want = step(xs[i], sl, caches[0]).clone()
        for gr, x, _, _ in graphs:
            x.copy_(xs[i])
        torch.cuda.synchronize()
        with torch.cuda.stream(other):
            graphs[1][0].replay()
        graphs[0][0].replay()
        torch.cuda.synchronize()
        assert torch.equal(graphs[0][3], want) and not torch.equal(graphs[1][3], want)


def test_non_default_stream(dev):
    c = Cache(4, 1, 2, 128, 4, 64, seed=6)
    q = queries(1, 3, 4, 128, 5)
    base = run(dev, c, q, [100], 3, 4, 2)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = run(dev, c, q, [100], 3, 4, 2)
    assert torch.equal(got, base)


@pytest.mark.parametrize("bits,hd,nq,nkv,W,lens,window,sinks", [
    (4, 128, 2, 2, 5, [70, 33], 0, 0), (4, 128, 8, 2, 1, [3000], 0, 0), (8, 128, 4, 2, 2, [300], 40, 4),
    (4, 256, 3, 1, 1, [64, 95], 40, 1), (8, 256, 2, 2, 4, [129], 64, 33), (4, 128, 2, 2, 5, [500], 33, 3)])
@pytest.mark.parametrize("poison", [False, True])
def test_few_rows_in_columns(dev, bits, hd, nq, nkv, W, lens, window, sinks, poison):
    """Up to five query rows per kv head, each in three columns; with an infinity or NaN in the newest token, which
    only the last row sees, and in the first row's last windowed key."""
    print(f"columns bits={bits} hd={hd} W={W} lens={lens} window={window} poison={poison}", flush=True)
    c = Cache(bits, len(lens), nkv, hd, -(-(max(lens) + W) // 64), 64, seed=9)
    if poison:
        for b, n in enumerate(lens):
            c.poison(b, torch.tensor([n + W - 1] + ([n - window + 1] if window else [])))
    q = queries(len(lens), W, nq, hd, 1)
    want, tol = reference(c, q, lens, W, nq, nkv, True, window, sinks, hd ** -0.5)
    check(run(dev, c, q, lens, W, nq, nkv, True, window, sinks), want, tol)


@pytest.mark.parametrize("bits,window,sinks,W", [(4, 0, 0, 1), (4, 0, 0, 90), (8, 100, 4, 9), (0, 100, 4, 1)])
def test_pages_past_32_bit_offsets(dev, bits, window, sinks, W):
    """The same pages at the end of pools of more than 4 GiB: append, attention and read-back bit for bit."""
    from mlx_dspark import ops

    nq, nkv, hd, page, n = 8, 2, 128, 64, 300
    kv = {0: ops.DSK_KV_BF16, 8: ops.DSK_KV_U8, 4: ops.DSK_KV_U4}[bits]
    width, dt = (hd // 2 if bits == 4 else hd), (torch.uint8 if bits else torch.bfloat16)
    far = (2 ** 32 + 2 ** 20) // (nkv * page * width * (1 if bits else 2))
    need = -(-(n + W) // page)
    inv = ops.rope_inv_freq(hd, 1e6, dev)
    x = torch.randn((1, n + W, (nq + 2 * nkv) * hd), generator=torch.Generator().manual_seed(4)).to(torch.bfloat16).to(dev)
    outs = []
    for first in (0, far):
        print(f"far bits={bits} W={W} first page {first}", flush=True)
        table = (first + torch.randperm(need, generator=torch.Generator().manual_seed(1))).to(torch.int32)[None].to(dev)
        pools = [torch.empty((first + need, nkv, page, width), dtype=dt, device=dev) for _ in range(2)]
        sbs = [torch.empty((first + need, nkv, page, hd // 64), dtype=torch.int32, device=dev) if bits else None for _ in range(2)]
        cache = (table, page, kv, *pools, *sbs)
        sl = torch.zeros(1, dtype=torch.int32, device=dev)
        ops.qkv_rope_append(x[0, :n].contiguous(), 1, n, nq, nkv, hd, None, None, 1e-6, inv, sl, *cache)
        sl.fill_(n)
        q = ops.qkv_rope_append(x[0, n:].contiguous(), 1, W, nq, nkv, hd, None, None, 1e-6, inv, sl, *cache)
        o = ops.attention(q, 1, W, nq, nkv, hd, hd ** -0.5, sl, n + W, *cache, window=window, sinks=sinks)
        k, v = ops.kv_read(torch.zeros(1, dtype=torch.int32, device=dev), n + W, nkv, hd, *cache)
        outs.append([t.cpu() for t in (q, o, k, v)])
        del pools, sbs, cache
    torch.cuda.empty_cache()
    assert all(torch.equal(a, b) for a, b in zip(*outs)) and all(t.float().abs().sum() > 0 for t in outs[0])


@pytest.mark.parametrize("bits,hd,nq,nkv,W,window,sinks", [
    (4, 128, 8, 2, 1, 0, 0), (4, 256, 4, 2, 20, 0, 0),
    *((bits, 128, 8, 2, W, window, sinks) for bits in (4, 0) for W, window, sinks in ((9, 40, 70), (100, 30, 4)))])
def test_table_entries_that_no_query_sees(dev, bits, hd, nq, nkv, W, window, sinks):
    """Table entries behind the rows' last pages, and the window's expired ones, may hold anything: here pages
    of another row."""
    lens = [150, 3]
    c = Cache(bits, 2, nkv, hd, 6, 64, seed=7)
    q = queries(2, W, nq, hd, 5)
    want, tol = reference(c, q, lens, W, nq, nkv, True, window, sinks, hd ** -0.5)
    for b, n in enumerate(lens):
        seen = {int(j) // 64 for j in torch.nonzero(visible(n, W, n + W, True, window, sinks).any(0)).view(-1)}
        for p in set(range(6)) - seen:
            c.table[b, p] = 0
    check(run(dev, c, q, lens, W, nq, nkv, True, window, sinks, rows=W > 64), want, tol)
