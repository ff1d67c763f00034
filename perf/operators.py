"""Operators of a 4-bit key/value cache and of windowed attention with sink tokens, as calls that can be
timed and checked one by one.

Every case is a plain dict; "op" says what it runs:
  append  ops.qkv_rope_append into a 4-bit paged cache (q/k RMSNorm, RoPE, K and V quantised as they are
          written) and ops.kv_read of the rows it wrote: the queries, and the values the cache stands for
  read    ops.kv_read of a cached context: the values of a 4-bit (8-bit, bf16) cache as bf16 rows
  attend  ops.attention (ops.attention_rows for prompts) over a 4-bit paged cache
  sinks   the same over any cache with a sliding window and the first tokens of the context visible

The 4-bit cache: affine codes in groups of 64 dims, a value is bf16(s c + b), c in 0..15, s and b bf16.
With lo, hi a group's least and largest value: s = bf16((hi - lo) / 15) (1 where that is not positive),
b = bf16(lo), c = round((v - b) / s) clamped to 0..15. Bytes of a page of one kv head, token t, dim d:
  K  token-major, hd / 2 bytes each: byte (d/128)*64 + ((d%32)/8)*16 + ((d%128)/32)*4 + (d%8)/2, the high
     half for odd d
  V  32-token blocks of 16 hd bytes: byte (d/64)*1024 + (d%16 + 16*((t%16)/4))*16 + ((d%64)/32)*8
     + 4*((t%32)/16) + t%4, the high half where (d%32)/16 is 1
  scale | bias << 16 words [page][kv head][token][hd/64], as the 8-bit cache's

Shapes are those of synthetic.TARGETS and of the benchmark: 16 heads of 128 (Qwen3-0.6B), 32 of 128
(Qwen3-8B), 16 of 256 (Gemma-style 12B, window 1024), each over 8 kv heads.
"""

import math
import random
import sys
import zlib
from pathlib import Path

import torch

own = False

_PKG = str(Path(__file__).resolve().parents[1] / "mlx-dspark_amd")
PAGE = 64
EPS = 1e-6
HEADS = {"q06": (16, 8, 128), "q8": (32, 8, 128), "g12": (16, 8, 256)}


def listed():
    return [
        # one decoded token of a small model: the split-K slices of its projection, latency counts
        dict(name="append_token", op="append", heads="q06", B=1, W=1, lo=311, hi=311, splits=2, room=16384),
        # a continuous batch's verify step: four conversations, 8 drafts and a bonus each
        dict(name="append_verify", op="append", heads="q8", B=4, W=9, lo=1024, hi=12288, splits=2, room=16384),
        # a prompt's piece, all of its rows at once
        dict(name="append_prompt", op="append", heads="q8", B=1, W=2048, lo=0, hi=0, splits=0, room=4096),
        # a short cached prefix read back (odd length, wide heads)
        dict(name="read_prefix", op="read", heads="g12", B=1, n=1027, bits=4, room=2048),
        # a whole long context read back
        dict(name="read_context", op="read", heads="q8", B=1, n=32768, bits=4, room=32768),
        # plain greedy decoding in a short chat, in a cache with room for a long one
        dict(name="decode_q06", op="attend", heads="q06", B=1, W=1, lo=311, hi=311, bits=4, room=16384),
        # the benchmark's verify step: a 16-position block over a 4096-token context
        dict(name="verify_q8", op="attend", heads="q8", B=1, W=16, lo=4096, hi=4096, bits=4, room=4160),
        # decoding four long documents at once, where the cache's bytes count
        dict(name="decode_long", op="attend", heads="q8", B=4, W=1, lo=16384, hi=65536, bits=4, room=66048),
        # a long prompt
        dict(name="prompt_q8", op="attend", heads="q8", B=1, W=4096, lo=0, hi=0, bits=4, room=4096),
        # a sliding layer of the Gemma-style shape in a verify step, bf16 cache
        dict(name="sinks_verify_g12", op="sinks", heads="g12", B=1, W=9, lo=8192, hi=8192, bits=0, window=1024,
             sinks=4, room=8448),
        # endless chats, window and sinks over an 8-bit cache, eight at once
        dict(name="sinks_decode", op="sinks", heads="q8", B=8, W=1, lo=2048, hi=32768, bits=8, window=4096,
             sinks=64, room=33024),
        # a prompt's piece after a context through a sliding layer, 4-bit cache
        dict(name="sinks_prompt", op="sinks", heads="g12", B=1, W=2048, lo=1000, hi=1000, bits=4, window=1024,
             sinks=4, room=4096),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random):
    op = rng.choice(["append", "read", "attend", "attend", "attend", "sinks", "sinks"])
    heads = rng.choice(sorted(HEADS))
    c = dict(op=op, heads=heads)
    if op == "read":
        n, B = _log_int(rng, 1, 16384), rng.choice([1, 1, 2])
        return dict(c, B=B, n=n, bits=rng.choice([4, 4, 8, 0]), room=n + rng.randint(0, 500))
    prompt = rng.random() < 0.3
    B = 1 if prompt else rng.choice([1, 1, 2, 3, 6])
    W = _log_int(rng, 65, 1500) if prompt else rng.choice([1, 1, rng.randint(2, min(17, 64 // B))])
    lo = _log_int(rng, 1, 2000 if prompt else 24000) - 1
    hi = lo if B == 1 else min(30000, lo * rng.randint(1, 5) + rng.randint(0, 40))
    c.update(B=B, W=W, lo=lo, hi=hi)
    if op == "append":
        c.update(splits=0 if prompt else rng.choice([0, 1, 2, 3]))
    elif op == "attend":
        c.update(bits=4)
    else:
        c.update(bits=rng.choice([0, 8, 4]), window=_log_int(rng, 16, 4096), sinks=rng.choice([1, 4, 4, 16, 70, 128]))
    return dict(c, room=hi + W + rng.choice([0, rng.randint(0, 200), rng.randint(0, 8000)]))


# ----------------------------------------------------------------------------- inputs
def _gen(seed, name):
    g = torch.Generator(device="cuda")
    g.manual_seed(zlib.crc32(f"{int(seed)}:{name}".encode()))
    return g


def _randn(shape, seed, name, std=1.0):
    return torch.randn(shape, generator=_gen(seed, name), device="cuda", dtype=torch.float32).mul_(std)


def _lengths(case):
    B, lo, hi = case["B"], max(1, case["lo"]), max(1, case["hi"])
    if B == 1 or case["hi"] == 0:
        return [case["lo"]] * B
    return [int(round(lo * (hi / lo) ** (b / (B - 1)))) for b in range(B)]


def _pool(case, seed, name, pages, nkv, hd, bits, std):
    """A cache's pages of seeded rows (every slot holds something, as after earlier use): the pool, and
    its scale | bias words."""
    dt, width = (torch.bfloat16, hd) if bits == 0 else (torch.uint8, hd if bits == 8 else hd // 2)
    pool = torch.empty((pages, nkv, PAGE, width), dtype=dt, device="cuda")
    words = torch.empty((pages, nkv, PAGE, hd // 64), dtype=torch.int32, device="cuda") if bits else None
    g = _gen(seed, name)
    for p0 in range(0, pages, 512):
        p1 = min(pages, p0 + 512)
        x = torch.randn((p1 - p0, nkv, PAGE, hd), generator=g, device="cuda").mul_(std)
        if bits == 0:
            pool[p0:p1] = x
            continue
        codes, words[p0:p1] = _codes(x, bits)
        pool[p0:p1] = codes if bits == 8 else (_k_bytes(codes) if name == "k" else _v_bytes(codes))
    return pool, words


def _codes(x, bits):
    """The codes (one per byte) and scale | bias words of rows x [..., hd]."""
    levels = float(2 ** bits - 1)
    g = x.view(*x.shape[:-1], -1, 64)
    lo, hi = g.amin(-1), g.amax(-1)
    s, b = ((hi - lo) / levels).to(torch.bfloat16), lo.to(torch.bfloat16)
    s = torch.where(s > 0, s, torch.ones_like(s))
    q = ((g - b.float()[..., None]) / s.float()[..., None]).round_().clamp_(0, levels)
    w = (s.view(torch.int16).to(torch.int32) & 0xFFFF) | (b.view(torch.int16).to(torch.int32) << 16)
    return q.view(x.shape).to(torch.uint8), w


def _k_bytes(codes):
    hd = codes.shape[-1]
    c = codes.view(*codes.shape[:-1], hd // 128, 4, 4, 4, 2).transpose(-4, -3)   # [half][dim/8 of 32][slab][byte][half byte]
    return (c[..., 0] | (c[..., 1] << 4)).reshape(*codes.shape[:-1], hd // 2)


def _v_bytes(codes):
    P, nkv, page, hd = codes.shape
    c = codes.view(P, nkv, page // 32, 2, 4, 4, hd // 64, 2, 2, 16)              # [tile, quad, key][chunk, pair, half, dim]
    c = c.permute(0, 1, 2, 6, 4, 9, 7, 3, 5, 8)
    return (c[..., 0] | (c[..., 1] << 4)).reshape(P, nkv, page, hd // 2)


def prepare(case, seed):
    nq, nkv, hd = HEADS[case["heads"]]
    B, bits = case["B"], case.get("bits", 4)
    max_pages = -(-case["room"] // PAGE)
    pages = B * max_pages + 2
    st = dict(case=dict(case), B=B, nq=nq, nkv=nkv, hd=hd, bits=bits, max_ctx=max_pages * PAGE)
    st["k_pool"], st["k_sb"] = _pool(case, seed, "k", pages, nkv, hd, bits, 1.0)
    st["v_pool"], st["v_sb"] = _pool(case, seed, "v", pages, nkv, hd, bits, 1.0)
    order = torch.randperm(pages, generator=_gen(seed, "pages"), device="cuda")
    st["table"] = order[:B * max_pages].view(B, max_pages).to(torch.int32).contiguous()
    if case["op"] == "read":
        st["lens"] = torch.zeros(B, dtype=torch.int32, device="cuda")
        return st
    W = st["W"] = case["W"]
    lens = _lengths(case)
    st["longest"] = max(lens) + W
    st["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    if case["op"] == "append":
        cols = (nq + 2 * nkv) * hd
        S = case["splits"]
        x = _randn((max(S, 1), B * W, cols), seed, "qkv").clamp_(-2.5, 2.5)   # activations without outliers
        st["qkv"] = x.mul_(S ** -0.5) if S else x[0].to(torch.bfloat16)
        st["q_norm"], st["k_norm"] = ((1 + _randn((hd,), seed, n, 0.1)).to(torch.bfloat16) for n in ("qn", "kn"))
        d = torch.arange(0, hd // 2, dtype=torch.float64)
        st["inv_freq"] = (1e6 ** (-2.0 * d / hd)).to(torch.float32).cuda()
    else:
        st["q"] = _randn((B * W, nq * hd), seed, "q", 1.5).to(torch.bfloat16)
    return st


# ----------------------------------------------------------------------------- plain forms
def _values(pool, words, hd, bits, v):
    """float32 values [P, nkv, page, hd] of pages of a cache."""
    if bits == 0:
        return pool.float()
    if bits == 4:
        P, nkv, page, _ = pool.shape
        c = torch.stack((pool & 15, pool >> 4), -1)
        if v:
            c = c.view(P, nkv, page // 32, hd // 64, 4, 16, 2, 2, 4, 2)          # [chunk][quad][dim][pair][tile][key][half]
            c = c.permute(0, 1, 2, 7, 4, 8, 3, 6, 9, 5)
        else:
            c = c.view(P, nkv, page, hd // 128, 4, 4, 8).transpose(-3, -2)
        pool = c.reshape(P, nkv, page, hd)
    s = (words << 16).view(torch.float32)
    b = (words & -65536).view(torch.float32)
    x = pool.float().view(*pool.shape[:-1], hd // 64, 64)
    return (x * s[..., None] + b[..., None]).to(torch.bfloat16).float().view(pool.shape)


def _context(st, n):
    """float32 keys and values [B, nkv, n, hd] of every row's first n positions."""
    t = st["table"][:, :-(-n // PAGE)].long()
    out = []
    for which in ("k", "v"):
        words = st[which + "_sb"]
        x = _values(st[which + "_pool"][t.reshape(-1)], None if words is None else words[t.reshape(-1)], st["hd"],
                    st["bits"], which == "v")
        x = x.view(st["B"], -1, st["nkv"], PAGE, st["hd"]).transpose(1, 2).reshape(st["B"], st["nkv"], -1, st["hd"])
        out.append(x[:, :, :n])
    return out


def _plain_attention(st):
    case, B, W, nq, nkv, hd = st["case"], st["B"], st["W"], st["nq"], st["nkv"], st["hd"]
    n, G = st["longest"], st["nq"] // st["nkv"]
    k, v = _context(st, n)
    q = st["q"].float().view(B, W, nkv, G, hd).permute(0, 2, 3, 1, 4).reshape(B, nkv, G * W, hd)
    s = (q @ k.transpose(2, 3).contiguous()).view(B, nkv, G, W, n) * hd ** -0.5
    j = torch.arange(n, device=q.device)
    pos = (st["lens"].long()[:, None] + torch.arange(W, device=q.device))[:, :, None]        # [B, W, 1]
    seen = j <= pos
    if case["op"] == "sinks":
        seen &= (j > pos - case["window"]) | (j < case["sinks"])
    s = s.masked_fill(~seen[:, None, None], float("-inf"))
    p = (s - s.amax(-1, keepdim=True)).exp()
    p = p / p.sum(-1, keepdim=True)
    o = (p.view(B, nkv, G * W, n) @ v.contiguous()).view(B, nkv, G, W, hd)
    return o.permute(0, 3, 1, 2, 4).reshape(B * W, nq * hd).to(torch.bfloat16)


def _plain_append(st):
    B, W, nq, nkv, hd = st["B"], st["W"], st["nq"], st["nkv"], st["hd"]
    x = st["qkv"].sum(0) if st["qkv"].dim() == 3 else st["qkv"].float()
    x = x.view(B, W, nq + 2 * nkv, hd)
    pos = st["lens"].long()[:, None] + torch.arange(W, device=x.device)
    ang = pos.double()[..., None] * st["inv_freq"].double()
    cos, sin = ang.cos().float()[:, :, None], ang.sin().float()[:, :, None]

    def roped(h, w):
        h = h * (h.square().mean(-1, keepdim=True) + EPS).rsqrt() * w.float()
        a, b = h[..., :hd // 2], h[..., hd // 2:]
        return torch.cat((a * cos - b * sin, b * cos + a * sin), -1)

    q = roped(x[:, :, :nq], st["q_norm"])
    at = (st["table"].gather(1, pos // PAGE).long()[..., None], torch.arange(nkv, device=x.device), (pos % PAGE)[..., None])
    out = [q.reshape(B * W, nq * hd).to(torch.bfloat16)]
    for which, rows in (("k", roped(x[:, :, nq:nq + nkv], st["k_norm"])), ("v", x[:, :, nq + nkv:])):
        codes, words = _codes(rows.contiguous(), 4)
        st[which + "_sb"][at] = words
        if which == "k":
            st["k_pool"][at] = _k_bytes(codes)
        else:
            t, c = (pos % PAGE)[..., None, None], codes.view(B, W, nkv, hd // 64, 2, 2, 16)
            off = (torch.arange(hd // 64, device=x.device)[:, None, None] * 1024
                   + torch.arange(2, device=x.device)[:, None] * 8 + torch.arange(16, device=x.device) * 16).view(-1)
            byte = (t // 32) * (16 * hd) + off + (t % 16 // 4) * 256 + (t % 32 // 16) * 4 + t % 4
            st["v_pool"].view(-1, nkv, PAGE * hd // 2)[at[0][..., None], at[1][:, None], byte] = (
                c[..., 0, :] | (c[..., 1, :] << 4)).view(B, W, nkv, hd // 2)
        g = codes.float().view(B, W, nkv, hd // 64, 64)
        g = g * (words << 16).view(torch.float32)[..., None] + (words & -65536).view(torch.float32)[..., None]
        out.append(g.to(torch.bfloat16).view(B, W, nkv, hd))
    return out


def _plain_read(st):
    n = st["case"]["n"]
    k, v = _context(st, n)
    return [k.transpose(1, 2).to(torch.bfloat16), v.transpose(1, 2).to(torch.bfloat16)]


# ----------------------------------------------------------------------------- one pass
def _own(st):
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    from mlx_dspark import ops

    case, kv = st["case"], {0: ops.DSK_KV_BF16, 8: ops.DSK_KV_U8, 4: ops.DSK_KV_U4}[st["bits"]]
    B, nq, nkv, hd = st["B"], st["nq"], st["nkv"], st["hd"]
    cache = (st["table"], PAGE, kv, st["k_pool"], st["v_pool"], st["k_sb"], st["v_sb"])
    if case["op"] == "read":
        return list(ops.kv_read(st["lens"], case["n"], nkv, hd, *cache))
    W = st["W"]
    if case["op"] == "append":
        q = ops.qkv_rope_append(st["qkv"], B, W, nq, nkv, hd, st["q_norm"], st["k_norm"], EPS, st["inv_freq"],
                                st["lens"], *cache)
        return [q, *ops.kv_read(st["lens"], W, nkv, hd, *cache)]
    mask = dict(window=case["window"], sinks=case["sinks"]) if case["op"] == "sinks" else {}
    attention = ops.attention if W <= 64 else ops.attention_rows
    return attention(st["q"], B, W, nq, nkv, hd, hd ** -0.5, st["lens"], st["max_ctx"], *cache, **mask)


def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    return (_plain_append if op == "append" else _plain_read if op == "read" else _plain_attention)(state)


def work(case):
    nq, nkv, hd = HEADS[case["heads"]]
    B, bits = case["B"], case.get("bits", 4)
    token = 2 * nkv * (hd * 2 if bits == 0 else hd * bits // 8 + hd // 16)     # K and V of one cached token
    row16 = 2 * nkv * hd * 2                                                   # the same as bf16 rows
    if case["op"] == "read":
        return dict(bytes=B * case["n"] * (token + row16), flops=B * case["n"] * 4 * nkv * hd)
    W = case["W"]
    if case["op"] == "append":
        cols = (nq + 2 * nkv) * hd
        each = cols * (4 * case["splits"] or 2) + nq * hd * 2 + token + row16
        return dict(bytes=B * W * each, flops=B * W * cols * (10 + case["splits"]))
    pairs, keys = 0, 0
    for n in _lengths(case):
        if case["op"] == "sinks":
            win, sk = case["window"], case["sinks"]
            pairs += sum(min(n + i + 1, win + min(sk, max(0, n + i + 1 - win))) for i in range(W))
            first = max(0, n + 1 - win)
            keys += n + W - first + min(sk, first)
        else:
            pairs += W * n + W * (W + 1) // 2
            keys += n + W
    return dict(bytes=keys * token + 2 * B * W * nq * hd * 2, flops=4 * hd * nq * pairs)


# ----------------------------------------------------------------------------- 64-bit results
def _at(st, which, b, j):
    """float64 values [nkv, len(j), hd] at positions j of row b, by the byte formulas above."""
    hd, nkv, bits = st["hd"], st["nkv"], st["bits"]
    page, t = st["table"][b].long()[j // PAGE], j % PAGE
    d = torch.arange(hd, device=j.device)
    pool = st[which + "_pool"]
    if bits != 4:
        x = pool[page[:, None], torch.arange(nkv, device=j.device), t[:, None]].double().transpose(0, 1)
    else:
        T = t[:, None]
        if which == "k":
            byte = T * (hd // 2) + d // 128 * 64 + d % 32 // 8 * 16 + d % 128 // 32 * 4 + d % 8 // 2
            high = (d % 2).expand_as(byte)
        else:
            byte = (T // 32 * (16 * hd) + d // 64 * 1024 + (d % 16 + 16 * (T % 16 // 4)) * 16 + d % 64 // 32 * 8
                    + T % 32 // 16 * 4 + T % 4)
            high = (d % 32 // 16).expand_as(byte)
        flat = pool.view(pool.shape[0], nkv, -1)
        raw = torch.stack([flat[page[:, None], h, byte] for h in range(nkv)])
        x = torch.where(high.bool(), raw >> 4, raw & 15).double()
    if bits == 0:
        return x
    w = st[which + "_sb"][page[:, None], torch.arange(nkv, device=j.device), t[:, None]].transpose(0, 1)   # [nkv, n, hd/64]
    s, b = (z.to(torch.int16).view(torch.bfloat16).double().repeat_interleave(64, -1) for z in (w, w >> 16))
    return (x * s + b).to(torch.bfloat16).double()


def exact(case, seed):
    st = prepare(case, seed)
    B, nq, nkv, hd = st["B"], st["nq"], st["nkv"], st["hd"]
    dev = "cuda"
    if case["op"] == "read":
        rows = [[_at(st, w, b, torch.arange(case["n"], device=dev)).transpose(0, 1) for b in range(B)] for w in ("k", "v")]
        return [torch.stack(r) for r in rows]
    W, G, lens = st["W"], nq // nkv, _lengths(case)
    if case["op"] == "append":
        x = st["qkv"].double()
        x = (x.sum(0) if x.dim() == 3 else x).view(B, W, nq + 2 * nkv, hd)
        out = [x[:, :, :nq].clone(), x[:, :, nq:nq + nkv].clone(), x[:, :, nq + nkv:].clone()]
        for h, w in zip(out[:2], (st["q_norm"], st["k_norm"])):
            h /= (h.pow(2).sum(-1, keepdim=True) / hd + EPS).sqrt()
            h *= w.double()
            for b in range(B):
                a = torch.outer(torch.arange(lens[b], lens[b] + W, device=dev).double(), st["inv_freq"].double())
                z = torch.complex(h[b, ..., :hd // 2], h[b, ..., hd // 2:]) * torch.polar(torch.ones_like(a), a)[:, None]
                h[b] = torch.cat((z.real, z.imag), -1)
        for r in out[1:]:
            for g in r.split(64, -1):
                lo = g.min(-1, keepdim=True).values
                s = ((g.max(-1, keepdim=True).values - lo) / 15).to(torch.bfloat16).double()
                s[s <= 0] = 1
                lo = lo.to(torch.bfloat16).double()
                g.copy_((((g - lo) / s).round().clamp(0, 15) * s + lo).to(torch.bfloat16))
        return [out[0].reshape(B * W, nq * hd), out[1], out[2]]
    res = torch.empty((B, W, nq, hd), dtype=torch.float64, device=dev)
    q = st["q"].double().view(B, W, nq, hd)
    for b, n in enumerate(lens):
        j = torch.arange(n + W, device=dev)
        i = torch.arange(n, n + W, device=dev)[:, None]
        hide = j > i
        if case["op"] == "sinks":
            hide = hide | ((j <= i - case["window"]) & (j >= case["sinks"]))
            j = torch.nonzero(~hide.all(0)).view(-1)
            hide = hide[:, j]
        k, v = _at(st, "k", b, j), _at(st, "v", b, j)
        for h in range(nq):
            s = (q[b, :, h] @ k[h // G].T) / math.sqrt(hd)
            res[b, :, h] = torch.softmax(s.masked_fill(hide, -math.inf), -1) @ v[h // G]
    return res.view(B * W, nq * hd)
