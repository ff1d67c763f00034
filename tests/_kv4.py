"""A 4-bit paged cache restated from its byte formulas, in plain torch on the CPU, for the tests."""

import numpy as np
import torch


def k_place(hd, t, d):
    """(byte, high half) of token t, dim d in a page of K of one head."""
    return t * (hd // 2) + d // 128 * 64 + d % 32 // 8 * 16 + d % 128 // 32 * 4 + d % 8 // 2, d % 2


def v_place(hd, t, d):
    return (t // 32 * 16 * hd + d // 64 * 1024 + (d % 16 + 16 * (t % 16 // 4)) * 16 + d % 64 // 32 * 8
            + t % 32 // 16 * 4 + t % 4), d % 32 // 16


def words(sb):
    """(scales, biases) float64 of int32 words."""
    w = sb.cpu().numpy().view(np.uint32)
    f = lambda h: torch.from_numpy((h.astype(np.uint32) << 16).view(np.float32).astype(np.float64))
    return f(w & 0xFFFF), f(w >> 16)


def decode(pool, sb, hd, which):
    """(codes, values) [pages, nkv, page, hd] of a 4-bit pool: int64 and float64 bf16(s c + b)."""
    pages, nkv, page, _ = pool.shape
    flat = pool.cpu().reshape(pages, nkv, -1).long()
    t, d = torch.arange(page)[:, None], torch.arange(hd)[None, :]
    byte, high = (k_place if which == "k" else v_place)(hd, t, d)
    raw = flat[:, :, byte.reshape(-1)].view(pages, nkv, page, hd)
    codes = torch.where(high.expand(page, hd) != 0, raw >> 4, raw & 15)
    s, b = words(sb)
    v = codes.double().view(pages, nkv, page, hd // 64, 64) * s[..., None] + b[..., None]
    return codes, v.to(torch.bfloat16).double().view(codes.shape)


def quantise(x):
    """float32 rows [..., hd] -> (codes, scale, bias) by the cache's rule in float32, as the engine states it."""
    g = x.float().view(*x.shape[:-1], -1, 64)
    lo, hi = g.amin(-1), g.amax(-1)
    s = ((hi - lo) / 15).to(torch.bfloat16).float()
    s = torch.where(s > 0, s, torch.ones_like(s))
    b = lo.to(torch.bfloat16).float()
    c = ((g - b[..., None]) / s[..., None]).round().clamp(0, 15)
    return c.long().view(x.shape), s, b


def fill(pool, sb, hd, which, x):
    """Write rows x [pages, nkv, page, hd] into a CPU pool; returns the values the cache stands for."""
    pages, nkv, page, _ = pool.shape
    c, s, b = quantise(x)
    t, d = torch.arange(page)[:, None], torch.arange(hd)[None, :]
    byte, high = (k_place if which == "k" else v_place)(hd, t, d)
    flat = torch.zeros((pages, nkv, page * hd // 2), dtype=torch.int64)
    at = byte.reshape(-1).expand(pages, nkv, -1)
    flat.scatter_add_(2, at, (c << (4 * high)).reshape(pages, nkv, -1))
    pool.copy_(flat.to(torch.uint8).view(pool.shape))
    bits = lambda f: f.to(torch.bfloat16).view(torch.int16).to(torch.int32)
    sb.copy_((bits(s) & 0xFFFF) | (bits(b) << 16))
    return decode(pool, sb, hd, which)[1]
