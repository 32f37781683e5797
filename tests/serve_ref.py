"""Plain 64-bit forms of the batched serving operators, for their tests: the 4-bit blocks, a
page's bytes, append, attention and the 8-bit product, in torch on any device, one sequence or
row at a time."""
from __future__ import annotations

import torch

EPS = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}   # half a step


def blocks(x):
    """x [..., hd] float64 -> (codes [..., hd] int64, scales [..., hd / 32] float16)."""
    b = x.unflatten(-1, (-1, 32))
    big = b.abs().amax(-1, keepdim=True)
    first = torch.argmax((b.abs() == big).to(torch.int8), -1, keepdim=True)
    m = torch.gather(b, -1, first)
    d = (m.float() * -0.125).half()
    bad = ~torch.isfinite(b).all(-1, keepdim=True) | ~torch.isfinite(d)
    safe = torch.where((m == 0) | bad, torch.ones_like(m), m)
    q = torch.floor(8.5 - 8 * torch.nan_to_num(b) / safe).clamp(0, 15)
    q = torch.where((m == 0) | bad, torch.full_like(q, 8), q).long()
    d = torch.where(bad, torch.full_like(d, float("nan")), d)
    return q.flatten(-2), d.squeeze(-1)


def held(x):
    """What the blocks of x stand for, float64."""
    q, d = blocks(x)
    return d.double().repeat_interleave(32, -1) * (q - 8)


def place(nkv, hd, page, kind, j, tok, d):
    """(byte, shift) of a code in its page, straight from the layout's description."""
    base = (j * (page // 16) + tok // 16) * 18 * hd + kind * 8 * hd
    t, b, i = tok % 16, d // 32, d % 32 // 8
    h = t // 8
    if kind == 0:
        g, c, e = t % 8, d % 8 // 2, d % 2
    else:
        g, c, e = d % 8, t % 8 // 2, t % 2
    return base + ((h * 8 + g) * 4 + c) * (hd // 8) + 4 * b + 2 * e + i // 2, 4 * (i % 2)


def scale_place(nkv, hd, page, kind, j, tok, b):
    t = tok % 16
    base = (j * (page // 16) + tok // 16) * 18 * hd + 16 * hd
    if kind == 0:
        return base + 2 * (t * (hd // 32) + b)
    return base + hd + 2 * ((((t // 8) * 4 + t % 8 // 2) * (hd // 32) + b) * 2 + t % 2)


class Cache:
    """Values [page][tok][kv head][hd] that a paged cache should hold, and its bytes."""

    def __init__(self, n_pages, nkv, hd, page, device="cpu"):
        self.nkv, self.hd, self.page = nkv, hd, page
        self.k = torch.zeros(n_pages, page, nkv, hd, dtype=torch.float64, device=device)
        self.v = torch.zeros_like(self.k)

    def pages(self, k, v):
        """The bytes of pages holding rows k, v [n][page][nkv][hd] (quantised here)."""
        nkv, hd, page, dev = self.nkv, self.hd, self.page, k.device
        out = torch.zeros(k.shape[0], nkv * (page // 16) * 18 * hd, dtype=torch.uint8, device=dev)
        tok = torch.arange(page, device=dev).view(-1, 1, 1)
        j = torch.arange(nkv, device=dev).view(1, -1, 1)
        d = torch.arange(hd, device=dev).view(1, 1, -1)
        for kind, x in ((0, k), (1, v)):
            q, s = blocks(x.double())
            at, shift = place(nkv, hd, page, kind, j, tok, d)
            at = at.expand(page, nkv, hd).reshape(-1)
            val = (q << shift.expand(page, nkv, hd)).reshape(k.shape[0], -1)
            acc = torch.zeros(out.shape, dtype=torch.int64, device=dev)
            acc.index_add_(1, at, val)
            sat = scale_place(nkv, hd, page, kind, j, tok, torch.arange(hd // 32, device=dev).view(1, 1, -1))
            pair = s.contiguous().view(torch.uint8).unflatten(-1, (-1, 2))
            sat = sat.expand(page, nkv, hd // 32).reshape(-1)
            acc[:, sat] = pair[..., 0].reshape(k.shape[0], -1).long()
            acc[:, sat + 1] = pair[..., 1].reshape(k.shape[0], -1).long()
            out |= acc.to(torch.uint8)
        return out


def rope(x, cos, sin):
    h = x.shape[-1] // 2
    a, b = x[..., :h], x[..., h:]
    return torch.cat((a * cos - b * sin, b * cos + a * sin), -1)


def norm_rope(x, w, eps, cos, sin):
    """x [T][heads][hd] float64; cos / sin [T][hd / 2] or None."""
    if w is not None:
        x = x * (1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)) * w.double()
    if cos is not None:
        x = rope(x, cos[:, None].double(), sin[:, None].double())
    return x


def attention(q, k, v, scale):
    """q [n][NH][hd], k / v [L][NKV][hd] float64; query i sees rows 0 .. L - n + i.  Returns the
    output, sum p |v|, the largest sum |q||k| scale and the largest |v|, per (query, head)."""
    n, nh, hd = q.shape
    L, nkv = k.shape[:2]
    out, spread = torch.zeros_like(q), torch.zeros_like(q)
    size = torch.zeros(n, nh, 1, dtype=q.dtype, device=q.device)
    top = torch.zeros_like(size)
    if not L:
        return out, spread, size, top
    seen = torch.arange(L, device=q.device)[None] <= (L - n + torch.arange(n, device=q.device))[:, None]
    for h in range(nh):
        j = h // (nh // nkv)
        s = (q[:, h] @ k[:, j].T * scale).masked_fill(~seen, float("-inf"))
        ok = seen.any(1)
        p = torch.softmax(s[ok], 1)
        out[ok, h], spread[ok, h] = p @ v[:, j], p @ v[:, j].abs()
        top[ok, h] = v[:, j].abs().max()
        size[ok, h] = ((q[ok, h].abs() @ k[:, j].abs().T) * scale).masked_fill(~seen[ok], 0).amax(1, keepdim=True)
    return out, spread, size, top


def i8_rows(x, norm=None, eps=0.0):
    """(codes float64, scales float64) of the rows of x."""
    x = x.double()
    y = x if norm is None else x * norm.double()
    top = y.abs().amax(1, keepdim=True)
    codes = torch.where(top > 0, torch.round(127 * y / torch.where(top > 0, top, torch.ones_like(top))), torch.zeros_like(y))
    s = top / 127
    if norm is not None:
        s = s / torch.sqrt((x * x).mean(1, keepdim=True) + eps)
    return codes, s
