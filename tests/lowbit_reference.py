"""64-bit forms of the low-bit operators for the tests, on the CPU: e4m3 values,
power-of-two block scales, append, attention, 4-bit projections."""
from __future__ import annotations

import math

import torch

PAGE, BLOCK = 64, 16


def e4m3_table():
    """The value of each of the 256 codes."""
    c = torch.arange(256, dtype=torch.int64)
    e, m = (c >> 3) & 15, c & 7
    v = torch.where(e > 0, (8 + m).double() * 2.0 ** (e.double() - 10), m.double() * 2.0 ** -9)
    v = torch.where((c & 127) == 127, torch.full_like(v, math.nan), v)
    return torch.where(c >= 128, -v, v)


def e4m3_round(x):
    """Nearest e4m3 value, ties to even, largest 448."""
    x = x.double()
    _, e = torch.frexp(x.abs().clamp(min=2.0 ** -30))
    step = torch.ldexp(torch.ones_like(x), (e - 1).clamp(min=-6) - 3)
    return (torch.round(x / step) * step).clamp(-448, 448)


def block_scale(amax):
    """Smallest 2^e, e >= -126, with amax <= 448 * 2^e."""
    e = torch.full_like(amax, -126.0)
    lo, e0 = torch.frexp(amax.double() / 448.0)
    want = torch.where(lo > 0.5, e0, e0 - 1).double()
    return torch.exp2(torch.where(amax > 0, torch.maximum(e.double(), want), e.double()))


def norm_rope(x, w, cos, sin, eps):
    """x [..., hd] in 64 bits, w [hd] or None, cos/sin [..., hd / 2]."""
    x = x.double()
    if w is not None:
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * w.double()
    a, b = x.chunk(2, -1)
    cos, sin = cos.double(), sin.double()
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


class Cache:
    """A cache on the host as values: codes [n_pages][layers][2][nkv][64][hd] (float64 e4m3 values), scales."""

    def __init__(self, codes, scales):
        self.codes = e4m3_table()[codes.long()]
        self.scales = scales.double()

    def append(self, layer, table_row, pos0, kv):
        """kv [2][nkv][n][hd] in 64 bits to positions pos0 ..."""
        n = kv.shape[2]
        p = pos0
        while p < pos0 + n:
            lo = p // BLOCK * BLOCK
            hi = min(lo + BLOCK, pos0 + n)
            page, b, o = int(table_row[lo // PAGE]), lo % PAGE // BLOCK, lo % PAGE
            new = kv[:, :, p - pos0:hi - pos0]
            amax = new.abs().amax((-1, -2))
            lost = ~torch.isfinite(new).all(-1).all(-1)
            s = block_scale(torch.where(lost, torch.zeros_like(amax), amax))
            if p > lo:
                had = self.scales[page, layer, :, :, b]
                s = torch.maximum(s, had)
                lost = lost | s.isnan()
                old = self.codes[page, layer, :, :, o:o + p - lo]
                self.codes[page, layer, :, :, o:o + p - lo] = torch.where(
                    (s > had)[..., None, None] & ~lost[..., None, None], e4m3_round(old * (had / s)[..., None, None]), old)
            codes = e4m3_round(torch.where(lost[..., None, None], torch.zeros_like(new), new / s[..., None, None]))
            self.codes[page, layer, :, :, o + p - lo:o + hi - lo] = codes
            self.scales[page, layer, :, :, b] = torch.where(lost, torch.full_like(s, math.nan), s)
            p = hi

    def read(self, layer, table_row, n):
        """[2][nkv][n][hd]"""
        pages = torch.as_tensor(table_row[: -(-n // PAGE)]).long()
        x = self.codes[pages, layer].unflatten(3, (PAGE // BLOCK, BLOCK)) * self.scales[pages, layer][..., None, None]
        return x.permute(1, 2, 0, 3, 4, 5).reshape(x.shape[1], x.shape[2], -1, x.shape[-1])[:, :, :n]


def attention(q, kv, pos):
    """q [nq][hd], kv [2][nkv][n][hd] in 64 bits, positions 0..pos seen. Returns the output and a bound of what an
    output in fp16 computed in fp32 with fp16 weights p may be off."""
    nq, hd = q.shape
    nkv = kv.shape[1]
    q = q.double().view(nkv, nq // nkv, hd)
    k, v = kv[0][:, :pos + 1], kv[1][:, :pos + 1]
    s = q @ k.transpose(1, 2) / math.sqrt(hd)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    total = p.sum(-1, keepdim=True)
    out = p @ v / total
    size = p @ v.abs() / total
    # p to fp16: half a step, 2^-11 of p, or 2^-25 where p is subnormal; the output to fp16: 2^-11 and 2^-25;
    # scores in fp32: products are exact, hd sums and two factors round (2^-23 counts truncating adders), their error
    # is the weights' relative error twice (numerator and total); exp2 and the sums: a few 2^-23 each.
    off = (q.abs() @ k.abs().transpose(1, 2) / math.sqrt(hd)).amax(-1, keepdim=True) * (hd + 4) * 2.0 ** -23
    tol = 2.0 ** -11 * out.abs() + 2.0 ** -25
    tol = tol + (2.0 ** -11 + 2 * off + 64 * 2.0 ** -23) * size + 2.0 ** -25 * v.abs().sum(1, keepdim=True) / total
    return out.reshape(nq, hd), tol.reshape(nq, hd)


def w4_weights(codes, scales, zeros, group):
    """[n][k] in 64 bits."""
    w = torch.stack([codes & 15, codes >> 4], -1).reshape(codes.shape[0], -1).double()
    z = 8.0 if zeros is None else zeros.double().repeat_interleave(group, 1)
    return (w - z) * scales.double().repeat_interleave(group, 1)
