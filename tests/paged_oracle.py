"""The paged 8-bit cache and windowed attention from their definitions, on the CPU.

A cache is taken as logical arrays (Held): codes and scale bytes by sequence, slot and head,
whatever pages they lie on.  Attention is in 64 bits; its bounds are derived in `bound`."""
from __future__ import annotations

import math

import torch

BLOCK = 64


def place(t: int) -> int:
    """Where token t of a block lies in a dimension's 64 bytes of V."""
    return 16 * (t % 16 // 4) + 4 * (t // 16) + t % 4


PLACE = torch.tensor([place(t) for t in range(BLOCK)])


class Held:
    """k, v uint8 [B, S, HKV, D]; ks, vs uint8 [B, S/64, HKV] of a cache's tensors."""

    def __init__(self, codes, scales, pages, DK):
        codes, scales, pages = codes.cpu(), scales.cpu(), pages.cpu().long()
        per = codes.shape[2]
        DV = codes.shape[3] // BLOCK - DK
        B, n = pages.shape
        ok = (pages >= 0) & (pages < codes.shape[0])
        at = pages.clamp(0, codes.shape[0] - 1)
        c = codes[at].permute(0, 1, 3, 2, 4).reshape(B, n * per, -1, codes.shape[3])  # [B, blocks, HKV, bytes]
        s = scales[at].permute(0, 1, 3, 2, 4).reshape(B, n * per, -1, 2)
        self.page = ok.repeat_interleave(per, 1)  # [B, blocks]: whether there is one
        k = c[..., :BLOCK * DK].unflatten(-1, (BLOCK, DK))
        v = c[..., BLOCK * DK:].unflatten(-1, (DV, BLOCK))[..., PLACE].transpose(-1, -2)
        self.k, self.v = (x.transpose(2, 3).flatten(1, 2).contiguous() for x in (k, v))
        for x in (self.k, self.v):  # a NaN has two codes
            x[x == 255] = 127
        self.ks, self.vs = s[..., 0].contiguous(), s[..., 1].contiguous()

    def values(self):
        """K and V [B, S, HKV, D] in 64 bits; zeros on no page."""
        out = []
        for c, s in ((self.k, self.ks), (self.v, self.vs)):
            x = value(c) * torch.exp2(s.double() - 127).repeat_interleave(BLOCK, 1).unsqueeze(-1)
            x[~self.page.repeat_interleave(BLOCK, 1)] = 0
            out.append(x)
        return out


def value(code):
    """What an e4m3 code stands for: s eeee mmm, bias 7, S.1111.111 no number."""
    c = code.long()
    e, m = (c >> 3) & 15, (c & 7).double()
    x = torch.where(e == 0, m / 512, (1 + m / 8) * torch.exp2(e.double() - 7))
    x = torch.where(c & 127 == 127, torch.nan, x)
    return torch.where(c >= 128, -x, x)


GRID = value(torch.arange(127, dtype=torch.uint8))  # 0 .. 448, ascending with the code


def encode(x, byte: int):
    """x (64 bits) / 2^(byte-127) to the nearest code, ties to the even one; Inf and NaN to 0x7f."""
    y = x.abs() * 2.0 ** (127 - byte)
    hi = torch.searchsorted(GRID, y.contiguous()).clamp(max=126)
    lo = (hi - 1).clamp(min=0)
    up = GRID[hi] - y < y - GRID[lo]
    tie = GRID[hi] - y == y - GRID[lo]
    c = torch.where(up | (tie & (hi % 2 == 0)), hi, lo)
    c = torch.where(y == GRID[hi], hi, c)
    c = c + 128 * torch.signbit(x).long()
    return torch.where(torch.isfinite(x), c, 127).to(torch.uint8)


def need(x) -> int:
    """Scale byte of new values: the least e with max <= 448 2^e."""
    top = float(torch.where(torch.isfinite(x), x, 0).abs().max()) if x.numel() else 0.0
    e = -117
    while e < 120 and top > 448 * 2.0 ** e:
        e += 1
    return e + 127


def rotate(x, cos, sin, at, pairs):
    """x [T, H, D] fp32, elementary operations in 32 bits."""
    x = x.float()
    R = 2 * cos.shape[1]
    c, s = cos[at].unsqueeze(1), sin[at].unsqueeze(1)
    a, b = (x[..., 0:R:2], x[..., 1:R:2]) if pairs else (x[..., :R // 2], x[..., R // 2:R])
    u, v = a * c - b * s, b * c + a * s
    y = torch.stack([u, v], -1).flatten(-2) if pairs else torch.cat([u, v], -1)
    return torch.cat([y, x[..., R:]], -1)


def append(h: Held, b: int, start: int, K, V) -> int:
    """K, V [n, HKV, D] fp32 (rotated) into slots start .. of sequence b; how many were lost."""
    n, S = K.shape[0], h.k.shape[1]
    lost = max(0, start + n - S)
    end = min(start + n, S)
    for blk in range(start // BLOCK, -(-end // BLOCK)):
        lo, hi = max(start, blk * BLOCK), min(end, (blk + 1) * BLOCK)
        if not h.page[b, blk]:
            lost += hi - lo
            continue
        for codes, scales, x in ((h.k, h.ks, K), (h.v, h.vs, V)):
            for j in range(x.shape[1]):
                new = x[lo - start:hi - start, j].double()
                e = need(new)
                if lo > blk * BLOCK:
                    old = int(scales[b, blk, j])
                    e = max(e, old)
                    if e > old:
                        held = codes[b, blk * BLOCK:lo, j]
                        codes[b, blk * BLOCK:lo, j] = encode(value(held) * 2.0 ** (old - 127), e)
                scales[b, blk, j] = e
                codes[b, lo:hi, j] = encode(new, e)
    return lost


def sees(n_all, t, s, window, sinks):
    """[len(t), len(s)]: whether the token at position t sees position s."""
    t, s = t.view(-1, 1), s.view(1, -1)
    ok = s <= t
    if window:
        ok = ok & ((s > t - window) | (s < sinks))
    return ok & (s < n_all)


def attention(q, k, v, ok, scale):
    """q [T, H, D], k, v [S, HKV, D] in 64 bits, ok [T, S] -> (O [T, H, DV], sum p |v|,
    largest sum |q k| scale of a row).  What is not seen is not read."""
    T, H, _ = q.shape
    G = H // k.shape[1]
    out = torch.full((T, H, v.shape[2]), math.nan, dtype=torch.float64)
    mass = torch.zeros_like(out)
    big = torch.zeros(T, H, 1, dtype=torch.float64)
    for t in range(T):
        at = ok[t].nonzero().view(-1)
        if not len(at):
            continue
        for j in range(k.shape[1]):
            rows = slice(j * G, (j + 1) * G)
            qq, kk, vv = q[t, rows].double(), k[at, j].double(), v[at, j].double()
            p = torch.softmax(qq @ kk.T * scale, -1)
            out[t, rows] = p @ vv
            mass[t, rows] = p @ vv.abs()
            big[t, rows, 0] = (qq.abs() @ kk.abs().T).amax(-1) * abs(scale)
    return out, mass, big


# p's rounding before its product with V: fp32 as two f16 pieces (2^-22 at least) or whole;
# 16-bit types over the cache as f16 (2^-11 halved: 2^-12); prompts in the inputs' own type.
def bound(dtype, n, D, mass, big, O, prompt: bool, vmax: float):
    """|error| of O against 64 bits.

    A logit is a sum of D products: at most (D + 8) 2^-24 big off (big: the sum of their
    magnitudes; the scale, the log2 factor and the row's power of two take the rest; Q as two
    f16 pieces 2^-22 big more in fp32), which moves p by as much relative to it, exp2 by 2^-22.
    p is rounded (r), the sums over n of p and of p v add at most (n + 8) 2^-24.
    Numerator and denominator may be off by all of it in opposite directions: twice.  f16
    pieces below its normal range are off by 2^-25 where the largest p is 1 at least.  The
    output's own rounding is half a step, and half the least subnormal of its type."""
    r = {torch.float32: 2.0 ** -22, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}[dtype]
    if not prompt and dtype != torch.float32:
        r = 2.0 ** -12
    eps = (D + 8) * 2.0 ** -24 * big + 2.0 ** -22 * big + 2.0 ** -21 + r + (n + 8) * 2.0 ** -24
    f = torch.finfo(dtype)
    return 2 * eps * mass + n * 2.0 ** -24 * vmax + O.abs() * (f.eps / 2) + f.smallest_normal * f.eps / 2
