"""The 4-bit cache and its operators in 64 bits, from their definitions, for the
tests (CPU or GPU tensors; no kernel of the library).

Bounds: u = 2^-24 is half a step of fp32.  A dot product of D products summed in
fp32 in any order is off by at most (D + 1) u sum|x y|; operands wider than the
matrix instruction's enter as pieces, whose products count each (PIECES: fp32 as
three of bf16, fp16 as two; of two fp32 operands the six largest, which leaves
out 2 u more); a logit adds the scale's rounding.  A logit off by d moves a probability by a factor within 1 +- (2 d +
d^2), normaliser included; an exponential by a few u; a probability held as two
bf16 pieces by 2^-16; sums over the slots run in chains of at most n/32 + 64
additions."""
from __future__ import annotations

import math

import torch

GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
U = 2.0 ** -24
PIECES = {torch.float32: 3, torch.float16: 2, torch.bfloat16: 1}


def decode(codes, scales):
    """codes [..., D/2] uint8, scales [..., D/32] uint8 -> float64 [..., D]."""
    lut = torch.tensor(GRID + tuple(-g for g in GRID), dtype=torch.float64, device=codes.device)
    v = torch.stack([lut[(codes & 15).long()], lut[(codes >> 4).long()]], -1).flatten(-2)
    s = torch.exp2(scales.double() - 127)
    s = torch.where(scales == 255, torch.full_like(s, math.nan), s)
    return (v.unflatten(-1, (-1, 32)) * s.unsqueeze(-1)).flatten(-2)


def quantise(x):
    """x [..., D] -> (codes, scales) as the format prescribes."""
    y = x.double().unflatten(-1, (-1, 32))
    top = y.abs().amax(-1)  # NaN where there is one
    bad = ~torch.isfinite(top)
    t = torch.where(bad | (top == 0), torch.ones_like(top), top)
    m, e = torch.frexp(t)  # t = m 2^e, 1/2 <= m < 1: the least e' with t < 7 2^e'
    e = torch.where(m < 0.875, e - 3, e - 2)
    e = torch.where(top == 0, torch.full_like(e, -1000), e).clamp(-125, 125)
    r = torch.where(bad.unsqueeze(-1), torch.zeros_like(y), y).abs() / torch.exp2(e.double()).unsqueeze(-1)
    dist = (r.unsqueeze(-1) - torch.tensor(GRID, dtype=torch.float64, device=x.device)).abs()
    near = dist.amin(-1, keepdim=True)
    hit = dist == near  # one code, or two neighbours of which the even one counts
    even = torch.arange(8, device=x.device) % 2 == 0
    code = torch.where(hit.sum(-1) > 1, (hit & even).int().argmax(-1), hit.int().argmax(-1))
    code = code + 8 * torch.signbit(torch.where(bad.unsqueeze(-1), torch.zeros_like(y), y)).int()
    code = torch.where(bad.unsqueeze(-1), torch.zeros_like(code), code).flatten(-2)
    byte = torch.where(bad, torch.full_like(e, 255), e + 127)
    return (code[..., 0::2] + 16 * code[..., 1::2]).to(torch.uint8), byte.to(torch.uint8)


def visible(length, count, Tq, S):
    """bool [B, Tq, S]: the slots each query sees."""
    length = length.clamp(0, S).view(-1, 1, 1)
    n = (torch.full_like(length, Tq) if count is None else count.clamp(0, Tq).view(-1, 1, 1))
    t = torch.arange(Tq, device=length.device).view(1, -1, 1)
    last = torch.where(t < n, length - n + t + 1, torch.zeros_like(length))
    return torch.arange(S, device=length.device) < last


def indexer(k_idx, length, q, w, count=None, span=None):
    """(scores float64 [B,Tq,span], bound on an fp32 computation's error)."""
    B, S, DI = k_idx.shape
    Tq, HI = q.shape[1:3]
    span = S if span is None else span
    k = k_idx[:, :span].double().transpose(1, 2).contiguous()
    qf = q.double().reshape(B, Tq * HI, DI)
    dots = torch.bmm(qf, k).view(B, Tq, HI, span)
    size = torch.bmm(qf.abs(), k.abs()).view(B, Tq, HI, span)
    wd = w.double().unsqueeze(-1)
    score = (wd * dots.clamp(min=0)).sum(2)
    bound = (wd.abs() * size).sum(2) * ((6 if q.dtype == torch.float32 else 1) * DI + HI + 6) * U
    ok = visible(length, count, Tq, S)[..., :span]
    return score.masked_fill(~ok, -math.inf), bound


def attention(codes, scales, DK, length, Q, slots=None, span=None, count=None, dtype=None):
    """(O float64 [B,Tq,HQ,DV], its bound, added weight [B,S], its bound); dtype: what the
    kernel had Q in, where that is not Q's here."""
    B, S, HKV = codes.shape[:3]
    Tq, HQ = Q.shape[1:3]
    G = HQ // HKV
    DV = 2 * codes.shape[3] - DK
    O = torch.full((B, Tq, HQ, DV), math.nan, dtype=torch.float64, device=codes.device)
    lim = torch.zeros_like(O)
    add = torch.zeros(B, S, dtype=torch.float64, device=codes.device)
    addlim = torch.zeros_like(add)
    ok = visible(length, count, Tq, S)
    for b in range(B):
        for t in range(Tq):
            at = torch.arange(S if span is None else span, device=codes.device)
            if slots is not None:
                at = slots[b, t].long()
                at = at[(at >= 0) & (at < S)]
            at = at[ok[b, t, at]]
            n = len(at)
            if n == 0:
                continue
            for h in range(HKV):
                K = decode(codes[b, at, h, :DK // 2], scales[b, at, h, :DK // 32])
                V = decode(codes[b, at, h, DK // 2:], scales[b, at, h, DK // 32:])
                q = Q[b, t, h * G:(h + 1) * G].double()
                lg = q @ K.t().contiguous() / math.sqrt(DK)
                d = ((PIECES[dtype or Q.dtype] * DK + 3) * U * (q.abs() @ K.abs().t().contiguous()) / math.sqrt(DK)).amax(-1, keepdim=True)
                p = torch.softmax(lg, -1)
                O[b, t, h * G:(h + 1) * G] = p @ V
                rel = 2 * d + d * d + 16 * U
                lim[b, t, h * G:(h + 1) * G] = (p @ V.abs()) * (rel + 2.0 ** -16 + 2 * (n / 32 + 64) * U)
                add[b].index_add_(0, at, p.sum(0))
                addlim[b].index_add_(0, at, (p * (rel + (n / 32 + 64) * U)).sum(0))
    return O, lim, add, addlim + add * (HQ * Tq) * U


def evict(length, seen, position, weight, keep, recent):
    """Per sequence: (src list, dst list, new length), by sorting."""
    out = []
    B, S = weight.shape
    for b in range(B):
        n = max(0, min(int(length[b]), S))
        if n <= keep:
            out.append(([], [], int(length[b])))
            continue

        def rank(s):
            w = float(weight[b, s])
            safe = int(position[b, s]) >= int(seen[b]) - recent
            return (not safe, 0 if safe or not math.isnan(w) else -1,
                    0.0 if safe or math.isnan(w) else -w, s)

        kept = set(sorted(range(n), key=rank)[:keep])
        src = [s for s in range(keep, n) if s in kept]
        dst = [s for s in range(min(keep, n)) if s not in kept]
        out.append((src, dst, keep))
    return out
