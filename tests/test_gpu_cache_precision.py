"""The 24 bits of the 4-bit cache's attention: that no bf16 piece of p or of Q is lost.

Inputs whose sums have few terms other than 0, all >= 0, so that a bound of some
u = 2^-24 can be derived and a lost third piece (of p 177 u on average) passes it.
N slots count; all others' logits lie so far below that their p is 0, in every tile,
wave and block of a long cache.  Dot products are exact in fp32.  With x a logit in
powers of 2, X = max |x|, R = max x - min x over the slots that count:

    x comes of a factor of three roundings (3 u |x|), loses u R against the running
    maximum, and u R in each of the factors of a moved maximum, of the waves' join and
    of the blocks': an exponential's factor is within ln 2 (3 X + 4 R) u;
    four exponentials are within 2 u each, and are multiplied (2 u and 1 u more in the
    joins): 10 u with them;
    the sum of p V has at most 5 N + 2 additions of terms other than 0 (three pieces a
    slot, the pieces' join, the waves' and the blocks'), each within 2 u of a partial sum;
    the sum of p has the exponentials' errors and 3 N additions within u;
    the division is within 3 u.
"""
from __future__ import annotations

import math

import pytest
import torch

import cache_oracle as C
import dsa_cache as D
from helpers import say

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
GRID = torch.tensor(C.GRID)
CASES = [  # S, HQ, HKV, DK, DV, Tq, listed: up to five rows and more, one block a row and many
    (200, 4, 4, 32, 32, 1, 0), (5000, 32, 8, 128, 128, 1, 0), (9000, 16, 1, 128, 128, 1, 0), (300, 24, 1, 64, 64, 1, 0),
    (5000, 8, 8, 64, 64, 1, 700), (5000, 16, 2, 96, 96, 2, 2100), (1100, 4, 2, 128, 128, 2, 0),
    (1100, 12, 2, 64, 64, 7, 0), (3000, 8, 2, 192, 128, 1, 0), (3000, 16, 1, 192, 192, 1, 0), (3000, 6, 2, 256, 256, 3, 0),
]


def limit(x, N):
    """x [..., N] fp64 logits in powers of 2: the bound, relative to sum p |V|."""
    X, R = x.abs().amax(-1), x.amax(-1) - x.amin(-1)
    return (2 * (math.log(2) * (3 * X + 4 * R) + 10) + 2 * (5 * N + 2) + 3 * N + 3) * C.U


def counted(S, HKV, DK, DV, Tq, seed, pieces_of_q, B=4, N=3):
    """K, V [B,S,HKV,D], Q's rows [B,Tq,64,DK], the slots that count [B,N] (on the CPU)."""
    g = torch.Generator().manual_seed(seed)
    K, V = torch.zeros(B, S, HKV, DK), GRID[torch.randint(1, 8, (B, S, HKV, DV), generator=g)]
    K[..., 0] = -12288.0  # a logit of -768 and below against Q's 1: p is 0
    at = torch.stack([torch.randperm(S - Tq, generator=g)[:N] for _ in range(B)])
    at[0, 0], at[1, -1] = 0, S - Tq
    Q = torch.randint(-16, 17, (B, Tq, 64, DK), generator=g) / 8.0
    for b in range(B):
        if pieces_of_q:  # one element of Q, with all its bits, against nothing
            K[b, at[b]] = 0
            K[b, at[b, 1], :, 1] = 1.0
            V[b, at[b, 1:]] = 0
        else:
            K[b, at[b]] = GRID[torch.randint(0, 8, (N, HKV, DK), generator=g)] / 8 * torch.randint(0, 2, (N, HKV, DK), generator=g).mul(2).sub(1)
            K[b, at[b], :, 0] = 0
    if pieces_of_q:
        Q[..., 1] = (3 + 2 * torch.rand(B, Tq, 64, generator=g)) * math.sqrt(DK)
    Q[..., 0] = 1.0
    return K, V, Q, at


def exact(K, V, Q, at, G):
    """(logits in powers of 2 [B,Tq,HQ,N], V [B,1,HQ,N,DV], O), 64 bits, of the slots that count."""
    b = torch.arange(len(K)).view(-1, 1)
    k, v = (x[b, at].double().transpose(1, 2).repeat_interleave(G, 1) for x in (K, V))  # [B,HQ,N,D]
    q = Q[:, :, :k.shape[1]].double()
    x = (q.unsqueeze(-2) * k.unsqueeze(1)).sum(-1) / math.sqrt(K.shape[-1]) / math.log(2)
    p = torch.exp2(x - x.amax(-1, keepdim=True))
    return x, v.unsqueeze(1), (p.unsqueeze(-1) * v.unsqueeze(1)).sum(-2) / p.sum(-1, keepdim=True)


def pieces(x, n):
    """fp32 x as the sum of its first n bf16 pieces, cut off."""
    total = torch.zeros_like(x)
    for _ in range(n):
        total += ((x - total).view(torch.int32) & -65536).view(torch.float32)
    return total


@pytest.mark.parametrize("of_q", [False, True])
@pytest.mark.parametrize("S, HQ, HKV, DK, DV, Tq, listed", CASES)
def test_the_bound_tells_two_pieces_from_three(S, HQ, HKV, DK, DV, Tq, listed, of_q):
    K, V, Q, at = counted(S, HKV, DK, DV, Tq, S + DK, of_q)
    x, v, O = exact(K, V, Q, at, HQ // HKV)
    lim = limit(x, 3).unsqueeze(-1) * O
    for n in (2, 3):
        if of_q:
            q = Q.clone()
            q[..., 1] = pieces(Q[..., 1].contiguous(), n)
            got = exact(K, V, q, at, HQ // HKV)[2]
        else:
            p = torch.exp2(x - x.amax(-1, keepdim=True)).float()
            got = (pieces(p, n).double().unsqueeze(-1) * v).sum(-2) / p.double().sum(-1, keepdim=True)
        beyond = ((got - O).abs() > lim).double().mean()
        assert beyond == 0 if n == 3 else beyond > 0.25, (n, beyond)


@pytest.mark.gpu
@pytest.mark.parametrize("of_q, dtype", [(False, F32), (False, BF16), (False, F16), (True, F32), (True, F16)])
@pytest.mark.parametrize("S, HQ, HKV, DK, DV, Tq, listed", CASES)
def test_every_piece_counts(dev, S, HQ, HKV, DK, DV, Tq, listed, of_q, dtype):
    say("pieces", S, HQ, HKV, DK, DV, Tq, listed, of_q, dtype)
    K, V, Q, at = counted(S, HKV, DK, DV, Tq, S + DK, of_q)
    Q = Q[:, :, :HQ].to(dtype)
    (kc, ks), (vc, vs) = C.quantise(K.to(dev)), C.quantise(V.to(dev))
    assert torch.equal(C.decode(kc, ks).float().cpu(), K) and torch.equal(C.decode(vc, vs).float().cpu(), V)
    cache = D.KV4Cache(torch.cat([kc, vc], -1), torch.cat([ks, vs], -1),
                       torch.full((len(K),), S, device=dev, dtype=torch.int32), DK=DK)
    slots = None
    if listed:  # what counts, once, among the others and entries that are none
        g = torch.Generator().manual_seed(listed)
        slots = torch.randint(-9, S + 9, (len(K), Tq, listed), generator=g, dtype=torch.int32)
        slots[(slots.unsqueeze(-1) == at.view(len(K), 1, 1, -1)).any(-1)] = -1
        for b in range(len(K)):
            for t in range(Tq):
                slots[b, t, torch.randperm(listed, generator=g)[:3]] = at[b].int()
        slots = slots.to(dev)
    x, _, O = exact(K, V, Q, at, HQ // HKV)
    rel = ((D.kv4_attention(cache, Q.to(dev), slots=slots).cpu().double() - O).abs() / O).amax(-1)
    worst = float((rel / limit(x, 3)).max())
    say(f"{worst:.3f} of the bound, {float(rel.max() / C.U):.1f} u")
    assert worst <= 1
