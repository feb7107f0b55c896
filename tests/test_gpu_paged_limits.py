"""GPU: the paged 8-bit cache and windowed attention (dsa_paged) at the limits of their number
formats: scales far apart or of pages of nobody, values near the largest, shares near the least, and
prompts that fill the card.  Against 64 bits, under paged_oracle's bounds."""
from __future__ import annotations

import math

import pytest
import torch

import dsa_paged as P
import paged_oracle as O
from test_gpu_paged import BF16, F16, F32, check_attention, check_window, filled, gen, ints, randn, state

pytestmark = pytest.mark.gpu


def unowned_poisoned(cache):
    """The same sequences in a pool whose first page and every other that is nobody's, and every
    block that no slot in use lies on, hold NaN with scales of 255."""
    per, page, lengths = cache.page // 64, cache.pages.cpu(), cache.length.tolist()
    keep = torch.zeros(cache.NP + 1, per, dtype=torch.bool)
    for b, n in enumerate(lengths):
        for blk in range(-(-n // 64)):
            keep[int(page[b, blk // per]) + 1, blk % per] = True
    codes = torch.cat([cache.codes[:1], cache.codes]).cpu().transpose(1, 2)
    scales = torch.cat([cache.scales[:1], cache.scales]).cpu().transpose(1, 2)
    codes[~keep], scales[~keep] = 0x7F, 0xFF
    dev = cache.device
    return P.KV8Cache(codes.transpose(1, 2).contiguous().to(dev), scales.transpose(1, 2).contiguous().to(dev),
                      cache.pages + 1, cache.length, DK=cache.DK)


# (own: a block's waves take slots of their own; shared: different rows of the same slots)
FEW = (2, [400, 390], 4, 1, 64, 4)      # own: B, lengths, HQ, HKV, D, Tq
SPLIT = (1, [9000], 4, 1, 64, 1)        # own, joined by a second launch
MANY = (8, [250 - b for b in range(8)], 64, 8, 128, 32)   # shared
PIECE = (1, [3100], 4, 1, 128, 1024)    # shared, joined; 16-bit types 32 rows a wave
LONG = (1, [6200], 4, 1, 64, 1024)      # own, 32 rows a wave, few splits joined by threads


@pytest.mark.parametrize("shape", [FEW, SPLIT, MANY, PIECE])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_pages_of_nobody_have_no_scale(dev, dtype, shape):
    """Ids that name no page among the slots that are seen: neither codes nor scales that lie
    elsewhere in the pool reach a row."""
    B, lengths, HQ, HKV, D, Tq = shape
    cache = unowned_poisoned(filled(dev, B, max(lengths) + 64, HKV, D, D, lengths, seed=D + Tq))
    for b, n in enumerate(lengths):
        blocks = -(-n // 64)
        cache.pages[b, 0 if b % 2 else blocks - 2] = cache.NP if b % 3 else -1
        cache.pages[b, blocks // 2] = -7
    Q = randn(gen(Tq), B, Tq, HQ, D, dtype=dtype)
    out, _ = check_attention(dev, cache, Q, dtype, None, 0)
    assert bool(out.isfinite().all())
    check_attention(dev, cache, Q, dtype, 150, 3)


def check_rows(dev, cache, Q, dtype, window):
    """check_attention, with a row's own largest |V|: among the slots that weigh more than 2^-60 in it
    (the tests' other ones weigh 2^-1000 and less, 0 in any p)."""
    B, Tq, HQ, D = Q.shape
    out = P.kv8_attention(cache, Q.to(dev), window=window).double().cpu()
    K, V = state(cache).values()
    G = HQ // cache.HKV
    for b, n in enumerate(cache.length.tolist()):
        ok = O.sees(n, n - Tq + torch.arange(Tq), torch.arange(cache.S), window, 0)
        ref, mass, big = O.attention(Q[b], K[b], V[b], ok, D ** -0.5)
        vmax = torch.zeros(Tq, HQ, 1, dtype=torch.float64)
        for h in range(HQ):
            p = torch.softmax((Q[b, :, h].double() @ K[b, :, h // G].nan_to_num().T * D ** -0.5).masked_fill(~ok, -math.inf), -1)
            vmax[:, h, 0] = torch.where(p > 2.0 ** -60, V[b, :, h // G].nan_to_num().abs().amax(-1), 0.0).amax(-1)
        lim = O.bound(dtype, n, D, mass, big, ref, False, vmax)
        err = (out[b] - ref).abs()
        assert bool((err <= lim).all()), (b, float((err / lim).max()))


@pytest.mark.parametrize("shape, window", [((2, [400, 400], 4, 1, 64, 2), 336), ((8, [200] * 8, 64, 8, 128, 32), 120)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_scales_that_weigh_nothing(dev, dtype, shape, window):
    """A block of very large values that some rows of a tile do not see, or in which no slot
    weighs anything for them, takes nothing from their small ones."""
    B, lengths, HQ, HKV, D, Tq = shape
    cache = filled(dev, B, 448, HKV, D, D, lengths, seed=D)
    first = cache.pages[:, 0].long()
    cache.scales[..., 1] -= 60
    cache.scales[first, :, 0, 1] += 160
    check_rows(dev, cache, randn(gen(Tq), B, Tq, HQ, D, dtype=dtype), dtype, window)
    # the block's keys all against the queries: logits of -14336 and less
    cache.codes[first, :, 0, :64 * D], cache.scales[first, :, 0, 0] = 0xFE, 127
    Q = 4.0 + 0.1 * randn(gen(Tq), B, Tq, HQ, D)
    check_rows(dev, cache, Q.to(dtype), dtype, None)


@pytest.mark.parametrize("shape", [FEW, SPLIT, MANY, PIECE, LONG])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_values_near_the_largest(dev, dtype, shape):
    """V up to 1.75 * 2^127, the largest that reads back as a number: a mean of them is one."""
    B, lengths, HQ, HKV, D, Tq = shape
    g = gen(D + Tq)
    S = -(-max(lengths) // 64) * 64
    cache = P.KV8Cache.empty(B, S, HKV, D, D, device=dev)
    K, V = randn(g, B, max(lengths), HKV, D), randn(g, B, max(lengths), HKV, D).clamp(-3.5, 3.5) * 2.0 ** 126
    V[:, :, :, 3] = 1.75 * 2.0 ** 127
    V[:, 5:, 0, 4] = -1.75 * 2.0 ** 127
    P.kv8_append(cache, K.to(dev), V.to(dev), count=ints(dev, lengths))
    Q = randn(gen(Tq), B, Tq, HQ, D, dtype=dtype)
    out, _ = check_attention(dev, cache, Q, dtype, None, 0)
    assert bool(out.isfinite().all()) and bool((out[..., 3].double() / (1.75 * 2.0 ** 127) - 1).abs().max() < 2.0 ** -8)


@pytest.mark.parametrize("B, HQ, D", [(1, 2, 32), (1, 2, 64), (1, 2, 128), (1, 2, 256), (16, 16, 64), (16, 16, 128)])
def test_small_shares_of_fp16_prompts(dev, B, HQ, D):
    """A first token 15 nats above all others, with a value of 0: what the others add, 2^-21.6 of
    their values each, keeps f16's precision.  Their logits are alike, so roundings of p add up.

    p is held as 2^10 and more times its share of the largest, so a share from 2^-24 on is a normal
    f16 and smaller ones are off by 2^-25 of the 2^10: n 2^-35 vmax in place of n 2^-24 vmax."""
    T = 500
    g = gen(D)
    Q = torch.ones(1, T, HQ, D)
    K = torch.zeros(1, T, 1, D)
    K[:, 0] = 15.0 / math.sqrt(D)
    V = 1.0 + 0.2 * randn(g, 1, T, 1, D)
    V[:, 0] = 0.0
    Q, K, V = Q.half(), K.half(), V.half()
    out = P.window_attention(*(x.to(dev).expand(B, -1, -1, -1) for x in (Q, K, V)))
    ref, mass, big = O.attention(Q[0], K[0], V[0], O.sees(T, torch.arange(T), torch.arange(T), None, 0), D ** -0.5)
    vmax = float(V.double().abs().max())
    lim = O.bound(F16, T, D, mass, big, ref, True, vmax * 2.0 ** -11)
    err = (out.double().cpu() - ref).abs() / lim
    assert float(err.max()) <= 1.0, float(err.max())


# Batches whose blocks fill the card, so that a block takes 128 queries (1024 blocks of 128 and more in 16
# bits, 512 in fp32), at windows that leave tiles which all queries of a block see whole.
@pytest.mark.parametrize("B, T, HQ, HKV, D, window, sinks, count, dtype", [
    (13, 520, 16, 2, 64, 400, 3, None, F16),
    (13, 520, 16, 2, 128, 391, 70, None, BF16),
    (13, 520, 16, 1, 128, None, 0, [520, 519, 1, 0, 64, 65, 128, 129, 200, 320, 400, 512, 513], F16),
    (13, 520, 16, 1, 64, None, 0, [513, 64, 520, 0, 449, 448, 447, 2, 257, 256, 255, 100, 384], BF16),
    (13, 520, 16, 1, 32, 330, 130, None, BF16),
    (13, 520, 8, 2, 64, 400, 3, None, F32),
    (13, 520, 8, 1, 32, None, 0, [520, 519, 1, 0, 64, 65, 128, 129, 200, 320, 400, 512, 513], F32),
])
def test_window_of_128_queries_a_block(dev, B, T, HQ, HKV, D, window, sinks, count, dtype):
    g = gen(B + T + D)
    Q, K, V = (randn(g, B, T, h, D, dtype=dtype) for h in (HQ, HKV, HKV))
    if count is not None:
        for b in range(B):
            Q[b, count[b]:], K[b, count[b]:], V[b, count[b]:] = math.nan, math.inf, math.nan
    check_window(dev, Q, K, V, dtype, window, sinks, count)


@pytest.mark.parametrize("D, dtype", [(32, BF16), (64, BF16), (64, F16), (128, BF16), (128, F16), (32, F32), (64, F32)])
def test_window_of_128_queries_keeps_what_is_not_seen_out(dev, D, dtype):
    """NaN and Inf in keys and values where a block takes 128 queries."""
    g = gen(D + 1)
    B, T, HQ, window = 13, 520, 8 if dtype == F32 else 16, 300
    Q, K, V = (randn(g, B, T, h, D, dtype=dtype) for h in (HQ, 2, 2))
    for b in range(0, B, 2):
        V[b, 30 + b, 0, 3], V[b, 100, 0, 7], V[b, 101, 0, 7], K[b, 170, 1, 5] = math.nan, math.inf, -math.inf, math.nan
        V[b, 1, 1, 2] = -math.inf
    out, _ = check_window(dev, Q, K, V, dtype, window, 2)
    half = HQ // 2
    assert bool(out[1::2].isfinite().all()) and bool(out[0, 30:330, :half, 3].isnan().all())
    assert bool(out[0, 100, :half, 7].isposinf().all()) and bool(out[0, 101:400, :half, 7].isnan().all()) and bool(out[0, 401:, :half].isfinite().all())
    assert bool((out[0, 1:170, half:, 2] == -math.inf).all()) and bool(out[0, 170:470, half:].isnan().all())
    assert bool((out[0, 470:, half:, 2] == -math.inf).all())


def test_windows_past_64_bits(dev):
    """A window or a number of first tokens that no 64-bit integer holds is all of them."""
    g = gen(5)
    Q, K, V = (randn(g, 1, 100, 2, 64, dtype=BF16).to(dev) for _ in range(3))
    every = P.window_attention(Q, K, V)
    for kw in (dict(window=2 ** 64 + 5), dict(window=2 ** 63), dict(window=3, sinks=2 ** 64), dict(window=3, sinks=2 ** 63 + 1)):
        assert torch.equal(P.window_attention(Q, K, V, **kw), every), kw
    cache = P.KV8Cache.empty(1, 128, 2, 64, 64, device=dev)
    P.kv8_append(cache, K, V)
    q = Q[:, -3:].contiguous()
    every = P.kv8_attention(cache, q)
    for kw in (dict(window=2 ** 64 + 5), dict(window=2 ** 63), dict(window=3, sinks=2 ** 64), dict(window=3, sinks=2 ** 63 + 1)):
        assert torch.equal(P.kv8_attention(cache, q, **kw), every), kw


@pytest.mark.parametrize("DK, DV, window, dtype", [(96, 96, None, BF16), (192, 192, 100, F32), (192, 128, None, F16)])
def test_prompts_over_the_pages(dev, DK, DV, window, dtype):
    """Whole prompts of a padded batch over the cache that they were appended to, at the head sizes
    that window_attention does not take."""
    g = gen(DK + DV)
    B, T, HQ, HKV, lengths = 3, 200, 4, 2, [200, 1, 130]
    rope = P.rope_tables(256, DK, device=dev)
    cache = P.KV8Cache.empty(B, 256, HKV, DK, DV, page=128, device=dev)
    Q, K, V = randn(g, B, T, HQ, DK, dtype=dtype), randn(g, B, T, HKV, DK, dtype=dtype), randn(g, B, T, HKV, DV, dtype=dtype)
    many = ints(dev, lengths)
    q, _ = P.kv8_append(cache, K.to(dev), V.to(dev), rope=rope, Q=Q.to(dev), count=many)
    check_attention(dev, cache, q.cpu(), dtype, window, 2, lengths)
