"""GPU: the paged 8-bit cache and windowed attention (dsa_paged) where offsets pass 32 bits, heads
are few, odd or many, and the work is split and joined: against 64 bits, or bit for bit against
the same values where they lie close together."""
from __future__ import annotations

import math

import pytest
import torch

import dsa_paged as P
import paged_oracle as O
from test_gpu_paged import BF16, F16, F32, check_attention, check_window, eq, filled, gen, ints, randn, same, state

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B, T, HKV, D, HQ, pairs, dtype", [
    (3, 200, 5, 32, 7, False, BF16),   # four heads side by side, the last alone
    (2, 131, 3, 64, 5, True, F32),     # two, likewise
    (1, 700, 1, 32, 1, False, F16),
    (40, 70, 9, 64, 2, False, F16),    # groups of several heads
    (70, 129, 6, 32, 11, False, BF16),
    (2, 5, 2, 256, 8, False, BF16),    # the shortest prompt
])
def test_prompts_of_odd_heads(dev, B, T, HKV, D, HQ, pairs, dtype):
    g = gen(HKV + D)
    S = 768
    cache = P.KV8Cache.empty(B, S, HKV, D, D, page=128, device=dev)
    want = state(cache)
    rope = P.rope_tables(S, D, device="cpu")
    K, V, Q = (randn(g, B, T, h, D, dtype=dtype) for h in (HKV, HKV, HQ))
    start = [(7 * b) % 66 for b in range(B)]
    count = [T - b % 3 for b in range(B)]
    q, k = P.kv8_append(cache, K.to(dev), V.to(dev), rope=tuple(x.to(dev) for x in rope), pairs=pairs, Q=Q.to(dev),
                        start=ints(dev, start), count=ints(dev, count), keys=True)
    for b in range(B):
        at = torch.arange(start[b], start[b] + T)
        kr = O.rotate(K[b], *rope, at, pairs)
        assert eq(k[b].cpu(), kr.to(dtype)) and eq(q[b].cpu(), O.rotate(Q[b], *rope, at, pairs).to(dtype)), b
        # (slots before start are taken as held: zeros of the least scale)
        assert O.append(want, b, start[b], kr[:count[b]], V[b, :count[b]].float()) == 0
    got = state(cache)
    assert cache.length.tolist() == [s + n for s, n in zip(start, count)] and not cache.lost.any()
    for n in ("ks", "vs", "k", "v"):
        assert eq(getattr(got, n), getattr(want, n)), n


@pytest.mark.parametrize("B, lengths, HQ, HKV, DK, DV, Tq, window, sinks, count, span, scale, dtype", [
    (2, [300, 111], 8, 2, 256, 256, 20, None, 0, None, None, None, BF16),   # 80 rows of 256
    (2, [300, 111], 8, 2, 256, 256, 9, 70, 2, [9, 4], None, None, F32),
    (1, [1400], 16, 1, 192, 192, 3, None, 0, None, None, None, F16),        # shared, split and joined
    (2, [500, 90], 6, 1, 192, 128, 30, 130, 5, None, None, None, BF16),     # 180 rows, two tiles
    (1, [20000], 4, 1, 64, 64, 1, None, 0, None, None, None, BF16),         # tens of splits
    (1, [20000], 4, 1, 64, 64, 1, 9000, 65, None, 19990, None, F32),
    (2, [900, 640], 4, 2, 96, 96, 17, None, 0, None, 700, -0.2, F16),       # the last tokens beyond the span
    (2, [300, 64], 4, 4, 128, 128, 2, None, 0, None, None, 0.0, F32),       # the mean of what is seen
    (3, [0, 64, 65], 3, 3, 32, 32, 1, 64, 0, None, None, None, F16),
])
def test_attention_of_more_shapes(dev, B, lengths, HQ, HKV, DK, DV, Tq, window, sinks, count, span, scale, dtype):
    S = -(-max(lengths) // 64) * 64 + 64
    cache = filled(dev, B, S, HKV, DK, DV, lengths, 64, seed=HQ + Tq)
    Q = randn(gen(Tq + DK), B, Tq, HQ, DK, dtype=dtype)
    check_attention(dev, cache, Q, dtype, window, sinks, count, span, scale)


@pytest.mark.parametrize("B, length, HQ, HKV, D, Tq, window, sinks, count, dtype", [
    (1, 6200, 4, 1, 64, 1024, None, 0, None, BF16),     # 32 rows a wave, waves of their own slots, four splits
    (1, 6200, 4, 1, 96, 1024, None, 0, [1000], F16),
    (1, 3100, 4, 1, 128, 1024, None, 0, None, BF16),    # 32 rows a wave, shared, sixteen splits
    (1, 3100, 4, 1, 128, 1024, None, 0, [1001], F32),
    (1, 2500, 8, 1, 128, 1024, 700, 70, None, F16),
    (1, 4200, 4, 1, 256, 512, 4000, 3, None, BF16),
    (1, 4200, 4, 1, 192, 512, None, 0, None, F32),
    (8, 200, 64, 8, 64, 32, None, 0, [32, 0, 1, 31, 32, 32, 17, 32], BF16),   # a few slots, shared
    (8, 150, 64, 8, 32, 32, 40, 1, None, F32),
    (8, 66, 64, 8, 96, 32, None, 0, None, F16),
    (8, 200, 64, 8, 128, 32, 64, 0, None, F32),
    (1, 300, 8, 1, 32, 600, None, 0, None, BF16),       # more tokens than slots, chunks fewer than XCDs
])
def test_pieces_of_many_rows(dev, B, length, HQ, HKV, D, Tq, window, sinks, count, dtype):
    """Pieces of prompts behind a cache.  NaN of a late slot's V reaches the rows that see it alone."""
    lengths = [length - 3 * b for b in range(B)]
    S = -(-length // 64) * 64 + 64
    cache = filled(dev, B, S, HKV, D, D, lengths, 64, seed=D + Tq)
    for b, at in enumerate(n - 5 for n in lengths):
        row = cache.codes[cache.pages[b, at // 64], 0, 0]
        row[64 * D:].view(D, 64)[::7, O.PLACE[at % 64]] = 0x7F
    Q = randn(gen(Tq + D), B, Tq, HQ, D, dtype=dtype)
    out, _ = check_attention(dev, cache, Q, dtype, window, sinks, count)
    assert bool(out[0, :2].isfinite().all()) or length < Tq


def test_pages_past_32_bits(dev):
    """Pages beyond 4 GiB of codes hold and give what the same tokens do in a small pool."""
    HKV, D, page, S, T = 8, 128, 4096, 8192, 5000
    NP = 560  # of 8 MiB
    g = gen(3)
    Q, K, V = (randn(g, 1, T, h, D, dtype=BF16).to(dev) for h in (16, HKV, HKV))
    rope = P.rope_tables(S, D, device=dev)
    small = P.KV8Cache.empty(1, S, HKV, D, D, page=page, device=dev)
    big = P.KV8Cache.empty(1, S, HKV, D, D, page=page, NP=NP, device=dev)
    assert big.codes.numel() > 1 << 32
    big.pages.copy_(ints(dev, [[NP - 1, NP - 2]]))
    outs = []
    for c in (small, big):
        q, _ = P.kv8_append(c, K[:, :T - 1], V[:, :T - 1], rope=rope, Q=Q[:, :T - 1])
        q1, _ = P.kv8_append(c, K[:, T - 1:], V[:, T - 1:], rope=rope, Q=Q[:, T - 1:])
        some = ints(dev, [[4999, 0, 4095, 4096, 77]])
        outs.append([P.kv8_attention(c, q1), P.kv8_attention(c, q1, window=1000, sinks=4), P.kv8_attention(c, q[:, -40:].contiguous()),
                     *P.kv8_rows(c, span=T, dtype=BF16), *P.kv8_rows(c, some)])
        c.check()
    for i, (a, b) in enumerate(zip(*outs)):
        assert same(a, b), i
    assert same(big.codes[NP - 1], small.codes[0]) and same(big.scales[NP - 2], small.scales[1])
    assert not big.codes[:NP - 2].any()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_strides_past_32_bits(dev, dtype):
    """Columns of rows so wide that a sequence's end lies past 4 GiB."""
    B, T, HQ, HKV, D = 1, 300, 2, 1, 64
    ld = (1 << 24) // (2 if dtype == F32 else 1)
    g = gen(4)
    data = randn(g, B, T, (HQ + 2 * HKV) * D, dtype=dtype).to(dev)
    wide = torch.empty(B, T, ld, dtype=dtype, device=dev)
    assert wide.numel() * wide.element_size() > 1 << 32
    wide[..., -data.shape[2]:] = data

    def columns(y):
        y = y[..., -data.shape[2]:]
        return (y[..., :HQ * D].unflatten(-1, (HQ, D)), y[..., HQ * D:(HQ + HKV) * D].unflatten(-1, (HKV, D)),
                y[..., (HQ + HKV) * D:].unflatten(-1, (HKV, D)))

    q, k, v = columns(wide)
    assert P._tokens(k, dtype)[1:] == (k.data_ptr(), ld)
    assert same(P.window_attention(q, k, v, window=90, sinks=3), P.window_attention(*(x.contiguous() for x in (q, k, v)), window=90, sinks=3))
    a, b = (P.KV8Cache.empty(B, 320, HKV, D, D, device=dev) for _ in range(2))
    rope = P.rope_tables(320, D, device=dev)
    x = P.kv8_append(a, k, v, rope=rope, Q=q, keys=True)
    y = P.kv8_append(b, k.contiguous(), v.contiguous(), rope=rope, Q=q.contiguous(), keys=True)
    assert same(a.codes, b.codes) and same(a.scales, b.scales) and same(x[0], y[0]) and same(x[1], y[1])


@pytest.mark.parametrize("B, T, HQ, HKV, D, window, sinks, count, dtype", [
    (2, 333, 4, 4, 256, 100, 33, [333, 31], F16),    # tiles of 32
    (1, 65, 2, 1, 256, 32, 0, None, BF16),
    (40, 130, 16, 2, 32, 64, 1, None, F16),          # 128 queries a block
    (24, 300, 16, 4, 128, 130, 2, None, BF16),
    (40, 129, 8, 8, 64, None, 0, None, F32),
    (11, 130, 10, 5, 64, None, 0, None, F32),        # 330 blocks, one team of waves each
    (11, 130, 10, 5, 128, 65, 2, None, F32),
    (12, 129, 9, 3, 32, 20, 0, None, F32),
    (1, 700, 9, 3, 128, 300, 0, None, BF16),         # K/V heads that are no multiple of 8
    (1, 64, 2, 1, 64, None, 0, None, F32),           # one tile of keys, two, three
    (1, 128, 2, 1, 64, None, 0, [127], F32),
    (1, 192, 2, 1, 64, None, 0, None, F32),
])
def test_window_of_more_shapes(dev, B, T, HQ, HKV, D, window, sinks, count, dtype):
    g = gen(B + T)
    Q, K, V = (randn(g, B, T, h, D, dtype=dtype) for h in (HQ, HKV, HKV))
    check_window(dev, Q, K, V, dtype, window, sinks, count)


@pytest.mark.parametrize("D, dtype", [(32, F32), (64, F32), (128, F32), (256, F32), (64, BF16), (128, F16)])
def test_window_of_many_blocks_keeps_what_is_not_seen_out(dev, D, dtype):
    """NaN and Inf in keys and values, in batches whose blocks fill the card."""
    g = gen(D + 1)
    B, T = 12, 150
    Q, K, V = (randn(g, B, T, h, D, dtype=dtype) for h in (8, 4, 4))
    for b in range(0, B, 2):
        V[b, 30 + b, 0, 3], V[b, 100, 1, 7], V[b, 101, 1, 7], K[b, 70, 2, 5] = math.nan, math.inf, -math.inf, math.nan
    out, _ = check_window(dev, Q, K, V, dtype, 40, 2)
    assert bool(out[1::2].isfinite().all()) and bool(out[0, 30:70, :2, 3].isnan().all()) and bool(out[0, :, 6:].isfinite().all())


def test_start_is_the_length(dev):
    """start=cache.length is the default: the length is read before it changes."""
    g = gen(6)
    caches = [P.KV8Cache.empty(2, 256, 2, 64, 64, device=dev) for _ in range(2)]
    for T in (70, 1, 5):
        K, V = randn(g, 2, T, 2, 64).to(dev), randn(g, 2, T, 2, 64).to(dev)
        P.kv8_append(caches[0], K, V)
        P.kv8_append(caches[1], K, V, start=caches[1].length)
    assert caches[0].length.tolist() == [76, 76]
    assert all(same(getattr(caches[0], n), getattr(caches[1], n)) for n in ("codes", "scales", "length", "lost"))


def test_count_is_the_length(dev):
    """count=cache.length: how much there is, written again."""
    g = gen(16)
    B, T, HKV, D = 40, 300, 8, 64
    K, V = randn(g, B, T, HKV, D).to(dev), randn(g, B, T, HKV, D).to(dev)
    many = ints(dev, [(17 * b) % (T + 1) for b in range(B)])
    zero = torch.zeros_like(many)
    caches = [P.KV8Cache.empty(B, 320, HKV, D, D, device=dev) for _ in range(2)]
    caches[0].length.copy_(many)
    P.kv8_append(caches[0], K, V, start=zero, count=caches[0].length)
    P.kv8_append(caches[1], K, V, start=zero, count=many)
    assert all(same(getattr(caches[0], n), getattr(caches[1], n)) for n in ("codes", "scales", "length", "lost"))
    assert eq(caches[0].length, many)


def test_work_on_another_stream(dev):
    """A chain of calls on a stream of its own, its temporaries freed meanwhile."""
    g = gen(8)
    B, T, HQ, HKV, D = 2, 150, 8, 2, 64
    Q, K, V = (randn(g, B, T + 6, h, D).to(dev) for h in (HQ, HKV, HKV))
    rope = P.rope_tables(256, D, device=dev)

    def chain():
        c = P.KV8Cache.empty(B, 256, HKV, D, D, device=dev)
        out = [P.window_attention(*P.kv8_append(c, K[:, :T], V[:, :T], rope=rope, Q=Q[:, :T], keys=True), V[:, :T], window=50)]
        for i in range(6):
            at = slice(T + i, T + i + 1)
            q, _ = P.kv8_append(c, K[:, at].double(), V[:, at].transpose(1, 2).contiguous().transpose(1, 2), rope=rope, Q=Q[:, at])
            out.append(P.kv8_attention(c, q, window=50, sinks=1))
        return out

    ref = chain()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = chain()
    s.synchronize()
    assert all(same(a, b) for a, b in zip(got, ref))
