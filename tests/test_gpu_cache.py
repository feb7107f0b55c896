"""GPU: the 4-bit decode cache (dsa_cache) against its definitions in 64 bits
(cache_oracle, which derives the bounds): append and rows bit for bit, indexer,
attention and its accumulated weights, eviction, and the step of all of them."""
from __future__ import annotations

import math

import pytest
import torch

import _dsa_lib as L
import cache_oracle as C
import dsa_cache as D
from helpers import say
from topk_threshold import topk_indices

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def gen(dev, seed):
    return torch.Generator(device=dev).manual_seed(seed)


def randn(g, *shape, dtype=F32):
    return torch.randn(shape, generator=g, device=g.device).to(dtype)


def ints(dev, v):
    return torch.tensor(v, device=dev, dtype=torch.int32)


def filled(dev, B, S, HKV, DK, DV, lengths, seed=0, DI=0, idx_dtype=BF16):
    """A cache of random tokens whose slots past the length hold NaN scales and
    index keys: nothing may read them into a result."""
    g = gen(dev, seed)
    codes, scales = zip(*(C.quantise(randn(g, B, S, HKV, d)) for d in (DK, DV)))
    codes, scales = torch.cat(codes, -1), torch.cat(scales, -1)
    length = ints(dev, lengths)
    behind = torch.arange(S, device=dev) >= length.view(-1, 1)
    scales[behind] = 255
    codes[behind] = 0x5A
    k_idx = None
    if DI:
        k_idx = randn(g, B, S, DI, dtype=idx_dtype)
        k_idx[behind] = math.nan
    weight = torch.rand(B, S, generator=g, device=dev)
    return D.KV4Cache(codes, scales, length, k_idx, weight=weight, DK=DK)


def bits(x):
    return x.contiguous().view(torch.uint8)


def same(a, b):
    """Equal bit for bit (a function, so that a failure does not print the tensors)."""
    return bool(torch.equal(bits(a), bits(b)))


def within(got, want, lim, what):
    got, want = got.double(), want.double()
    assert bool((torch.isnan(got) == torch.isnan(want)).all()), f"{what}: NaN in other places"
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf]) and not torch.isinf(got[~inf]).any(), f"{what}: Inf"
    fine = torch.isfinite(want)
    err, lim = (got - want).abs()[fine], lim.expand_as(want)[fine]
    worst = float((err / lim.clamp(min=1e-300)).max()) if err.numel() else 0.0
    say(f"{what}: {worst:.3f} of the bound")
    assert bool((err <= lim).all()), f"{what}: {worst} times the bound"


# --- append and rows ----------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("B, T, S, HKV, DK, DV, DI, counts", [
    (1, 1, 4, 1, 32, 32, 0, None),
    (3, 1, 8, 4, 64, 64, 32, [1, 0, 1]),
    (2, 5, 9, 3, 96, 32, 64, [5, 2]),
    (2, 37, 64, 8, 128, 128, 128, None),
    (4, 130, 131, 2, 192, 128, 0, [130, 0, 77, 500]),
    (1, 257, 300, 5, 256, 256, 256, None),
])
def test_append_and_rows(dev, dtype, B, T, S, HKV, DK, DV, DI, counts):
    say("append", dtype, B, T, S, HKV, DK, DV, DI)
    g = gen(dev, 7)
    idx_dtype = dtype
    had = [min(2, S - T)] * B
    cache = filled(dev, B, S, HKV, DK, DV, had, 3, DI, idx_dtype)
    cache.weight.fill_(5.0)
    want_c, want_s, want_w = cache.codes.clone(), cache.scales.clone(), cache.weight.clone()
    want_i = cache.k_idx.clone() if DI else None
    K, V = randn(g, B, T, HKV, DK, dtype=dtype) * 3, randn(g, B, T, HKV, DV, dtype=dtype)
    V[0, 0, 0] = 0
    K[0, T - 1, HKV - 1, :4] = 1e-3
    new = randn(g, B, T, DI, dtype=idx_dtype) if DI else None
    w = torch.rand(B, T, generator=g, device=dev) if T > 1 else None
    D.kv4_append(cache, K, V, new, count=ints(dev, counts) if counts else None, weight=w)
    (kc, ks), (vc, vs) = C.quantise(K), C.quantise(V)
    for b in range(B):
        n, h = min(counts[b], T) if counts else T, had[b]
        want_c[b, h:h + n] = torch.cat([kc, vc], -1)[b, :n]
        want_s[b, h:h + n] = torch.cat([ks, vs], -1)[b, :n]
        want_w[b, h:h + n] = w[b, :n] if w is not None else 0.0
        if DI:
            want_i[b, h:h + n] = new[b, :n]
        assert int(cache.length[b]) == h + n == int(cache.seen[b]) and int(cache.lost[b]) == 0
        assert cache.position[b, :h + n].tolist() == list(range(h + n))
    assert torch.equal(cache.codes, want_c) and torch.equal(cache.scales, want_s)
    assert torch.equal(cache.weight, want_w)
    if DI:  # bit for bit, the NaN behind the tokens too
        assert same(cache.k_idx, want_i)
    ok = (torch.arange(S, device=dev) < cache.length.view(-1, 1)).view(B, S, 1, 1)
    wk, wv = (torch.where(ok, C.decode(c, s), 0.0) for c, s in
              ((want_c[..., :DK // 2], want_s[..., :DK // 32]), (want_c[..., DK // 2:], want_s[..., DK // 32:])))
    for out in (F32, BF16, F16):
        k, v = D.kv4_rows(cache, dtype=out)
        assert torch.equal(k, wk.to(out)) and torch.equal(v, wv.to(out)), out
    pick = torch.randint(-3, S + 3, (B, 11), generator=g, device=dev, dtype=torch.int32)
    pick[:, 4] = pick[:, 3]
    k, v = D.kv4_rows(cache, pick)
    at = pick.clamp(0, S - 1).long()
    b = torch.arange(B, device=dev).view(-1, 1)
    keep = (pick == at).view(B, 11, 1, 1)
    assert torch.equal(k, torch.where(keep, wk[b, at], 0.0).float())
    assert torch.equal(v, torch.where(keep, wv[b, at], 0.0).float())


def test_append_values_at_the_edges(dev):
    """Ties, magnitudes at 7 * 2^e and one step either side, the ends of fp32's range, -0,
    subnormals, Inf and NaN: the codes of the rule, bit for bit."""
    vals = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, -0.0, 0.0]
    rows = []
    for e in (-149, -140, -127, -126, -125, -124, -20, 0, 5, 100, 124, 125):
        for top in (7.0, math.nextafter(7.0, 0), 7.0 * (1 + 2.0 ** -23), 4.0, 6.0, 3.5):
            r = torch.tensor(vals + [top] + [0.1] * 21, dtype=torch.float64)
            rows.append((r * 2.0 ** e * (1 if len(rows) % 2 else -1)).float())
    for bad in (math.inf, -math.inf, math.nan):
        rows.append(torch.tensor([1.0] * 31 + [bad]))
    rows.append(torch.full((32,), 3.4028234e38))
    x = torch.stack(rows).to(dev)
    n = len(rows)
    cache = D.KV4Cache.empty(1, n, 1, 32, 32, device=dev)
    K = x.view(1, n, 1, 32)
    D.kv4_append(cache, K, K.flip(-1).contiguous())
    for x, half in ((K, slice(0, 16)), (K.flip(-1), slice(16, 32))):
        codes, scales = C.quantise(x.cpu())
        assert torch.equal(cache.codes[..., half].cpu(), codes)
        assert torch.equal(cache.scales[..., half.start // 16].cpu(), scales[..., 0])
        k = D.kv4_rows(cache)[0 if half.start == 0 else 1]
        want = C.decode(codes, scales).float()
        assert torch.equal(torch.nan_to_num(k.cpu(), nan=1e9), torch.nan_to_num(want, nan=1e9))


def test_append_from_other_layouts(dev):
    """Views of a fused projection, a transposed batch, and an unaligned slice."""
    g = gen(dev, 5)
    B, T, HKV, DK, DV = 2, 6, 2, 64, 32
    fused = randn(g, B, T, HKV * (DK + DV) + 1, dtype=BF16)
    K = fused[..., 1:1 + HKV * DK].view(B, T, HKV, DK)
    V = fused[..., 1 + HKV * DK:].view(B, T, HKV, DV)
    a, b = (D.KV4Cache.empty(B, 8, HKV, DK, DV, device=dev) for _ in range(2))
    D.kv4_append(a, K, V)
    D.kv4_append(b, K.contiguous(), V.contiguous())
    assert torch.equal(a.codes, b.codes) and torch.equal(a.scales, b.scales)
    Kt = K.transpose(0, 1).contiguous().transpose(0, 1)
    D.kv4_append(a, Kt, V.float(), restart=True)  # mixed types go as fp32
    assert torch.equal(a.codes[:, :T], b.codes[:, :T])


def test_append_past_the_end(dev):
    g = gen(dev, 6)
    cache = filled(dev, 3, 10, 1, 32, 32, [10, 8, 0])
    before = cache.codes.clone()
    D.kv4_append(cache, randn(g, 3, 4, 1, 32), randn(g, 3, 4, 1, 32), count=ints(dev, [4, 4, 0]))
    assert cache.length.tolist() == [10, 10, 0] and cache.lost.tolist() == [4, 2, 0]
    assert cache.seen.tolist() == [14, 12, 0]
    assert torch.equal(before[0], cache.codes[0]) and torch.equal(before[1, :8], cache.codes[1, :8])
    with pytest.raises(RuntimeError, match="6 tokens"):
        cache.check()
    D.kv4_append(cache, randn(g, 3, 0, 1, 32), randn(g, 3, 0, 1, 32), restart=True)
    assert not cache.length.any() and not cache.seen.any()
    cache.check()


# --- the indexer -----------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("S, Tq, HI, DI, lengths, counts, span", [
    (1, 1, 1, 32, [1], None, None),
    (5, 1, 4, 32, [0, 1, 5], None, None),
    (67, 1, 64, 128, [67, 66, 3], None, None),
    (300, 2, 12, 64, [300, 1, 0, 257], [2, 1, 2, 0], None),
    (1029, 3, 17, 64, [1029, 600], None, 1000),
    (530, 1, 256, 128, [530], None, 513),
    (4100, 1, 8, 256, [4100, 100], None, None),
    (200, 65, 5, 32, [200, 64], None, None),
])
def test_indexer(dev, dtype, S, Tq, HI, DI, lengths, counts, span):
    say("indexer", dtype, S, Tq, HI, DI, lengths)
    B = len(lengths)
    cache = filled(dev, B, S, 1, 32, 32, lengths, 1, DI, dtype)
    g = gen(dev, 2)
    q, w = randn(g, B, Tq, HI, DI, dtype=dtype), randn(g, B, Tq, HI, dtype=dtype)
    count = ints(dev, counts) if counts else None
    got = D.kv4_indexer_scores(cache, q, w, span=span, count=count)
    want, lim = C.indexer(torch.nan_to_num(cache.k_idx), cache.length, q, w, count, span)
    within(got, want, lim, "scores")


def test_indexer_fp32_with_16_wide_keys_and_no_codes(dev):
    g = gen(dev, 3)
    k = randn(g, 2, 77, 16)
    cache = D.KV4Cache(None, None, ints(dev, [77, 40]), k)
    q, w = randn(g, 2, 1, 4, 16), randn(g, 2, 1, 4)
    want, lim = C.indexer(k, cache.length, q, w)
    within(D.kv4_indexer_scores(cache, q, w), want, lim, "scores")
    with pytest.raises(AssertionError, match="index keys only"):
        D.kv4_attention(cache, q)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_indexer_values_of_every_size(dev, dtype):
    """Rows and keys of widely different magnitudes, zeros, and one Inf or NaN, which
    shows in the scores that take it in and in no others."""
    g = gen(dev, 4)
    S, HI, DI = 70, 4, 32
    k = randn(g, 1, S, DI) * torch.exp2(torch.randint(-30, 30, (1, S, 1), generator=g, device=dev).float())
    q = randn(g, 1, 2, HI, DI) * torch.exp2(torch.randint(-30, 30, (1, 2, HI, 1), generator=g, device=dev).float())
    k, q, w = k.to(dtype), q.to(dtype), randn(g, 1, 2, HI, dtype=dtype)
    k[0, 9] = 0
    cache = D.KV4Cache(None, None, ints(dev, [S]), k)
    want, lim = C.indexer(k, cache.length, q, w)
    within(D.kv4_indexer_scores(cache, q, w), want, lim, "scores")
    k[0, 5, 3], k[0, 6, 3] = math.nan, math.inf
    got = D.kv4_indexer_scores(cache, q, w)
    assert torch.isnan(got[0, :, 5]).all() and not torch.isfinite(got[0, :, 6]).any()
    keep = [s for s in range(S) if s not in (5, 6)]
    within(got[..., keep], want[..., keep], lim[..., keep], "the others")


# --- attention ---------------------------------------------------------------------------------------
def attend(cache, Q, what, **kw):
    before = cache.weight.clone()
    out = D.kv4_attention(cache, Q, accumulate=True, **kw)
    O, lim, add, addlim = C.attention(cache.codes, cache.scales, cache.DK, cache.length, Q, **kw)
    within(out, O, lim, what)
    # every addition onto a weight rounds by at most u of a partial sum, and no partial
    # sum exceeds the last (all addends are >= 0): one addition per token and listing
    times = torch.full_like(before, Q.shape[1])
    if (slots := kw.get("slots")) is not None:
        at = slots.flatten(1).long()
        ok = (at >= 0) & (at < cache.S)
        times = torch.zeros_like(before).scatter_add_(1, torch.where(ok, at, 0), ok.float())
    w = before.double() + add
    within(cache.weight, w, addlim + (times + 1) * C.U * w.abs(), what + " weights")
    again = D.kv4_attention(cache, Q, **kw)
    assert same(torch.nan_to_num(again), torch.nan_to_num(out)), "another result without the weights"
    return out


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("HQ, HKV, DK, DV", [
    (1, 1, 32, 32), (4, 4, 32, 32), (8, 2, 64, 64), (6, 2, 96, 96), (16, 1, 128, 128),
    (32, 8, 128, 128), (24, 1, 128, 128), (40, 2, 192, 192), (8, 2, 192, 128), (9, 3, 256, 256),
])
def test_attention_heads(dev, dtype, HQ, HKV, DK, DV):
    say("attention", dtype, HQ, HKV, DK, DV)
    lengths = [77, 1, 0, 130]
    cache = filled(dev, 4, 130, HKV, DK, DV, lengths, 11)
    attend(cache, randn(gen(dev, 12), 4, 1, HQ, DK, dtype=dtype), "out")


@pytest.mark.parametrize("S", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 257, 511, 1023, 2049, 5000])
@pytest.mark.parametrize("HQ, HKV, D", [(4, 4, 32), (16, 4, 128)])
def test_attention_lengths(dev, S, HQ, HKV, D):
    say("attention", S, HQ, HKV, D)
    cache = filled(dev, 2, S, HKV, D, D, [S, (S + 1) // 2], S)
    attend(cache, randn(gen(dev, S), 2, 1, HQ, D, dtype=BF16), "out")


@pytest.mark.parametrize("B, S, HQ, HKV, D", [(1, 40000, 8, 8, 64), (1, 33000, 16, 1, 128), (6, 9001, 8, 2, 32)])
def test_attention_over_long_caches(dev, B, S, HQ, HKV, D):
    say("attention", B, S, HQ, HKV, D)
    cache = filled(dev, B, S, HKV, D, D, [S - 1000 * b for b in range(B)], 5)
    attend(cache, randn(gen(dev, 6), B, 1, HQ, D, dtype=F16) * 2, "out")


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("Tq, lengths, counts", [
    (2, [50, 2, 1, 0], None), (3, [400, 7, 3, 90], [3, 1, 0, 2]), (70, [333, 70, 12, 69], [70, 70, 12, 500]),
])
def test_attention_of_several_tokens(dev, dtype, Tq, lengths, counts):
    say("attention", dtype, Tq, lengths, counts)
    cache = filled(dev, 4, 400, 2, 64, 64, lengths, 21)
    count = ints(dev, counts) if counts else None
    attend(cache, randn(gen(dev, 22), 4, Tq, 8, 64, dtype=dtype), "out", count=count)


def test_attention_span(dev):
    cache = filled(dev, 3, 300, 2, 64, 64, [300, 100, 7], 23)
    Q = randn(gen(dev, 24), 3, 1, 4, 64)
    attend(cache, Q, "out", span=131)
    assert torch.isnan(D.kv4_attention(cache, Q, span=0)).all()


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("k, Tq, HQ, HKV, DH", [
    (1, 1, 4, 4, 32), (31, 1, 8, 2, 64), (100, 2, 16, 1, 128), (255, 1, 16, 4, 128), (700, 3, 4, 2, 192), (64, 1, 4, 1, 256),
])
def test_attention_over_listed_slots(dev, dtype, k, Tq, HQ, HKV, DH):
    """Slots in no order, some of them twice, some past the length, past S, negative."""
    say("listed", dtype, k, Tq, HQ, HKV, DH)
    g = gen(dev, k)
    B, S = 4, 500
    cache = filled(dev, B, S, HKV, DH, DH, [500, 37, 3, 0], 31)
    slots = torch.randint(-20, S + 20, (B, Tq, k), generator=g, device=dev, dtype=torch.int32)
    slots[0, 0, 0] = -2 ** 31
    slots[0, :, k // 2] = 2 ** 31 - 1
    slots[1, :, : k // 3] = torch.randint(0, 37, (Tq, k // 3), generator=g, device=dev, dtype=torch.int32)
    attend(cache, randn(g, B, Tq, HQ, DH, dtype=dtype), "out", slots=slots)
    wide = torch.full((B, Tq, k + 3), 7, device=dev, dtype=torch.int32)
    wide[..., :k] = slots
    Q = randn(g, B, Tq, HQ, DH, dtype=dtype)
    a, b = D.kv4_attention(cache, Q, slots=wide[..., :k]), D.kv4_attention(cache, Q, slots=slots)
    assert same(torch.nan_to_num(a), torch.nan_to_num(b))  # a view of a wider list
    attend(cache, Q, "long list", slots=torch.randint(0, 500, (B, Tq, 3000), generator=g, device=dev, dtype=torch.int32))


def test_attention_of_listed_all_is_attention(dev):
    g = gen(dev, 41)
    cache = filled(dev, 2, 200, 2, 128, 128, [200, 150], 42)
    Q = randn(g, 2, 1, 8, 128, dtype=BF16)
    slots = torch.arange(200, device=dev, dtype=torch.int32).flip(0).expand(2, 1, 200)
    O, lim, _, _ = C.attention(cache.codes, cache.scales, 128, cache.length, Q)
    within(D.kv4_attention(cache, Q, slots=slots), O, lim, "listed")
    assert torch.isnan(D.kv4_attention(cache, Q, slots=slots[..., :0])).all()


@pytest.mark.parametrize("HQ, HKV, DK, DV, Tq, dtype", [
    (1, 1, 64, 64, 2, F32), (2, 2, 128, 128, 5, BF16), (8, 2, 64, 64, 2, F16), (8, 4, 32, 32, 3, F32),
    (12, 2, 128, 128, 7, BF16), (5, 1, 96, 96, 3, BF16), (12, 4, 192, 128, 11, F16), (3, 3, 256, 256, 33, BF16),
    (20, 1, 64, 64, 4, F32), (4, 1, 192, 192, 40, F32)])
def test_attention_of_tokens_together(dev, HQ, HKV, DK, DV, Tq, dtype):
    """Tokens that share the cache's tiles: their own last slots on both sides of a
    tile's edge, row tiles that begin inside a token's heads, padded batches."""
    cache = filled(dev, 5, 1100, HKV, DK, DV, [1100, 1056 + Tq // 2, 1025, Tq - 1, 0], 46)
    Q = randn(gen(dev, 47), 5, Tq, HQ, DK, dtype=dtype)
    attend(cache, Q, "all tokens")
    attend(cache, Q, "padded", count=ints(dev, [Tq, 1, Tq - 1, 1, 0]))
    attend(cache, Q, "the first slots", span=1057)


@pytest.mark.parametrize("D_", [32, 128, 192])
def test_nan_of_tokens_together(dev, D_):
    """A later token's NaN value, and an earlier one's, among tokens that share tiles:
    NaN exactly in the blocks of 32 of the queries that see it."""
    g, Tq, n = gen(dev, 48), 6, 1058
    cache = filled(dev, 1, 1100, 2, D_, D_, [n], 49)
    per = D_ // 32
    cache.scales[0, n - 2, 0, per] = 255       # V of the last token but one: block 0 of head 0
    cache.scales[0, n - 5, 1, 2 * per - 1] = 255  # V of the second: the last block of head 1
    cache.scales[0, n - 1, 1, 0] = 255         # K of the last: its own query of head 1 alone
    out = D.kv4_attention(cache, randn(g, 1, Tq, 4, D_)).view(Tq, 2, 2, per, 32)
    want = torch.zeros(Tq, 2, 2, per, 32, dtype=torch.bool, device=dev)
    want[Tq - 2:, 0, :, 0] = True
    want[1:, 1, :, per - 1] = True
    want[Tq - 1, 1] = True
    assert torch.equal(torch.isnan(out), want)


def test_attention_nan_where_it_belongs(dev):
    """A NaN block of a later token's or an unlisted slot reaches no other query; a seen one does."""
    g = gen(dev, 43)
    cache = filled(dev, 1, 64, 2, 64, 64, [40], 44)
    cache.scales[0, 39] = 255  # the last token: K and V are NaN
    Q = randn(g, 1, 2, 4, 64)
    out = D.kv4_attention(cache, Q, accumulate=True)
    assert torch.isfinite(out[:, 0]).all() and torch.isnan(out[:, 1]).all()
    assert torch.isnan(cache.weight[0, :40]).all() and torch.isfinite(cache.weight[0, 40:]).all()
    slots = torch.arange(39, device=dev, dtype=torch.int32).expand(1, 2, 39)
    assert torch.isfinite(D.kv4_attention(cache, Q, slots=slots)).all()
    cache = filled(dev, 1, 64, 2, 64, 64, [40], 44)
    cache.scales[0, 3, 1, 2:] = 255  # the value of one slot of head 1
    out = D.kv4_attention(cache, Q)
    assert torch.isfinite(out[0, 1, :2]).all() and torch.isnan(out[0, 1, 2:]).all()
    Q[0, 1, 0] = math.inf
    Q[0, 0, 1, 5] = math.nan
    out = D.kv4_attention(filled(dev, 1, 64, 2, 64, 64, [40], 44), Q)
    assert torch.isnan(out[0, 1, 0]).all() and torch.isnan(out[0, 0, 1]).all()
    assert torch.isfinite(out[0, 0, 0]).all() and torch.isfinite(out[0, 0, 2:]).all() and torch.isfinite(out[0, 1, 1:]).all()


@pytest.mark.parametrize("size", [2.0 ** -60, 2.0 ** 8, 2.0 ** 40])
def test_attention_large_and_small_values(dev, size):
    """Logits of hundreds (one slot takes all) and values far from 1."""
    g = gen(dev, 45)
    S, D_ = 150, 64
    cache = filled(dev, 2, S, 2, D_, D_, [150, 33], 46)
    step = int(math.log2(size))
    cache.scales[..., D_ // 32:] = (cache.scales[..., D_ // 32:].int() + step).clamp(2, 252).to(torch.uint8)
    attend(cache, randn(g, 2, 1, 4, D_) * 40, "out")


def test_attention_all_logits_minus_infinity(dev):
    """exp over -inf alone is 0/0, and beside a finite logit it is 0."""
    cache = D.KV4Cache.empty(1, 40, 1, 32, 32, device=dev)
    K = torch.zeros(1, 40, 1, 32, device=dev)
    K[..., 0] = 2.0 ** 100
    V = torch.ones(1, 40, 1, 32, device=dev)
    D.kv4_append(cache, K, V)
    Q = torch.zeros(1, 1, 1, 32, device=dev)
    Q[..., 0] = -2.0 ** 100
    assert torch.isnan(D.kv4_attention(cache, Q)).all()
    K[0, 35] = 0
    D.kv4_append(cache, K, V * torch.arange(40, device=dev).view(1, 40, 1, 1), restart=True)
    assert torch.equal(D.kv4_attention(cache, Q), D.kv4_rows(cache)[1][:, 35:36])


def test_attention_past_32_bit_offsets(dev):
    """Batches whose codes lie past 4 GiB, sequences near 2 GiB."""
    B, S, HKV, D_ = 3, (1 << 21) - 1, 8, 128
    if torch.cuda.mem_get_info(dev)[0] < 12 << 30:
        pytest.skip("needs 12 GiB")
    cache = D.KV4Cache.empty(B, S, HKV, D_, D_, device=dev)
    small = filled(dev, B, 300, HKV, D_, D_, [300] * B, 51)
    at = S - 300
    cache.codes[:, at:], cache.scales[:, at:] = small.codes, small.scales
    cache.length.fill_(S)
    Q = randn(gen(dev, 52), B, 1, 16, D_, dtype=BF16)
    pick = torch.arange(300, device=dev, dtype=torch.int32).expand(B, 1, 300)
    O, lim, add, addlim = C.attention(small.codes, small.scales, D_, small.length, Q)
    out = D.kv4_attention(cache, Q, slots=pick + at, accumulate=True)
    within(out, O, lim, "listed at the end")
    within(cache.weight[:, at:], add, addlim + C.U * add, "weights")
    # the whole: a prefix of zero keys has logit 0 and value 0
    lg = torch.einsum("bhgd,bshd->bhgs", Q.double().view(B, HKV, 2, D_),
                      C.decode(small.codes[..., :64], small.scales[..., :4])) / math.sqrt(D_)
    e = lg.exp()
    O = torch.einsum("bhgs,bshd->bhgd", e, C.decode(small.codes[..., 64:], small.scales[..., 4:]))
    size = torch.einsum("bhgs,bshd->bhgd", e, C.decode(small.codes[..., 64:], small.scales[..., 4:]).abs())
    total = e.sum(-1, keepdim=True) + at
    # chains of S/32 additions of ones, exact below 2^24, then 300 other slots
    within(D.kv4_attention(cache, Q), (O / total).view(B, 1, 16, D_),
           (size / total).view(B, 1, 16, D_) * (2.0 ** -16 + 600 * C.U + 1e-5), "whole")
    K, V = D.kv4_rows(cache, (pick + at)[:, 0].contiguous())
    assert torch.equal(K, C.decode(small.codes[..., :64], small.scales[..., :4]).float())
    src, dst = D.kv4_evict(cache, S - 5, 0)
    assert src.shape == dst.shape == (B, 5) and cache.length.tolist() == [S - 5] * B


# --- eviction ----------------------------------------------------------------------------------------
def check_evict(cache, keep, recent, what):
    say("evict", what)
    want = C.evict(cache.length.cpu(), cache.seen.cpu(), cache.position.cpu(), cache.weight.cpu(), keep, recent)
    names = ("codes", "scales", "position", "weight", "k_idx")
    before = {n: getattr(cache, n).clone() for n in names if getattr(cache, n) is not None}
    moved = torch.stack(D.kv4_evict(cache, keep, recent)).cpu()
    M = max(0, min(keep, cache.S - keep))
    assert moved.shape == (2, cache.B, M)
    for b, (src, dst, n) in enumerate(want):
        assert len(src) == len(dst) <= M
        assert moved[0, b].tolist() == src + [-1] * (M - len(src)), (what, b)
        assert moved[1, b].tolist() == dst + [-1] * (M - len(dst)), (what, b)
        assert int(cache.length[b]) == n
        for x in before.values():
            if src:
                x[b, torch.tensor(dst, device=x.device)] = x[b, torch.tensor(src, device=x.device)].clone()
    for name, x in before.items():  # moved, and nothing else touched
        assert same(getattr(cache, name), x), (what, name)


@pytest.mark.parametrize("S, lengths, keep, recent", [
    (1, [1, 0], 0, 0), (2, [2, 1], 1, 1), (9, [9, 8, 7, 3], 8, 2), (64, [64, 0, 33], 32, 0),
    (65, [65, 64], 64, 64), (1000, [1000, 999, 700, 5], 300, 50), (1000, [1000, 950], 900, 0),
    (5000, [5000, 1], 4999, 4999), (5000, [4097, 5000], 17, 3), (20000, [20000, 12345], 8192, 128),
    (70001, [70001, 66000], 30000, 1000), (64, [64], 64, 1), (64, [64], 100, 0),
])
def test_evict(dev, S, lengths, keep, recent):
    cache = filled(dev, len(lengths), S, 2, 32, 32, lengths, S, 32)
    check_evict(cache, keep, recent, "random weights")
    cache = filled(dev, len(lengths), S, 1, 64, 32, lengths, S)
    g = gen(dev, S + 1)
    cache.weight.copy_(torch.randint(0, 3, cache.weight.shape, generator=g, device=dev).float())
    # positions as they stand after evictions: no order
    order = torch.rand(cache.B, S, generator=g, device=dev).argsort(1).to(torch.int32)
    cache.position.copy_(order)
    cache.seen.fill_(S)
    check_evict(cache, keep, recent, "ties, shuffled positions")
    cache = filled(dev, len(lengths), S, 1, 32, 32, lengths, S)
    cache.weight.zero_()
    check_evict(cache, keep, recent, "all equal")


def test_evict_orders_every_float(dev):
    S = 400
    cache = filled(dev, 2, S, 1, 32, 32, [S, S - 1], 3)
    g = gen(dev, 4)
    w = torch.randn(2, S, generator=g, device=dev) * torch.exp2(torch.randint(-140, 100, (2, S), generator=g, device=dev).float())
    w[:, ::7] = 0.0
    w[:, 3::14] = -0.0
    w[:, 5::50], w[:, 6::50], w[:, 8::50] = math.inf, -math.inf, math.nan
    cache.weight.copy_(w)
    for keep in (350, 200, 60, 8, 1):
        check_evict(cache, keep, min(keep, 3), f"keep {keep}")


def test_evict_of_more_recent_than_kept(dev):
    """Positions that a caller set so that more slots count as recent than stay."""
    cache = filled(dev, 1, 100, 1, 32, 32, [100], 3)
    cache.position.fill_(99)
    check_evict(cache, 40, 5, "all recent")


# --- together ----------------------------------------------------------------------------------------
def step_inputs(g, B, Tq, HI, DI, HQ, HKV, DK, DV, dtype):
    return (randn(g, B, Tq, HI, DI, dtype=dtype), randn(g, B, Tq, DI, dtype=dtype), randn(g, B, Tq, HI, dtype=dtype),
            randn(g, B, Tq, HQ, DK, dtype=dtype), randn(g, B, Tq, HKV, DK, dtype=dtype), randn(g, B, Tq, HKV, DV, dtype=dtype))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_decode_steps(dev, dtype):
    """Prompts, then steps that fill the cache, evict and go on: at every step the
    output, weights and eviction of the cache as it then is."""
    g = gen(dev, 61)
    B, S, HI, DI, HQ, HKV, DK, DV, keep, recent, k = 3, 41, 4, 32, 8, 2, 64, 64, 38, 4, 12
    cache = D.KV4Cache.empty(B, S, HKV, DK, DV, DI, idx_dtype=dtype, device=dev)
    _, ki, _, _, K, V = step_inputs(g, B, 30, HI, DI, HQ, HKV, DK, DV, dtype)
    D.kv4_append(cache, K, V, ki, count=ints(dev, [30, 17, 1]), restart=True)
    seen = [30, 17, 1]
    for step in range(24):
        Tq = 1 + step % 3
        x = step_inputs(g, B, Tq, HI, DI, HQ, HKV, DK, DV, dtype)
        # the same step from its parts on a copy
        copy = D.KV4Cache(*(getattr(cache, n).clone() for n in ("codes", "scales", "length", "k_idx", "position", "weight", "seen", "lost")), DK=DK)
        out = D.dsa_decode(cache, *x, top_k=k, keep=keep, recent=recent)
        D.kv4_append(copy, x[4], x[5], x[1])
        scores = D.kv4_indexer_scores(copy, x[0], x[2])
        want, lim = C.indexer(torch.nan_to_num(copy.k_idx), copy.length, x[0], x[2])
        within(scores, want, lim, "scores")
        _, slots = topk_indices(scores, k)
        before = copy.weight.clone()
        O, lim, add, addlim = C.attention(copy.codes, copy.scales, DK, copy.length, x[3], slots=slots)
        within(out, O, lim, f"step {step}")
        D.kv4_attention(copy, x[3], slots=slots, accumulate=True)
        w = before.double() + add
        within(copy.weight, w, addlim + (Tq + 1) * C.U * w.abs(), "weights")
        check_evict(copy, keep, recent, f"step {step}")
        seen = [n + Tq for n in seen]
        for n in ("codes", "scales", "length", "k_idx", "position", "weight", "seen", "lost"):
            assert same(getattr(cache, n), getattr(copy, n)), n
        assert cache.seen.tolist() == seen
        for b in range(B):  # the newest tokens are there, every position once
            n = int(cache.length[b])
            pos = cache.position[b, :n].tolist()
            assert n == min(seen[b], keep) and len(set(pos)) == n
            assert set(range(max(0, seen[b] - recent), seen[b])) <= set(pos)
    cache.check()


def test_decode_top_k_past_the_span_attends_to_all(dev):
    g = gen(dev, 62)
    cache = filled(dev, 2, 50, 2, 64, 64, [30, 7], 63, 32)
    cache.scales[cache.scales == 255] = 127
    x = step_inputs(g, 2, 1, 4, 32, 4, 2, 64, 64, BF16)
    out = D.dsa_decode(cache, *x, top_k=40, span=40)
    O, lim, _, _ = C.attention(cache.codes, cache.scales, 64, cache.length, x[3])
    within(out, O, lim, "all")


def test_decode_of_a_padded_batch(dev):
    """Sequences with fewer tokens than the batch's: their other rows see nothing and
    change nothing."""
    g = gen(dev, 64)
    cache = filled(dev, 3, 60, 2, 64, 64, [30, 7, 0], 65, 32)
    x = step_inputs(g, 3, 3, 4, 32, 4, 2, 64, 64, BF16)
    out = D.dsa_decode(cache, *x, top_k=9, count=ints(dev, [3, 1, 0]), keep=50)
    assert cache.length.tolist() == [33, 8, 0] and cache.seen.tolist() == [33, 8, 0]
    nan = torch.isnan(out).flatten(2)
    assert [[bool(nan[b, t].all()) for t in range(3)] for b in range(3)] == \
        [[False] * 3, [False, True, True], [True] * 3]
    assert not nan[0].any() and not nan[1, 0].any()
    assert torch.isfinite(cache.weight).all()


def test_decode_captured_and_replayed(dev):
    """Two captured graphs over one cache and one over another, replayed in turn with
    eager work between: each replay is the eager step, bit for bit."""
    g = gen(dev, 66)
    B, S, args = 2, 300, (1, 4, 64, 8, 2, 128, 128, BF16)
    x = step_inputs(g, B, *args)
    caches = [filled(dev, B, S, 2, 128, 128, [200, 150], 67, 64) for _ in range(3)]
    eager, one, other = caches
    kw = dict(top_k=40, keep=220, recent=8)

    def step(c, inputs):
        return D.dsa_decode(c, *inputs, **kw)

    warm = filled(dev, B, S, 2, 128, 128, [200, 150], 67, 64)
    step(warm, x)
    torch.cuda.synchronize()
    graphs = []
    for c in (one, one, other):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = step(c, x)
        graphs.append((gr, out))
    for i in range(30):
        for t, new in zip(x, step_inputs(g, B, *args)):
            t.copy_(new)
        gr, out = graphs[i % 2]
        gr.replay()
        got = out.clone()
        graphs[2][0].replay()
        torch.randn(1000, 1000, device=dev).sum()
        want = step(eager, x)
        torch.cuda.synchronize()
        assert torch.equal(got, want) and torch.equal(graphs[2][1], want), i
        for c in (one, other):
            for n in ("codes", "scales", "length", "k_idx", "position", "weight", "seen"):
                a, b = getattr(c, n), getattr(eager, n)
                assert same(a, b), (i, n)


def test_two_streams_at_once(dev):
    """Steps of two caches on two streams, neither of them the default."""
    g = gen(dev, 68)
    args = (1, 4, 64, 8, 2, 64, 64, F32)
    xs = [step_inputs(g, 2, *args) for _ in range(12)]
    make = lambda: filled(dev, 2, 400, 2, 64, 64, [380, 17], 69, 64, F32)  # noqa: E731
    alone = make()
    want = [D.dsa_decode(alone, *x, top_k=30, keep=380, recent=5) for x in xs]
    caches, streams, got = [make(), make()], [torch.cuda.Stream(dev) for _ in range(2)], [[], []]
    torch.cuda.synchronize()
    for x in xs:
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(D.dsa_decode(caches[i], *x, top_k=30, keep=380, recent=5))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(a, b) for a, b in zip(got[i], want))


@pytest.mark.parametrize("scale", [-0.125, 0.0, 0.5])
@pytest.mark.parametrize("HQ", [2, 16])
def test_any_finite_scale(dev, scale, HQ):
    """The C entry's scale: of either sign, and 0 (a plain mean of the visible slots)."""
    g = gen(dev, 70)
    cache = filled(dev, 2, 90, 1, 64, 64, [77, 2], 71)
    Q = randn(g, 2, 1, HQ, 64)
    out, lib = torch.empty(2, 1, HQ, 64, device=dev), L.lib()
    nws = lib.dsa_kv4_attention_workspace_bytes(cache._ref, 1, HQ, 0, 90, 1)
    ws = torch.empty(nws, device=dev, dtype=torch.uint8)
    before = cache.weight.clone()
    args = (cache._ref, Q.data_ptr(), L.DSA_F32, None, None, 1, HQ, 90, 1, scale, out.data_ptr(), ws.data_ptr())
    assert lib.dsa_kv4_attention(*args, nws - 1, L.stream_ptr(dev)) == L.DSA_EINVAL
    L.check(lib.dsa_kv4_attention(*args, nws, L.stream_ptr(dev)), "attention")
    # the same logits come of Q * scale * sqrt(64) at the usual scale
    O, lim, add, addlim = C.attention(cache.codes, cache.scales, 64, cache.length, Q.double() * scale * 8, dtype=F32)
    within(out, O, lim, "out")
    w = before.double() + add
    within(cache.weight, w, addlim + 2 * C.U * w.abs(), "weights")


def test_buffers_stay(dev):
    cache = filled(dev, 2, 20, 1, 32, 32, [20, 4])
    for name in D.KV4Cache._BUFFERS:
        with pytest.raises(AttributeError):
            setattr(cache, name, None)
    cache.length.copy_(ints(dev, [5, 0]))  # back to an earlier token
    Q = randn(gen(dev, 1), 2, 1, 2, 32)
    O, lim, _, _ = C.attention(cache.codes, cache.scales, 32, ints(dev, [5, 0]), Q)
    within(D.kv4_attention(cache, Q), O, lim, "out")


def test_nothing_in_nothing_out(dev):
    """No sequences, no tokens: empty results, and nothing changes."""
    none = D.KV4Cache.empty(0, 8, 2, 64, 64, 32, device=dev)
    z = lambda *s: torch.zeros(s, device=dev)  # noqa: E731
    D.kv4_append(none, z(0, 3, 2, 64), z(0, 3, 2, 64), z(0, 3, 32))
    assert D.kv4_attention(none, z(0, 1, 4, 64), accumulate=True).shape == (0, 1, 4, 64)
    assert D.kv4_indexer_scores(none, z(0, 1, 4, 32), z(0, 1, 4)).shape == (0, 1, 8)
    assert D.kv4_rows(none)[0].shape == (0, 8, 2, 64) and D.kv4_evict(none, 4)[0].shape == (0, 4)
    cache = filled(dev, 2, 20, 2, 64, 64, [20, 4], DI=32)
    before = [getattr(cache, n).clone() for n in D.KV4Cache._BUFFERS]
    D.kv4_append(cache, z(2, 0, 2, 64), z(2, 0, 2, 64), z(2, 0, 32))
    assert D.kv4_attention(cache, z(2, 0, 4, 64), accumulate=True).shape == (2, 0, 4, 64)
    assert D.kv4_indexer_scores(cache, z(2, 0, 4, 32), z(2, 0, 4)).shape == (2, 0, 20)
    D.kv4_evict(cache, 20)
    assert all(same(a, getattr(cache, n)) for a, n in zip(before, D.KV4Cache._BUFFERS))


def test_refused_steps_change_nothing(dev):
    """A step that one of its later calls would refuse is refused before the append."""
    g = gen(dev, 72)
    cache = filled(dev, 2, 40, 2, 64, 64, [20, 4], 73, 32)
    q, ki, w, Q, K, V = step_inputs(g, 2, 1, 4, 32, 4, 2, 64, 64, BF16)
    odd = filled(dev, 2, 40, 1, 160, 160, [20, 4], 74)  # no attention kernel for it
    caches = [cache, odd]
    before = [[getattr(c, n).clone() for n in D.KV4Cache._BUFFERS if getattr(c, n) is not None] for c in caches]
    wide = randn(g, 2, 1, 257, 32)
    rows = randn(g, 2, 1, 1, 160)
    for args, kw in [((q, ki, w, Q, K, V, 8), dict(keep=30, recent=31)),
                     ((q, ki, w, Q, K, V, 8), dict(keep=-1)),
                     ((q, ki, w, Q, K, V, 8), dict(span=41)),
                     ((q, ki, w, Q[:, :, :3], K, V, 8), {}),
                     ((q, ki, w, Q[..., :32], K, V, 8), {}),
                     ((q, ki, w, Q.expand(2, 2, 4, 64), K, V, 8), {}),
                     ((q, ki, w[..., :3], Q, K, V, 8), {}),
                     ((q[..., :16], ki, w, Q, K, V, 8), {}),
                     ((wide, ki, wide[..., 0], Q, K, V, 8), {}),
                     ((q.expand(2, 2, 4, 32), ki, w.expand(2, 2, 4), Q, K, V, 8), {})]:
        with pytest.raises(AssertionError):
            D.dsa_decode(cache, *args, **kw)
    with pytest.raises(AssertionError):  # scores of a cache without index keys
        D.dsa_decode(odd, q, None, w, rows, rows, rows, 8)
    with pytest.raises(L.DSAUnsupported):
        D.dsa_decode(odd, q, None, w, rows, rows, rows, 40)
    for c, old in zip(caches, before):
        now = [getattr(c, n) for n in D.KV4Cache._BUFFERS if getattr(c, n) is not None]
        assert all(same(a, b) for a, b in zip(now, old))
    D.dsa_decode(cache, q, ki, w, Q, K, V, 8, keep=30, recent=30)
    assert cache.length.tolist() == [21, 5]


def test_python_refusals(dev):
    cache = D.KV4Cache.empty(2, 16, 2, 64, 32, 32, device=dev)
    K, V, ki = (torch.zeros(2, 1, *s, device=dev) for s in ((2, 64), (2, 32), (32,)))
    bad = [
        lambda: D.kv4_append(cache, K, V),                                   # no index keys
        lambda: D.kv4_append(cache, V, K, ki),
        lambda: D.kv4_append(cache, K[:1], V[:1], ki[:1]),
        lambda: D.kv4_append(cache, K.cpu(), V, ki),
        lambda: D.kv4_append(cache, K, V, ki, count=torch.ones(2, device=dev)),
        lambda: D.kv4_append(cache, K, V, ki, weight=torch.ones(2, 2, device=dev)),
        lambda: D.kv4_rows(cache, torch.zeros(3, 1, device=dev, dtype=torch.int32)),
        lambda: D.kv4_rows(cache, dtype=torch.int8),
        lambda: D.kv4_rows(cache, span=17),
        lambda: D.kv4_indexer_scores(cache, torch.zeros(2, 1, 4, 64, device=dev), torch.zeros(2, 1, 4, device=dev)),
        lambda: D.kv4_indexer_scores(cache, torch.zeros(2, 1, 4, 32, device=dev), torch.zeros(2, 1, 5, device=dev)),
        lambda: D.kv4_attention(cache, torch.zeros(2, 1, 4, 64, device=dev)),  # DK 64 with DV 32
        lambda: D.kv4_evict(cache, 4, 5),
        lambda: D.kv4_evict(cache, -1),
        lambda: D.dsa_decode(cache, *[K] * 6, top_k=0),
        lambda: D.dsa_decode(cache, *[K] * 6, top_k=4, keep=16),  # no room for a token
        lambda: D.KV4Cache(cache.codes[:, ::2], cache.scales[:, ::2], cache.length, DK=64),
        lambda: D.KV4Cache(cache.codes, cache.scales, cache.length.long(), DK=64),
        lambda: D.KV4Cache.empty(1, 4, 1, 48, 32, device=dev),
        lambda: D.KV4Cache.empty(1, 4, 1, 32, 32, 32, idx_dtype=torch.float8_e4m3fn, device=dev),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(AssertionError):
            f()
            say(i)
    even = D.KV4Cache.empty(2, 16, 2, 64, 64, device=dev)
    Q = torch.zeros(2, 1, 4, 64, device=dev)
    for f in (lambda: D.kv4_attention(even, Q[..., :32]), lambda: D.kv4_attention(even, Q[:, :, :3]),
              lambda: D.kv4_attention(even, Q, span=20),
              lambda: D.kv4_attention(even, Q, slots=torch.zeros(2, 1, 3, device=dev)),
              lambda: D.kv4_attention(even, Q, slots=torch.zeros(2, 2, 3, device=dev, dtype=torch.int32)),
              lambda: D.kv4_attention(even, Q, out=torch.zeros(2, device=dev)),
              lambda: D.kv4_indexer_scores(even, Q, Q[..., 0])):
        with pytest.raises(AssertionError):
            f()
    assert not cache.length.any()
