"""GPU: the paged 8-bit cache and windowed attention (dsa_paged) against their definitions in
64 bits (paged_oracle, which derives the bounds): append and rows bit for bit, attention over
pages and of prompts, and a run of them together."""
from __future__ import annotations

import math

import pytest
import torch

import _dsa_lib as L
import dsa_paged as P
import paged_oracle as O
from helpers import say

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def gen(seed):
    return torch.Generator().manual_seed(seed)


def randn(g, *shape, dtype=F32):
    return torch.randn(shape, generator=g).to(dtype)


def ints(dev, v):
    return torch.tensor(v, device=dev, dtype=torch.int32)


def dealt(dev, B, n, NP, g):
    """A page table of distinct pages in no order."""
    return torch.randperm(NP, generator=g)[:B * n].view(B, n).to(torch.int32).to(dev)


def filled(dev, B, S, HKV, DK, DV, lengths, page=64, seed=0, behind=0x7F):
    """A cache of random tokens; codes of slots past the length and of pages of nobody are
    `behind` (NaN), their scales too: nothing may read them into a result."""
    g = gen(seed)
    n = -(-S // page)
    NP = B * n + 3
    per = page // 64
    codes = torch.full((NP, HKV, per, 64 * (DK + DV)), behind, dtype=torch.uint8)
    scales = torch.full((NP, HKV, per, 2), 127, dtype=torch.uint8)
    pages = torch.randperm(NP, generator=g)[:B * n].view(B, n)
    for b in range(B):
        for blk in range(-(-lengths[b] // 64)):
            many = min(64, lengths[b] - 64 * blk)
            for h in range(HKV):
                row = codes[pages[b, blk // per], h, blk % per]
                for at, D, which in ((0, DK, 0), (64 * DK, DV, 1)):
                    x = randn(g, many, D).double() * 2.0 ** int(torch.randint(-3, 4, (1,), generator=g))
                    e = O.need(x)
                    c = O.encode(x, e)
                    part = row[at:at + 64 * D]
                    if which:
                        part.view(D, 64)[:, O.PLACE[:many]] = c.T
                    else:
                        part.view(64, D)[:many] = c
                    scales[pages[b, blk // per], h, blk % per, which] = e
    return P.KV8Cache(codes.to(dev), scales.to(dev), pages.to(torch.int32).to(dev), ints(dev, lengths), DK=DK)


def state(cache):
    return O.Held(cache.codes, cache.scales, cache.pages, cache.DK)


def same(a, b):
    return bool(torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8)))


def eq(a, b):
    """Equal; else the first places that are not (in place of the whole tensors)."""
    if torch.equal(a, b):
        return True
    say("shapes", tuple(a.shape), tuple(b.shape))
    if a.shape == b.shape:
        at = (a != b).nonzero()
        say(len(at), "differ:", [(i.tolist(), a[tuple(i)].item(), b[tuple(i)].item()) for i in at[:8]])
    return False


# --- append and rows -----------------------------------------------------------------------------
SIZES = [  # B, S, page, HKV, DK, DV, HQ, R, pairs, dtype
    (2, 256, 64, 2, 32, 32, 4, 32, False, F32),
    (1, 256, 128, 1, 64, 64, 0, 16, True, BF16),
    (3, 192, 64, 3, 96, 96, 3, 48, False, F16),
    (2, 512, 256, 2, 128, 128, 8, 128, False, BF16),
    (2, 256, 64, 2, 128, 128, 2, 64, True, F32),
    (1, 256, 64, 2, 192, 192, 2, 192, True, F16),
    (2, 256, 128, 1, 192, 128, 1, 64, False, F32),
    (1, 256, 64, 2, 256, 256, 4, 256, False, F32),
    (1, 256, 64, 1, 256, 256, 1, 0, False, BF16),
]


@pytest.mark.parametrize("B, S, page, HKV, DK, DV, HQ, R, pairs, dtype", SIZES)
def test_appends_bit_for_bit(dev, B, S, page, HKV, DK, DV, HQ, R, pairs, dtype):
    """A prompt, single tokens that make scales grow, a piece across blocks, tokens taken back,
    tokens past the last slot: codes, scales, counters and rotated rows after each."""
    g = gen(DK + HKV + page)
    cache = filled(dev, B, S, HKV, DK, DV, [0] * B, page, seed=1, behind=0x55)
    rope = P.rope_tables(S + 5, R, device="cpu") if R else None
    turn = tuple(x.to(dev) for x in rope) if rope else None
    lost = [0] * B
    where = [0] * B
    for i, (T, start, count, size) in enumerate([
            (70, None, None, 1.0), (1, None, None, 16.0), (1, None, None, 1e4), (2, None, [2] * B, 1e-3),
            (0, None, None, 1.0), (65, None, [65 - 7 * b for b in range(B)], 3.0), (3, [64] * B, [2] * B, 1.0),
            (5, [63 - b for b in range(B)], [0] * B, 1.0), (130, [100] * B, None, 30.0),
            (100, [S - 30] * B, [99] * B, 1.0), (1, [S] * B, None, 1.0)]):
        say("append", i, T, start, count, dtype)
        K, V = (randn(g, B, T, HKV, D) * size for D in (DK, DV))
        if i == 5 and T:
            K[0, 0, 0, :3] = torch.tensor([math.nan, math.inf, -math.inf])
            V[0, 1, 0, -2:] = torch.tensor([math.inf, 0.0])
            V[:, :, -1] = 0.0  # a head of zeros
        K, V = K.to(dtype), V.to(dtype)
        Q = randn(g, B, T, HQ, DK, dtype=dtype) if HQ else None
        want = state(cache)
        first = start if start is not None else where
        many = count if count is not None else [T] * B
        Kr = K.float()
        if rope:
            at = [torch.arange(T) + first[b] for b in range(B)]
            Kr = torch.stack([O.rotate(K[b], *rope, at[b].clamp(max=S - 1), pairs) for b in range(B)])
        for b in range(B):
            lost[b] += O.append(want, b, first[b], Kr[b, :many[b]], V[b, :many[b]].float())
            where[b] = min(S, first[b] + many[b])
        q, k = P.kv8_append(cache, K.to(dev), V.to(dev), rope=turn, pairs=pairs, Q=Q.to(dev) if HQ else None,
                            start=ints(dev, start) if start is not None else None,
                            count=ints(dev, count) if count is not None else None, keys=True)
        got = state(cache)
        assert cache.length.tolist() == where and cache.lost.tolist() == lost, (i, cache.length, where, cache.lost, lost)
        for n in ("ks", "vs", "k", "v"):
            assert eq(getattr(got, n), getattr(want, n)), (i, n)
        if rope:
            past = torch.stack([a >= S for a in at]).view(B, T, 1, 1)
            assert eq(k.cpu().nan_to_num(7.0), Kr.masked_fill(past, math.nan).to(dtype).nan_to_num(7.0)), i
            if HQ:
                qr = torch.stack([O.rotate(Q[b], *rope, at[b].clamp(max=S - 1), pairs) for b in range(B)])
                assert eq(q.cpu().nan_to_num(7.0), qr.masked_fill(past, math.nan).to(dtype).nan_to_num(7.0)), i
        elif HQ:
            assert eq(q.cpu(), Q) and eq(k.cpu().nan_to_num(7.0), K.nan_to_num(7.0)), i
    with pytest.raises(RuntimeError, match="lost|found no slot"):
        cache.check()
    # every slot back as values
    K64, V64 = want.values()
    for dt in (F32, BF16):
        k, v = P.kv8_rows(cache, dtype=dt)
        behind = (torch.arange(S).view(1, S) >= cache.length.cpu().view(-1, 1)).view(B, S, 1, 1)
        for x, y in ((k, K64), (v, V64)):
            y = y.masked_fill(behind, 0.0)
            assert eq(x.double().cpu().nan_to_num(9.0), y.nan_to_num(9.0))
    pick = torch.tensor([[3, -1, S, 3, 64, 127, 2 ** 31 - 1]] * B, dtype=torch.int32)
    k, v = P.kv8_rows(cache, pick.to(dev), dtype=F16)
    ok = (pick >= 0) & (pick < cache.length.cpu().view(-1, 1))
    for x, y in ((k, K64), (v, V64)):
        y = torch.stack([y[b, pick[b].clamp(0, S - 1).long()] for b in range(B)]).masked_fill(~ok.view(B, -1, 1, 1), 0.0)
        assert eq(x.cpu().nan_to_num(9.0), y.to(F16).nan_to_num(9.0))


def test_append_on_bad_pages(dev):
    """Tokens on ids that name no page are counted and written nowhere; the rest goes in."""
    cache = filled(dev, 2, 512, 2, 64, 64, [0, 0], seed=3, behind=0)
    cache.pages[0, 1], cache.pages[0, 2], cache.pages[1, 0] = -1, cache.NP, 2 ** 31 - 1
    g = gen(5)
    K, V = randn(g, 2, 300, 2, 64), randn(g, 2, 300, 2, 64)
    want = state(cache)
    before = cache.codes.clone()
    lost = [O.append(want, b, 0, K[b], V[b]) for b in range(2)]
    P.kv8_append(cache, K.to(dev), V.to(dev))
    assert lost == [128, 64] and cache.lost.tolist() == lost and cache.length.tolist() == [300, 300]
    got = state(cache)
    held = want.page.repeat_interleave(64, 1)
    assert eq(got.k[held], want.k[held]) and eq(got.v[held], want.v[held])
    used = set(cache.pages.flatten().tolist())
    for p in range(cache.NP):
        if p not in used:
            assert eq(cache.codes[p], before[p]), p
    k, _ = P.kv8_rows(cache, span=320)
    assert not k[0, 64:192].any() and not k[1, :64].any() and not k[:, 300:].any() and bool(k[0, :64].any())


def test_columns_of_a_projection(dev):
    """q, k and v as the columns of one tensor go in as they are, and give what copies give."""
    g = gen(9)
    B, T, HQ, HKV, D = 2, 150, 4, 2, 64
    y = randn(g, B, T, (HQ + 2 * HKV) * D, dtype=BF16).to(dev)
    Q = y[..., :HQ * D].unflatten(-1, (HQ, D))
    K = y[..., HQ * D:(HQ + HKV) * D].unflatten(-1, (HKV, D))
    V = y[..., (HQ + HKV) * D:].unflatten(-1, (HKV, D))
    assert P._tokens(K, BF16)[1:] == (K.data_ptr(), (HQ + 2 * HKV) * D)
    rope = P.rope_tables(192, D, device=dev)
    out = []
    for copy in (False, True):
        q, k, v = (x.contiguous() if copy else x for x in (Q, K, V))
        cache = P.KV8Cache.empty(B, 192, HKV, D, D, device=dev)
        qr, kr = P.kv8_append(cache, k, v, rope=rope, Q=q, keys=True)
        out.append((cache.codes, cache.scales, qr, kr, P.window_attention(q, k, v, window=70, sinks=2)))
    assert all(same(a, b) for a, b in zip(*out))
    # other orders: heads before tokens, every second token, a reversed batch
    ref = P.window_attention(Q.contiguous(), K.contiguous(), V.contiguous(), window=33)
    assert same(P.window_attention(Q.transpose(1, 2).contiguous().transpose(1, 2), K, V, window=33), ref)
    two = torch.stack([y, y], 2).flatten(1, 2)[:, ::2]
    assert same(P.window_attention(two[..., :HQ * D].unflatten(-1, (HQ, D)), K, V, window=33), ref)
    f = y.flip(0)
    assert same(P.window_attention(Q.flip(0), f[..., HQ * D:(HQ + HKV) * D].unflatten(-1, (HKV, D)), V.flip(0), window=33), ref.flip(0))


# --- attention over the cache --------------------------------------------------------------------
ATTENTION = [  # B, lengths, page, HQ, HKV, DK, DV, Tq, window, sinks, count, dtype
    (1, [1], 64, 4, 4, 32, 32, 1, None, 0, None, F32),
    (2, [129, 64], 64, 4, 4, 32, 32, 1, None, 0, None, F32),
    (2, [500, 65], 128, 8, 2, 64, 64, 1, None, 0, None, F16),
    (3, [700, 1, 0], 64, 16, 1, 128, 128, 1, None, 0, None, BF16),
    (2, [300, 257], 256, 4, 2, 96, 96, 3, None, 0, None, F32),
    (2, [333, 200], 64, 6, 2, 192, 192, 2, 100, 3, None, BF16),
    (1, [400], 64, 2, 1, 192, 128, 1, None, 0, None, F32),
    (2, [300, 130], 64, 4, 2, 256, 256, 2, 64, 0, None, F32),
    (2, [640, 639], 64, 32, 2, 128, 128, 1, 65, 4, None, BF16),
    (2, [640, 70], 64, 8, 1, 64, 64, 20, 1, 0, None, F16),
    (2, [512, 300], 128, 4, 1, 64, 64, 40, 90, 70, None, F32),
    (3, [200, 100, 50], 64, 4, 2, 64, 64, 5, None, 0, [5, 2, 0], BF16),
    (2, [1500, 1100], 64, 5, 1, 128, 128, 1, None, 0, None, F32),
    (1, [1600], 64, 2, 2, 64, 64, 33, 700, 1, [17], F16),
    (2, [90, 40], 64, 4, 4, 64, 64, 60, None, 0, None, F32),  # more new tokens than slots of one
]


def check_attention(dev, cache, Q, dtype, window, sinks, count=None, span=None, scale=None, want=None):
    lengths = [max(0, min(x, cache.S)) for x in cache.length.tolist()]
    B, Tq, HQ, DK = Q.shape
    out = P.kv8_attention(cache, Q.to(dev), window=window, sinks=sinks, span=span, scale=scale,
                          count=ints(dev, count) if count is not None else None)
    assert out.dtype == dtype and out.shape == (B, Tq, HQ, cache.DV)
    h = want or state(cache)
    K, V = h.values()
    page = h.page.repeat_interleave(64, 1)
    n = cache.S if span is None else span
    worst = 0.0
    for b in range(B):
        many = Tq if count is None else max(0, min(count[b], Tq))
        t = lengths[b] - many + torch.arange(Tq)
        ok = O.sees(min(lengths[b], n), t, torch.arange(cache.S), window, sinks) & page[b].view(1, -1)
        ok[many:] = False
        ref, mass, big = O.attention(Q[b], K[b], V[b], ok, scale if scale is not None else 1 / math.sqrt(DK))
        got = out[b].double().cpu()
        assert eq(got.isnan(), ref.isnan()), b
        vmax = float(V[b][:lengths[b]].nan_to_num().abs().max()) if lengths[b] else 0.0
        lim = O.bound(dtype, lengths[b], DK, mass, big, ref, False, vmax)
        # beyond the type's largest number the result is Inf
        over = ref.abs() > torch.finfo(dtype).max
        assert bool((got[over] == ref[over].sign() * math.inf).all())
        fine = ~ref.isnan() & ~over
        err = (got - ref).abs()[fine] / lim[fine]
        if err.numel():
            worst = max(worst, float(err.max()))
    assert worst <= 1.0, worst
    return out, worst


@pytest.mark.parametrize("B, lengths, page, HQ, HKV, DK, DV, Tq, window, sinks, count, dtype", ATTENTION)
def test_attention(dev, B, lengths, page, HQ, HKV, DK, DV, Tq, window, sinks, count, dtype):
    say("attention", lengths, page, HQ, HKV, DK, DV, Tq, window, sinks, count, dtype)
    S = -(-(max(lengths) + 1) // page) * page
    cache = filled(dev, B, S, HKV, DK, DV, lengths, page, seed=DK + Tq)
    Q = randn(gen(Tq), B, Tq, HQ, DK).to(dtype)
    _, worst = check_attention(dev, cache, Q, dtype, window, sinks, count)
    say("  worst share of the bound", worst)
    check_attention(dev, cache, Q, dtype, window, sinks, count, span=max(0, max(lengths) - 30), scale=0.3)
    out = torch.empty(B, Tq, HQ, DV, device=dev, dtype=dtype)
    c = ints(dev, count) if count is not None else None
    a = P.kv8_attention(cache, Q.to(dev), window=window, sinks=sinks, count=c, out=out)
    assert a is out and same(a, P.kv8_attention(cache, Q.to(dev), window=window, sinks=sinks, count=c))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_attention_scales_far_apart(dev, dtype):
    """Blocks of very small and very large values, rows of Q of very different sizes: every
    one keeps its precision, and a large V that weighs nothing takes none from a small one."""
    cache = filled(dev, 1, 320, 1, 64, 64, [300], seed=11)
    at = cache.pages[0].long()
    cache.scales[at[0], 0, 0, 1] += 60
    cache.scales[at[1], 0, 0, 1] -= 60
    cache.scales[at[2], 0, 0, 0] -= 20
    Q = randn(gen(3), 1, 1, 6, 64) * torch.tensor([1e-30, 1e-4, 1.0, 3.0, 1e4 if dtype == F16 else 1e10, 0.0]).view(1, 1, 6, 1)
    check_attention(dev, cache, Q.to(dtype), dtype, None, 0)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_what_is_not_seen_does_not_count(dev, dtype):
    """NaN in slots that some tokens see and others do not, in slots before the window, on
    pages of nobody; ids that name no page inside and outside the window."""
    cache = filled(dev, 2, 512, 1, 64, 64, [400, 390], seed=13)
    page = cache.pages.cpu()

    def spoil(b, slot, v):
        row = cache.codes[page[b, slot // 64], 0, 0]
        if v:
            row[64 * 64 + 5 * 64 + O.place(slot % 64)] = 0xFF
        else:
            row[(slot % 64) * 64 + 7] = 0x7F

    for b, slot in ((0, 399), (0, 398), (1, 389), (0, 250)):  # the newest, and one before the window
        spoil(b, slot, True)
    spoil(1, 388, False)
    cache.pages[0, 1] = -1          # behind the window: never looked at
    cache.pages[1, 5] = cache.NP    # inside it: holds nothing
    Q = randn(gen(1), 2, 4, 4, 64).to(dtype)
    out, _ = check_attention(dev, cache, Q, dtype, 130, 2)
    nan = out.isnan().cpu()
    # only dimension 5 of the tokens that see the slots; all of those that see a NaN key
    assert nan[0, :2].sum() == 0 and nan[0, 2:, :, 5].all() and nan[0].sum() == 2 * 4
    assert nan[1, 0:2].sum() == 0 and nan[1, 2:].all()
    check_attention(dev, cache, Q, dtype, None, 0)


def test_rows_of_q_that_are_not_finite(dev):
    cache = filled(dev, 1, 192, 2, 64, 64, [150], seed=2)
    for dtype in (F32, BF16, F16):
        Q = randn(gen(4), 1, 2, 4, 64).to(dtype)
        ref = P.kv8_attention(cache, Q.to(dev))
        bad = Q.clone()
        bad[0, 0, 1, 3], bad[0, 1, 2, 0], bad[0, 1, 3, 9] = math.nan, math.inf, -math.inf
        out = P.kv8_attention(cache, bad.to(dev))
        rows = torch.zeros(1, 2, 4, dtype=torch.bool)
        rows[0, 0, 1] = rows[0, 1, 2] = rows[0, 1, 3] = True
        assert out[rows.to(dev)].isnan().all() and same(out[~rows.to(dev)], ref[~rows.to(dev)])


def test_lengths_out_of_range_and_empty_calls(dev):
    cache = filled(dev, 2, 128, 1, 64, 64, [100, 60], seed=6)
    Q = randn(gen(0), 2, 1, 2, 64).to(dev)
    ref = P.kv8_attention(cache, Q)
    cache.length.copy_(ints(dev, [-5, 1000]))
    out = P.kv8_attention(cache, Q)
    assert out[0].isnan().all()
    cache.length.copy_(ints(dev, [100, 60]))
    assert same(P.kv8_attention(cache, Q), ref)
    assert P.kv8_attention(cache, Q[:, :0]).shape == (2, 0, 2, 64)
    assert P.kv8_attention(cache, Q, span=0).isnan().all()
    none = P.KV8Cache.empty(0, 64, 1, 64, 64, device=dev)
    x = torch.empty(0, 1, 1, 64, device=dev)
    P.kv8_append(none, x, x)
    assert P.kv8_attention(none, x).shape == (0, 1, 1, 64) and P.kv8_rows(none)[0].shape == (0, 64, 1, 64)
    assert P.window_attention(x, x, x).shape == (0, 1, 1, 64)
    y = torch.empty(2, 0, 1, 64, device=dev)
    assert P.window_attention(y, y, y, window=3).shape == (2, 0, 1, 64)
    P.kv8_append(cache, y, y, start=ints(dev, [7, 9]))
    assert cache.length.tolist() == [7, 9]


# --- prompts -------------------------------------------------------------------------------------
WINDOW = [  # B, T, HQ, HKV, D, window, sinks, count, dtype
    (1, 1, 2, 1, 64, 1, 0, None, BF16),
    (1, 100, 4, 4, 32, 32, 4, None, F32),
    (2, 130, 4, 2, 32, None, 0, None, BF16),
    (2, 257, 4, 1, 64, 100, 1, [257, 200], F16),
    (2, 300, 2, 2, 64, 64, 70, [129, 0], F32),
    (1, 400, 4, 2, 128, 129, 130, None, BF16),
    (2, 333, 2, 1, 128, 1, 0, [333, 128], F16),
    (1, 200, 2, 1, 128, 63, 5, None, F32),
    (1, 260, 2, 1, 256, 128, 4, None, BF16),
    (1, 190, 2, 1, 256, 65, 1, [150], F32),
    (9, 70, 3, 3, 64, 17, 2, [70, 1, 2, 63, 64, 65, 0, 33, 70], BF16),
    (1, 600, 1, 1, 64, 600, 3, None, F16),
    (1, 384, 1, 1, 64, 1 << 40, 1 << 40, None, F32),
]


def check_window(dev, Q, K, V, dtype, window, sinks, count=None, scale=None):
    B, T, HQ, D = Q.shape
    out = P.window_attention(Q.to(dev), K.to(dev), V.to(dev), window=window, sinks=sinks, scale=scale,
                             count=ints(dev, count) if count is not None else None)
    assert out.dtype == dtype and out.shape == Q.shape
    worst = 0.0
    for b in range(B):
        n = T if count is None else count[b]
        ok = O.sees(n, torch.arange(T), torch.arange(T), window, sinks)
        ok[n:] = False
        ref, mass, big = O.attention(Q[b], K[b], V[b], ok, scale if scale is not None else 1 / math.sqrt(D))
        got = out[b].double().cpu()
        assert eq(got.isnan(), ref.isnan()), b
        inf = ref.isinf()
        assert eq(got[inf], ref[inf])
        fine = ref.isfinite()
        finite = V[b, :n].double()
        lim = O.bound(dtype, n, D, mass, big, ref, True, float(finite[finite.isfinite()].abs().max()) if n else 0.0)
        err = (got - ref).abs()[fine] / lim[fine]
        if err.numel():
            worst = max(worst, float(err.max()))
    assert worst <= 1.0, worst
    return out, worst


@pytest.mark.parametrize("B, T, HQ, HKV, D, window, sinks, count, dtype", WINDOW)
def test_window(dev, B, T, HQ, HKV, D, window, sinks, count, dtype):
    say("window", B, T, HQ, HKV, D, window, sinks, count, dtype)
    g = gen(T + D)
    Q, K, V = randn(g, B, T, HQ, D, dtype=dtype), randn(g, B, T, HKV, D, dtype=dtype), randn(g, B, T, HKV, D, dtype=dtype)
    if count is not None:  # a padded batch's rows behind the tokens
        for b in range(B):
            Q[b, count[b]:], K[b, count[b]:], V[b, count[b]:] = math.nan, math.inf, math.nan
    _, worst = check_window(dev, Q, K, V, dtype, window, sinks, count)
    say("  worst share of the bound", worst)
    check_window(dev, Q * 4, K, V, dtype, window, sinks, count, scale=0.4)


@pytest.mark.parametrize("D, dtype", [(64, BF16), (64, F16), (128, BF16), (64, F32), (256, F16), (128, F32)])
def test_window_keeps_what_is_not_seen_out(dev, D, dtype):
    """NaN and Inf in keys and values behind the window and ahead of a token reach only the
    rows that see them; Inf in V gives Inf, both signs NaN."""
    g = gen(D)
    T = 400
    Q, K, V = (randn(g, 1, T, 2, D, dtype=dtype) for _ in range(3))
    V[0, 200, 0, 3], V[0, 260, 0, 7], V[0, 261, 0, 7] = math.nan, math.inf, -math.inf
    V[0, 310, 1, 0], K[0, 150, 1, 5], V[0, 1, 1, 2] = math.inf, math.nan, -math.inf
    out, _ = check_window(dev, Q, K, V, dtype, 50, 2)
    odd = (~out.isfinite()).cpu()
    assert odd[0, :200, 0].sum() == 0 and odd[0, 200:250, 0, 3].all() and odd[0, 250:260, 0].sum() == 0
    assert odd[0, 260:311, 0, 7].all() and odd[0, 311:, 0].sum() == 0
    assert odd[0, 0, 1].sum() == 0 and (out[0, 1:150, 1, 2] == -math.inf).all() and out[0, 150:200, 1].isnan().all()


def test_window_small_values(dev):
    """Logits far below the others', values near the least of the type, one key's worth of mass."""
    g = gen(8)
    for dtype in (F32, BF16, F16):
        Q, K, V = (randn(g, 1, 300, 2, 64) for _ in range(3))
        Q[0, 100:] *= 20
        V[0, :, 1] *= 1e-4 if dtype == F16 else 1e-30
        check_window(dev, Q.to(dtype), K.to(dtype), V.to(dtype), dtype, 90, 3)


def test_refused_by_the_python_layer(dev):
    x = torch.zeros(2, 8, 4, 64, device=dev)
    for bad in (dict(window=0), dict(window=-1), dict(sinks=-1), dict(scale=math.inf),
                dict(count=ints(dev, [1])), dict(count=torch.tensor([1, 2], device=dev)), dict(count=torch.tensor([1, 2], dtype=torch.int32)),
                dict(out=torch.empty(2, 8, 4, 64, device=dev, dtype=BF16)), dict(out=torch.empty(2, 8, 4, 32, device=dev)),
                dict(out=torch.empty(2, 8, 64, 4, device=dev).transpose(2, 3))):
        with pytest.raises(AssertionError):
            P.window_attention(x, x, x, **bad)
    for q, k in ((x[:, :, :3], x[:, :, :2]), (x, x[:, :7]), (x[0], x[0]), (x[..., :48], x[..., :48])):
        with pytest.raises(AssertionError):
            P.window_attention(q, k, k)
    cache = P.KV8Cache.empty(2, 128, 2, 64, 64, device=dev)
    k, rope = x[:, :, :2], P.rope_tables(128, 64, device=dev)
    before = cache.codes.clone()
    for bad in (dict(rope=P.rope_tables(127, 64, device=dev)), dict(rope=P.rope_tables(128, 24, device=dev)),
                dict(rope=P.rope_tables(128, 80, device=dev)), dict(rope=(rope[0], rope[1][:5])), dict(rope=tuple(t.double() for t in rope)),
                dict(start=ints(dev, [1])), dict(start=torch.zeros(2, device=dev)), dict(count=torch.tensor([1, 1], dtype=torch.int32)),
                dict(Q=x[:, :7], rope=rope), dict(Q=x[..., :32], rope=rope), dict(rope=tuple(t.cpu() for t in rope))):
        with pytest.raises(AssertionError):
            P.kv8_append(cache, k, k, **bad)
    for kk, vv in ((x, x), (k[:1], k[:1]), (k, k[:, :3]), (k[..., :32], k), (k.cpu(), k)):
        with pytest.raises(AssertionError):
            P.kv8_append(cache, kk, vv)
    assert eq(cache.codes, before) and cache.length.tolist() == [0, 0]
    for bad in (dict(window=0), dict(sinks=-2), dict(span=129), dict(span=-1), dict(scale=math.nan), dict(count=ints(dev, [1, 2, 3])),
                dict(out=torch.empty(2, 8, 4, 64, device=dev, dtype=F16))):
        with pytest.raises(AssertionError):
            P.kv8_attention(cache, x, **bad)
    for q in (x[:, :, :3], x[:1], x[..., :32], x.cpu()):
        with pytest.raises(AssertionError):
            P.kv8_attention(cache, q)
    with pytest.raises(AssertionError):
        P.kv8_rows(cache, ints(dev, [[1]]))
    with pytest.raises(AssertionError):
        P.kv8_rows(cache, dtype=torch.float64)
    with pytest.raises(AttributeError):
        cache.length = cache.length.clone()
    for sizes in (dict(DK=48, DV=48), dict(page=96), dict(page=32), dict(HKV=0)):
        with pytest.raises(AssertionError):
            P.KV8Cache.empty(**{**dict(B=1, S=64, HKV=1, DK=64, DV=64, device=dev), **sizes})
    with pytest.raises(L.DSAUnsupported):
        P.KV8Cache.empty(1, 64, 1, 64, 128, device=dev)


# --- together ------------------------------------------------------------------------------------
def step_reference(K, V, want, b, t0, T, rope):
    """Rotated keys of T tokens from t0 on, into the oracle's cache."""
    kr = O.rotate(K[b, t0:t0 + T], *rope, torch.arange(t0, t0 + T), False)
    assert O.append(want, b, t0, kr, V[b, t0:t0 + T].float()) == 0
    return kr


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_prompt_and_steps_together(dev, dtype):
    """A padded batch's prompt (append, attention on the rotated rows), then steps of one and
    of three drafted tokens, one of them taken back, pages dealt out as they are needed and
    taken back behind the window: against 64 bits at each."""
    g = gen(21)
    B, HQ, HKV, D, page, window, sinks, N = 2, 4, 2, 64, 64, 100, 3, 330
    rope = P.rope_tables(384, D, device="cpu")
    turn = tuple(x.to(dev) for x in rope)
    Q, K, V = randn(g, B, N, HQ, D, dtype=dtype), randn(g, B, N, HKV, D, dtype=dtype), randn(g, B, N, HKV, D, dtype=dtype)
    cache = P.KV8Cache.empty(B, 384, HKV, D, D, page=page, NP=9, device=dev)
    free = list(range(9))

    def deal(lengths):
        for b in range(B):
            for i in range(6):
                used = i * page < lengths[b] and (i == 0 or (i + 1) * page > lengths[b] - window - 8)
                have = int(cache.pages[b, i])
                if used and have < 0:
                    cache.pages[b, i] = free.pop()
                elif not used and have >= 0:
                    cache.pages[b, i] = -1
                    free.append(have)

    # the oracle's own cache has every page
    want = O.Held(torch.zeros(12, HKV, 1, 128 * D, dtype=torch.uint8), torch.zeros(12, HKV, 1, 2, dtype=torch.uint8),
                  torch.arange(12).view(B, 6), D)
    lengths = [200, 77]
    for b in range(B):
        for i in range(-(-lengths[b] // page)):
            cache.pages[b, i] = free.pop()
    T = 200
    qr, kr = P.kv8_append(cache, K[:, :T].to(dev), V[:, :T].to(dev), rope=turn, Q=Q[:, :T].to(dev), count=ints(dev, lengths), keys=True)
    o = P.window_attention(qr, kr, V[:, :T].to(dev), window=window, sinks=sinks, count=ints(dev, lengths))
    for b in range(B):
        k = step_reference(K, V, want, b, 0, lengths[b], rope)
        ok = O.sees(lengths[b], torch.arange(T), torch.arange(T), window, sinks)
        ok[lengths[b]:] = False
        full = torch.zeros(T, HKV, D)
        full[:lengths[b]] = k.to(dtype).float()
        q = O.rotate(Q[b, :T], *rope, torch.arange(T), False).to(dtype)
        ref, mass, big = O.attention(q, full, V[b, :T], ok, 1 / math.sqrt(D))
        lim = O.bound(dtype, T, D, mass, big, ref, True, float(V[b].double().abs().max()))
        got = o[b].double().cpu()
        assert eq(got.isnan(), ref.isnan())
        assert bool(((got - ref).abs() <= lim)[~ref.isnan()].all()), b
    for i, (Tq, back) in enumerate([(1, 0), (1, 0), (3, 1), (1, 0), (3, 0)] + [(3, 0)] * 12):
        deal([n + Tq for n in lengths])
        idx = [slice(n, n + Tq) for n in lengths]
        q, k, v = (torch.stack([x[b, idx[b]] for b in range(B)]).to(dev) for x in (Q, K, V))
        qr, _ = P.kv8_append(cache, k, v, rope=turn, Q=q)
        o = P.kv8_attention(cache, qr, window=window, sinks=sinks)
        for b in range(B):
            step_reference(K, V, want, b, lengths[b], Tq, rope)
            lengths[b] += Tq
            kk, vv = want.values()
            t = lengths[b] - Tq + torch.arange(Tq)
            ref, mass, big = O.attention(qr[b].cpu(), kk[b], vv[b], O.sees(lengths[b], t, torch.arange(384), window, sinks), 1 / math.sqrt(D))
            lim = O.bound(dtype, lengths[b], D, mass, big, ref, False, float(vv[b].abs().max()))
            assert bool(((o[b].double().cpu() - ref).abs() <= lim).all()), (i, b)
        if back:
            lengths = [n - back for n in lengths]
            cache.length.copy_(ints(dev, lengths))
    assert cache.length.tolist() == lengths
    cache.check()


def test_captured_steps(dev):
    """A step captured into a graph advances the cache with each replay, as eager calls do,
    with the program's own work between them."""
    g = gen(31)
    B, HQ, HKV, D, T0, n = 2, 8, 2, 128, 700, 6
    rope = P.rope_tables(1024, D, device=dev)
    K, V, Q = (randn(g, B, T0 + n, h, D, dtype=BF16).to(dev) for h in (HKV, HKV, HQ))

    def fresh():
        c = P.KV8Cache.empty(B, 1024, HKV, D, D, page=128, device=dev)
        P.kv8_append(c, K[:, :T0], V[:, :T0], rope=rope, count=ints(dev, [T0, T0 - 60]))
        return c

    def step(c, q, k, v):
        qr, _ = P.kv8_append(c, k, v, rope=rope, Q=q)
        return P.kv8_attention(c, qr), P.kv8_attention(c, qr, window=200, sinks=2)

    eager, c = fresh(), fresh()
    q, k, v = Q[:, :1].clone(), K[:, :1].clone(), V[:, :1].clone()
    start = c.length.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(c, q, k, v)
    torch.cuda.current_stream().wait_stream(side)
    c.length.copy_(start)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = step(c, q, k, v)
    c.length.copy_(start)
    for i in range(n):
        for dst, src in ((q, Q), (k, K), (v, V)):
            dst.copy_(src[:, T0 + i:T0 + i + 1])
        graph.replay()
        ref = step(eager, Q[:, T0 + i:T0 + i + 1], K[:, T0 + i:T0 + i + 1], V[:, T0 + i:T0 + i + 1])
        torch.cuda.synchronize()
        assert eq(c.length, eager.length)
        assert all(same(a, b) for a, b in zip(o, ref)), i
    wgraph = torch.cuda.CUDAGraph()
    x, y, z = Q[:, :300].clone(), K[:, :300].clone(), V[:, :300].clone()
    P.window_attention(x, y, z, window=77)
    with torch.cuda.graph(wgraph):
        w = P.window_attention(x, y, z, window=77)
    for i in range(3):
        x.copy_(Q[:, i:i + 300])
        wgraph.replay()
        assert same(w, P.window_attention(x, y, z, window=77))


def test_two_calls_at_once(dev):
    """Calls on two streams with workspaces of their own, over one cache that both read."""
    cache = filled(dev, 2, 1536, 2, 64, 64, [1500, 1300], seed=17)
    Q = [randn(gen(s), 2, 1, 8, 64, dtype=BF16).to(dev) for s in range(2)]
    ref = [P.kv8_attention(cache, q) for q in Q]
    streams = [torch.cuda.Stream() for _ in Q]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    outs = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[i].append(P.kv8_attention(cache, Q[i]))
    torch.cuda.synchronize()
    assert all(same(o, ref[i]) for i in range(2) for o in outs[i])
