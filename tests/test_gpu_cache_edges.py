"""GPU: calls of the 4-bit decode cache at the edges of what they allow."""
from __future__ import annotations

import math

import pytest
import torch

import _dsa_lib as L
import cache_oracle as C
import dsa_cache as D
from helpers import say
from test_gpu_cache import BF16, F16, F32, attend, check_evict, filled, gen, ints, randn, same, step_inputs, within
from topk_threshold import topk_indices

pytestmark = pytest.mark.gpu


# --- the indexer -----------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("HI, DI", [(1, 32), (4, 32), (12, 64), (16, 32), (17, 128), (63, 128), (250, 128)])
def test_infinite_index_keys(dev, dtype, HI, DI):
    """An Inf in a key gives what the sum gives: +-Inf where a head's product is +Inf,
    and nothing where the ReLU takes all of them away, whatever HI pads to."""
    say("infinite keys", dtype, HI, DI)
    g, S = gen(dev, HI), 70
    q, k = randn(g, 1, 2, HI, DI, dtype=dtype), randn(g, 1, S, DI, dtype=dtype)
    q[..., 0] = q[..., 0].abs() + 0.5
    q[..., 1] = -q[..., 0]
    q[:, :, HI - 1, 1] = 1.0  # the last head alone
    w = randn(g, 1, 2, HI).abs() + 0.5
    w[:, 1] *= -1
    w = w.to(dtype)
    clean = D.kv4_indexer_scores(D.KV4Cache(None, None, ints(dev, [S]), k.clone()), q, w)
    k[0, 5, 0], k[0, 6, 0], k[0, 7, 1], k[0, 69, 0] = math.inf, -math.inf, math.inf, math.inf
    got = D.kv4_indexer_scores(D.KV4Cache(None, None, ints(dev, [S]), k), q, w)
    inf = math.inf
    assert got[0, :, [5, 6, 7]].tolist() == [[inf, 0.0, inf], [-inf, 0.0, -inf]]
    assert got[0, 1, 69].item() == -inf and got[0, 0, 69].item() == -inf  # the second token sees it, the first does not
    keep = [s for s in range(S - 1) if s not in (5, 6, 7)]
    assert torch.equal(got[..., keep], clean[..., keep])


@pytest.mark.parametrize("cached", [BF16, F16])
@pytest.mark.parametrize("q_dtype, w_dtype", [(F32, F32), (None, F32), (F32, None), (BF16, F16), (torch.float64, F32)])
@pytest.mark.parametrize("HI, DI, Tq", [(4, 32, 1), (17, 64, 3), (64, 128, 2), (9, 256, 1), (250, 128, 1)])
def test_mixed_types_of_the_indexer(dev, cached, q_dtype, w_dtype, HI, DI, Tq):
    """Queries and weights of another type than the cached keys' lose none of their bits:
    mixed types go as fp32 (None: the cache's own)."""
    q_dtype, w_dtype = q_dtype or cached, w_dtype or cached
    say("mixed", cached, q_dtype, w_dtype, HI, DI, Tq)
    lengths, S = [333, 40, 1, 0], 333
    cache = filled(dev, 4, S, 1, 32, 32, lengths, 1, DI, cached)
    g = gen(dev, HI)
    q, w = randn(g, 4, Tq, HI, DI, dtype=q_dtype), randn(g, 4, Tq, HI, dtype=w_dtype)
    if q_dtype is F32:
        q[0] *= 1e5  # past fp16's range
    for kw in ({}, dict(count=ints(dev, [Tq, 1, 0, 1]), span=300)):
        want, lim = C.indexer(torch.nan_to_num(cache.k_idx), cache.length, q.float(), w.float(), **kw)
        within(D.kv4_indexer_scores(cache, q, w, **kw), want, lim, "scores")


def test_infinite_keys_and_mixed_types(dev):
    g, S, HI = gen(dev, 1), 40, 12
    q, w, k = randn(g, 1, 1, HI, 64).abs() + 0.5, randn(g, 1, 1, HI).abs(), randn(g, 1, S, 64, dtype=BF16)
    k[0, 3, 9], k[0, 4, 9], k[0, 5, 63] = math.inf, -math.inf, math.nan
    got = D.kv4_indexer_scores(D.KV4Cache(None, None, ints(dev, [S]), k), q, w)[0, 0]
    assert got[3].item() == math.inf and got[4].item() == 0.0 and torch.isnan(got[5])
    assert torch.isfinite(got[6:]).all()


# --- attention ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("HQ", [1, 16])
@pytest.mark.parametrize("low", [-2048.0, -2.0 ** 100])
@pytest.mark.parametrize("listed", [False, True])
def test_nan_value_beside_a_far_larger_logit(dev, HQ, low, listed):
    """A visible slot's NaN value is NaN in the output however small its probability
    (0 * NaN), also where blocks share a long cache and its block's sums weigh nothing."""
    S, D_ = 5000, 64
    say("far below", HQ, low, listed)
    K, V = torch.zeros(1, S, 1, D_, device=dev), torch.ones(1, S, 1, D_, device=dev)
    K[..., 0] = low
    K[0, 7] = 0
    V[0, 4000, 0, 3] = math.nan  # the first 32 columns
    cache = D.KV4Cache.empty(1, S, 1, D_, D_, device=dev)
    D.kv4_append(cache, K, V)
    Q = torch.zeros(1, 1, HQ, D_, device=dev)
    Q[..., 0] = 8.0 if low > -1e6 else 2.0 ** 100
    slots = torch.arange(S, device=dev, dtype=torch.int32).flip(0).expand(1, 1, S) if listed else None
    out = D.kv4_attention(cache, Q, slots=slots)
    assert torch.isnan(out[..., :32]).all() and bool((out[..., 32:] == 1).all())
    cache.length.fill_(4000)  # the NaN is behind the last slot
    assert bool((D.kv4_attention(cache, Q, slots=slots) == 1).all())


# --- the step ----------------------------------------------------------------------------------------
NAMES = ("codes", "scales", "length", "k_idx", "position", "weight", "seen", "lost")


def copy_of(c):
    return D.KV4Cache(*(getattr(c, n).clone() for n in NAMES[:4]),
                      **{n: getattr(c, n).clone() for n in NAMES[4:]}, DK=c.DK)


@pytest.mark.parametrize("S, length, Tq, keep, recent", [
    (10, 10, 1, 6, 2), (10, 9, 2, 6, 0), (10, 10, 2, 8, 8), (300, 300, 3, 100, 7), (300, 298, 3, 297, 0),
    (400, 390, 70, 200, 20), (20000, 19999, 2, 17000, 64),
])
def test_step_of_a_full_cache(dev, S, length, Tq, keep, recent):
    """A prompt that left no room: the step first evicts down to it, so that every new
    token is stored and sees itself."""
    say("full", S, length, Tq, keep)
    g = gen(dev, S + Tq)
    cache = filled(dev, 1, S, 2, 64, 64, [length], S, 32)
    apart = copy_of(cache)
    x = step_inputs(g, 1, Tq, 4, 32, 4, 2, 64, 64, BF16)
    k = min(8, S - 1)
    out = D.dsa_decode(cache, *x, top_k=k, keep=keep, recent=recent)
    D.kv4_evict(apart, S - Tq, recent)
    D.kv4_append(apart, x[4], x[5], x[1])
    assert int(apart.length) == S and not int(apart.lost)
    _, slots = topk_indices(D.kv4_indexer_scores(apart, x[0], x[2]), k)
    want = D.kv4_attention(apart, x[3], slots=slots, accumulate=True)
    D.kv4_evict(apart, keep, recent)
    assert same(out, want)
    for n in NAMES:
        assert same(getattr(cache, n), getattr(apart, n)), n
    cache.check()


@pytest.mark.parametrize("S, Tq", [(40, 3), (40, 40), (500, 100), (17000, 2)])
def test_room_is_made_by_sequence(dev, S, Tq):
    """Each sequence down to S - its own tokens; those with room stay as they are, and so
    does what no kept slot moves into."""
    lengths = [S, S - 1, S - Tq, S - Tq + 1 if Tq > 1 else S, S, 0, S]
    counts = [Tq, 1, Tq, Tq, 0, Tq, Tq + 9]
    for count in (counts, None):
        cache = filled(dev, 7, S, 2, 32, 32, lengths, S + Tq, 32)
        moved = torch.empty(2, 7, Tq, device=dev, dtype=torch.int32)
        names = ("codes", "scales", "k_idx", "position", "weight")
        before = {n: getattr(cache, n).clone() for n in names}
        want = []
        for b in range(7):
            one = slice(b, b + 1)
            room = S - (Tq if count is None else min(count[b], Tq))
            want += C.evict(cache.length[one].cpu(), cache.seen[one].cpu(), cache.position[one].cpu(),
                            cache.weight[one].cpu(), room, 2)
        n = ints(dev, count) if count else None
        L.check(L.lib().dsa_kv4_make_room(cache._ref, n.data_ptr() if count else None, Tq, 2, moved[0].data_ptr(),
                                          moved[1].data_ptr(), L.stream_ptr(dev)), "room")
        for b, (src, dst, length) in enumerate(want):
            assert moved[0, b].tolist() == src + [-1] * (Tq - len(src)), b
            assert moved[1, b].tolist() == dst + [-1] * (Tq - len(dst)), b
            assert int(cache.length[b]) == length
            for x in before.values():
                if src:
                    x[b, torch.tensor(dst, device=dev)] = x[b, torch.tensor(src, device=dev)].clone()
        for name, x in before.items():
            assert same(getattr(cache, name), x), name


def test_steps_of_a_padded_full_batch(dev):
    """Room is made for a sequence's own tokens alone, and a captured step makes it too."""
    g, S, lengths = gen(dev, 90), 60, [60, 59, 60, 20]
    args = (3, 4, 32, 4, 2, 64, 64, BF16)
    caches = [filled(dev, 4, S, 2, 64, 64, lengths, 91, 32) for _ in range(2)]
    x, count = step_inputs(g, 4, *args), ints(dev, [3, 1, 0, 2])
    kw = dict(top_k=9, count=count, keep=57, recent=3)
    warm = filled(dev, 4, S, 2, 64, 64, lengths, 91, 32)
    D.dsa_decode(warm, *x, **kw)
    assert not warm.lost.any() and warm.seen.tolist() == [63, 60, 60, 22] and warm.length.tolist() == [57, 57, 57, 22]
    for b, n in enumerate([3, 1, 0, 2]):  # the newest tokens are there
        assert set(range(lengths[b], lengths[b] + n)) <= set(warm.position[b, :int(warm.length[b])].tolist())
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        out = D.dsa_decode(caches[0], *x, **kw)
    for i in range(6):
        for t, new in zip(x, step_inputs(g, 4, *args)):
            t.copy_(new)
        if i == 3:  # full again
            for c in caches:
                c.length.fill_(S)
        gr.replay()
        got = out.clone()
        torch.randn(500, 500, device=dev).sum()
        want = D.dsa_decode(caches[1], *x, **kw)
        torch.cuda.synchronize()
        assert same(torch.nan_to_num(got), torch.nan_to_num(want)), i
        for n in NAMES:
            assert same(getattr(caches[0], n), getattr(caches[1], n)), (i, n)
    caches[1].check()


def test_refused_steps_of_a_full_cache_make_no_room(dev):
    """What the append refuses is refused before room is made for it."""
    g = gen(dev, 95)
    cache = filled(dev, 2, 40, 2, 64, 64, [40, 39], 96, 32)
    before = [getattr(cache, n).clone() for n in NAMES]
    q, ki, w, Q, K, V = step_inputs(g, 2, 2, 4, 32, 4, 2, 64, 64, BF16)
    for args, kw in [((q, None, w, Q, K, V, 8), {}), ((q, ki[..., :16], w, Q, K, V, 8), {}),
                     ((q, ki, w, Q, K, V[:, :1], 8), {}), ((q, ki, w, Q, K[..., :32], V, 8), {}),
                     ((q, ki, w, Q, K, V, 8), dict(count=torch.ones(2, device=dev)))]:
        with pytest.raises(AssertionError):
            D.dsa_decode(cache, *args, keep=30, **kw)
    assert all(same(getattr(cache, n), old) for n, old in zip(NAMES, before))


def test_steps_refused_for_a_device_or_for_room_change_nothing(dev):
    g = gen(dev, 92)
    cache = filled(dev, 2, 40, 2, 64, 64, [20, 4], 93, 32)
    before = [getattr(cache, n).clone() for n in NAMES]
    x = step_inputs(g, 2, 1, 4, 32, 4, 2, 64, 64, BF16)
    for i in range(6):
        bad = [t.cpu() if j == i else t for j, t in enumerate(x)]
        with pytest.raises(AssertionError, match="cache's GPU"):
            D.dsa_decode(cache, *bad, 8)
    with pytest.raises(AssertionError, match="cache's GPU"):
        D.kv4_attention(cache, x[3].cpu())
    with pytest.raises(AssertionError, match="cache's GPU"):
        D.kv4_indexer_scores(cache, x[0], x[2].cpu())
    with pytest.raises(AssertionError, match="count"):
        D.dsa_decode(cache, *x, 8, count=torch.ones(2, dtype=torch.int32))
    with pytest.raises(AssertionError, match="do not fit"):
        D.dsa_decode(cache, *x, 8, keep=40)
    assert all(same(getattr(cache, n), old) for n, old in zip(NAMES, before))
    D.dsa_decode(cache, *x, 8, keep=39)
    assert cache.length.tolist() == [21, 5]


@pytest.mark.parametrize("keep", [40, 390])  # moves by a launch of their own, and by the selecting block
def test_scales_at_any_multiple_of_four_bytes(dev, keep):
    """The C entries take scales that are 4-byte aligned, also where a slot's are 16 bytes."""
    S = 400
    cache = filled(dev, 2, S, 4, 64, 64, [S, S - 7], 94, 32)
    room = torch.zeros(cache.scales.numel() + 16, device=dev, dtype=torch.uint8)
    for shift in (4, 8, 12):
        apart = copy_of(cache)
        moved = room[shift:shift + cache.scales.numel()]
        moved.copy_(cache.scales.flatten())
        c = copy_of(cache)
        D.kv4_evict(apart, keep, 5)
        out = torch.empty(2, 2, min(keep, S - keep), device=dev, dtype=torch.int32)
        c._c.scales = moved.data_ptr()
        L.check(L.lib().dsa_kv4_evict(c._ref, keep, 5, out[0].data_ptr(), out[1].data_ptr(), L.stream_ptr(dev)), "evict")
        assert same(moved, apart.scales.flatten()) and same(c.codes, apart.codes), shift


# --- sizes -------------------------------------------------------------------------------------------
@pytest.mark.parametrize("HQ, HKV, D_, Tq, listed", [(1024, 1024, 32, 1, 0), (1024, 1, 64, 1, 0), (1024, 4, 32, 3, 0),
                                                     (1024, 2, 32, 1, 90), (1023, 341, 64, 2, 50)])
def test_attention_of_the_most_heads(dev, HQ, HKV, D_, Tq, listed):
    say("most heads", HQ, HKV, D_, Tq, listed)
    g = gen(dev, HQ + HKV)
    cache = filled(dev, 2, 70, HKV, D_, D_, [70, 33], 97)
    slots = torch.randint(-2, 72, (2, Tq, listed), generator=g, device=dev, dtype=torch.int32) if listed else None
    attend(cache, randn(g, 2, Tq, HQ, D_, dtype=BF16), "out", slots=slots)


def test_steps_of_nothing_and_of_one_slot(dev):
    """No sequences, no tokens, and a cache whose one slot each step takes over."""
    g = gen(dev, 98)
    none = D.KV4Cache.empty(0, 8, 2, 64, 64, 32, device=dev)
    assert D.dsa_decode(none, *step_inputs(g, 0, 1, 4, 32, 4, 2, 64, 64, BF16), 4, keep=7).shape == (0, 1, 4, 64)
    cache = filled(dev, 2, 20, 2, 64, 64, [20, 4], 99, 32)
    assert D.dsa_decode(cache, *step_inputs(g, 2, 0, 4, 32, 4, 2, 64, 64, BF16), 4, keep=20).shape == (2, 0, 4, 64)
    assert cache.length.tolist() == [20, 4] and not cache.lost.any()
    one = D.KV4Cache.empty(2, 1, 2, 64, 64, 32, device=dev)
    x = step_inputs(g, 2, 1, 4, 32, 4, 2, 64, 64, BF16)
    D.kv4_append(one, x[4], x[5], x[1])
    for i in range(3):
        x = step_inputs(g, 2, 1, 4, 32, 4, 2, 64, 64, BF16)
        out = D.dsa_decode(one, *x, 1, keep=0)
        V = C.decode(*C.quantise(x[5])).repeat_interleave(2, 2)
        assert torch.equal(out.double(), V)  # p = 1
        assert one.length.tolist() == [0, 0] and one.seen.tolist() == [i + 2] * 2 and not one.lost.any()


@pytest.mark.parametrize("S, T", [(300, 200)])
def test_rows_of_the_widest_heads(dev, S, T):
    """DK and DV up to 1024, which append, rows and eviction take."""
    g = gen(dev, 100)
    cache = D.KV4Cache.empty(2, S, 3, 1024, 32, device=dev)
    K, V = randn(g, 2, T, 3, 1024, dtype=BF16), randn(g, 2, T, 3, 32, dtype=BF16)
    D.kv4_append(cache, K, V, weight=torch.rand(2, T, generator=g, device=dev))
    k, v = D.kv4_rows(cache, span=T)
    assert torch.equal(k.double(), C.decode(*C.quantise(K))) and torch.equal(v.double(), C.decode(*C.quantise(V)))
    check_evict(cache, 90, 7, "wide")
