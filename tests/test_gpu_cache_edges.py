"""GPU: calls of the 4-bit decode cache at the edges of what they allow."""
from __future__ import annotations

import math

import pytest
import torch

import cache_oracle as C
import dsa_cache as D
from helpers import say
from test_gpu_cache import BF16, F16, F32, filled, gen, ints, randn, within

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
