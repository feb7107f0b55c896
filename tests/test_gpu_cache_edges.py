"""GPU: calls of the 4-bit decode cache at the edges of what they allow."""
from __future__ import annotations

import math

import pytest
import torch

import dsa_cache as D
from helpers import say
from test_gpu_cache import BF16, F16, F32, gen, ints, randn

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
