"""GPU: the paged 8-bit cache and windowed attention (dsa_paged) at the limits of their number
formats: scales far apart or of pages of nobody, values near the largest, shares near the least, and
prompts that fill the card.  Against 64 bits, under paged_oracle's bounds."""
from __future__ import annotations

import pytest
import torch

import dsa_paged as P
from test_gpu_paged import BF16, F32, check_attention, filled, gen, randn

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
