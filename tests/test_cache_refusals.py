"""CPU: what else the 4-bit cache's C entries refuse before any HIP call."""
from __future__ import annotations

import pytest

import _dsa_lib as L
from test_cache_host import CALLS, FAKE, cache, call, put


@pytest.mark.parametrize("changes, needle", [
    (dict(_0=None), "null"), (dict(_0=FAKE + 8), "aligned"), (dict(_1=None), "null"), (dict(_3=-1), "Tq"),
    (dict(_4=0), "HI"), (dict(_4=257), "HI"), (dict(_5=65), "span"), (dict(_6=None), "null"),
])
def test_fp32_indexer_refusals(changes, needle):
    name, args = "dsa_kv4_indexer_scores_f32", CALLS["dsa_kv4_indexer_scores"]
    rc, msg = call(name, cache(), *put(args, **changes))
    assert rc == L.DSA_EINVAL and needle in msg, (rc, msg)
    assert call(name, None, *args)[0] == L.DSA_EINVAL
    assert call(name, cache(DI=16), *args)[0] == L.DSA_EUNSUPPORTED  # 16 bits have no kernel of 16
    assert call(name, cache(k_idx=None), *args)[0] == L.DSA_EINVAL
    assert call(name, cache(), *put(args, _3=0))[0] == L.DSA_OK


ROOM = (None, 4, 2, FAKE, FAKE, None)


@pytest.mark.parametrize("changes", [dict(_1=-1), dict(_1=65), dict(_2=-1), dict(_3=None), dict(_4=None),
                                     dict(_3=FAKE + 2), dict(_4=FAKE + 1), dict(_0=FAKE + 2)])
def test_make_room_refusals(changes):
    name = "dsa_kv4_make_room"
    rc, msg = call(name, cache(), *put(ROOM, **changes))
    assert rc == L.DSA_EINVAL and msg, (rc, msg)
    assert call(name, None, *ROOM)[0] == L.DSA_EINVAL
    assert call(name, cache(codes=None), *ROOM)[0] == L.DSA_EINVAL
    assert call(name, cache(), *put(ROOM, _1=0))[0] == L.DSA_OK
    assert call(name, cache(B=0), *ROOM)[0] == L.DSA_OK


@pytest.mark.parametrize("name", ["dsa_kv4_indexer_scores", "dsa_kv4_indexer_scores_f32"])
@pytest.mark.parametrize("B, Tq, span", [(16, 1 << 30, 1 << 30), (1 << 15, 1 << 30, 1 << 19), (1, 1 << 23, 64)])
def test_sizes_of_the_indexer_whose_product_overflows(name, B, Tq, span):
    """B * Tq * span is 2^64 in the first two."""
    c = cache(B=B, S=1 << 30, codes=None)
    rc, msg = call(name, c, *put(CALLS["dsa_kv4_indexer_scores"], _3=Tq, _5=span))
    assert rc == L.DSA_EINVAL and "2^23" in msg, (rc, msg)
    assert call(name, c, *put(CALLS["dsa_kv4_indexer_scores"], _3=Tq, _5=0))[0] == L.DSA_OK


def test_append_of_more_blocks_than_a_launch_holds():
    """Two tokens a block of 256 threads: 2^25 - 1 of them are 2^32 threads."""
    rc, msg = call("dsa_kv4_append", cache(), *put(CALLS["dsa_kv4_append"], _6=(1 << 25) - 1))
    assert rc == L.DSA_EINVAL and "T=" in msg, (rc, msg)
