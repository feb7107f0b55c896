"""CPU: the 4-bit cache's C entries refuse what they cannot take before any HIP
call, and the Python layer raises the framework's error classes.  No kernel is
launched here."""
from __future__ import annotations

import ctypes

import pytest
import torch

import _dsa_lib as L
import cache_oracle as C
import dsa_cache as D

FAKE = 0x1000  # never dereferenced: validation fails first


def cache(**kw):
    c = dict(codes=FAKE, scales=FAKE, k_idx=FAKE, length=FAKE, seen=FAKE, lost=FAKE, position=FAKE,
             weight=FAKE, B=2, S=64, HKV=4, DK=64, DV=64, DI=64, idx_dtype=L.DSA_BF16)
    c.update(kw)
    return L.Kv4Cache(**c)


def call(name, c, *args):
    rc = getattr(L.lib(), name)(ctypes.addressof(c) if c is not None else None, *args)
    return rc, L.lib().dsa_last_error().decode()


APPEND = (FAKE, FAKE, L.DSA_BF16, FAKE, None, None, 4, 0, None)
ROWS = (None, 8, L.DSA_F32, FAKE, FAKE, None)
INDEX = (FAKE, FAKE, None, 1, 8, 64, FAKE, None)
ATTN = (FAKE, L.DSA_BF16, None, None, 1, 8, 64, 0, 0.125, FAKE, FAKE, 1 << 40, None)
EVICT = (16, 4, FAKE, FAKE, None)
CALLS = {"dsa_kv4_append": APPEND, "dsa_kv4_rows": ROWS, "dsa_kv4_indexer_scores": INDEX,
         "dsa_kv4_attention": ATTN, "dsa_kv4_evict": EVICT}


@pytest.mark.parametrize("name", CALLS)
def test_every_entry_checks_the_cache(name):
    def refused(code, needle, **kw):
        rc, msg = call(name, cache(**kw), *CALLS[name])
        assert rc == code and needle in msg, (name, kw, rc, msg)

    assert call(name, None, *CALLS[name])[0] == L.DSA_EINVAL
    refused(L.DSA_EINVAL, "B=", B=-1)
    refused(L.DSA_EINVAL, "S=", S=0)
    refused(L.DSA_EINVAL, "65535", B=65536)
    refused(L.DSA_EINVAL, "2^31", S=1 << 31)
    refused(L.DSA_EINVAL, "null length", length=None)
    refused(L.DSA_EINVAL, "aligned", length=FAKE + 2)
    refused(L.DSA_EINVAL, "aligned", k_idx=FAKE + 8)
    refused(L.DSA_EINVAL, "dtype", idx_dtype=L.DSA_FP8)
    refused(L.DSA_EUNSUPPORTED, "DI=", DI=16)
    if name != "dsa_kv4_indexer_scores":
        refused(L.DSA_EINVAL, "HKV", HKV=0)
        refused(L.DSA_EUNSUPPORTED, "DK=", DK=48)
        refused(L.DSA_EUNSUPPORTED, "DV=", DV=0)
        refused(L.DSA_EINVAL, "2^31", S=1 << 24, HKV=2)
        for part in ("codes", "scales", "seen", "lost", "position", "weight"):
            refused(L.DSA_EINVAL, "null", **{part: None})
        refused(L.DSA_EINVAL, "aligned", codes=FAKE + 8)
        refused(L.DSA_EINVAL, "aligned", scales=FAKE + 2)
    else:
        refused(L.DSA_EINVAL, "no index keys", k_idx=None)


def put(args, **at):
    args = list(args)
    for i, v in at.items():
        args[int(i[1:])] = v
    return args


@pytest.mark.parametrize("name, changes, code", [
    ("dsa_kv4_append", dict(_2=7), L.DSA_EINVAL),
    ("dsa_kv4_append", dict(_2=L.DSA_FP8), L.DSA_EINVAL),
    ("dsa_kv4_append", dict(_6=-1), L.DSA_EINVAL),
    ("dsa_kv4_append", dict(_0=None), L.DSA_EINVAL),
    ("dsa_kv4_append", dict(_1=FAKE + 8), L.DSA_EINVAL),
    ("dsa_kv4_append", dict(_3=None), L.DSA_EINVAL),      # the cache holds index keys
    ("dsa_kv4_append", dict(_5=FAKE + 1), L.DSA_EINVAL),
    ("dsa_kv4_rows", dict(_1=-1), L.DSA_EINVAL),
    ("dsa_kv4_rows", dict(_2=9), L.DSA_EINVAL),
    ("dsa_kv4_rows", dict(_3=None), L.DSA_EINVAL),
    ("dsa_kv4_rows", dict(_4=FAKE + 4), L.DSA_EINVAL),
    ("dsa_kv4_rows", dict(_0=FAKE + 1), L.DSA_EINVAL),
    ("dsa_kv4_indexer_scores", dict(_0=None), L.DSA_EINVAL),
    ("dsa_kv4_indexer_scores", dict(_0=FAKE + 8), L.DSA_EINVAL),
    ("dsa_kv4_indexer_scores", dict(_3=-1), L.DSA_EINVAL),
    ("dsa_kv4_indexer_scores", dict(_4=0), L.DSA_EINVAL),
    ("dsa_kv4_indexer_scores", dict(_4=257), L.DSA_EINVAL),
    ("dsa_kv4_indexer_scores", dict(_5=65), L.DSA_EINVAL),
    ("dsa_kv4_indexer_scores", dict(_6=None), L.DSA_EINVAL),
    ("dsa_kv4_attention", dict(_1=L.DSA_FP8), L.DSA_EINVAL),
    ("dsa_kv4_attention", dict(_4=-1), L.DSA_EINVAL),
    ("dsa_kv4_attention", dict(_5=6), L.DSA_EINVAL),      # HQ % HKV
    ("dsa_kv4_attention", dict(_5=2048), L.DSA_EINVAL),
    ("dsa_kv4_attention", dict(_6=65), L.DSA_EINVAL),     # n > S without slots
    ("dsa_kv4_attention", dict(_8=float("nan")), L.DSA_EINVAL),
    ("dsa_kv4_attention", dict(_9=None), L.DSA_EINVAL),
    ("dsa_kv4_attention", dict(_0=FAKE + 2), L.DSA_EINVAL),
    ("dsa_kv4_attention", dict(_11=-1), L.DSA_EINVAL),
    ("dsa_kv4_evict", dict(_0=-1, _1=0), L.DSA_EINVAL),
    ("dsa_kv4_evict", dict(_1=17), L.DSA_EINVAL),
    ("dsa_kv4_evict", dict(_1=-1), L.DSA_EINVAL),
    ("dsa_kv4_evict", dict(_2=None), L.DSA_EINVAL),
    ("dsa_kv4_evict", dict(_3=FAKE + 2), L.DSA_EINVAL),
])
def test_wrong_arguments(name, changes, code):
    rc, msg = call(name, cache(), *put(CALLS[name], **changes))
    assert rc == code and msg, (rc, msg)


def test_head_sizes_without_an_attention_kernel():
    for DK, DV in ((160, 160), (64, 128), (512, 512)):
        assert call("dsa_kv4_attention", cache(DK=DK, DV=DV), *ATTN)[0] == L.DSA_EUNSUPPORTED


def test_nothing_to_do_is_no_error():
    none = dict.fromkeys(("codes", "scales", "k_idx", "length", "seen", "lost", "position", "weight"))
    for name, args in CALLS.items():
        c = cache(B=0) if name == "dsa_kv4_indexer_scores" else cache(B=0, **none)
        assert call(name, c, *args)[0] == L.DSA_OK, (name, L.lib().dsa_last_error())
    assert call("dsa_kv4_append", cache(), *put(APPEND, _6=0))[0] == L.DSA_OK
    assert call("dsa_kv4_evict", cache(), *put(EVICT, _0=64))[0] == L.DSA_OK  # keep = S


def test_python_layer_raises_assertion_errors():
    with pytest.raises(AssertionError):  # no CPU path
        D.KV4Cache.empty(1, 8, 1, 32, 32, device="cpu")
    with pytest.raises(AssertionError):
        D.KV4Cache(None, None, torch.zeros(1, dtype=torch.int32))


def test_the_oracles_format():
    """The worked values of the format's rule, and codes against their values."""
    x = torch.zeros(9, 32)
    x[0, 0], x[1, 0], x[2, 0] = 6.0, 6.99, 7.0       # scales 1, 1, 2
    x[3, 0], x[4, 0] = float("nan"), float("inf")
    x[6, 0], x[7, 0] = 3.4e38, 1e-45
    x[8] = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -0.26] + [4.0] * 24)
    codes, scales = C.quantise(x)
    assert scales[:, 0].tolist() == [127, 127, 128, 255, 255, 2, 252, 2, 127]
    v = C.decode(codes, scales)
    assert v[0, 0] == 6 and v[1, 0] == 6 and v[2, 0] == 8 and torch.isnan(v[3:5]).all()
    assert v[6, 0] == 6 * 2.0 ** 125 and not v[7].any() and not v[5].any()
    assert v[8, :8].tolist() == [0, 1, 1, 2, 2, 4, 4, -0.5]
    y = torch.randn(1000, 32, generator=torch.Generator().manual_seed(1))
    c, s = C.quantise(y)
    step = torch.exp2(s.double() - 127)
    assert ((C.decode(c, s) - y).abs() <= step).all()  # half of the widest step
