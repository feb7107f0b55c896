"""CPU: the paged 8-bit cache's and windowed attention's C entries refuse what they cannot
take before any HIP call, and the Python layer raises the framework's error classes; the
oracle's format against torch's own.  No kernel is launched here."""
from __future__ import annotations

import ctypes

import pytest
import torch

import _dsa_lib as L
import dsa_paged as P
import paged_oracle as O

FAKE = 0x1000  # never dereferenced: validation fails first


def cache(**kw):
    c = dict(codes=FAKE, scales=FAKE, pages=FAKE, length=FAKE, lost=FAKE, B=2, NP=8, max_pages=4, HKV=4,
             DK=64, DV=64, page=64)
    c.update(kw)
    return L.Kv8Cache(**c)


def call(name, c, args):
    rc = getattr(L.lib(), name)(ctypes.addressof(c) if c is not None else None, *args)
    return rc, L.lib().dsa_last_error().decode()


def put(args, **at):
    args = list(args)
    for k, v in at.items():
        args[int(k[1:])] = v
    return tuple(args)


#         K     V     Q     dtype       T  HQ ldk  ldv  ldq  cos   sin   rows R   pairs start count K_out Q_out stream
APPEND = (FAKE, FAKE, FAKE, L.DSA_BF16, 4, 8, 256, 256, 512, FAKE, FAKE, 256, 64, 0, None, None, FAKE, FAKE, None)
ROWS = (None, 8, L.DSA_F32, FAKE, FAKE, None)
#       Q     dtype       count Tq HQ n    window sinks scale  out   ws    bytes    stream
ATTN = (FAKE, L.DSA_BF16, None, 1, 8, 256, 100, 4, 0.125, FAKE, FAKE, 1 << 40, None)
CALLS = {"dsa_kv8_append": APPEND, "dsa_kv8_rows": ROWS, "dsa_kv8_attention": ATTN}


@pytest.mark.parametrize("name", CALLS)
def test_every_entry_checks_the_cache(name):
    def refused(code, needle, **kw):
        rc, msg = call(name, cache(**kw), CALLS[name])
        assert rc == code and needle in msg, (name, kw, rc, msg)

    assert call(name, None, CALLS[name])[0] == L.DSA_EINVAL
    refused(L.DSA_EINVAL, "B=", B=-1)
    refused(L.DSA_EINVAL, "65535", B=65536)
    refused(L.DSA_EINVAL, "NP=", NP=0)
    refused(L.DSA_EINVAL, "max_pages=", max_pages=0)
    for page in (0, 32, 96, 192, 1 << 17):
        refused(L.DSA_EINVAL, "page=", page=page)
    refused(L.DSA_EINVAL, "2^31", max_pages=1 << 25)
    refused(L.DSA_EINVAL, "2^31", max_pages=(1 << 31) - 1, page=65536)
    refused(L.DSA_EINVAL, "HKV", HKV=0)
    refused(L.DSA_EINVAL, "HKV", HKV=1025)
    for d in (dict(DK=48), dict(DV=0), dict(DK=128), dict(DK=160, DV=160), dict(DK=128, DV=192)):
        refused(L.DSA_EUNSUPPORTED, "DK=", **d)
    for part in ("codes", "scales", "pages", "length", "lost"):
        refused(L.DSA_EINVAL, "null", **{part: None})
    refused(L.DSA_EINVAL, "aligned", codes=FAKE + 8)
    refused(L.DSA_EINVAL, "aligned", scales=FAKE + 1)
    for part in ("pages", "length", "lost"):
        refused(L.DSA_EINVAL, "aligned", **{part: FAKE + 2})


@pytest.mark.parametrize("changes, needle", [
    (dict(_0=None), "null"), (dict(_1=None), "null"), (dict(_2=None), "Q goes"), (dict(_17=None), "Q goes"),
    (dict(_3=L.DSA_FP8), "dtype"), (dict(_3=9), "dtype"), (dict(_4=-1), "T="), (dict(_4=1 << 29), "2^23"),
    (dict(_4=(1 << 62)), "T="), (dict(_5=0), "HQ"), (dict(_5=1025, _8=65600), "HQ"), (dict(_6=255), "strides"),
    (dict(_6=260), "strides"), (dict(_7=248), "strides"), (dict(_7=(1 << 24) + 8), "strides"),
    (dict(_8=511), "stride"), (dict(_8=516), "stride"), (dict(_9=None), "null"), (dict(_10=None), "null"),
    (dict(_11=255), "rows"), (dict(_12=-16), "R="), (dict(_12=8), "R="), (dict(_12=80), "R="),
    (dict(_0=FAKE + 8), "aligned"), (dict(_1=FAKE + 2), "aligned"), (dict(_2=FAKE + 4), "aligned"),
    (dict(_9=FAKE + 4), "aligned"), (dict(_10=FAKE + 8), "aligned"), (dict(_16=FAKE + 8), "aligned"),
    (dict(_17=FAKE + 8), "aligned"), (dict(_14=FAKE + 2), "aligned"), (dict(_15=FAKE + 1), "aligned"),
    (dict(_4=1 << 21, _5=1024, _8=65536), "2^31"),
])
def test_append_refusals(changes, needle):
    rc, msg = call("dsa_kv8_append", cache(), put(APPEND, **changes))
    assert rc == L.DSA_EINVAL and needle in msg, (rc, msg)
    assert call("dsa_kv8_append", cache(B=0), APPEND)[0] == L.DSA_OK


@pytest.mark.parametrize("changes, needle", [
    (dict(_1=-1), "N="), (dict(_1=1 << 40), "N="), (dict(_1=1 << 28), "2^24"), (dict(_2=L.DSA_FP8), "dtype"),
    (dict(_3=None), "null"), (dict(_4=None), "null"), (dict(_3=FAKE + 8), "aligned"), (dict(_0=FAKE + 2), "aligned"),
])
def test_rows_refusals(changes, needle):
    rc, msg = call("dsa_kv8_rows", cache(), put(ROWS, **changes))
    assert rc == L.DSA_EINVAL and needle in msg, (rc, msg)
    assert call("dsa_kv8_rows", cache(), put(ROWS, _1=0))[0] == L.DSA_OK


@pytest.mark.parametrize("changes, needle", [
    (dict(_0=None), "null"), (dict(_1=L.DSA_FP8), "dtype"), (dict(_2=FAKE + 2), "aligned"), (dict(_3=-1), "Tq"),
    (dict(_3=1 << 40), "Tq"), (dict(_3=1 << 19), "2^23"), (dict(_4=0), "HQ"), (dict(_4=6), "HQ"), (dict(_4=2048), "HQ"),
    (dict(_5=-1), "n="), (dict(_5=257), "n="), (dict(_6=-1), "window"), (dict(_7=-1), "sinks"),
    (dict(_8=float("inf")), "scale"), (dict(_8=float("nan")), "scale"), (dict(_9=None), "null"),
    (dict(_9=FAKE + 4), "aligned"), (dict(_0=FAKE + 2), "aligned"),
])
def test_attention_refusals(changes, needle):
    rc, msg = call("dsa_kv8_attention", cache(), put(ATTN, **changes))
    assert rc == L.DSA_EINVAL and needle in msg, (rc, msg)
    assert call("dsa_kv8_attention", cache(), put(ATTN, _3=0))[0] == L.DSA_OK
    assert call("dsa_kv8_attention", cache(B=0), ATTN)[0] == L.DSA_OK


def test_attention_workspace():
    def need(c, *args):
        return L.lib().dsa_kv8_attention_workspace_bytes(ctypes.addressof(c), *args)

    long = cache(max_pages=1024)
    nws = need(long, 1, 8, 65536, 0, 0)
    assert nws > 0
    assert need(long, 1, 8, 64, 0, 0) == 0 and need(long, 1, 8, 65536, 1, 0) == 0  # a wave each at most
    assert need(long, 1, 8, 65536, 1 << 62, 1 << 62) == nws  # a window past the slots is none
    for changes in (dict(_10=None), dict(_11=nws - 1), dict(_10=FAKE + 8), dict(_11=-1)):
        rc, msg = call("dsa_kv8_attention", long, put(ATTN, _5=65536, _6=0, _11=nws, **{k: v for k, v in changes.items() if k != "_11"})
                       if "_11" not in changes else put(ATTN, _5=65536, _6=0, **changes))
        assert rc == L.DSA_EINVAL and "workspace" in msg, (changes, rc, msg)
    assert need(cache(HKV=0), 1, 8, 64, 0, 0) == L.DSA_EINVAL


#         Q     K     V     dtype       count B  T   HQ HKV D  ldq  ldk  ldv  window sinks scale out stream
WINDOW = (FAKE, FAKE, FAKE, L.DSA_BF16, None, 2, 64, 8, 4, 64, 512, 256, 256, 16, 4, 0.125, FAKE, None)


@pytest.mark.parametrize("changes, needle", [
    (dict(_0=None), "null"), (dict(_1=None), "null"), (dict(_2=None), "null"), (dict(_16=None), "null"),
    (dict(_3=L.DSA_FP8), "dtype"), (dict(_4=FAKE + 2), "aligned"), (dict(_5=-1), "B="), (dict(_6=-1), "T="),
    (dict(_6=1 << 31), "T="), (dict(_7=6), "HQ"), (dict(_7=0), "HQ"), (dict(_8=0), "HKV"), (dict(_7=2048), "HQ"),
    (dict(_10=504), "strides"), (dict(_11=255), "strides"), (dict(_12=260), "strides"), (dict(_10=(1 << 24) + 8), "strides"),
    (dict(_13=0), "window"), (dict(_13=-5), "window"), (dict(_14=-1), "sinks"), (dict(_15=float("inf")), "scale"),
    (dict(_0=FAKE + 8), "aligned"), (dict(_1=FAKE + 2), "aligned"), (dict(_2=FAKE + 8), "aligned"), (dict(_16=FAKE + 4), "aligned"),
    (dict(_5=1 << 30), "2^24"), (dict(_6=1 << 30), "2^24"),
    (dict(_5=1 << 21), "2^24"), (dict(_5=1 << 30, _6=1 << 30, _7=1024, _8=1024, _10=1 << 17, _11=1 << 17, _12=1 << 17), "2^24"),  # 2^21 * 8; 2^64
])
def test_window_refusals(changes, needle):
    rc = L.lib().dsa_window_attention(*put(WINDOW, **changes))
    msg = L.lib().dsa_last_error().decode()
    assert rc == L.DSA_EINVAL and needle in msg, (rc, msg)
    assert L.lib().dsa_window_attention(*put(WINDOW, _9=96)) == L.DSA_EUNSUPPORTED
    assert L.lib().dsa_window_attention(*put(WINDOW, _6=0)) == L.DSA_OK
    assert L.lib().dsa_window_attention(*put(WINDOW, _5=0)) == L.DSA_OK


def test_python_refuses_cpu_tensors():
    x = torch.zeros(1, 4, 2, 64)
    with pytest.raises(AssertionError, match="GPU"):
        P.window_attention(x, x, x)
    with pytest.raises(AssertionError, match="GPU"):
        P.KV8Cache(torch.zeros(4, 2, 1, 8192, dtype=torch.uint8), torch.zeros(4, 2, 1, 2, dtype=torch.uint8),
                   torch.zeros(1, 4, dtype=torch.int32), torch.zeros(1, dtype=torch.int32))


def test_rope_tables_of_far_positions():
    cos, sin = P.rope_tables(1 << 17, 64, 500.0, device="cpu")
    p, j = (1 << 17) - 1, 3
    angle = p * 500.0 ** (-2 * j / 64)
    import math
    assert abs(float(cos[p, j]) - math.cos(angle)) < 2.0 ** -24 + 1e-10 and abs(float(sin[p, j]) - math.sin(angle)) < 2.0 ** -24 + 1e-10
    for bad in ((0, 64), (4, 0), (4, 3)):
        with pytest.raises(AssertionError):
            P.rope_tables(*bad, device="cpu")


def test_oracle_format():
    """The oracle's codes against torch's own e4m3 and its scales against their definition."""
    codes = torch.arange(256, dtype=torch.uint8)
    ours, theirs = O.value(codes), codes.view(torch.float8_e4m3fn).double()
    assert torch.equal(ours.isnan(), theirs.isnan()) and torch.equal(ours[~ours.isnan()], theirs[~theirs.isnan()])
    x = torch.cat([torch.linspace(-448, 448, 9001), torch.randn(4000) * 2.0 ** torch.randint(-14, 7, (4000,))]).double().clamp(-448, 448)
    mid = (O.GRID[1:] + O.GRID[:-1]) / 2
    x = torch.cat([x, mid, -mid, O.GRID, -O.GRID])
    assert torch.equal(O.encode(x, 127), x.float().to(torch.float8_e4m3fn).view(torch.uint8))
    for top, e in ((448.0, 0), (448.1, 1), (1.0, -8), (0.0, -117), (2.0 ** -130, -117), (3.0e38, 120)):
        assert O.need(torch.tensor([top, -top / 2, float("nan"), float("inf")])) == e + 127, top
    assert sorted(O.PLACE.tolist()) == list(range(64))
