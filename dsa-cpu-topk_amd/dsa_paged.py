"""Layers beside the sparse ones: attention over a sliding window (or all) of a prompt, and
of single tokens over a paged cache held in 8 bits.

    window_attention   a prompt's attention: a sliding window, and the first tokens
    kv8_append         tokens into the pages, keys (and queries) rotated by their position
    kv8_attention      attention of the newest tokens over the pages, windowed or not
    kv8_rows           slots back as values
    rope_tables        cosines and sines of the position rotation

A prompt's keys are rotated as they go into the cache (kv8_append gives the rotated
queries and keys back), its attention runs on those, and each step after it appends and
attends. The 4-bit cache of dsa_cache is one buffer a sequence, evicted by attention; here a
slot is a position, pages come from a pool that the caller deals out (and takes back,
behind a window), and 8 bits with a scale per 64 tokens and head hold four mantissa
bits of every value.

Every function enqueues gfx950 kernels of libdsa_amd.so on torch's current stream of its
tensors' device and returns without synchronising; none moves anything to the host.  All
can be captured into HIP graphs (replays advance the cache, whose counters live on the
GPU).  Like the forwards they have no backward.  The reference has no counterpart: its
attention sees what the indexer selects, and it has no cache.
"""
from __future__ import annotations

import ctypes
import math

import torch

import _dsa_lib as L


def rope_tables(positions: int, R: int, base: float = 10000.0, device="cuda"):
    """(cos, sin), fp32 [positions, R/2]: the angle of position p and pair j is
    p * base^(-2j/R), taken in 64 bits, which far positions need."""
    assert positions >= 1 and R >= 2 and R % 2 == 0, f"positions={positions} R={R}"
    j = torch.arange(R // 2, device=device, dtype=torch.float64)
    angle = torch.arange(positions, device=device, dtype=torch.float64).unsqueeze(1) * base ** (-2 * j / R)
    return angle.cos().float(), angle.sin().float()


_TYPES = {torch.float32: L.DSA_F32, torch.bfloat16: L.DSA_BF16, torch.float16: L.DSA_F16}


def _tokens(x: torch.Tensor, dtype: torch.dtype):
    """(x, its address, token stride): [B, T, H, D] in `dtype` as the kernels take it: a token's
    heads side by side, tokens a stride of 16 bytes' multiple apart (the columns of one
    projection's output), batch elements T of them; a contiguous copy of anything else."""
    at = x.data_ptr()
    if x.dtype is dtype and at & 15 == 0:
        B, T, H, D = x.shape
        if x.is_contiguous():
            return x, at, H * D
        sb, st, sh, sd = x.stride()
        if x.numel() and sd == 1 and (H == 1 or sh == D) and H * D <= st <= 1 << 24 and st * x.element_size() % 16 == 0 \
                and (B == 1 or sb == T * st):
            return x, at, st
    x = L.prep(x, dtype)
    return x, x.data_ptr(), x.shape[2] * x.shape[3]


def _span_args(window: int | None, sinks: int):
    W = 0 if window is None else int(window)
    n = int(sinks)
    assert window is None or W >= 1, f"window={window} must be >= 1 (None: all)"
    assert n >= 0, f"sinks={sinks} must be >= 0"
    return min(W, 1 << 62), min(n, 1 << 62)  # (ctypes keeps an integer's low 64 bits)


def _out(out, shape, dtype, like):
    """The caller's `out`, checked, or a new tensor of that shape (`like`: one on its GPU)."""
    if out is None:
        if like.dtype is dtype and like.shape == shape and like.is_contiguous():
            return torch.empty_like(like)
        return like.new_empty(shape, dtype=dtype)
    assert out.dtype is dtype and out.shape == shape and out.is_contiguous() and out.device == like.device \
        and out.data_ptr() % 16 == 0, \
        f"out: contiguous 16-byte aligned {dtype} {tuple(shape)} on {like.device} (got {out.dtype} {tuple(out.shape)} on {out.device})"
    return out


def window_attention(Q: torch.Tensor, K: torch.Tensor, V: torch.Tensor, *, window: int | None = None,
                     sinks: int = 0, count: torch.Tensor | None = None, scale: float | None = None,
                     out: torch.Tensor | None = None) -> torch.Tensor:
    """Causal attention of whole prompts over a sliding window: token t sees the positions
    s <= t with s > t - window, and of the others the first `sinks`.  O [B,T,HQ,D].

    Q [B,T,HQ,D], K, V [B,T,HKV,D], HQ a multiple of HKV (query head h reads K/V head
    h // (HQ/HKV)), D in {32, 64, 128, 256}.  One type for all (fp32, bf16 or fp16; mixed ones go
    as fp32), which is the output's.  Columns of one projection's output go in as they
    are.  window None: every earlier token.  count int32 [B]: how many of
    a sequence's T rows are tokens (a padded batch); the others get NaN.  scale: of the
    logits, default 1/sqrt(D).  What a token does not see does not reach its row, NaN
    and Inf included.  (Prompts of the cache's other head sizes, 96 and 192, go over the pages,
    by kv8_attention after their append.)"""
    if not (Q.is_cuda and K.is_cuda and V.is_cuda):
        L.require_gpu(Q, K, V)
    shape, kv = Q.shape, K.shape
    assert len(shape) == 4 and len(kv) == 4, "Q [B,T,HQ,D], K and V [B,T,HKV,D]"
    B, T, HQ, D = shape
    HKV = kv[2]
    assert kv[0] == B and kv[1] == T and kv[3] == D and V.shape == kv, \
        f"K {tuple(kv)} and V {tuple(V.shape)} must be {(B, T, HKV, D)}"
    index = Q.get_device()
    assert K.get_device() == index and V.get_device() == index, "Q, K and V must be on one GPU"
    W, sinks = _span_args(window, sinks)
    dt = L.common_dtype(Q, K, V)
    q, q_ptr, ldq = _tokens(Q, dt)
    k, k_ptr, ldk = _tokens(K, dt)
    v, v_ptr, ldv = _tokens(V, dt)
    count_ptr = None
    if count is not None:
        assert count.dtype is torch.int32 and count.shape == (B,) and count.get_device() == index, \
            f"count: int32 {(B,)} on {Q.device} (got {count.dtype} {tuple(count.shape)} on {count.device})"
        count = count.contiguous()
        count_ptr = count.data_ptr()
    out = _out(out, shape, dt, Q)
    with L.on_device(Q.device):
        rc = L.lib().dsa_window_attention(
            q_ptr, k_ptr, v_ptr, _TYPES[dt], count_ptr, B, T, HQ, HKV, D, ldq, ldk, ldv, W or max(T, 1), sinks,
            D ** -0.5 if scale is None else float(scale), out.data_ptr(), L.stream_ptr(Q.device))
    if rc != L.DSA_OK:
        L.check(rc, "window_attention")
    return out


class KV8Cache:
    """The pages of B sequences' caches (include/dsa_amd.h, dsa_kv8_cache), all contiguous on
    one GPU and written in place:

      codes uint8 [NP, HKV, page/64, 64*(DK+DV)]   scales uint8 [NP, HKV, page/64, 2]
      pages int32 [B, max_pages]   length, lost int32 [B]

    A pool of NP pages of `page` slots (64 times a power of two); pages[b, i] is the page of
    sequence b's slots i*page and on, any id outside [0, NP) none.  The caller deals pages
    out: pages.copy_(...) or pages[b, i] = id before the append that needs them, and an id of
    -1 where a window has left a page behind.  length: slots in use (a slot is a position);
    length.copy_(...) takes tokens back, and sets a sequence up anew.  lost: tokens that found
    no slot or no page (check() raises where there are any).  The calls go by the buffers'
    addresses: write into a buffer, it cannot be replaced."""

    _BUFFERS = ("codes", "scales", "pages", "length", "lost")

    def __setattr__(self, name, value):
        if name in self._BUFFERS and name in self.__dict__:
            raise AttributeError(f"KV8Cache.{name} is written in place, not replaced")
        super().__setattr__(name, value)

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, pages: torch.Tensor, length: torch.Tensor,
                 lost: torch.Tensor | None = None, DK: int | None = None):
        L.require_gpu(codes)
        assert codes.dim() == 4 and pages.dim() == 2, "codes [NP,HKV,page/64,64*(DK+DV)], pages [B,max_pages]"
        NP, HKV, per, row = codes.shape
        B, max_pages = pages.shape
        device = codes.device
        assert row % 64 == 0, f"codes' rows of {row} bytes must be 64*(DK+DV)"
        DK = row // 128 if DK is None else int(DK)
        DV = row // 64 - DK
        if lost is None:
            lost = torch.zeros(B, device=device, dtype=torch.int32)
        self._is("codes", codes, (NP, HKV, per, row), torch.uint8, device, 16)
        self._is("scales", scales, (NP, HKV, per, 2), torch.uint8, device, 2)
        self._is("pages", pages, (B, max_pages), torch.int32, device, 4)
        self._is("length", length, (B,), torch.int32, device, 4)
        self._is("lost", lost, (B,), torch.int32, device, 4)
        self.codes, self.scales, self.pages, self.length, self.lost = codes, scales, pages, length, lost
        self.B, self.NP, self.max_pages, self.page = B, NP, max_pages, 64 * per
        self.S, self.HKV, self.DK, self.DV = max_pages * 64 * per, HKV, DK, DV
        self.device, self.index = device, device.index
        self.scale = 1.0 / math.sqrt(DK) if DK > 0 else 0.0
        self._workspace = {}  # bytes of kv8_attention's, by its sizes
        self._c = L.Kv8Cache(codes.data_ptr(), scales.data_ptr(), pages.data_ptr(), length.data_ptr(),
                             lost.data_ptr(), B, NP, max_pages, HKV, DK, DV, 64 * per)
        self._ref = ctypes.addressof(self._c)
        self._lib = L.lib()
        # sizes that no call takes are refused here
        _workspace_bytes(self, 0, HKV, 0, 0, 0)

    @staticmethod
    def _is(name, x, shape, dtype, device, align):
        assert x.device == device and x.dtype == dtype and tuple(x.shape) == shape \
            and x.is_contiguous() and (x.data_ptr() % align == 0 or not x.numel()), \
            f"{name}: contiguous {align}-byte aligned {dtype} {shape} on {device} " \
            f"(got {x.dtype} {tuple(x.shape)} on {x.device})"

    @classmethod
    def empty(cls, B: int, S: int, HKV: int, DK: int, DV: int, page: int = 64, NP: int | None = None,
              device="cuda") -> "KV8Cache":
        """A cache with nothing in it for up to S slots a sequence.  NP None: a pool with pages
        for all of them, dealt out; else a pool of NP pages and none dealt out (ids of -1)."""
        assert page >= 64 and page % 64 == 0 and S >= 1, f"S={S} page={page}: whole pages of 64 * 2^j slots"
        dev = torch.device(device)
        if dev.type == "cuda" and dev.index is None:
            dev = torch.device("cuda", torch.cuda.current_device())
        n = -(-S // page)
        if NP is None:
            NP = max(1, B * n)
            pages = torch.arange(B * n, device=dev, dtype=torch.int32).view(B, n)
        else:
            pages = torch.full((B, n), -1, device=dev, dtype=torch.int32)
        return cls(torch.zeros(NP, HKV, page // 64, 64 * (DK + DV), device=dev, dtype=torch.uint8),
                   torch.zeros(NP, HKV, page // 64, 2, device=dev, dtype=torch.uint8), pages,
                   torch.zeros(B, device=dev, dtype=torch.int32), DK=DK)

    def check(self) -> None:
        """RuntimeError if a token found no slot or no page (waits for the GPU)."""
        if self.B and int(self.lost.max()) > 0:
            raise RuntimeError(f"KV8Cache: {int(self.lost.sum())} tokens found no slot (S={self.S}) or no page")


def _ints(x: torch.Tensor, shape, name: str, cache: KV8Cache) -> torch.Tensor:
    """An int32 tensor of the caller's; a contiguous copy where it is not."""
    assert x.dtype is torch.int32 and x.shape == shape and x.get_device() == cache.index, \
        f"{name}: int32 {shape} on {cache.device} (got {x.dtype} {tuple(x.shape)} on {x.device})"
    return x if x.is_contiguous() else x.contiguous()


def _here(cache: KV8Cache, *xs: torch.Tensor) -> None:
    for x in xs:
        assert x.get_device() == cache.index, f"inputs must be on the cache's GPU {cache.device} (got {x.device})"


def _workspace_bytes(cache: KV8Cache, Tq: int, HQ: int, n: int, window: int, sinks: int) -> int:
    """What dsa_kv8_attention needs of these sizes; raises where it would refuse them."""
    sizes = (Tq, HQ, n, window, sinks)
    nws = cache._workspace.get(sizes)
    if nws is None:
        if len(cache._workspace) >= 64:  # spans of a growing cache
            cache._workspace.clear()
        with L.on_device(cache.device):
            nws = L.lib().dsa_kv8_attention_workspace_bytes(cache._ref, Tq, HQ, n, window, sinks)
        if nws < 0:
            L.check(nws, "kv8_attention")
        cache._workspace[sizes] = nws
    return nws


def _call(cache: KV8Cache, what: str, fn, *args) -> None:
    """fn(cache, *args, stream) on the cache's GPU.  Single-token calls are bound by
    the host, so the usual case enters no context."""
    if torch.cuda.current_device() == cache.index:
        rc = fn(cache._ref, *args, L.stream_ptr(cache.device))
    else:
        with torch.cuda.device(cache.device):
            rc = fn(cache._ref, *args, L.stream_ptr(cache.device))
    if rc != L.DSA_OK:
        L.check(rc, what)


def kv8_append(cache: KV8Cache, K: torch.Tensor, V: torch.Tensor, *, rope=None, pairs: bool = False,
               Q: torch.Tensor | None = None, start: torch.Tensor | None = None,
               count: torch.Tensor | None = None, keys: bool = False):
    """T new tokens a sequence into the cache's pages, keys rotated by their position on the way.
    Returns (rotated Q or None, rotated K or None).

    K [B,T,HKV,DK], V [B,T,HKV,DV] (one type of fp32, bf16 or fp16; mixed ones go as fp32),
    the columns of one projection's output as they are.  The tokens' positions, and slots, are
    start[b] + i, start int32 [B] (default: the cache's length, which then grows; 0 for new
    prompts, less than the length to take drafted tokens back; outside [0, S] the nearer end).  count int32 [B]: how many of
    the T are tokens (a padded batch; default all).  Tokens past the last slot or on no page
    are not stored but counted in cache.lost.
    rope: (cos, sin) fp32 [>= S, R/2] (rope_tables), R a multiple of 16 up to DK: the first R
    dimensions turn, as two halves, or with pairs neighbour by neighbour; None: nothing turns.
    Q [B,T,HQ,DK]: rotated too; keys: K's rotated rows are returned as well.  Both are of all T
    rows, NaN at positions past the last slot, in the one type that K, V and Q have (fp32 where
    their types differ).  Without rope they come back as they are."""
    kv = K.shape
    assert len(kv) == 4, "K [B,T,HKV,DK], V [B,T,HKV,DV]"
    B, T = kv[0], kv[1]
    assert B == cache.B and kv[2] == cache.HKV and kv[3] == cache.DK, \
        f"K shape {tuple(kv)} != {(cache.B, T, cache.HKV, cache.DK)}"
    assert V.shape == (B, T, cache.HKV, cache.DV), \
        f"V shape {tuple(V.shape)} != {(cache.B, T, cache.HKV, cache.DV)}"
    _here(cache, K, V)
    HQ = 0
    if Q is not None:
        assert Q.dim() == 4 and (Q.shape[0], Q.shape[1], Q.shape[3]) == (B, T, cache.DK), \
            f"Q shape {tuple(Q.shape)}: B={B}, T={T}, DK={cache.DK}"
        _here(cache, Q)
        HQ = Q.shape[2]
    dt = L.common_dtype(K, V) if Q is None or rope is None else L.common_dtype(K, V, Q)
    k, k_ptr, ldk = _tokens(K, dt)
    v, v_ptr, ldv = _tokens(V, dt)
    R = rows = ldq = 0
    cos_ptr = sin_ptr = start_ptr = count_ptr = q_ptr = q_out = k_out = q_out_ptr = k_out_ptr = None
    if rope is not None:
        cos, sin = rope
        assert cos.dim() == 2 and cos.shape == sin.shape and cos.dtype is torch.float32 and sin.dtype is torch.float32, \
            "rope: (cos, sin), fp32 [positions, R/2] each"
        _here(cache, cos, sin)
        rows, R = cos.shape[0], 2 * cos.shape[1]
        cos, sin = L.prep(cos, torch.float32), L.prep(sin, torch.float32)
        cos_ptr, sin_ptr = cos.data_ptr(), sin.data_ptr()
        if Q is not None:
            q, q_ptr, ldq = _tokens(Q, dt)
            q_out = _out(None, Q.shape, dt, Q)
            q_out_ptr = q_out.data_ptr()
        if keys:
            k_out = _out(None, kv, dt, K)
            k_out_ptr = k_out.data_ptr()
    if start is not None:
        start = _ints(start, (B,), "start", cache)
        start_ptr = start.data_ptr()
    if count is not None:
        count = _ints(count, (B,), "count", cache)
        count_ptr = count.data_ptr()
    _call(cache, "kv8_append", cache._lib.dsa_kv8_append, k_ptr, v_ptr, q_ptr, _TYPES[dt], T, HQ, ldk, ldv, ldq,
          cos_ptr, sin_ptr, rows, R, 1 if pairs else 0, start_ptr, count_ptr, k_out_ptr, q_out_ptr)
    if rope is None:
        return Q, (K if keys else None)
    return q_out, k_out


def kv8_rows(cache: KV8Cache, slots: torch.Tensor | None = None, *, span: int | None = None,
             dtype: torch.dtype = torch.float32):
    """The values that slots stand for: (K [B,N,HKV,DK], V [B,N,HKV,DV]).

    slots int32 [B,N], or the first `span` slots (default all).  Slots that hold
    nothing give zeros.  Exact in fp32 and bf16."""
    slots_ptr = None
    if slots is not None:
        assert span is None, "slots or span, not both"
        assert slots.dim() == 2, "slots: int32 [B, N]"
        N = slots.shape[1]
        slots = _ints(slots, (cache.B, N), "slots", cache)
        slots_ptr = slots.data_ptr()
    else:
        N = _span(cache, span)
    code = _TYPES.get(dtype)
    assert code is not None, f"unsupported dtype {dtype}"
    K = cache.codes.new_empty((cache.B, N, cache.HKV, cache.DK), dtype=dtype)
    V = torch.empty_like(K) if cache.DV == cache.DK else cache.codes.new_empty((cache.B, N, cache.HKV, cache.DV), dtype=dtype)
    _call(cache, "kv8_rows", cache._lib.dsa_kv8_rows, slots_ptr, N, code, K.data_ptr(), V.data_ptr())
    return K, V


def _span(cache: KV8Cache, span: int | None) -> int:
    if span is None:
        return cache.S
    n = int(span)
    assert 0 <= n <= cache.S, f"span={n} outside [0, S={cache.S}]"
    return n


def kv8_attention(cache: KV8Cache, Q: torch.Tensor, *, window: int | None = None, sinks: int = 0,
                  span: int | None = None, count: torch.Tensor | None = None, scale: float | None = None,
                  out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of each sequence's last Tq appended tokens over its pages: O [B,Tq,HQ,DV] of
    Q's type.

    Q [B,Tq,HQ,DK] (fp32, bf16 or fp16), HQ a multiple of HKV.  A token sees its own and the
    earlier slots: with a window the last `window` of them, and of the others the first `sinks`.
    span: only the first span slots count (default S; where the caller knows that no sequence has
    more in use, fewer blocks join).  count int32 [B]: how many of the Tq are tokens, as
    kv8_append's; the others see nothing.  A token that sees nothing gets NaN; slots on no
    page count for nothing.  scale: of the logits, default 1/sqrt(DK)."""
    shape = Q.shape
    assert len(shape) == 4 and shape[0] == cache.B and shape[3] == cache.DK, \
        f"Q shape {tuple(shape)}: B={cache.B}, DK={cache.DK}"
    B, Tq, HQ, _ = shape
    _here(cache, Q)
    W, sinks = _span_args(window, sinks)
    n = _span(cache, span)
    dt, q = Q.dtype, Q
    if dt not in _TYPES:
        dt = torch.float32
    q_ptr = Q.data_ptr()
    if q_ptr & 15 or Q.dtype is not dt or not Q.is_contiguous():
        q = L.prep(Q, dt)
        q_ptr = q.data_ptr()
    count_ptr = None
    if count is not None:
        count = _ints(count, (B,), "count", cache)
        count_ptr = count.data_ptr()
    if cache.DV != cache.DK:
        shape = (B, Tq, HQ, cache.DV)
    out = _out(out, shape, dt, q)
    nws = _workspace_bytes(cache, Tq, HQ, n, W, sinks)
    ws_ptr = None
    if nws:
        ws = cache.codes.new_empty(nws)
        ws_ptr = ws.data_ptr()
    _call(cache, "kv8_attention", cache._lib.dsa_kv8_attention, q_ptr, _TYPES[dt], count_ptr, Tq, HQ, n, W, sinks,
          cache.scale if scale is None else float(scale), out.data_ptr(), ws_ptr, nws)
    return out
