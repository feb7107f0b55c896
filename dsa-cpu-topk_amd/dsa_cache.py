"""DSA decode over a cache held in 4 bits: what follows the prompt.

The forwards of dsa_attention take whole sequences.  Here a sequence's keys and
values stay on the GPU between calls, in OCP MXFP4 (e2m1 codes, one power-of-two
scale per 32 elements: 4.25 bits a value), and each new token is appended,
attends, and the slots that drew the least attention make room:

    kv4_append           tokens into the cache (and index keys beside them)
    kv4_indexer_scores   lightning indexer of the new tokens against the cached index keys
    kv4_attention        attention over the whole cache, or over the slots that the
                         select chose (topk_threshold.topk_indices of the scores);
                         accumulates each slot's attention weight
    kv4_evict            down to a budget, by that weight, the newest tokens kept
    kv4_rows             slots back as values
    dsa_decode           a DSA step of all of them

Every function enqueues gfx950 kernels of libdsa_amd.so on torch's current
stream of the cache's device and returns without synchronising; none moves
anything to the host.  All can be captured into HIP graphs (replays advance the
cache, whose counters live on the GPU).  Like the forwards they have no backward.
The reference has no counterpart: it has no cache and no single-token form.
"""
from __future__ import annotations

import ctypes
import math

import torch

import _dsa_lib as L
from topk_threshold import topk_indices


class KV4Cache:
    """The buffers of B sequences' caches of S slots (include/dsa_amd.h,
    dsa_kv4_cache), all contiguous on one GPU and written in place:

      codes uint8 [B, S, HKV, (DK+DV)/2]   scales uint8 [B, S, HKV, (DK+DV)/32]
      k_idx [B, S, DI] fp32, bf16 or fp16 (None: no index keys)
      length, seen, lost int32 [B]   position int32 [B, S]   weight fp32 [B, S]

    length: slots in use; seen: tokens appended so far; lost: tokens that found
    no free slot (check() raises where there are any); weight: attention weight
    accumulated by kv4_attention.  Made from buffers in use, what is not given
    starts as after an append of `length` tokens.  A cache of index keys alone
    (codes None) serves kv4_indexer_scores.  The calls go by the buffers' addresses:
    write into a buffer (cache.length.copy_(...), and seen with it where tokens are
    taken back), it cannot be replaced."""

    _BUFFERS = ("codes", "scales", "k_idx", "length", "seen", "lost", "position", "weight")

    def __setattr__(self, name, value):
        if name in self._BUFFERS and name in self.__dict__:
            raise AttributeError(f"KV4Cache.{name} is written in place, not replaced")
        super().__setattr__(name, value)

    def __init__(self, codes: torch.Tensor | None, scales: torch.Tensor | None,
                 length: torch.Tensor, k_idx: torch.Tensor | None = None,
                 position: torch.Tensor | None = None, weight: torch.Tensor | None = None,
                 seen: torch.Tensor | None = None, lost: torch.Tensor | None = None,
                 DK: int | None = None):
        first = codes if codes is not None else k_idx
        assert first is not None, "a cache needs codes or index keys"
        L.require_gpu(first)
        assert first.dim() == (4 if codes is not None else 3), "codes [B,S,HKV,(DK+DV)/2], k_idx [B,S,DI]"
        B, S = first.shape[:2]
        device = first.device
        HKV = DV = DI = 0
        if codes is not None:
            HKV, row = codes.shape[2], codes.shape[3]
            DK = row if DK is None else int(DK)
            DV = 2 * row - DK
            assert DK > 0 and DV > 0 and DK % 32 == 0 and DV % 32 == 0, \
                f"DK={DK} DV={DV} must be multiples of 32"
            assert scales is not None, "codes go with scales"
            if position is None:
                position = torch.arange(S, device=device, dtype=torch.int32).repeat(B, 1)
            if weight is None:
                weight = torch.zeros(B, S, device=device)
            if seen is None:
                seen = length.clone()
            if lost is None:
                lost = torch.zeros(B, device=device, dtype=torch.int32)
            self._is("codes", codes, (B, S, HKV, row), torch.uint8, device)
            self._is("scales", scales, (B, S, HKV, row // 16), torch.uint8, device)
            self._is("position", position, (B, S), torch.int32, device)
            self._is("weight", weight, (B, S), torch.float32, device)
            self._is("seen", seen, (B,), torch.int32, device)
            self._is("lost", lost, (B,), torch.int32, device)
        self._is("length", length, (B,), torch.int32, device)
        idx_dtype = torch.float32
        if k_idx is not None:
            DI, idx_dtype = k_idx.shape[2], k_idx.dtype
            assert idx_dtype in (torch.float32, torch.bfloat16, torch.float16), \
                f"index keys: fp32, bf16 or fp16 (got {idx_dtype})"
            self._is("k_idx", k_idx, (B, S, DI), idx_dtype, device)
        self.codes, self.scales, self.k_idx = codes, scales, k_idx
        self.length, self.seen, self.lost = length, seen, lost
        self.position, self.weight = position, weight
        self.B, self.S, self.HKV, self.DK, self.DV, self.DI = B, S, HKV, DK or 0, DV, DI
        self.device, self.index, self.idx_dtype = device, device.index, idx_dtype
        self.scale = 1.0 / math.sqrt(self.DK) if self.DK else 0.0

        def at(x):
            return x.data_ptr() if x is not None else None

        self._workspace = {}  # bytes of kv4_attention's, by its sizes
        self._c = L.Kv4Cache(at(codes), at(scales), at(k_idx), at(length), at(seen), at(lost),
                             at(position), at(weight), B, S, HKV, self.DK, DV, DI,
                             L.dtype_code(idx_dtype))
        self._ref = ctypes.addressof(self._c)

    @staticmethod
    def _is(name, x, shape, dtype, device):
        assert x.device == device and x.dtype == dtype and tuple(x.shape) == shape \
            and x.is_contiguous() and (x.data_ptr() % 16 == 0 or not x.numel()), \
            f"{name}: contiguous 16-byte aligned {dtype} {shape} on {device} " \
            f"(got {x.dtype} {tuple(x.shape)} on {x.device})"

    @classmethod
    def empty(cls, B: int, S: int, HKV: int, DK: int, DV: int, DI: int = 0,
              idx_dtype: torch.dtype = torch.bfloat16, device="cuda") -> "KV4Cache":
        """A cache with nothing in it (DI = 0: without index keys, which are held in idx_dtype)."""
        assert DK > 0 and DV > 0 and DK % 32 == 0 and DV % 32 == 0, \
            f"DK={DK} DV={DV} must be multiples of 32"
        dev = torch.device(device)
        if dev.type == "cuda" and dev.index is None:
            dev = torch.device("cuda", torch.cuda.current_device())
        return cls(torch.zeros(B, S, HKV, (DK + DV) // 2, device=dev, dtype=torch.uint8),
                   torch.zeros(B, S, HKV, (DK + DV) // 32, device=dev, dtype=torch.uint8),
                   torch.zeros(B, device=dev, dtype=torch.int32),
                   torch.zeros(B, S, DI, device=dev, dtype=idx_dtype) if DI else None, DK=DK)

    def check(self) -> None:
        """RuntimeError if a token found no free slot (waits for the GPU)."""
        if self.lost is not None and self.B and int(self.lost.max()) > 0:
            raise RuntimeError(f"KV4Cache: {int(self.lost.sum())} tokens found no free slot "
                               f"(S={self.S}): evict before appending")


def _stored(cache: KV4Cache) -> None:
    assert cache.codes is not None, "this cache holds index keys only"


def _ints(x: torch.Tensor, shape, name: str, cache: KV4Cache) -> torch.Tensor:
    """An int32 tensor of the caller's; a contiguous copy where it is not."""
    assert x.dtype is torch.int32 and x.shape == shape and x.get_device() == cache.index, \
        f"{name}: int32 {shape} on {cache.device} (got {x.dtype} {tuple(x.shape)} on {x.device})"
    return x if x.is_contiguous() else x.contiguous()


def _here(cache: KV4Cache, *xs: torch.Tensor) -> None:
    for x in xs:
        assert x.get_device() == cache.index, \
            f"inputs must be on the cache's GPU {cache.device} (got {x.device})"


def _ready(dtype: torch.dtype, cache: KV4Cache, *xs: torch.Tensor):
    """`xs` as the kernels take them (L.prep) and their pointers."""
    _here(cache, *xs)
    ptrs = L.ready_ptrs(dtype, xs)
    if ptrs is None:
        xs = [L.prep(x, dtype) for x in xs]
        ptrs = [x.data_ptr() for x in xs]
    return xs, ptrs


def _span(cache: KV4Cache, span: int | None) -> int:
    if span is None:
        return cache.S
    n = int(span)
    assert 0 <= n <= cache.S, f"span={n} outside [0, S={cache.S}]"
    return n


def _queries(cache: KV4Cache, Q: torch.Tensor):
    _stored(cache)
    assert Q.dim() == 4 and (Q.shape[0], Q.shape[3]) == (cache.B, cache.DK), \
        f"Q shape {tuple(Q.shape)}: B={cache.B}, DK={cache.DK}"
    return Q.shape


def _index_queries(cache: KV4Cache, q_idx: torch.Tensor, w_idx: torch.Tensor):
    assert cache.k_idx is not None, "this cache holds no index keys"
    assert q_idx.dim() == 4 and (q_idx.shape[0], q_idx.shape[3]) == (cache.B, cache.DI), \
        f"q_idx shape {tuple(q_idx.shape)}: B={cache.B}, DI={cache.DI}"
    assert 1 <= q_idx.shape[2] <= 256, f"HI={q_idx.shape[2]} outside [1,256]"
    assert w_idx.shape == q_idx.shape[:3], f"w_idx shape {tuple(w_idx.shape)} != {tuple(q_idx.shape[:3])}"
    return q_idx.shape


def _workspace_bytes(cache: KV4Cache, Tq: int, HQ: int, listed: bool, n: int, acc: int) -> int:
    """What dsa_kv4_attention needs of these sizes; raises where it would refuse them."""
    sizes = (Tq, HQ, listed, n, acc)
    nws = cache._workspace.get(sizes)
    if nws is None:
        if len(cache._workspace) >= 64:  # spans of a growing cache
            cache._workspace.clear()
        with L.on_device(cache.device):
            nws = L.lib().dsa_kv4_attention_workspace_bytes(cache._ref, Tq, HQ, int(listed), n, acc)
        if nws < 0:
            L.check(nws, "kv4_attention")
        cache._workspace[sizes] = nws
    return nws


def _call(cache: KV4Cache, what: str, fn, *args) -> None:
    """fn(cache, *args, stream) on the cache's GPU.  Single-token calls are bound by
    the host, so the usual case enters no context."""
    if torch.cuda.current_device() == cache.index:
        rc = fn(cache._ref, *args, L.stream_ptr(cache.device))
    else:
        with torch.cuda.device(cache.device):
            rc = fn(cache._ref, *args, L.stream_ptr(cache.device))
    if rc != L.DSA_OK:
        L.check(rc, what)


def _append_args(cache: KV4Cache, K, V, k_idx, count, weight):
    """dsa_kv4_append's arguments up to T, and what they point into."""
    _stored(cache)
    B, T = K.shape[:2]
    assert K.shape == (cache.B, T, cache.HKV, cache.DK), \
        f"K shape {tuple(K.shape)} != {(cache.B, T, cache.HKV, cache.DK)}"
    assert V.shape == (cache.B, T, cache.HKV, cache.DV), \
        f"V shape {tuple(V.shape)} != {(cache.B, T, cache.HKV, cache.DV)}"
    assert (k_idx is None) == (cache.k_idx is None), "index keys go with a cache that holds them"
    dt = L.common_dtype(K, V)
    kv, (k_ptr, v_ptr) = _ready(dt, cache, K, V)
    idx_ptr = weight_ptr = count_ptr = None
    if k_idx is not None:
        assert k_idx.shape == (B, T, cache.DI), f"k_idx shape {tuple(k_idx.shape)} != {(B, T, cache.DI)}"
        k_idx, (idx_ptr,) = _ready(cache.idx_dtype, cache, k_idx)
    if weight is not None:
        assert weight.shape == (B, T), f"weight shape {tuple(weight.shape)} != {(B, T)}"
        weight, (weight_ptr,) = _ready(torch.float32, cache, weight)
    if count is not None:
        count = _ints(count, (B,), "count", cache)
        count_ptr = count.data_ptr()
    return (k_ptr, v_ptr, L.dtype_code(dt), idx_ptr, weight_ptr, count_ptr, T), (kv, k_idx, weight, count)


def kv4_append(cache: KV4Cache, K: torch.Tensor, V: torch.Tensor, k_idx: torch.Tensor | None = None,
               *, count: torch.Tensor | None = None, weight: torch.Tensor | None = None,
               restart: bool = False) -> None:
    """Quantise T new tokens a sequence into the cache's next slots.

    K [B,T,HKV,DK], V [B,T,HKV,DV] (fp32, bf16 or fp16), k_idx [B,T,DI] where the
    cache holds index keys, stored in the type of its buffer (idx_dtype: other types
    are rounded to it, past fp16's range to Inf).  count int32 [B]: how many of the T are tokens (a
    padded batch; default all).  weight fp32 [B,T]: the new slots' first weights,
    e.g. what a prompt's own attention gave them (default 0).  restart: the
    sequences begin anew, at slot 0 and position 0 (a new batch of prompts).
    Tokens past slot S - 1 are not stored but counted in cache.lost."""
    args, held = _append_args(cache, K, V, k_idx, count, weight)
    _call(cache, "kv4_append", L.lib().dsa_kv4_append, *args, 1 if restart else 0)


def kv4_rows(cache: KV4Cache, slots: torch.Tensor | None = None, *, span: int | None = None,
             dtype: torch.dtype = torch.float32):
    """The values that slots stand for: (K [B,N,HKV,DK], V [B,N,HKV,DV]).

    slots int32 [B,N], or the first `span` slots (default all).  Slots that hold
    nothing give zeros.  Exact in fp32 and bf16."""
    _stored(cache)
    slots_ptr = None
    if slots is not None:
        assert span is None, "slots or span, not both"
        assert slots.dim() == 2, "slots: int32 [B, N]"
        N = slots.shape[1]
        slots = _ints(slots, (cache.B, N), "slots", cache)
        slots_ptr = slots.data_ptr()
    else:
        N = _span(cache, span)
    code = L.dtype_code(dtype)
    K = torch.empty((cache.B, N, cache.HKV, cache.DK), device=cache.device, dtype=dtype)
    V = torch.empty((cache.B, N, cache.HKV, cache.DV), device=cache.device, dtype=dtype)
    _call(cache, "kv4_rows", L.lib().dsa_kv4_rows, slots_ptr, N, code, K.data_ptr(), V.data_ptr())
    return K, V


def kv4_indexer_scores(cache: KV4Cache, q_idx: torch.Tensor, w_idx: torch.Tensor, *,
                       span: int | None = None, count: torch.Tensor | None = None) -> torch.Tensor:
    """Lightning indexer of the last Tq appended tokens against the cached index
    keys: [B,Tq,span] fp32, -inf where a token does not see the slot (its own and
    the earlier slots it sees, the later tokens' it does not).

    q_idx [B,Tq,HI,DI], w_idx [B,Tq,HI].  Types other than the cached keys' (or each
    other's) go as fp32: nothing is rounded to the keys' type.  span: only the first span slots (default
    all S).  count int32 [B]: how many of the Tq are tokens, as kv4_append's; the
    others' rows are -inf."""
    B, Tq, HI, _ = _index_queries(cache, q_idx, w_idx)
    n = _span(cache, span)
    dt, fn = cache.idx_dtype, L.lib().dsa_kv4_indexer_scores
    if q_idx.dtype is not dt or w_idx.dtype is not dt:
        dt, fn = torch.float32, L.lib().dsa_kv4_indexer_scores_f32
    qw, (q_ptr, w_ptr) = _ready(dt, cache, q_idx, w_idx)
    count_ptr = None
    if count is not None:
        count = _ints(count, (B,), "count", cache)
        count_ptr = count.data_ptr()
    scores = torch.empty((B, Tq, n), device=cache.device, dtype=torch.float32)
    _call(cache, "kv4_indexer_scores", fn, q_ptr, w_ptr, count_ptr, Tq, HI, n, scores.data_ptr())
    return scores


def kv4_attention(cache: KV4Cache, Q: torch.Tensor, *, slots: torch.Tensor | None = None,
                  span: int | None = None, count: torch.Tensor | None = None,
                  accumulate: bool = False, out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of the last Tq appended tokens over the cache: O [B,Tq,HQ,DV] fp32.

    Q [B,Tq,HQ,DK] (fp32, bf16 or fp16), HQ a multiple of HKV (query head h reads
    K/V head h // (HQ/HKV)); scale 1/sqrt(DK).  Over all slots that a token sees
    (its own and the earlier ones) among the first `span`, or only those listed
    in slots int32 [B,Tq,k] (topk_indices of kv4_indexer_scores); entries that it
    does not see count for nothing.  A token that sees nothing gets NaN.
    count int32 [B]: how many of the Tq are tokens; the others see nothing.
    accumulate: add each slot's probabilities, over tokens and heads, to
    cache.weight (what kv4_evict goes by)."""
    B, Tq, HQ, _ = _queries(cache, Q)
    slots_ptr = count_ptr = None
    if slots is not None:
        assert slots.dim() == 3, "slots: int32 [B, Tq, k]"
        assert span is None, "slots or span, not both"
        n = slots.shape[2]
        slots = _ints(slots, (B, Tq, n), "slots", cache)
        slots_ptr = slots.data_ptr()
    else:
        n = _span(cache, span)
    if count is not None:
        count = _ints(count, (B,), "count", cache)
        count_ptr = count.data_ptr()
    dt = L.common_dtype(Q)
    q, (q_ptr,) = _ready(dt, cache, Q)
    if out is None:
        out = torch.empty((B, Tq, HQ, cache.DV), device=cache.device, dtype=torch.float32)
    else:
        L.check_out(out, B * Tq * HQ * cache.DV, cache.device)
    acc = 1 if accumulate else 0
    lib = L.lib()
    nws = _workspace_bytes(cache, Tq, HQ, slots is not None, n, acc)
    ws = torch.empty(nws, device=cache.device, dtype=torch.uint8) if nws else None
    _call(cache, "kv4_attention", lib.dsa_kv4_attention, q_ptr, L.dtype_code(dt), slots_ptr, count_ptr,
          Tq, HQ, n, acc, cache.scale, out.data_ptr(), ws.data_ptr() if nws else None, nws)
    return out


def kv4_evict(cache: KV4Cache, keep: int, recent: int = 0):
    """Evict every sequence that has more than `keep` slots down to them: the
    `recent` newest tokens stay, then those of the largest accumulated weight
    (among equals the lowest slot).

    Kept slots at or past `keep` move into the freed ones.  Returns (from, to), int32
    [B,M] each, M = min(keep, S - keep): the slots that moved, in order, -1 past the
    last (for buffers of the caller's that go by slot)."""
    _stored(cache)
    keep, recent = int(keep), int(recent)
    M = max(0, min(keep, cache.S - keep))
    moved = torch.empty((2, cache.B, M), device=cache.device, dtype=torch.int32)
    src = moved.data_ptr()
    _call(cache, "kv4_evict", L.lib().dsa_kv4_evict, keep, recent, src, src + 4 * cache.B * M)
    return moved.unbind(0)


def _make_room(cache: KV4Cache, count_ptr: int | None, Tq: int, recent: int) -> None:
    """Evict what leaves no room for the next append: down to S - count[b] (default S - Tq)."""
    moved = torch.empty((2, cache.B, Tq), device=cache.device, dtype=torch.int32)
    src = moved.data_ptr()
    _call(cache, "kv4_make_room", L.lib().dsa_kv4_make_room, count_ptr, Tq, recent, src, src + 4 * cache.B * Tq)


def dsa_decode(cache: KV4Cache, q_idx, k_idx, w_idx, Q, K, V, top_k: int, *,
               span: int | None = None, count: torch.Tensor | None = None,
               keep: int | None = None, recent: int = 0) -> torch.Tensor:
    """A DSA step of Tq new tokens a sequence: append them, score the cached index
    keys, select the top_k slots of each token, attend to those, and (with `keep`)
    accumulate their weights and evict down to `keep` slots.  O [B,Tq,HQ,DV] fp32.

    q_idx [B,Tq,HI,DI]  k_idx [B,Tq,DI]  w_idx [B,Tq,HI]  Q [B,Tq,HQ,DK]
    K [B,Tq,HKV,DK]  V [B,Tq,HKV,DV].  Exactly top_k slots a token (the lowest
    slot wins ties), all it sees where it sees fewer.  span: no sequence has more
    slots than that in use (default S); where top_k >= span all of them are
    attended to and nothing is scored.  With keep (keep + Tq <= S) a sequence that has
    no room for its new tokens, after a prompt, is evicted down to it before the append;
    without, the caller sees to the room and cache.check() says whether tokens were lost."""
    assert top_k >= 1, "top_k must be >= 1"
    n = _span(cache, span)
    # what the later calls would refuse, before the first one changes the cache
    B, Tq, HQ, _ = _queries(cache, Q)
    assert K.shape[:2] == (B, Tq), f"K shape {tuple(K.shape)}: {Tq} tokens in Q"
    listed = top_k < n
    _here(cache, Q)
    if listed:
        assert _index_queries(cache, q_idx, w_idx)[1] == Tq, f"q_idx shape {tuple(q_idx.shape)}: {Tq} tokens in Q"
        _here(cache, q_idx, w_idx)
    if keep is not None:
        assert 0 <= recent <= keep, f"keep={keep} recent={recent} must be 0 <= recent <= keep"
        assert keep + Tq <= cache.S, f"keep={keep} slots and {Tq} new tokens do not fit S={cache.S}"
    _workspace_bytes(cache, Tq, HQ, listed, int(top_k) if listed else n, 0 if keep is None else 1)
    with L.on_device(cache.device):
        args, held = _append_args(cache, K, V, k_idx, count, None)
        if keep is not None:
            _make_room(cache, args[5], Tq, int(recent))
        _call(cache, "kv4_append", L.lib().dsa_kv4_append, *args, 0)
        slots = None
        if listed:
            scores = kv4_indexer_scores(cache, q_idx, w_idx, span=n, count=count)
            _, slots = topk_indices(scores, int(top_k))
        out = kv4_attention(cache, Q, slots=slots, span=None if slots is not None else n,
                            count=count, accumulate=keep is not None)
        if keep is not None:
            kv4_evict(cache, keep, recent)
    return out
