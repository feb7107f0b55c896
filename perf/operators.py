"""Cases of the 4-bit decode cache: its attention, its indexer, what is appended to it, what is
evicted from it.

A sequence's keys and values are held in slots, in OCP MXFP4: codes of e2m1 elements (the even
element of a pair in the low nibble) and one E8M0 scale byte per 32 of them,
    codes [B, S, HKV, (DK+DV)/2]   scales [B, S, HKV, (DK+DV)/32]     (K, then V, of each head).
`run` computes each operator in torch's elementary operations in 32 bits where `own` is false, and
calls the framework where it is true; `exact` computes it in 64 bits.
"""
from __future__ import annotations

import math
import os
import sys

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}


def _attention(name, B, S, HQ, HKV, D, dtype, Tq=1, k=0, ragged=True, weights=False):
    return {"name": name, "kind": "attention", "B": B, "S": S, "HQ": HQ, "HKV": HKV, "D": D,
            "dtype": dtype, "Tq": Tq, "k": k, "ragged": ragged, "weights": weights}


def _indexer(name, B, S, HI, DI, dtype, Tq=1, ragged=True):
    return {"name": name, "kind": "indexer", "B": B, "S": S, "HI": HI, "DI": DI, "dtype": dtype,
            "Tq": Tq, "ragged": ragged}


def _append(name, B, T, HKV, D, DI, dtype, ragged=True):
    return {"name": name, "kind": "append", "B": B, "T": T, "HKV": HKV, "D": D, "DI": DI,
            "dtype": dtype, "ragged": ragged}


def _evict(name, B, T, keep, recent, HKV, D, DI, dtype, prompt):
    return {"name": name, "kind": "evict", "B": B, "T": T, "keep": keep, "recent": recent,
            "HKV": HKV, "D": D, "DI": DI, "dtype": dtype, "prompt": prompt}


def listed():
    return [
        # The smallest call: one user's first tokens after a short prompt, where latency counts.
        _attention("attention_one_short", 1, 129, 4, 4, 32, "fp32", ragged=False),
        # A serving batch at the long-row configuration's head sizes (one K/V head per query head).
        _attention("attention_batch", 16, 4096, 8, 8, 64, "bf16"),
        # Grouped heads over long caches: the most bytes of any call.
        _attention("attention_long", 16, 32768, 32, 8, 128, "bf16"),
        # One K/V head for all queries, two tokens a sequence (one drafted), weights for eviction.
        _attention("attention_one_kv_head", 8, 10007, 16, 1, 128, "fp16", Tq=2, weights=True),
        # Sparse decode: the 2048 slots that the indexer chose out of a long cache, and their weights.
        _attention("attention_sparse", 32, 16384, 16, 4, 128, "bf16", k=2048, weights=True),
        # Sparse decode in fp32 with a small odd selection.
        _attention("attention_sparse_fp32", 4, 4000, 8, 8, 64, "fp32", k=255),
        # The indexer of one new token: one short sequence, and a batch of long ones.
        _indexer("indexer_one_short", 1, 512, 4, 32, "fp32", ragged=False),
        _indexer("indexer_long", 8, 32768, 64, 128, "bf16"),
        # Prompts put into 4 bits: a padded batch of no particular lengths, and a long one.
        _append("append_prompts", 8, 1001, 8, 64, 64, "fp32"),
        _append("append_long", 2, 16384, 8, 128, 128, "bf16", ragged=False),
        # A decode step of full caches: a token each goes in, the least attended to goes out.
        _evict("evict_step", 32, 1, 2048, 64, 8, 128, 128, "bf16", prompt=False),
        # Prompts cut to a budget by the weights that their own attention gave.
        _evict("evict_prompts", 8, 4099, 1024, 32, 8, 128, 64, "fp16", prompt=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attention"] * 5 + ["indexer"] * 2 + ["append", "evict", "evict"])
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    D = rng.choice([32, 64, 64, 128, 128, 128, 256])
    if kind == "indexer":
        S, HI, DI, Tq = _log(rng, 64, 32768), rng.choice([1, 4, 8, 12, 32, 64]), rng.choice([32, 64, 128]), rng.choice([1, 1, 1, 2, 4])
        most = (1 << 36) // (S * HI * DI * Tq * (4 if dtype == "fp32" else 1))
        return _indexer("", max(1, min(_log(rng, 1, 32), most)), S, HI, DI, dtype, Tq, rng.random() < 0.7)
    HKV = rng.choice([1, 2, 4, 8])
    row = HKV * D  # bytes of one token's codes
    if kind == "append":
        T = _log(rng, 1, 16384)
        B = max(1, min(_log(rng, 1, 32), (1 << 25) // (T * row)))
        return _append("", B, T, HKV, D, rng.choice([32, 64, 128]), dtype, rng.random() < 0.7)
    if kind == "evict":
        prompt = rng.random() < 0.5
        T = _log(rng, 64, 8192) if prompt else rng.randint(1, 8)
        keep = max(8, int(T * rng.uniform(0.1, 0.9))) if prompt else _log(rng, 64, 8192)
        B = max(1, min(_log(rng, 1, 32), (1 << 26) // ((T + keep) * row)))
        return _evict("", B, T, keep, rng.randint(0, keep // 4), HKV, D, rng.choice([32, 64, 128]), dtype, prompt)
    S, Tq = _log(rng, 1, 32768), rng.choice([1, 1, 1, 1, 2, 3])
    B = max(1, min(_log(rng, 1, 64), (1 << 28) // (S * row * Tq)))
    k = max(1, min(S, _log(rng, 16, 2048))) if rng.random() < 0.4 else 0
    return _attention("", B, max(S, Tq), HKV * rng.choice([1, 2, 4, 8, 16]), HKV, D, dtype, Tq, k,
                      rng.random() < 0.7, rng.random() < 0.4)


def _pure(c):
    return {k: v for k, v in c.items() if k != "name"}


def _lengths(c, B, n, least):
    """How full each sequence is: `n`, or for a ragged batch from there down to half of it."""
    if not c.get("ragged"):
        return [n] * B
    return [max(least, n - (b * 977) % (n // 2 + 1)) for b in range(B)]


# --- the format ------------------------------------------------------------------------------
def _encode(x):
    """x [..., D] -> (codes [..., D/2], scale bytes [..., D/32])."""
    x = x.float().unflatten(-1, (-1, 32))
    top = x.abs().amax(-1)
    e = (((top.view(torch.int32) + 0x200000) >> 23) - 2).clamp(2, 252)
    r = x.abs() * ((254 - e) << 23).view(torch.float32).unsqueeze(-1)
    code = ((r > 0.25).int() + (r >= 0.75).int() + (r > 1.25).int() + (r >= 1.75).int()
            + (r > 2.5).int() + (r >= 3.5).int() + (r > 5.0).int())
    code = (code + 8 * (x < 0).int()).flatten(-2)
    return (code[..., 0::2] + 16 * code[..., 1::2]).to(torch.uint8), e.to(torch.uint8)


def _decode(codes, scales):
    """The values that codes [..., D/2] and scale bytes [..., D/32] stand for, fp32."""
    e2m1 = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, 0, -.5, -1, -1.5, -2, -3, -4, -6], device=codes.device)
    v = e2m1[torch.stack([codes & 15, codes >> 4], -1).int()].flatten(-2)
    s = (scales.int() << 23).view(torch.float32)
    return (v.unflatten(-1, (-1, 32)) * s.unsqueeze(-1)).flatten(-2)


def _kv(codes, scales, D):
    return (_decode(codes[..., :D // 2], scales[..., :D // 32]),
            _decode(codes[..., D // 2:], scales[..., D // 32:]))


# --- inputs ----------------------------------------------------------------------------------
def _randn(g, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def _ints(v):
    return torch.tensor(v, device="cuda", dtype=torch.int32)


def _filled(g, B, S, HKV, D):
    """Buffers of a cache in use: keys with a few strong channels, values N(0,1)."""
    codes = torch.empty(B, S, HKV, D, device="cuda", dtype=torch.uint8)
    scales = torch.empty(B, S, HKV, D // 16, device="cuda", dtype=torch.uint8)
    strong = 1 + 3 * (torch.rand(HKV, D, generator=g, device="cuda") < 0.05)
    for b in range(B):
        for at, x in ((0, _randn(g, S, HKV, D) * strong), (1, _randn(g, S, HKV, D))):
            c, s = _encode(x)
            codes[b, :, :, at * D // 2:(at + 1) * D // 2] = c
            scales[b, :, :, at * D // 32:(at + 1) * D // 32] = s
    return codes, scales


def prepare(case, seed):
    c, kind, B = _pure(case), case["kind"], case["B"]
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[c["dtype"]]
    if kind == "indexer":
        S, Tq, HI, DI = c["S"], c["Tq"], c["HI"], c["DI"]
        return dict(case=c, length=_ints(_lengths(c, B, S, Tq)), k_idx=_randn(g, B, S, DI, dtype=dt),
                    q_idx=_randn(g, B, Tq, HI, DI, dtype=dt), w_idx=_randn(g, B, Tq, HI, dtype=dt, scale=HI ** -0.5))
    HKV, D = c["HKV"], c["D"]
    if kind == "attention":
        S, Tq, k = c["S"], c["Tq"], c["k"]
        lengths = _lengths(c, B, S, Tq)
        codes, scales = _filled(g, B, S, HKV, D)
        s = dict(case=c, codes=codes, scales=scales, length=_ints(lengths),
                 weight=torch.rand(B, S, generator=g, device="cuda"),
                 Q=_randn(g, B, Tq, c["HQ"], D, dtype=dt))
        if k:  # ascending, as the select gives them, and slots past the length where it has too few
            score = torch.rand(B, Tq, S, generator=g, device="cuda")
            score.masked_fill_(torch.arange(S, device="cuda") >= s["length"].view(B, 1, 1), -1.0)
            s["slots"] = score.topk(k, dim=-1).indices.sort(-1).values.to(torch.int32)
        return s
    T, DI = c["T"], c["DI"]
    held = 0 if kind == "append" or c["prompt"] else c["keep"]
    S = held + T
    s = dict(case=c, K=_randn(g, B, T, HKV, D, dtype=dt), V=_randn(g, B, T, HKV, D, dtype=dt),
             new_idx=_randn(g, B, T, DI, dtype=dt), k_idx=_randn(g, B, S, DI, dtype=dt),
             count=_ints(_lengths(c, B, T, 1)))
    s["codes"], s["scales"] = _filled(g, B, S, HKV, D)
    s["length"], s["seen"] = _ints([held] * B), _ints([held] * B)
    s["position"] = torch.arange(S, device="cuda", dtype=torch.int32).expand(B, S).contiguous()
    s["weight"] = torch.rand(B, S, generator=g, device="cuda")
    if kind == "evict" and c["prompt"]:
        s["new_weight"] = torch.rand(B, T, generator=g, device="cuda")
    return s


# --- the operators, plainly --------------------------------------------------------------------
def _visible(s, S, Tq):
    """[B, Tq, S]: the slots that each of the last Tq tokens sees."""
    last = s["length"].view(-1, 1, 1) - Tq + 1 + torch.arange(Tq, device="cuda").view(1, -1, 1)
    return torch.arange(S, device="cuda") < last


def _plain_indexer(s):
    c = s["case"]
    B, S, Tq, HI, DI = (c[x] for x in ("B", "S", "Tq", "HI", "DI"))
    dots = torch.bmm(s["q_idx"].float().view(B, Tq * HI, DI), s["k_idx"].float().transpose(1, 2).contiguous())
    score = (dots.clamp(min=0).view(B, Tq, HI, S) * s["w_idx"].float().unsqueeze(-1)).sum(2)
    return score.masked_fill(~_visible(s, S, Tq), float("-inf"))


def _plain_attention(s):
    c = s["case"]
    B, S, Tq, HQ, HKV, D = (c[x] for x in ("B", "S", "Tq", "HQ", "HKV", "D"))
    G, codes, scales, ok = HQ // HKV, s["codes"], s["scales"], _visible(s, S, Tq)
    if c["k"]:  # one row of keys for each query token
        at = s["slots"].long()
        b = torch.arange(B, device="cuda").view(-1, 1, 1)
        codes, scales, ok = codes[b, at].flatten(0, 1), scales[b, at].flatten(0, 1), ok.gather(2, at)
    K, V = _kv(codes, scales, D)
    n, rows = K.shape[1], Tq * G if not c["k"] else G
    K = K.permute(0, 2, 3, 1).reshape(-1, D, n)
    V = V.permute(0, 2, 1, 3).reshape(-1, n, D)
    q = s["Q"].float().view(B, Tq, HKV, G, D)
    q = q.permute(0, 2, 1, 3, 4) if not c["k"] else q
    score = torch.bmm(q.reshape(-1, rows, D), K) / math.sqrt(D)
    score = score.view(B, HKV, Tq, G, n) if not c["k"] else score.view(B, Tq, HKV, G, n).transpose(1, 2)
    score = score.masked_fill(~ok.view(B, 1, Tq, 1, n), float("-inf"))
    p = (score - score.amax(-1, keepdim=True)).exp()
    p = p / p.sum(-1, keepdim=True)
    p_rows = p.reshape(-1, rows, n) if not c["k"] else p.transpose(1, 2).reshape(-1, rows, n)
    O = torch.bmm(p_rows, V)
    O = O.view(B, HKV, Tq, G, D).permute(0, 2, 1, 3, 4) if not c["k"] else O
    if not c["weights"]:
        return O.reshape(B, Tq, HQ, D)
    per = p.sum((1, 3))  # [B, Tq, n]
    if c["k"]:
        s["weight"].scatter_add_(1, at.flatten(1), per.flatten(1))
    else:
        s["weight"] += per.sum(1)
    return O.reshape(B, Tq, HQ, D), s["weight"]


def _plain_append(s, restart, weight):
    c = s["case"]
    B, T = c["B"], c["T"]
    S = s["codes"].shape[1]
    if restart:
        s["length"].zero_()
        s["seen"].zero_()
    i = torch.arange(T, device="cuda").view(1, T)
    new = i < s["count"].view(B, 1)
    at = (s["length"].view(B, 1) + i).clamp(max=S - 1).long()
    b = torch.arange(B, device="cuda").view(B, 1)
    kc, ks = _encode(s["K"])
    vc, vs = _encode(s["V"])
    for name, x in (("codes", torch.cat([kc, vc], -1)), ("scales", torch.cat([ks, vs], -1)),
                    ("k_idx", s["new_idx"]), ("position", (s["seen"].view(B, 1) + i).int()),
                    ("weight", weight if weight is not None else torch.zeros(B, T, device="cuda"))):
        m = new.view(B, T, *[1] * (x.dim() - 2))
        s[name][b, at] = torch.where(m, x, s[name][b, at])
    s["length"] += s["count"]
    s["seen"] += s["count"]


def _plain_rows(s, at):
    """K and V of the slots `at` [B, N], zeros for those that hold nothing."""
    b = torch.arange(at.shape[0], device="cuda").view(-1, 1)
    ok = ((at >= 0) & (at < s["length"].view(-1, 1))).view(*at.shape, 1, 1)
    at = at.clamp(min=0).long()
    dt = DTYPES[s["case"]["dtype"]]
    return tuple((x * ok).to(dt) for x in _kv(s["codes"][b, at], s["scales"][b, at], s["case"]["D"]))


def _plain_evict(s, keep, recent):
    B, S = s["weight"].shape
    M = min(keep, S - keep)
    slot = torch.arange(S, device="cuda").expand(B, S)
    n = s["length"].view(B, 1)
    rank_of = s["weight"].masked_fill(s["position"] >= s["seen"].view(B, 1) - recent, float("inf"))
    rank_of = rank_of.masked_fill(slot >= n, float("-inf"))
    order = rank_of.sort(dim=1, descending=True, stable=True).indices
    kept = torch.zeros(B, S, dtype=torch.bool, device="cuda").scatter_(1, order[:, :keep], True)
    kept = (kept | (n <= keep)) & (slot < n)
    away, free = kept & (slot >= keep), ~kept & (slot < keep) & (slot < n)
    many = away.sum(1, keepdim=True)
    i = torch.arange(M, device="cuda")
    src, dst = ((~m).int().sort(dim=1, stable=True).indices[:, :M] for m in (away, free))
    b = torch.arange(B, device="cuda").view(B, 1)
    u, v = torch.where(i < many, src, S - 1), torch.where(i < many, dst, S - 1)
    for name in ("codes", "scales", "k_idx", "position", "weight"):
        s[name][b, v] = s[name][b, u]
    s["length"].clamp_(max=keep)
    return torch.where(i < many, src, -1).int(), torch.where(i < many, dst, -1).int()


# --- the framework's calls -----------------------------------------------------------------------
def _held(s):
    """The framework's handle on the state's buffers, which a program makes once and keeps."""
    if "cache" not in s:
        pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "dsa-cpu-topk_amd")
        if pkg not in sys.path:
            sys.path.insert(0, pkg)
        import dsa_cache

        buffers = {k: s.get(k) for k in ("codes", "scales", "k_idx", "position", "weight", "seen")}
        s["module"], s["cache"] = dsa_cache, dsa_cache.KV4Cache(length=s["length"], **buffers)
    return s["module"], s["cache"]


def run(state):
    s, c = state, state["case"]
    if c["kind"] == "indexer":
        if not own:
            return _plain_indexer(s)
        m, cache = _held(s)
        return m.kv4_indexer_scores(cache, s["q_idx"], s["w_idx"])
    if c["kind"] == "attention":
        if not own:
            return _plain_attention(s)
        m, cache = _held(s)
        O = m.kv4_attention(cache, s["Q"], slots=s.get("slots"), accumulate=c["weights"])
        return (O, s["weight"]) if c["weights"] else O
    # What went into the 4 bits comes back as the values that it stands for.
    names = ("k_idx", "position", "weight", "length", "seen")
    if c["kind"] == "append":
        if own:
            m, cache = _held(s)
            m.kv4_append(cache, s["K"], s["V"], s["new_idx"], count=s["count"], restart=True)
            K, V = m.kv4_rows(cache, dtype=DTYPES[c["dtype"]])
        else:
            _plain_append(s, True, None)
            K, V = _plain_rows(s, torch.arange(c["T"], device="cuda").expand(c["B"], -1))
        return {"K": K, "V": V, **{k: s[k] for k in names}}
    prompt = c["prompt"]
    if own:
        m, cache = _held(s)
        m.kv4_append(cache, s["K"], s["V"], s["new_idx"], count=s["count"], restart=prompt,
                     weight=s.get("new_weight"))
        src, dst = m.kv4_evict(cache, c["keep"], c["recent"])
        K, V = m.kv4_rows(cache, dst, dtype=DTYPES[c["dtype"]])
    else:
        _plain_append(s, prompt, s.get("new_weight"))
        src, dst = _plain_evict(s, c["keep"], c["recent"])
        K, V = _plain_rows(s, dst)
    return {"src": src, "dst": dst, "K": K, "V": V, **{k: s[k] for k in names}}


# --- what a pass cannot do without ---------------------------------------------------------------
def work(case):
    c, kind, B = case, case["kind"], case["B"]
    es = BYTES[c["dtype"]]
    if kind == "indexer":
        S, Tq, HI, DI = c["S"], c["Tq"], c["HI"], c["DI"]
        held = sum(_lengths(c, B, S, Tq))
        return {"bytes": held * DI * es + 4.0 * B * Tq * S + es * B * Tq * HI * (DI + 1),
                "flops": 2.0 * Tq * held * HI * (DI + 1)}
    HKV, D = c["HKV"], c["D"]
    row = HKV * D * 17 / 16  # codes and scales of one token
    if kind == "attention":
        S, Tq, k = c["S"], c["Tq"], c["k"]
        # a listed slot is read once for each token that lists it; a full cache once for all
        read = [Tq * min(n, k) if k else n for n in _lengths(c, B, S, Tq)]
        pairs = sum(read) if k else Tq * sum(read)
        io = (es + 4.0) * B * Tq * c["HQ"] * D + (4.0 * B * Tq * k)
        return {"bytes": sum(read) * (row + (8 if c["weights"] else 0)) + io, "flops": 4.0 * pairs * c["HQ"] * D}
    T, DI = c["T"], c["DI"]
    tokens = sum(_lengths(c, B, T, 1))
    put = tokens * (es * (2 * HKV * D + 2 * DI) + row + 8)
    if kind == "append":
        return {"bytes": put + tokens * row + es * 2.0 * B * T * HKV * D, "flops": 4.0 * tokens * HKV * D}
    keep = c["keep"]
    S = T if c["prompt"] else keep + T
    M = min(keep, S - keep)
    # as many survivors lie past the budget as chance puts there
    moved = B * (keep * (S - keep) / S if c["prompt"] else min(T, c["recent"]))
    return {"bytes": put + 8.0 * B * S + moved * 2 * (row + DI * es + 8) + moved * row + es * 2.0 * B * M * HKV * D,
            "flops": 4.0 * tokens * HKV * D + B * S}


# --- 64 bits -------------------------------------------------------------------------------------
def _value64(nibble, byte):
    """sign * {0, 1/2, 1, 3/2, 2, 3, 4, 6} * 2^(byte-127), by the bits of e2m1: s ee m."""
    nibble = nibble.to(torch.int64)
    e, m = (nibble >> 1) & 3, (nibble & 1).double()
    mag = torch.where(e == 0, m / 2, (1 + m / 2) * torch.exp2(e.double() - 1))
    return torch.where(nibble >= 8, -mag, mag) * torch.exp2(byte.double() - 127)


def _unpack64(codes, scales, at, D):
    """One head's D elements from `at` on: codes [n, bytes], scales [n, blocks] -> [n, D] float64."""
    j = torch.arange(D, device="cuda")
    byte = codes[:, (at + j) // 2]
    nibble = torch.where(j % 2 == 0, byte & 15, byte >> 4)
    return _value64(nibble, scales[:, (at + j) // 32])


def _quantised64(x):
    """The values that x [..., 32 n] becomes in the cache, by comparing distances on the grid."""
    y = x.double().unflatten(-1, (-1, 32))
    top = y.abs().amax(-1, keepdim=True)
    e = torch.floor(torch.log2(top.clamp(min=2.0 ** -130) / 7)) + 1  # the least with top < 7 * 2^e
    e = torch.where(top >= 7 * torch.exp2(e), e + 1, torch.where(top < 7 * torch.exp2(e - 1), e - 1, e)).clamp(-125, 125)
    r = (y.abs() / torch.exp2(e)).clamp(max=6)
    step = torch.where(r < 2, 0.5, torch.where(r < 4, 1.0, 2.0))
    r = torch.round(r / step) * step  # ties to the even multiple, which is the even code
    return (torch.sign(y) * r * torch.exp2(e)).flatten(-2)


def _exact_attention(s):
    c = s["case"]
    B, S, Tq, HQ, HKV, D = (c[x] for x in ("B", "S", "Tq", "HQ", "HKV", "D"))
    G = HQ // HKV
    out = torch.empty(B, Tq, HQ, D, device="cuda", dtype=torch.float64)
    weight = s["weight"].double()
    for b in range(B):
        n = int(s["length"][b])
        for t in range(Tq):
            at = torch.arange(n - Tq + t + 1, device="cuda")
            if c["k"]:
                at = s["slots"][b, t].long()
                at = at[at < n - Tq + t + 1]
            for h in range(HKV):
                K = _unpack64(s["codes"][b, at, h], s["scales"][b, at, h], 0, D)
                V = _unpack64(s["codes"][b, at, h], s["scales"][b, at, h], D, D)
                p = torch.softmax(s["Q"][b, t, h * G:(h + 1) * G].double() @ K.t() / math.sqrt(D), -1)
                out[b, t, h * G:(h + 1) * G] = p @ V
                weight[b].index_add_(0, at, p.sum(0))
    return (out, weight) if c["weights"] else out


def _exact_indexer(s):
    c = s["case"]
    B, S, Tq = c["B"], c["S"], c["Tq"]
    out = torch.full((B, Tq, S), float("-inf"), device="cuda", dtype=torch.float64)
    for b in range(B):
        for t in range(Tq):
            n = int(s["length"][b]) - Tq + t + 1
            dots = s["q_idx"][b, t].double() @ s["k_idx"][b, :n].double().t()
            out[b, t, :n] = s["w_idx"][b, t].double() @ dots.clamp(min=0)
    return out


def _exact_cache(s):
    """Append and eviction on the values themselves, a sequence at a time."""
    c = s["case"]
    B, T, D = c["B"], c["T"], c["D"]
    evict = c["kind"] == "evict"
    S = s["codes"].shape[1]
    restart = not evict or c["prompt"]
    M = min(c["keep"], S - c["keep"]) if evict else T
    K = torch.zeros(B, M, c["HKV"], D, device="cuda", dtype=torch.float64)
    V = torch.zeros_like(K)
    k_idx, weight = s["k_idx"].double(), s["weight"].double()
    for b in range(B):
        n0, new = 0 if restart else int(s["length"][b]), int(s["count"][b])
        n = n0 + new
        k_idx[b, n0:n] = s["new_idx"][b, :new].double()
        weight[b, n0:n] = s["new_weight"][b, :new].double() if "new_weight" in s else 0.0
        if not evict:
            K[b, :new], V[b, :new] = _quantised64(s["K"][b, :new]), _quantised64(s["V"][b, :new])
            continue
        if n <= c["keep"]:
            continue
        value = weight[b, :n].clone()
        value[max(0, n - c["recent"]):] = float("inf")  # slots are still in the order of positions
        kept = value.sort(descending=True, stable=True).indices[:c["keep"]].sort().values
        free = torch.ones(c["keep"], dtype=torch.bool, device="cuda")
        free[kept[kept < c["keep"]]] = False
        src, dst = kept[kept >= c["keep"]], free.nonzero().view(-1)
        k_idx[b, dst], weight[b, dst] = k_idx[b, src], weight[b, src]
        # what moves was appended now: a full cache held only the slots below the budget
        m = len(src)
        K[b, :m], V[b, :m] = _quantised64(s["K"][b, src - n0]), _quantised64(s["V"][b, src - n0])
    return K, V, k_idx, weight


def exact(case, seed):
    c = case
    if c["kind"] == "attention" and c["B"] * c["Tq"] * c["HKV"] > 4096:
        return None  # minutes of small products
    s = prepare(case, seed)
    if c["kind"] == "indexer":
        return _exact_indexer(s)
    if c["kind"] == "attention":
        return _exact_attention(s)
    K, V, k_idx, weight = _exact_cache(s)
    got = {"K": K, "V": V, "k_idx": k_idx, "weight": weight}
    none = ("src", "dst", "position", "length", "seen") if c["kind"] == "evict" else ("position", "length", "seen")
    return {**got, **{k: None for k in none}}
