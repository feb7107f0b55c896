"""Cases of attention with a sliding window and of the paged 8-bit cache: what goes into the cache, with
the position rotation on the way, the attention over it, and the attention of prompts.

A sequence's keys and values are held in pages of a pool, in blocks of 64 tokens of one head: e4m3 codes
and one E8M0 scale byte each for the block's K and V,
    codes [pages, HKV, page/64, 64*(D+D)]   scales [pages, HKV, page/64, 2]
K token by token, then V dimension by dimension, a dimension's 64 tokens in the order of `_order`.
A token at position t sees position s where s <= t and (s > t - window or s < sinks); window 0: all.
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
BLOCK = 64


def _append(name, B, T, HQ, HKV, D, dtype, held=0, page=64, R=None, pairs=False, ragged=True):
    """held: slots in use before; HQ query heads rotated along (0: none); R rotated dimensions (0: none);
    pairs: neighbours rotate together, else the two halves of the R."""
    return {"name": name, "kind": "append", "B": B, "T": T, "HQ": HQ, "HKV": HKV, "D": D, "dtype": dtype,
            "held": held, "page": page, "R": D if R is None else R, "pairs": pairs, "ragged": ragged}


def _attention(name, B, S, HQ, HKV, D, dtype, Tq=1, window=0, sinks=0, page=64, ragged=True):
    return {"name": name, "kind": "attention", "B": B, "S": S, "HQ": HQ, "HKV": HKV, "D": D, "dtype": dtype,
            "Tq": Tq, "window": window, "sinks": sinks, "page": page, "ragged": ragged}


def _window(name, B, T, HQ, HKV, D, dtype, window, sinks, ragged=True):
    return {"name": name, "kind": "window", "B": B, "T": T, "HQ": HQ, "HKV": HKV, "D": D, "dtype": dtype,
            "window": window, "sinks": sinks, "ragged": ragged}


def listed():
    return [
        # A decode step of a serving batch: a token each into pages in use, its queries rotated with it.
        _append("append_step", 32, 1, 32, 8, 128, "bf16", held=2040),
        # A padded batch of prompts of no particular lengths, half of each head rotated, by neighbours.
        _append("append_prompts", 8, 1001, 8, 8, 64, "fp32", page=128, R=32, pairs=True),
        # Long prompts, the most bytes of any append.
        _append("append_long", 2, 16384, 32, 8, 128, "bf16", ragged=False),
        # The smallest call: one user's token after a short prompt, where latency counts.
        _attention("attention_one_short", 1, 129, 4, 4, 32, "fp32", ragged=False),
        # Grouped heads over long caches: the most bytes of any call.
        _attention("attention_long", 16, 32768, 32, 8, 128, "bf16"),
        # A serving batch of short sequences, one K/V head for each query head.
        _attention("attention_batch", 64, 2001, 8, 8, 64, "fp16", page=128),
        # A layer with a sliding window over long caches, the first tokens kept.
        _attention("attention_window", 32, 16384, 16, 4, 128, "bf16", window=4096, sinks=4, page=256),
        # A piece of 48 prompt tokens (or as many drafted ones) behind a cache, one K/V head for all.
        _attention("attention_piece", 4, 8191, 16, 1, 128, "bf16", Tq=48),
        # The smallest prompt: latency.
        _window("window_one_short", 1, 100, 4, 4, 32, "fp32", 32, 4, ragged=False),
        # A padded batch of prompts, grouped heads.
        _window("window_prompts", 4, 1777, 16, 4, 64, "fp16", 500, 4),
        # fp32 at the head sizes of the long-row configuration.
        _window("window_fp32", 2, 4096, 8, 8, 64, "fp32", 1024, 1, ragged=False),
        # The most work: a long prompt, grouped heads.
        _window("window_long", 1, 32768, 32, 8, 128, "bf16", 2048, 16, ragged=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append"] * 3 + ["attention"] * 5 + ["window"] * 4)
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    HKV, page, ragged = rng.choice([1, 2, 4, 8]), rng.choice([64, 64, 128, 256]), rng.random() < 0.7
    if kind == "window":
        D, HQ = rng.choice([32, 64, 64, 128, 128, 128, 256]), HKV * rng.choice([1, 2, 4])
        T, W, sinks = _log(rng, 1, 16384), _log(rng, 1, 4096), rng.choice([0, 1, 4, 4, 16, 100])
        if T <= 4096 and rng.random() < 0.25:
            W, sinks = 0, 0
        # fp32 costs about eight times as much a pair
        one = (min(W or T, T) + sinks) * HQ * max(D, 64) * (8 if dtype == "fp32" else 1)
        T = max(1, min(T, (1 << 37) // one))
        return _window("", max(1, min(_log(rng, 1, 16), (1 << 37) // (one * T))), T, HQ, HKV, D, dtype, W, sinks, ragged)
    D = rng.choice([32, 64, 64, 96, 128, 128, 128, 192, 256])
    if kind == "append":
        HQ = HKV * rng.choice([0, 1, 2, 4, 8])
        one = (2 * HKV + HQ) * D
        T = min(_log(rng, 1, 16384), (1 << 27) // one)
        B = max(1, min(_log(rng, 1, 64), (1 << 26) // (T * one)))
        held = rng.choice([0, 1, 63, 64, rng.randint(2, 2000), rng.randint(2, 2000)])
        return _append("", B, T, HQ, HKV, D, dtype, held, page, rng.choice([0, D // 2, D, D]), rng.random() < 0.4, ragged)
    S, Tq, G = _log(rng, 1, 32768), rng.choice([1, 1, 1, 1, 2, 3, rng.randint(4, 80)]), rng.choice([1, 2, 4, 8, 16])
    Tq = max(1, min(Tq, (1 << 33) // (S * HKV * G * D)))
    B = max(1, min(_log(rng, 1, 64), (1 << 28) // (S * HKV * D * max(1, Tq * G // 16))))
    W, sinks = (_log(rng, 1, 8192), rng.choice([0, 1, 4, 16, 100])) if rng.random() < 0.4 else (0, 0)
    return _attention("", B, max(S, Tq), HKV * G, HKV, D, dtype, Tq, W, sinks, page, ragged)


def _pure(c):
    return {k: v for k, v in c.items() if k != "name"}


def _lengths(c, B, n, least):
    """How full each sequence is: `n`, or for a ragged batch from there down to half of it."""
    if not c["ragged"]:
        return [n] * B
    return [max(least, n - (b * 977) % (n // 2 + 1)) for b in range(B)]


# --- the format ------------------------------------------------------------------------------
def _order():
    """Where token t of a block lies in each dimension's 64 bytes of V."""
    t = torch.arange(BLOCK, device="cuda")
    return (t // 4 % 4) * 16 + (t // 16) * 4 + t % 4


def _split(codes, D):
    """codes [..., 64*(D+D)] -> K and V codes [..., 64, D]."""
    k = codes[..., :BLOCK * D].unflatten(-1, (BLOCK, D))
    return k, codes[..., BLOCK * D:].unflatten(-1, (D, BLOCK))[..., _order()].transpose(-1, -2)


def _joined(k, v):
    """The inverse of _split."""
    back = torch.argsort(_order())
    return torch.cat([k.flatten(-2), v.transpose(-1, -2)[..., back].flatten(-2)], -1)


def _need(x):
    """Scale byte of a block [..., 64, D]: the least 2^e with max|x| <= 448 2^e."""
    bits = x.abs().amax((-1, -2)).view(torch.int32)
    return (((bits + 0x1FFFFF) >> 23) - 8).clamp(10, 247)


def _encode(x, byte):
    inverse = ((254 - byte.int()) << 23).view(torch.float32)
    return (x * inverse[..., None, None]).to(torch.float8_e4m3fn).view(torch.uint8)


def _decode(codes, byte):
    return codes.view(torch.float8_e4m3fn).float() * (byte.int() << 23).view(torch.float32)[..., None, None]


# --- inputs ----------------------------------------------------------------------------------
def _randn(g, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def _ints(v):
    return torch.tensor(v, device="cuda", dtype=torch.int32)


def _pool(c, g, B, S):
    """Pages in use, in no particular order: keys with a few strong channels, values N(0,1)."""
    HKV, D, page = c["HKV"], c["D"], c["page"]
    n, per = -(-S // page), page // BLOCK
    pages = torch.randperm(B * n, generator=g, device="cuda").to(torch.int32).view(B, n)
    codes = torch.empty(B * n, HKV, per, 2 * BLOCK * D, device="cuda", dtype=torch.uint8)
    scales = torch.empty(B * n, HKV, per, 2, device="cuda", dtype=torch.uint8)
    strong = 1 + 3 * (torch.rand(HKV, 1, 1, D, generator=g, device="cuda") < 0.05)
    step = max(1, (1 << 26) // (HKV * page * D))
    for i in range(0, B * n, step):
        m = min(step, B * n - i)
        k = _randn(g, m, HKV, per, BLOCK, D) * strong
        v = _randn(g, m, HKV, per, BLOCK, D)
        ks, vs = _need(k), _need(v)
        codes[i:i + m] = _joined(_encode(k, ks), _encode(v, vs))
        scales[i:i + m] = torch.stack([ks, vs], -1).to(torch.uint8)
    return pages, codes, scales


def _angles(positions, R):
    """Angles of position p and pair j, p * 10000^(-2j/R), in 64 bits."""
    j = torch.arange(R // 2, device="cuda", dtype=torch.float64)
    return torch.arange(positions, device="cuda", dtype=torch.float64).view(-1, 1) * torch.pow(10000.0, -2 * j / R)


def prepare(case, seed):
    c, kind, B = _pure(case), case["kind"], case["B"]
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt, HQ, HKV, D = DTYPES[c["dtype"]], c["HQ"], c["HKV"], c["D"]
    if kind == "window":
        T = c["T"]
        s = dict(case=c, Q=_randn(g, B, T, HQ, D, dtype=dt), K=_randn(g, B, T, HKV, D, dtype=dt),
                 V=_randn(g, B, T, HKV, D, dtype=dt))
        if c["ragged"]:
            s["count"] = _ints(_lengths(c, B, T, 1))
        return s
    if kind == "attention":
        pages, codes, scales = _pool(c, g, B, c["S"])
        return dict(case=c, pages=pages, codes=codes, scales=scales, Q=_randn(g, B, c["Tq"], HQ, D, dtype=dt),
                    length=_ints(_lengths(c, B, c["S"], c["Tq"])))
    T, held = c["T"], c["held"]
    start = _lengths(c, B, held, 0)
    pages, codes, scales = _pool(c, g, B, held + T)
    # the keys' strong channels; the tokens' sizes differ, so that some blocks' scales have to grow
    size = torch.exp2(torch.randint(-1, 3, (B, T, 1, 1), generator=g, device="cuda").float())
    strong = 1 + 3 * (torch.rand(HKV, D, generator=g, device="cuda") < 0.05)
    s = dict(case=c, pages=pages, codes=codes, scales=scales, start=_ints(start),
             K=(_randn(g, B, T, HKV, D) * strong * size).to(dt), V=(_randn(g, B, T, HKV, D) * size).to(dt),
             count=_ints(_lengths(c, B, T, 1)), length=_ints(start))
    if HQ:
        s["Q"] = _randn(g, B, T, HQ, D, dtype=dt)
    if c["R"]:
        angles = _angles(pages.shape[1] * c["page"], c["R"])
        s["cos"], s["sin"] = angles.cos().float(), angles.sin().float()
    # the slots that the append touches: from its first block's first one to its last token's
    first = s["start"] // BLOCK * BLOCK
    most = max(x % BLOCK for x in start) + T
    s["slots"] = (first.view(B, 1) + torch.arange(most, device="cuda", dtype=torch.int32)).contiguous()
    return s


# --- the operators, plainly --------------------------------------------------------------------
def _rotated(x, s, at):
    """x [B, T, H, D] in 32 bits, rotated by its positions `at` [B, T]."""
    c, x = s["case"], x.float()
    R = c["R"]
    if not R:
        return x
    cos, sin = (s[n][at].unsqueeze(2) for n in ("cos", "sin"))
    a, b = (x[..., 0:R:2], x[..., 1:R:2]) if c["pairs"] else (x[..., :R // 2], x[..., R // 2:R])
    a, b = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack([a, b], -1).flatten(-2) if c["pairs"] else torch.cat([a, b], -1)
    return torch.cat([turned, x[..., R:]], -1)


def _plain_append(s):
    c, start = s["case"], s["start"]
    B, T, HKV, D, per = c["B"], c["T"], c["HKV"], c["D"], c["page"] // BLOCK
    i = torch.arange(T, device="cuda")
    at = start.view(B, 1).long() + i
    k = _rotated(s["K"], s, at)
    out = {"rotated_K": k.to(s["K"].dtype)}
    if c["HQ"]:
        out["rotated_Q"] = _rotated(s["Q"], s, at).to(s["Q"].dtype)
    # the blocks that the call touches, [B, n, HKV]
    b = torch.arange(B, device="cuda").view(B, 1)
    n = -(-(BLOCK - 1 + T) // BLOCK)
    block = start.view(B, 1).long() // BLOCK + torch.arange(n, device="cuda")
    last = s["pages"].shape[1] * per - 1
    page, sub = s["pages"][b, (block.clamp(max=last) // per)].long(), block % per
    old_codes, old_scales = s["codes"][page, :, sub], s["scales"][page, :, sub].int()
    off = start.view(B, 1).long() % BLOCK
    token = torch.arange(n * BLOCK, device="cuda")
    held = (token < off).view(B, n, 1, BLOCK, 1)
    new = ((token >= off) & (token < off + s["count"].view(B, 1))).view(B, n, 1, BLOCK, 1)
    codes = []
    scales = []
    for x, old, which in zip((k, s["V"].float()), _split(old_codes, D), (0, 1)):
        put = torch.zeros(B, n * BLOCK, HKV, D, device="cuda")
        put[b, off + i] = x
        put = put.view(B, n, BLOCK, HKV, D).transpose(2, 3) * new
        need, before = _need(put), old_scales[..., which]
        e = torch.where(held.any(3).view(B, n, 1), torch.maximum(need, before), need)
        e = torch.where(new.any(3).view(B, n, 1), e, before)
        moved = _encode(_decode(old, before), e)
        codes.append(torch.where(new, _encode(put, e), torch.where(held, moved, old)))
        scales.append(e)
    ok = (block <= last).nonzero(as_tuple=True)
    s["codes"][page[ok], :, sub[ok]] = _joined(*codes)[ok]
    s["scales"][page[ok], :, sub[ok]] = torch.stack(scales, -1).to(torch.uint8)[ok]
    s["length"].copy_(start + s["count"])
    return out


def _plain_rows(s, at, dtype):
    """K and V of the slots `at` [B, N], zeros behind the length."""
    c, B = s["case"], s["case"]["B"]
    D, per = c["D"], c["page"] // BLOCK
    ok = (at < s["length"].view(B, 1)).view(B, -1, 1, 1)
    at = at.clamp(max=s["pages"].shape[1] * c["page"] - 1).long()
    page = s["pages"].gather(1, at // c["page"]).long()
    sub, t = at // BLOCK % per, at % BLOCK
    d = torch.arange(D, device="cuda")
    codes, scales = s["codes"], (s["scales"].int() << 23).view(torch.float32)
    h = torch.arange(c["HKV"], device="cuda").view(1, 1, -1, 1)
    page, sub, t = (x.view(B, -1, 1, 1) for x in (page, sub, t))
    k = codes[page, h, sub, t * D + d].view(torch.float8_e4m3fn).float() * scales[page, h, sub, 0]
    v = codes[page, h, sub, BLOCK * D + d * BLOCK + _order()[t]].view(torch.float8_e4m3fn).float() * scales[page, h, sub, 1]
    return (k * ok).to(dtype), (v * ok).to(dtype)


def _plain_attention(s):
    c = s["case"]
    B, S, Tq, HQ, HKV, D, W, sinks = (c[x] for x in ("B", "S", "Tq", "HQ", "HKV", "D", "window", "sinks"))
    G, length = HQ // HKV, s["length"].view(B, 1).long()
    if W and sinks + W + Tq < S:  # the slots that any of the tokens sees
        first = (length - Tq + 1 - W).clamp(min=0)
        near = first + torch.arange(W + Tq - 1, device="cuda")
        at = torch.cat([torch.arange(sinks, device="cuda").expand(B, -1), near], 1)
        once = torch.cat([torch.ones(B, sinks, device="cuda", dtype=torch.bool), near >= sinks], 1)
        K, V = _plain_rows(s, at, torch.float32)
    else:
        at = torch.arange(S, device="cuda").expand(B, -1)
        once = torch.ones(B, S, device="cuda", dtype=torch.bool)
        blocks = torch.arange(-(-S // BLOCK), device="cuda")
        per = c["page"] // BLOCK
        page = s["pages"][:, blocks // per].long()
        k, v = _split(s["codes"][page, :, blocks % per], D)
        e = s["scales"][page, :, blocks % per]
        K, V = (_decode(x, e[..., w]).permute(0, 1, 3, 2, 4).flatten(1, 2)[:, :S] for x, w in ((k, 0), (v, 1)))
    n = at.shape[1]
    t = (length - Tq + torch.arange(Tq, device="cuda")).view(B, Tq, 1)
    at = at.view(B, 1, n)
    ok = (at <= t) & once.view(B, 1, n)
    if W:
        ok &= (at > t - W) | (at < sinks)
    K = K.permute(0, 2, 3, 1).reshape(-1, D, n)
    V = (V * ok.any(1).view(B, n, 1, 1)).permute(0, 2, 1, 3).reshape(-1, n, D)
    q = s["Q"].float().view(B, Tq, HKV, G, D).permute(0, 2, 1, 3, 4).reshape(-1, Tq * G, D)
    score = (torch.bmm(q, K) / math.sqrt(D)).view(B, HKV, Tq, G, n)
    score = score.masked_fill(~ok.view(B, 1, Tq, 1, n), float("-inf"))
    p = (score - score.amax(-1, keepdim=True)).exp()
    p = p / p.sum(-1, keepdim=True)
    O = torch.bmm(p.view(-1, Tq * G, n), V)
    return O.view(B, HKV, Tq, G, D).permute(0, 2, 1, 3, 4).reshape(B, Tq, HQ, D).to(s["Q"].dtype)


def _plain_window(s):
    """Queries in blocks of C, each against the keys that any of them sees."""
    c = s["case"]
    B, T, HQ, HKV, D, W, sinks = (c[x] for x in ("B", "T", "HQ", "HKV", "D", "window", "sinks"))
    G, dt = HQ // HKV, s["Q"].dtype
    W = min(W, T) or T
    sinks = min(sinks, T)
    C = T if W >= T else min(T, max(64, W))
    n = -(-T // C)
    pad = n * C - T
    q = torch.nn.functional.pad(s["Q"].float(), (0, 0, 0, 0, 0, pad)).view(B, n, C, HKV, G, D)
    q = q.permute(0, 3, 1, 4, 2, 5).reshape(B * HKV * n, G * C, D) / math.sqrt(D)
    k, v = (s[x].float().transpose(1, 2) for x in ("K", "V"))  # [B, HKV, T, D]
    near = [torch.nn.functional.pad(x, (0, 0, W - 1, pad)).unfold(2, W - 1 + C, C) for x in (k, v)]
    wide = W - 1 + C
    t = torch.arange(n * C, device="cuda").view(n, 1, C, 1)
    at = (torch.arange(n, device="cuda") * C - W + 1).view(n, 1, 1, 1) + torch.arange(wide, device="cuda")
    ok = (at >= 0) & (at <= t) & (at > t - W) & (at < T)
    score = torch.bmm(q, near[0].reshape(B * HKV * n, D, wide)).view(B * HKV, n, G, C, wide)
    score = score.masked_fill(~ok, float("-inf"))
    if sinks:
        first = k[:, :, :sinks].transpose(2, 3).unsqueeze(2).expand(-1, -1, n, -1, -1)
        far = torch.bmm(q, first.reshape(-1, D, sinks)).view(B * HKV, n, G, C, sinks)
        score = torch.cat([score, far.masked_fill(torch.arange(sinks, device="cuda") > t - W, float("-inf"))], -1)
    p = (score - score.amax(-1, keepdim=True)).exp()
    del score
    p /= p.sum(-1, keepdim=True)
    O = torch.bmm(p[..., :wide].reshape(-1, G * C, wide), near[1].transpose(3, 4).reshape(-1, wide, D))
    if sinks:
        first = v[:, :, :sinks].unsqueeze(2).expand(-1, -1, n, -1, -1).reshape(-1, sinks, D)
        O += torch.bmm(p[..., wide:].reshape(-1, G * C, sinks), first)
    O = O.view(B, HKV, n, G, C, D).permute(0, 2, 4, 1, 3, 5).reshape(B, n * C, HQ, D)[:, :T]
    if "count" in s:  # a padded row sees nothing: 0 / 0
        O = O.masked_fill((torch.arange(T, device="cuda") >= s["count"].view(B, 1)).view(B, T, 1, 1), float("nan"))
    return O.to(dt)


# --- the framework's calls -----------------------------------------------------------------------
def _framework():
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "dsa-cpu-topk_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import dsa_paged

    return dsa_paged


def _held(s):
    """The framework's handle on the state's buffers, which a program makes once and keeps."""
    if "cache" not in s:
        s["cache"] = _framework().KV8Cache(s["codes"], s["scales"], s["pages"], s["length"])
    return s["cache"]


def run(state):
    s, c = state, state["case"]
    if c["kind"] == "window":
        if not own:
            return _plain_window(s)
        return _framework().window_attention(s["Q"], s["K"], s["V"], window=c["window"] or None, sinks=c["sinks"],
                                             count=s.get("count"))
    if c["kind"] == "attention":
        if not own:
            return _plain_attention(s)
        return _framework().kv8_attention(_held(s), s["Q"], window=c["window"] or None, sinks=c["sinks"])
    # What went into the 8 bits comes back as the values that it stands for, which bf16 holds exactly.
    if own:
        m, cache = _framework(), _held(s)
        rope = (s["cos"], s["sin"]) if c["R"] else None
        q, k = m.kv8_append(cache, s["K"], s["V"], rope=rope, pairs=c["pairs"], Q=s.get("Q"), start=s["start"],
                            count=s["count"], keys=True)
        out = {"rotated_K": k, **({"rotated_Q": q} if c["HQ"] else {})}
        K, V = m.kv8_rows(cache, s["slots"], dtype=torch.bfloat16)
    else:
        out = _plain_append(s)
        K, V = _plain_rows(s, s["slots"], torch.bfloat16)
    return {**out, "K": K, "V": V, "length": s["length"]}


# --- what a pass cannot do without ---------------------------------------------------------------
def _pairs(n, T, W, sinks):
    """Pairs (t, s) with n - T <= t < n that see each other."""
    W = W or n
    total = 0
    for t in range(n - T, n):
        total += min(t + 1, W) + max(0, min(sinks, t + 1 - W))
    return total


def work(case):
    c, kind, B = case, case["kind"], case["B"]
    es, HQ, HKV, D = BYTES[c["dtype"]], c["HQ"], c["HKV"], c["D"]
    row = 2 * HKV * D  # bytes of one token's codes
    if kind == "window":
        many = _lengths(c, B, c["T"], 1)
        return {"bytes": sum(many) * es * (2.0 * HKV * D + HQ * D) + es * B * c["T"] * HQ * D,
                "flops": sum(4.0 * HQ * D * _pairs(n, n, c["window"], c["sinks"]) for n in many)}
    if kind == "attention":
        S, Tq, W = c["S"], c["Tq"], c["window"]
        lengths = _lengths(c, B, S, Tq)
        near = [min(n, W + Tq - 1) if W else n for n in lengths]
        read = sum(m + min(c["sinks"], n - m) for m, n in zip(near, lengths))
        return {"bytes": read * (row + row / (BLOCK * D)) + 2.0 * es * B * Tq * HQ * D,
                "flops": sum(4.0 * HQ * D * _pairs(n, Tq, W, c["sinks"]) for n in lengths)}
    T, held = c["T"], _lengths(c, B, c["held"], 0)
    tokens = sum(_lengths(c, B, T, 1))
    back = tokens + sum(n % BLOCK for n in held)  # a first block's held tokens come back too
    rows = B * (max(n % BLOCK for n in held) + T)  # of values, zeros behind the last token
    moved = 2 * B * T * (HKV + HQ) * D + tokens * HKV * D
    return {"bytes": es * float(moved) + (tokens + back + 2.0 * rows) * row + 4.0 * c["R"] * T,
            "flops": 3.0 * B * T * c["R"] * (HKV + HQ) + 2.0 * tokens * row}


# --- 64 bits -------------------------------------------------------------------------------------
def _value64(code, byte):
    """Of e4m3: s eeee mmm, bias 7, 1111 111 no number; times 2^(byte - 127)."""
    code = code.to(torch.int64)
    e, m = (code >> 3) & 15, (code & 7).double()
    mag = torch.where(e == 0, m / 512, (1 + m / 8) * torch.exp2(e.double() - 7))
    return torch.where(code >= 128, -mag, mag) * torch.exp2(byte.double() - 127)


def _held64(s, b, h, n):
    """K and V [n, D] of one head's first n slots."""
    c = s["case"]
    D, per = c["D"], c["page"] // BLOCK
    at = torch.arange(n, device="cuda")
    page, sub, t = s["pages"][b, at // c["page"]].long(), at // BLOCK % per, at % BLOCK
    d = torch.arange(D, device="cuda")
    row = s["codes"][page, h, sub]
    k = row.gather(1, (t * D).view(-1, 1) + d)
    # bytes of a dimension: tokens 0-3 16-19 32-35 48-51 4-7 20-23 ...
    place = torch.tensor([16 * (x % 16 // 4) + 4 * (x // 16) + x % 4 for x in range(BLOCK)], device="cuda")[t]
    v = row.gather(1, BLOCK * D + d * BLOCK + place.view(-1, 1))
    e = s["scales"][page, h, sub]
    return _value64(k, e[:, :1]), _value64(v, e[:, 1:])


def _exact_attention(s):
    c = s["case"]
    B, Tq, HQ, HKV, D, W = (c[x] for x in ("B", "Tq", "HQ", "HKV", "D", "window"))
    G = HQ // HKV
    out = torch.empty(B, Tq, HQ, D, device="cuda", dtype=torch.float64)
    for b in range(B):
        n = int(s["length"][b])
        at = torch.arange(n, device="cuda")
        t = (n - Tq + torch.arange(Tq, device="cuda")).view(-1, 1, 1)
        ok = (at <= t) & ((at > t - W) | (at < c["sinks"]) if W else True)
        for h in range(HKV):
            K, V = _held64(s, b, h, n)
            score = s["Q"][b, :, h * G:(h + 1) * G].double() @ K.t() / math.sqrt(D)
            out[b, :, h * G:(h + 1) * G] = torch.softmax(score.masked_fill(~ok, float("-inf")), -1) @ V
    return out


def _exact_window(s):
    c = s["case"]
    B, T, HQ, HKV, D, sinks = (c[x] for x in ("B", "T", "HQ", "HKV", "D", "sinks"))
    W, G = c["window"] or c["T"], HQ // HKV
    out = torch.full((B, T, HQ, D), float("nan"), device="cuda", dtype=torch.float64)
    for b in range(B):
        n = int(s["count"][b]) if "count" in s else T
        for t0 in range(0, n, 512):
            t = torch.arange(t0, min(t0 + 512, n), device="cuda").view(-1, 1)
            lo = max(0, t0 - W + 1)
            at = torch.cat([torch.arange(min(sinks, lo), device="cuda"), torch.arange(lo, int(t[-1]) + 1, device="cuda")])
            ok = (at <= t) & ((at > t - W) | (at < sinks))
            for h in range(HKV):
                K, V = s["K"][b, at, h].double(), s["V"][b, at, h].double()
                q = s["Q"][b, t0:t0 + len(t), h * G:(h + 1) * G].double().transpose(0, 1)
                score = (q @ K.t() / math.sqrt(D)).masked_fill(~ok, float("-inf"))
                out[b, t0:t0 + len(t), h * G:(h + 1) * G] = (torch.softmax(score, -1) @ V).transpose(0, 1)
    return out


def _grid64(x, byte):
    """x to the nearest of e4m3's values times 2^(byte - 127), ties to the even code."""
    y = x.abs() * torch.exp2(127 - byte.double())
    e = torch.floor(torch.log2(y.clamp(min=2.0 ** -20))).clamp(-6, 8)
    e = torch.where(y >= torch.exp2(e + 1), e + 1, torch.where(y < torch.exp2(e), e - 1, e)).clamp(-6, 8)
    step = torch.exp2(e - 3)
    return torch.sign(x) * torch.round(y / step) * step * torch.exp2(byte.double() - 127)


def _turn64(x, s, at):
    """x [T, H, D] at positions `at`, each pair as a complex number times cos + i sin."""
    c, x = s["case"], x.double().clone()
    R = c["R"]
    if not R:
        return x
    unit = torch.complex(s["cos"][at].double(), s["sin"][at].double()).unsqueeze(1)
    i = torch.arange(R // 2, device="cuda")
    real, imag = (2 * i, 2 * i + 1) if c["pairs"] else (i, i + R // 2)
    z = torch.complex(x[..., real], x[..., imag]) * unit
    x[..., real], x[..., imag] = z.real, z.imag
    return x


def _exact_append(s):
    """A sequence and a block at a time, on the values themselves."""
    c = s["case"]
    B, T, HQ, HKV, D, N = c["B"], c["T"], c["HQ"], c["HKV"], c["D"], s["slots"].shape[1]
    K = torch.zeros(B, N, HKV, D, device="cuda", dtype=torch.float64)
    V = torch.zeros_like(K)
    turned_k = torch.empty(B, T, HKV, D, device="cuda", dtype=torch.float64)
    turned_q = torch.empty(B, T, HQ, D, device="cuda", dtype=torch.float64)
    for b in range(B):
        n0, new = int(s["start"][b]), int(s["count"][b])
        at = n0 + torch.arange(T, device="cuda")
        turned_k[b] = _turn64(s["K"][b], s, at)
        if HQ:
            turned_q[b] = _turn64(s["Q"][b], s, at)
        begin = n0 // BLOCK * BLOCK
        off = n0 - begin
        for which, out, fresh in ((0, K, turned_k[b, :new]), (1, V, s["V"][b, :new].double())):
            x = torch.zeros(-(-(off + new) // BLOCK) * BLOCK, HKV, D, device="cuda", dtype=torch.float64)
            x[off:off + new] = fresh
            top = x.view(-1, BLOCK, HKV, D).abs().amax((1, 3))  # [blocks, HKV]
            e = torch.ceil(torch.log2(top.clamp(min=2.0 ** -130) / 448))
            e = torch.where(top > 448 * torch.exp2(e), e + 1, torch.where(top <= 448 * torch.exp2(e - 1), e - 1, e))
            byte = (e + 127).clamp(10, 247)
            if off:
                page, sub = int(s["pages"][b, n0 // c["page"]]), n0 // BLOCK % (c["page"] // BLOCK)
                byte[0] = torch.maximum(byte[0], s["scales"][page, :, sub, which].double())
                for h in range(HKV):
                    x[:off, h] = _held64(s, b, h, n0)[which][begin:]
            x = _grid64(x, byte.repeat_interleave(BLOCK, 0).unsqueeze(-1))
            out[b, :off + new] = x[:off + new]
    got = {"rotated_K": turned_k, "K": K, "V": V, "length": None}
    return {**got, "rotated_Q": turned_q} if HQ else got


def exact(case, seed):
    c = case
    if c["kind"] == "attention" and c["B"] * c["HKV"] > 2048:
        return None  # minutes of small products
    s = prepare(case, seed)
    return {"append": _exact_append, "attention": _exact_attention, "window": _exact_window}[c["kind"]](s)
