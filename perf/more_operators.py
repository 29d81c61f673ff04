"""Cases of the attention operators over a paged cache of keys and values:

  rope       norm and position rotation of queries and keys, head by head
  append     keys (normed and rotated) and values of new tokens into the paged cache, their queries rotated on the way
  attention  new tokens of each sequence over its cached keys and values: causal, grouped heads, optionally with
             a sliding window and a few first tokens that stay visible

`run` computes them in plain torch operations, or (own = True) through the
framework's entry points.  Queries and keys are N(0, 1), as after a norm, with a
per-head key offset and a louder first key, so that attention is not flat; a
sequence's pages are scattered over the cache in random order.
"""
import math
import random
import sys

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


def _nxq():
    """The framework's binding, initialised on the first GPU."""
    if "nexus-inference-engine-_b200" not in sys.path:
        sys.path.insert(0, "nexus-inference-engine-_b200")
    import nxq

    nxq.init(0)
    return nxq


# ---- cases -------------------------------------------------------------------
# new_lo .. new_hi: new tokens per sequence; ctx_lo .. ctx_hi: tokens already in the cache.

def listed():
    return [
        # The queries and keys of one decode step of one sequence (Llama-3-8B's heads), with their norms.
        {"name": "rope-1", "op": "rope", "T": 1, "Hq": 32, "Hk": 8, "D": 128, "dims": 128, "layout": "half", "scaling": "none",
         "norm": True, "x": "f16", "y": "f16", "far": 8192},
        # A prompt batch at far positions, half of each head rotated, frequencies scaled for long contexts.
        {"name": "rope-8192", "op": "rope", "T": 8192, "Hq": 32, "Hk": 8, "D": 128, "dims": 64, "layout": "interleaved", "scaling": "yarn",
         "norm": False, "x": "bf16", "y": "bf16", "far": 1000000},
        # A decode step of 48 sequences, straight from fp32 projections.
        {"name": "append-48", "op": "append", "S": 48, "new_lo": 1, "new_hi": 1, "ctx_lo": 100, "ctx_hi": 500, "Hq": 32, "Hk": 8, "D": 128,
         "page": 32, "order": "heads", "dims": 128, "layout": "half", "scaling": "blend", "norm": True, "x": "f32", "y": "bf16"},
        # Ragged prompts going in, 11 sequences of 1000 to 2000 tokens.
        {"name": "append-ragged", "op": "append", "S": 11, "new_lo": 1000, "new_hi": 2000, "ctx_lo": 0, "ctx_hi": 300, "Hq": 64, "Hk": 8, "D": 128,
         "page": 64, "order": "tokens", "dims": 128, "layout": "half", "scaling": "none", "norm": False, "x": "bf16", "y": "bf16"},
        # One sequence's next token with a short history: latency.
        {"name": "decode-1-short", "op": "attention", "S": 1, "new_lo": 1, "new_hi": 1, "ctx_lo": 999, "ctx_hi": 999, "Hq": 32, "Hk": 8, "D": 128,
         "page": 16, "order": "heads", "window": 0, "sinks": 0, "x": "f16", "y": "f16"},
        # One sequence's next token with a long history (128 query heads over 8, the 405B-shaped layer).
        {"name": "decode-1-long", "op": "attention", "S": 1, "new_lo": 1, "new_hi": 1, "ctx_lo": 131071, "ctx_hi": 131071, "Hq": 128, "Hk": 8, "D": 128,
         "page": 64, "order": "heads", "window": 0, "sinks": 0, "x": "bf16", "y": "bf16"},
        # A served batch's decode step, ragged histories.
        {"name": "decode-64-ragged", "op": "attention", "S": 64, "new_lo": 1, "new_hi": 1, "ctx_lo": 200, "ctx_hi": 8000, "Hq": 32, "Hk": 8, "D": 128,
         "page": 16, "order": "tokens", "window": 0, "sinks": 0, "x": "bf16", "y": "bf16"},
        # Drafted tokens of 24 sequences, up to six each, on their way to verification; five query heads per key head.
        {"name": "drafted-24", "op": "attention", "S": 24, "new_lo": 2, "new_hi": 6, "ctx_lo": 1000, "ctx_hi": 5000, "Hq": 40, "Hk": 8, "D": 128,
         "page": 32, "order": "heads", "window": 0, "sinks": 0, "x": "f16", "y": "f16"},
        # A served batch's decode step with a window and sinks over long histories.
        {"name": "decode-32-window", "op": "attention", "S": 32, "new_lo": 1, "new_hi": 1, "ctx_lo": 10000, "ctx_hi": 40000, "Hq": 64, "Hk": 8, "D": 64,
         "page": 32, "order": "heads", "window": 2048, "sinks": 4, "x": "bf16", "y": "bf16"},
        # A whole prompt.
        {"name": "prompt-8192", "op": "attention", "S": 1, "new_lo": 8192, "new_hi": 8192, "ctx_lo": 0, "ctx_hi": 0, "Hq": 32, "Hk": 8, "D": 128,
         "page": 64, "order": "heads", "window": 0, "sinks": 0, "x": "bf16", "y": "bf16"},
        # Chunks of six prompts, some long in the cache already, in one step.
        {"name": "chunks-6", "op": "attention", "S": 6, "new_lo": 37, "new_hi": 1500, "ctx_lo": 500, "ctx_hi": 16000, "Hq": 32, "Hk": 8, "D": 128,
         "page": 16, "order": "heads", "window": 0, "sinks": 0, "x": "f16", "y": "f16"},
        # Ragged prompts through a windowed layer with sinks.
        {"name": "prompts-window", "op": "attention", "S": 4, "new_lo": 2000, "new_hi": 6000, "ctx_lo": 0, "ctx_hi": 3000, "Hq": 32, "Hk": 4, "D": 64,
         "page": 32, "order": "tokens", "window": 1024, "sinks": 4, "x": "bf16", "y": "bf16"},
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rope", "append", "attention", "attention", "attention"])
    Hk = rng.choice([1, 2, 4, 8])
    Hq = Hk * rng.choice([1, 2, 3, 4, 5, 7, 8, 16])
    D = rng.choice([64, 80, 96, 128, 128])
    x = rng.choice(["f16", "bf16"])
    if op == "rope":
        return {"op": op, "T": _log(rng, 1, max(1, min(8192, 8192 * 40 * 128 // ((Hq + Hk) * D)))), "Hq": Hq, "Hk": Hk, "D": D,
                "dims": rng.choice([D, D, D // 2]), "layout": rng.choice(["half", "interleaved"]), "scaling": rng.choice(["none", "yarn", "blend"]),
                "norm": rng.random() < 0.5, "x": rng.choice(["f32", x]), "y": x, "far": _log(rng, 100, 1000000)}
    page = rng.choice([8, 16, 24, 32, 64, 128, 256])
    base = {"op": op, "Hq": Hq, "Hk": Hk, "D": D, "page": page, "order": rng.choice(["heads", "tokens"]), "x": x, "y": rng.choice([x, x, "f32"])}
    if op == "append":
        S = _log(rng, 1, 64)
        most = max(1, 1500 * 11 * 80 * 128 // (S * (Hq + 2 * Hk) * D))
        new = _log(rng, 1, min(2000, most))
        ctx = _log(rng, 1, 500)
        return {**base, "S": S, "new_lo": max(1, new // 2), "new_hi": new, "ctx_lo": ctx // 4, "ctx_hi": ctx, "dims": rng.choice([D, D // 2]),
                "layout": rng.choice(["half", "interleaved"]), "scaling": rng.choice(["none", "blend"]), "norm": rng.random() < 0.5,
                "x": rng.choice(["f32", x]), "y": x}
    window, sinks = rng.choice([(0, 0), (0, 0), (_log(rng, 64, 4096), rng.choice([0, 1, 4, 33]))])
    kind = rng.choice(["decode", "drafted", "chunk"])
    S = _log(rng, 1, 64 if kind != "chunk" else 12)
    ctx = _log(rng, 1, max(1, min(131072, 64 * 8000 // S)))
    if kind == "decode":
        lo = hi = 1
    elif kind == "drafted":
        lo, hi = 1, rng.randint(2, 16)
    else:
        hi = _log(rng, 17, 8192)
        # As many scores as a whole prompt of 8192 tokens at most.
        while S * hi * (ctx + hi) * Hq * D > 8192 * 8192 * 32 * 128 // 2 and hi > 1:
            hi = (hi + 1) // 2
            ctx = max(1, ctx // 2) if ctx > 4 * hi else ctx
        lo = max(1, hi // 3)
    return {**base, "S": S, "new_lo": lo, "new_hi": hi, "ctx_lo": ctx // 5, "ctx_hi": ctx, "window": window, "sinks": sinks}


def _lengths(case):
    """New tokens and cached tokens of every sequence: the same for every seed, as a timing wants them."""
    rng = random.Random("%(S)d %(new_lo)d %(new_hi)d %(ctx_lo)d %(ctx_hi)d" % case)
    new = [rng.randint(case["new_lo"], case["new_hi"]) for _ in range(case["S"])]
    return new, [rng.randint(case["ctx_lo"], case["ctx_hi"]) for _ in range(case["S"])]


# ---- inputs -------------------------------------------------------------------

def _frequencies(dims, scaling):
    """Radians per position of every pair, as a model's loader computes them, and the factor on sine and cosine."""
    inv = [10000.0 ** (-2.0 * i / dims) for i in range(dims // 2)]
    if scaling == "none":
        return inv, 1.0
    factor, trained, out = 8.0, 8192.0, []
    for i, f in enumerate(inv):
        if scaling == "yarn":  # slow pairs are divided, fast ones kept, a ramp over the pair's index between
            turns = lambda b: dims * math.log(trained / (b * 2 * math.pi)) / (2 * math.log(10000.0))  # noqa: E731
            lo, hi = max(math.floor(turns(32.0)), 0), min(math.ceil(turns(1.0)), dims - 1)
            ramp = min(max((i - lo) / max(hi - lo, 0.001), 0.0), 1.0)
            out.append(f / factor * ramp + f * (1 - ramp))
        else:  # the same by wavelength, between 1/4 and 1 of the trained length
            smooth = min(max((trained * f / (2 * math.pi) - 1.0) / 3.0, 0.0), 1.0)
            out.append((1 - smooth) * f / factor + smooth * f)
    return out, (0.1 * math.log(factor) + 1.0 if scaling == "yarn" else 1.0)


def _cache(case, g, pages, dtype):
    """Keys and values [pages][heads][slots][D], or [pages][slots][heads][D] for order "tokens"."""
    Hk, D, page = case["Hk"], case["D"], case["page"]
    shape = (pages, Hk, page, D) if case["order"] == "heads" else (pages, page, Hk, D)
    mean = 0.5 * torch.randn((Hk, 1, D) if case["order"] == "heads" else (Hk, D), device="cuda", generator=g)
    k = torch.randn(shape, device="cuda", generator=g).add_(mean).to(dtype)
    v = torch.randn(shape, device="cuda", generator=g).to(dtype)
    return k, v


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op, s = case["op"], {"case": case}
    Hq, Hk, D, x = case["Hq"], case["Hk"], case["D"], DTYPES[case["x"]]
    n = s["nxq"] = _nxq() if own else None
    if op != "attention":
        s["inv"], s["factor"] = _frequencies(case["dims"], case["scaling"])
        s["freq"] = torch.tensor(s["inv"], dtype=torch.float64, device="cuda")
        s["norms"] = [1 + 0.1 * torch.randn(D, device="cuda", generator=g) if case["norm"] else None for _ in range(2)]
        if own:
            s["rope"] = n.Rope(s["inv"], layout=case["layout"], scale=s["factor"])
    if op == "rope":
        T = case["T"]
        # Queries and keys as they lie in the projection's output: one row of both per token.
        s["qk"] = torch.randn((T, Hq + Hk, D), device="cuda", generator=g).to(x)
        s["q"], s["k"] = s["qk"][:, :Hq], s["qk"][:, Hq:]
        s["positions"] = torch.randint(0, case["far"], (T,), device="cuda", generator=g)
        return s
    new, ctx = _lengths(case)
    T, S, page = sum(new), case["S"], case["page"]
    total = [a + b for a, b in zip(new, ctx)]
    s["new"], s["total"] = new, total
    need = [-(-t // page) for t in total]
    pages = sum(need) + 3
    order = torch.randperm(pages, device="cuda", generator=g).to(torch.int32)
    table = torch.full((S, max(need)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for i, c in enumerate(need):
        table[i, :c] = order[at:at + c]
        at += c
    s["table"] = table
    s["kv_lens"] = torch.tensor(total, dtype=torch.int32, device="cuda")
    s["q_offsets"] = torch.tensor([0] + new, device="cuda").cumsum(0).to(torch.int32)
    y = DTYPES[case["y"]]
    if op == "append":
        s["cache"] = _cache(case, g, pages, y)
        s["qkv"] = torch.randn((T, Hq + 2 * Hk, D), device="cuda", generator=g).to(x)
        s["q"], s["k"], s["v"] = s["qkv"][:, :Hq], s["qkv"][:, Hq:Hq + Hk], s["qkv"][:, Hq + Hk:]
    else:
        s["cache"] = _cache(case, g, pages, x)
        k, first = s["cache"][0], table[:, 0].long()
        at = (first, slice(None), 0) if case["order"] == "heads" else (first, 0)
        k[at] = k[at] * 1.5  # the first key of a sequence draws more than its share
        s["q"] = (1.5 * torch.randn((T, Hq, D), device="cuda", generator=g)).to(x)
        if case["window"]:  # pages that no query sees any more went back to the pool
            for i in range(S):
                gone = (ctx[i] - case["window"] + 1) // page
                kept = -(-case["sinks"] // page)
                if gone > kept:
                    table[i, kept:gone] = -1
    if own:
        s["kv"] = n.KVCache(*s["cache"], order=case["order"])
    return s


# ---- one pass -----------------------------------------------------------------

def _angles(positions, freq):
    """Sine and cosine of position * frequency: the angle in 64 bits, rounded once."""
    a = positions.double()[:, None] * freq
    return torch.sin(a).float()[:, None], torch.cos(a).float()[:, None]


def _turn(x, norm, sin, cos, dims, layout, factor):
    """Norm over the head and rotation of x [T][H][D], in float32."""
    x = x.float()
    if norm is not None:
        x = x * torch.rsqrt((x * x).mean(dim=-1, keepdim=True) + 1e-6) * norm
    r, rest = x[..., :dims], x[..., dims:]
    a, b = (r[..., :dims // 2], r[..., dims // 2:]) if layout == "half" else (r[..., 0::2], r[..., 1::2])
    c, d = (a * cos - b * sin) * factor, (a * sin + b * cos) * factor
    r = torch.cat([c, d], dim=-1) if layout == "half" else torch.stack([c, d], dim=-1).flatten(-2)
    return torch.cat([r, rest], dim=-1)


def _positions(s):
    """Position of every new token and its place (page, slot) in the cache."""
    lens, off = s["kv_lens"].long(), s["q_offsets"].long()
    t = torch.arange(sum(s["new"]), device="cuda")
    i = torch.searchsorted(off[1:], t, right=True)
    p = lens[i] - (off[i + 1] - t)
    page = s["case"]["page"]
    return p, s["table"][i, p // page].long(), p % page


def _gather(s, which, i, lo, hi):
    """Keys or values lo .. hi - 1 of sequence i as [heads][keys][D] in float32."""
    page, c = s["case"]["page"], s["cache"][which]
    first = lo // page
    rows = c[s["table"][i, first:-(-hi // page)].long()].float()
    rows = rows.transpose(0, 1) if s["case"]["order"] == "heads" else rows.permute(2, 0, 1, 3)
    return rows.reshape(rows.shape[0], -1, rows.shape[-1])[:, lo - first * page:hi - first * page]


def _attend(s):
    case, q = s["case"], s["q"]
    Hq, Hk, D, W, sinks = (case[n] for n in ("Hq", "Hk", "D", "window", "sinks"))
    out = torch.empty(q.shape, dtype=DTYPES[case["y"]], device="cuda")
    scale, at, group = 1 / math.sqrt(D), 0, Hq // Hk
    for i, (n, total) in enumerate(zip(s["new"], s["total"])):
        for t0 in range(0, n, 512):  # queries in pieces, so that their scores stay small
            t1 = min(n, t0 + 512)
            hi = total - n + t1
            lo = max(0, total - n + t0 - W + 1) if W else 0
            k, v = _gather(s, 0, i, lo, hi), _gather(s, 1, i, lo, hi)
            j = torch.arange(lo, hi, device="cuda")
            head = min(sinks, lo)
            if head:
                k, v = torch.cat([_gather(s, 0, i, 0, head), k], dim=1), torch.cat([_gather(s, 1, i, 0, head), v], dim=1)
                j = torch.cat([torch.arange(head, device="cuda"), j])
            p = torch.arange(total - n + t0, hi, device="cuda")[:, None]
            seen = j <= p
            if W:
                seen &= (j > p - W) | (j < sinks)
            x = q[at + t0:at + t1].float().view(t1 - t0, Hk, group, D).permute(1, 2, 0, 3).reshape(Hk, -1, D)
            a = (x @ k.transpose(1, 2)).view(Hk, group, t1 - t0, -1) * scale
            a = a.masked_fill(~seen, -math.inf)
            a = torch.exp(a - a.amax(dim=-1, keepdim=True))
            z = a.sum(dim=-1, keepdim=True)
            o = (a.view(Hk, group * (t1 - t0), -1) @ v).view(Hk, group, t1 - t0, D) / z
            out[at + t0:at + t1] = o.permute(2, 0, 1, 3).reshape(t1 - t0, Hq, D).to(out.dtype)
        at += n
    return out


def run(s):
    case, op, n = s["case"], s["case"]["op"], s["nxq"]
    y = DTYPES[case["y"]]
    if op == "rope":
        if own:
            q, k = n.rope(s["rope"], s["positions"], s["q"], s["k"], q_norm=s["norms"][0], k_norm=s["norms"][1], out_dtype=y)
            return {"q": q, "k": k}
        sin, cos = _angles(s["positions"], s["freq"])
        q, k = (_turn(x, w, sin, cos, case["dims"], case["layout"], s["factor"]) for x, w in zip((s["q"], s["k"]), s["norms"]))
        return {"q": q.to(y), "k": k.to(y)}
    if op == "append":
        if own:
            q = n.kv_append(s["kv"], s["k"], s["v"], s["q_offsets"], s["kv_lens"], s["table"], rope=s["rope"], q=s["q"],
                            q_norm=s["norms"][0], k_norm=s["norms"][1], out_dtype=y)
            return {"q": q, "keys": s["cache"][0], "values": s["cache"][1]}
        p, page, slot = _positions(s)
        sin, cos = _angles(p, s["freq"])
        q, k = (_turn(x, w, sin, cos, case["dims"], case["layout"], s["factor"]) for x, w in zip((s["q"], s["k"]), s["norms"]))
        for c, x in zip(s["cache"], (k, s["v"].float())):
            if case["order"] == "heads":
                c[page, :, slot] = x.to(c.dtype)
            else:
                c[page, slot] = x.to(c.dtype)
        return {"q": q.to(y), "keys": s["cache"][0], "values": s["cache"][1]}
    if own:
        return n.paged_attention(s["q"], s["kv"], s["q_offsets"], s["kv_lens"], s["table"], window=case["window"], sinks=case["sinks"],
                                 max_new=case["new_hi"], out_dtype=y)
    return _attend(s)


# ---- work and exact values ------------------------------------------------------

def work(case):
    Hq, Hk, D, x, y = case["Hq"], case["Hk"], case["D"], SIZE[case["x"]], SIZE[case["y"]]
    if case["op"] == "rope":
        rows = case["T"] * (Hq + Hk)
        return {"bytes": rows * D * (x + y) + 8 * case["T"], "flops": rows * (3 * case["dims"] + (3 * D if case["norm"] else 0))}
    new, ctx = _lengths(case)
    T = sum(new)
    if case["op"] == "append":
        return {"bytes": T * (Hq + 2 * Hk) * D * (x + y) + 8 * case["S"], "flops": T * (Hq + Hk) * (3 * case["dims"] + (3 * D if case["norm"] else 0))}
    W, sinks, keys, pairs = case["window"], case["sinks"], 0, 0
    for n, c in zip(new, ctx):
        if not W:
            keys += n + c
            pairs += n * c + n * (n + 1) // 2
            continue
        lo = max(0, c - W + 1)
        keys += n + c - lo + min(sinks, lo)
        for p in range(c, c + n):
            first = max(0, p - W + 1)
            pairs += p + 1 - first + min(sinks, first)
    return {"bytes": 2 * keys * Hk * D * x + T * Hq * D * (x + y) + 8 * case["S"], "flops": 4 * pairs * Hq * D}


def _exact_turn(x, norm, positions, s):
    """Rotation as a complex product, in 64 bits."""
    case = s["case"]
    x = x.double()
    if norm is not None:
        x = x / ((x ** 2).sum(-1, keepdim=True) / case["D"] + 1e-6).sqrt() * norm.double()
    dims = case["dims"]
    pick = torch.arange(dims // 2, device="cuda")
    a, b = (pick, pick + dims // 2) if case["layout"] == "half" else (2 * pick, 2 * pick + 1)
    angle = positions.double()[:, None, None] * s["freq"]
    z = torch.complex(x[..., a], x[..., b]) * torch.polar(torch.full_like(angle, s["factor"]), angle)
    out = x.clone()
    out[..., a], out[..., b] = z.real, z.imag
    return out


def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    if case["op"] == "rope":
        return {"q": _exact_turn(s["q"], s["norms"][0], s["positions"], s), "k": _exact_turn(s["k"], s["norms"][1], s["positions"], s)}
    if case["op"] == "append":
        p = torch.cat([torch.arange(t - n, t, device="cuda") for n, t in zip(s["new"], s["total"])])
        q, k = _exact_turn(s["q"], s["norms"][0], p, s), _exact_turn(s["k"], s["norms"][1], p, s)
        out = [c.double() for c in s["cache"]]
        at = 0
        for i, (n, t) in enumerate(zip(s["new"], s["total"])):
            where = torch.arange(t - n, t, device="cuda")
            pages, slots = s["table"][i].long()[where // case["page"]], where % case["page"]
            for c, x in zip(out, (k, s["v"].double())):
                (c if case["order"] == "tokens" else c.transpose(1, 2))[pages, slots] = x[at:at + n]
            at += n
        return {"q": q, "keys": out[0], "values": out[1]}
    # Attention head by head: the plain definition over the keys that a query sees, all of a sequence's keys laid out first.
    Hq, Hk, W, sinks = (case[n] for n in ("Hq", "Hk", "window", "sinks"))
    keys, values = (c if case["order"] == "tokens" else c.transpose(1, 2) for c in s["cache"])
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    at = 0
    for i, (n, t) in enumerate(zip(s["new"], s["total"])):
        j = torch.arange(t, device="cuda")
        pages = s["table"][i].long()[j // case["page"]]
        live = pages >= 0
        flat = pages.clamp(min=0) * case["page"] + j % case["page"]
        for q0 in range(0, n, 1024):
            q1 = min(n, q0 + 1024)
            pos = (t - n + torch.arange(q0, q1, device="cuda"))[:, None]
            hidden = (j > pos) | ~live
            if W:
                hidden |= (pos - j >= W) & (j >= sinks)
            use = (~hidden).any(dim=0).nonzero()[:, 0]
            for h in range(Hk):
                k, v = (c[:, :, h].reshape(-1, case["D"])[flat[use]].double() for c in (keys, values))
                for m in range(h * (Hq // Hk), (h + 1) * (Hq // Hk)):
                    a = (s["q"][at + q0:at + q1, m].double() @ k.T) * case["D"] ** -0.5
                    a[hidden[:, use]] = -math.inf
                    out[at + q0:at + q1, m] = torch.softmax(a, dim=1) @ v
        at += n
    return out
