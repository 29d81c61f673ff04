"""Cases of the mixture-of-experts and embedding operators over block-quantized weights:

  route      top-k softmax routing of logits [T][E], and the order of the choices by expert
  ragged     products grouped by expert with ragged sizes, y[s] = x[rows[s]] W_e^T
  swiglu     the same with a gate and an up projection, h = silu(x Wg^T) * (x Wu^T)
  combine    weighted sum of the experts' outputs per token, plus the residual
  embedding  scaled lookup of rows of a quantized table

`run` computes them in plain torch operations, or (own = True) through the
framework's entry points.  Weights are GGUF blocks of random codes whose scales
make the decoded weights about N(0, 0.02), as trained projections are;
activations are N(0, 1), as after a norm; routing logits carry a bias per
expert, so some experts get several times the rows of others.
"""
import math
import sys

import torch

own = False

# Elements per block and bytes per block of the GGUF types used here.
GEOMETRY = {"Q4_0": (32, 18), "Q8_0": (32, 34), "Q3_K": (256, 110), "Q4_K": (256, 144), "Q6_K": (256, 210)}
TYPE_IDS = {"Q4_0": 2, "Q8_0": 8, "Q3_K": 11, "Q4_K": 12, "Q6_K": 14}
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _nxq():
    """The framework's binding, initialised on the first GPU."""
    if "nexus-inference-engine-_b200" not in sys.path:
        sys.path.insert(0, "nexus-inference-engine-_b200")
    import nxq

    nxq.init(0)
    return nxq


# ---- cases -------------------------------------------------------------------

def listed():
    return [
        # One decode step's token embedding: a row of a 64k-entry table.
        {"name": "embedding-1-q6k", "op": "embedding", "type": "Q6_K", "V": 65536, "K": 4096, "T": 1, "y": "bf16"},
        # The embedding of a long prompt batch, scaled by sqrt(K).
        {"name": "embedding-8192-q4k", "op": "embedding", "type": "Q4_K", "V": 65536, "K": 4096, "T": 8192, "y": "f32"},
        # Routing of one decode step with one sequence.
        {"name": "route-1-e128", "op": "route", "T": 1, "E": 128, "k": 8, "x": "f32", "norm": True, "masked": 0.0},
        # Routing of a prefill batch; a few padded tokens have every expert masked.
        {"name": "route-16384-e256", "op": "route", "T": 16384, "E": 256, "k": 8, "x": "bf16", "norm": True, "masked": 0.02},
        # Down projection of a decode step with three sequences, 24 ragged slots.
        {"name": "ragged-24-q6k", "op": "ragged", "type": "Q6_K", "E": 128, "N": 2048, "K": 768, "T": 3, "k": 8, "x": "f16", "y": "bf16", "gather": False},
        # A batched decode step: 256 sequences over 64 experts, 16 rows each on average; Llama-3-8B's hidden size.
        {"name": "ragged-1024-q4k", "op": "ragged", "type": "Q4_K", "E": 64, "N": 4096, "K": 2048, "T": 256, "k": 4, "x": "bf16", "y": "bf16", "gather": False},
        # Down projection of a prefill batch.
        {"name": "ragged-32768-q4k", "op": "ragged", "type": "Q4_K", "E": 64, "N": 4096, "K": 2048, "T": 8192, "k": 4, "x": "f16", "y": "bf16", "gather": False},
        # Gate and up of one decode step with one sequence: eight experts, one row each.
        {"name": "swiglu-8-q4k", "op": "swiglu", "type": "Q4_K", "E": 128, "N": 768, "K": 2048, "T": 1, "k": 8, "x": "f16", "y": "bf16", "gather": True},
        # Few large experts (Llama-3-8B's MLP shape), a ragged batch of 37 sequences.
        {"name": "swiglu-74-q4_0", "op": "swiglu", "type": "Q4_0", "E": 8, "N": 14336, "K": 4096, "T": 37, "k": 2, "x": "f16", "y": "bf16", "gather": True},
        # Gate and up of a prefill batch.
        {"name": "swiglu-32768-q4k", "op": "swiglu", "type": "Q4_K", "E": 64, "N": 2048, "K": 4096, "T": 8192, "k": 4, "x": "bf16", "y": "bf16", "gather": True},
        # The experts' outputs of one decode step into the residual stream.
        {"name": "combine-1", "op": "combine", "N": 4096, "T": 1, "k": 8, "x": "bf16", "y": "f32", "masked": 0.0},
        # The same for a prefill batch with padded tokens.
        {"name": "combine-8192", "op": "combine", "N": 4096, "T": 8192, "k": 8, "x": "bf16", "y": "f32", "masked": 0.02},
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["embedding", "route", "ragged", "ragged", "swiglu", "swiglu", "combine"])
    types = ["Q4_0", "Q8_0", "Q3_K", "Q4_K", "Q6_K"]
    if op == "embedding":
        t = rng.choice(types)
        return {"op": op, "type": t, "V": _log(rng, 1000, 65536), "K": GEOMETRY[t][0] * _log(rng, 1, 4096 // GEOMETRY[t][0]),
                "T": _log(rng, 1, 8192), "y": rng.choice(["f32", "f16", "bf16"])}
    if op == "route":
        E = _log(rng, 2, 256)
        return {"op": op, "T": _log(rng, 1, 16384), "E": E, "k": rng.randint(1, min(8, E)), "x": rng.choice(["f32", "f16", "bf16"]),
                "norm": rng.random() < 0.5, "masked": rng.choice([0.0, 0.1])}
    if op == "combine":
        return {"op": op, "N": _log(rng, 1, 4096), "T": _log(rng, 1, 8192), "k": rng.randint(1, 8), "x": rng.choice(["f16", "bf16"]),
                "y": rng.choice(["f32", "bf16"]), "masked": rng.choice([0.0, 0.1])}
    t = rng.choice(types)
    qk = GEOMETRY[t][0]
    E = _log(rng, 2, 128)
    N, K = _log(rng, 64, 4096), qk * _log(rng, max(1, 256 // qk), 4096 // qk)
    N = max(64, min(N, 64 * 4096 * 2048 // (E * K)))  # the experts' weights stay within the largest listed case's
    k = rng.randint(1, min(8, E))
    most = max(1, min(8192, 32768 * 4096 * 2048 // (k * N * K)))
    return {"op": op, "type": t, "E": E, "N": N, "K": K, "T": _log(rng, 1, most), "k": k, "x": rng.choice(["f16", "bf16"]),
            "y": "bf16", "gather": op == "swiglu" or rng.random() < 0.5}


# ---- inputs -------------------------------------------------------------------

def _blocks(g, type_, n, K):
    """n rows of K / QK GGUF blocks [n][K/QK][bytes] on the GPU: uniform codes, fp16 scale fields that
    make the decoded weights about N(0, 0.02)."""
    qk, bb = GEOMETRY[type_]
    nb = n * (K // qk)
    b = torch.randint(0, 256, (nb, bb), dtype=torch.uint8, device="cuda", generator=g)

    def half(off, v):
        b[:, off:off + 2] = v.to(torch.float16).view(torch.uint8).view(nb, 2)

    d = torch.empty((nb, 1), dtype=torch.float32, device="cuda").uniform_(0.7, 1.3, generator=g)
    if type_ == "Q4_0":
        half(0, d * 4.3e-3)
    elif type_ == "Q8_0":
        half(0, d * 2.7e-4)
    elif type_ == "Q3_K":
        half(108, d * 4.7e-4)
    elif type_ == "Q4_K":  # the min term takes the mean of the codes off, as a fitted block's does
        half(0, d * 8e-5)
        half(2, d * 6e-4)
    else:
        half(208, d * 1.4e-5)
    return b.view(n, K // qk, bb)


def _choices(case, g):
    """The experts of T tokens: k distinct ones each, by logits with a bias per expert."""
    E = case["E"]
    bias = 0.35 * torch.randn(E, device="cuda", generator=g)
    logits = torch.randn((case["T"], E), device="cuda", generator=g) + bias
    return torch.sort(logits, dim=1, descending=True, stable=True)[1][:, :case["k"]]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op, s = case["op"], {"case": case}
    if op == "embedding":
        s["table"] = _blocks(g, case["type"], case["V"], case["K"])
        s["ids"] = torch.randint(0, case["V"], (case["T"],), device="cuda", generator=g)
        s["scale"] = math.sqrt(case["K"])
        if own:
            s["nxq"] = _nxq()
            s["weight"] = s["nxq"].Weight.register_device(s["table"], case["type"], case["V"], case["K"])
    elif op == "route":
        T, E = case["T"], case["E"]
        l = 1.5 * torch.randn((T, E), device="cuda", generator=g) + 0.35 * torch.randn(E, device="cuda", generator=g)
        l[torch.rand(T, device="cuda", generator=g) < case["masked"]] = -math.inf
        s["logits"] = l.to(DTYPES[case["x"]])
        if own:
            s["nxq"] = _nxq()
    elif op == "combine":
        T, k, N = case["T"], case["k"], case["N"]
        s["h"] = torch.randn((T * k, N), device="cuda", generator=g).to(DTYPES[case["x"]])
        slots = torch.randperm(T * k, device="cuda", generator=g).to(torch.int32).view(T, k)
        w = torch.softmax(1.5 * torch.randn((T, k), device="cuda", generator=g), dim=1)
        out = torch.rand(T, device="cuda", generator=g) < case["masked"]
        s["slots"] = torch.where(out[:, None], torch.full_like(slots, -1), slots)
        s["w"] = torch.where(out[:, None], torch.zeros_like(w), w)
        s["res"] = torch.randn((T, N), device="cuda", generator=g)
        if own:
            s["nxq"] = _nxq()
    else:
        E, N, K, T, k = (case[n] for n in ("E", "N", "K", "T", "k"))
        flat = _choices(case, g).reshape(-1)
        order = torch.sort(flat, stable=True)[1]
        counts = torch.bincount(flat, minlength=E)
        s["offsets"] = torch.cat([counts.new_zeros(1), counts.cumsum(0)]).to(torch.int32)
        s["most"] = int(counts.max())  # the largest expert's rows
        s["rows"] = (order // k).to(torch.int32) if case["gather"] else None
        s["x"] = torch.randn((T if case["gather"] else T * k, K), device="cuda", generator=g).to(DTYPES[case["x"]])
        s["blocks"] = [_blocks(g, case["type"], E * N, K).view(E, N, K // GEOMETRY[case["type"]][0], -1)
                       for _ in range(2 if op == "swiglu" else 1)]
        if own:
            n = s["nxq"] = _nxq()
            s["experts"] = [n.Experts([n.Weight.register_device(b[e], case["type"], N, K) for e in range(E)]) for b in s["blocks"]]
    if own:  # a program that ends with its weights gives them back
        s["keep"] = _Keep(s.get("experts"), s.get("weight"))
    return s


class _Keep:
    """Releases a state's registered weights with the state."""

    def __init__(self, experts, weight):
        self.experts, self.weight = experts, weight

    def __del__(self):
        try:
            for e in self.experts or []:
                ws = e.weights
                e.release()
                [w.release() for w in ws]
            if self.weight is not None:
                self.weight.release()
        except Exception:
            pass


# ---- one pass -----------------------------------------------------------------

def _half(b, off):
    return b[..., off:off + 2].contiguous().view(torch.float16).float()


def decode(type_, b):
    """GGUF blocks [..., blocks, bytes] as float32 values [..., blocks * QK]."""
    lead = b.shape[:-2]
    if type_ == "Q4_0":
        q = b[..., 2:]
        w = (torch.cat([q & 15, q >> 4], dim=-1).float() - 8) * _half(b, 0)
    elif type_ == "Q8_0":
        w = b[..., 2:].view(torch.int8).float() * _half(b, 0)
    elif type_ == "Q4_K":
        s, e = b[..., 4:12], b[..., 12:16]
        sc = (s & 63).float()
        mn = ((s >> 6) | (torch.cat([e & 15, e >> 4], dim=-1) << 2)).float()
        q = b[..., 16:]
        q = torch.stack([q & 15, q >> 4], dim=-1).view(*b.shape[:-1], 8, 32).float()
        w = q * (sc * _half(b, 0))[..., None] - (mn * _half(b, 2))[..., None]
    elif type_ == "Q3_K":
        shift2 = torch.arange(0, 8, 2, dtype=torch.uint8, device=b.device)
        shift1 = torch.arange(8, dtype=torch.uint8, device=b.device)
        hi = ((b[..., 0:32, None] >> shift1) & 1).flatten(-2)
        lo = ((b[..., 32:96, None] >> shift2) & 3).flatten(-2)
        s, e = b[..., 96:104], b[..., 104:108]
        pair = torch.stack([e & 15, e >> 4], dim=-1).flatten(-2)  # one nibble for scales i and i + 8
        sc = torch.cat([(s & 15) | ((pair & 3) << 4), (s >> 4) | ((pair >> 2) << 4)], dim=-1).float() - 32
        q = ((lo | (hi << 2)).float() - 4).view(*b.shape[:-1], 16, 16)
        w = q * (sc * _half(b, 108))[..., None]
    else:  # Q6_K
        lo = torch.stack([b[..., 0:128] & 15, b[..., 0:128] >> 4], dim=-1).flatten(-2)
        shift2 = torch.arange(0, 8, 2, dtype=torch.uint8, device=b.device)
        hi = ((b[..., 128:192, None] >> shift2) & 3).flatten(-2)
        q = ((lo | (hi << 4)).float() - 32).view(*b.shape[:-1], 16, 16)
        sc = b[..., 192:208].view(torch.int8).float()
        w = q * (sc * _half(b, 208))[..., None]
    return w.reshape(*lead, -1)


def _products(s, weights):
    """x[rows[slot]] W_e^T of every slot for each of the quantized `weights`, in float32."""
    case, off = s["case"], s["offsets"].long()
    R = case["T"] * case["k"]
    slot = torch.arange(R, device="cuda")
    e = torch.searchsorted(off[1:], slot, right=True)
    x = (s["x"] if s["rows"] is None else s["x"][s["rows"].long()]).float()
    if R <= case["E"]:  # few rows: only the experts that have any are decoded
        return [(decode(case["type"], b[e]) @ x[:, :, None])[:, :, 0] for b in weights]
    padded = x.new_zeros((case["E"], s["most"], case["K"]))
    padded[e, slot - off[e]] = x
    return [(padded @ decode(case["type"], b).transpose(1, 2))[e, slot - off[e]] for b in weights]


def run(s):
    case, op = s["case"], s["case"]["op"]
    y_type = DTYPES[case.get("y", "f32")]
    if op == "embedding":
        if own:
            return s["nxq"].embedding(s["weight"], s["ids"], scale=s["scale"], out_dtype=y_type)
        return (decode(case["type"], s["table"][s["ids"]]) * s["scale"]).to(y_type)
    if op == "route":
        if own:
            ids, w, offsets, rows, slots = s["nxq"].moe_route(s["logits"], case["k"], normalize=case["norm"])
            return {"ids": ids, "weights": w, "offsets": offsets, "rows": rows, "slots": slots}
        return _route(s["logits"].float(), case["k"], case["norm"])
    if op == "combine":
        if own:
            return s["nxq"].moe_combine(s["h"], s["slots"], s["w"], res=s["res"], out_dtype=y_type)
        h = s["h"][s["slots"].long().clamp(min=0)].float()
        w = torch.where(s["slots"] >= 0, s["w"], torch.zeros_like(s["w"]))
        return ((h * w[:, :, None]).sum(dim=1) + s["res"]).to(y_type)
    if op == "ragged":
        if own:
            return s["nxq"].qmatmul_ragged(s["experts"][0], s["x"], s["offsets"], rows=s["rows"], out_dtype=y_type)
        return _products(s, s["blocks"])[0].to(y_type)
    if own:
        return s["nxq"].qmatmul_ragged_swiglu(s["experts"][0], s["experts"][1], s["x"], s["offsets"], rows=s["rows"], out_dtype=y_type)
    gate, up = _products(s, s["blocks"])
    return (gate / (1 + torch.exp(-gate)) * up).to(y_type)


def _route(l, k, norm):
    T, E = l.shape
    top, ids = torch.sort(l, dim=1, descending=True, stable=True)
    top, ids = top[:, :k], ids[:, :k]
    ok = top > -math.inf
    m = top[:, :1].clamp(min=-3e38)
    p = torch.exp(top - m)
    z = p.sum(1, keepdim=True) if norm else torch.exp(l - m).sum(1, keepdim=True)
    w = torch.where(ok, p / z, torch.zeros_like(p))
    flat = torch.where(ok, ids, torch.full_like(ids, E)).reshape(-1)
    order = torch.sort(flat, stable=True)[1]
    counts = (flat[:, None] == torch.arange(E, device=l.device)).sum(0)
    offsets = torch.cat([counts.new_zeros(1), counts.cumsum(0)])
    place = torch.arange(T * k, device=l.device)
    slots = torch.empty_like(order)
    slots[order] = place
    minus = torch.full_like(place, -1)
    rows = torch.where(place < offsets[E], order // k, minus)
    slots = torch.where(flat < E, slots, minus).view(T, k)
    out = {"ids": torch.where(ok, ids, torch.full_like(ids, -1)), "offsets": offsets, "rows": rows, "slots": slots}
    return {**{n: v.to(torch.int32) for n, v in out.items()}, "weights": w}


# ---- work and exact values ------------------------------------------------------

def _row_bytes(case):
    qk, bb = GEOMETRY[case["type"]]
    return case["K"] // qk * bb


def work(case):
    size = {"f32": 4, "f16": 2, "bf16": 2}
    op, T = case["op"], case["T"]
    if op == "embedding":
        return {"bytes": T * (8 + _row_bytes(case) + case["K"] * size[case["y"]]), "flops": T * case["K"]}
    if op == "route":
        return {"bytes": T * case["E"] * size[case["x"]] + T * case["k"] * 16 + 4 * (case["E"] + 1), "flops": 3 * T * case["E"]}
    k, N = case["k"], case["N"]
    if op == "combine":
        return {"bytes": T * k * (8 + N * size[case["x"]]) + T * N * (4 + size[case["y"]]), "flops": 2 * T * k * N}
    mats = 2 if op == "swiglu" else 1
    # Experts with a row: all of them when the rows are many, an expected share of them when few.
    active = case["E"] * (1 - (1 - k / case["E"]) ** T)
    x_rows = T if case["gather"] else T * k
    return {"bytes": mats * active * N * _row_bytes(case) + x_rows * case["K"] * size[case["x"]] + T * k * N * size[case["y"]]
            + 4 * (case["E"] + 1) + (4 * T * k if case["gather"] else 0),
            "flops": 2 * mats * T * k * N * case["K"]}


def _decode64(type_, rows):
    """Blocks [n][blocks][bytes] in float64, element by element from the definition: code index, scale index
    and shift of each element of a block are written out as index tables."""
    qk, _ = GEOMETRY[type_]
    i = torch.arange(qk, device=rows.device)
    b = rows.to(torch.int32)

    def f16(off):
        u = (b[..., off] | (b[..., off + 1] << 8)).to(torch.int64)
        sign, ex, man = 1 - 2 * (u >> 15), (u >> 10) & 31, u & 1023
        v = torch.where(ex == 0, man.double() * 2.0 ** -24, (1024 + man).double() * torch.pow(2.0, (ex - 25).double()))
        return (sign.double() * v)[..., None]

    def signed(v):
        return torch.where(v > 127, v - 256, v).double()

    if type_ == "Q4_0":  # element i < 16: low nibble of byte i; else the high nibble of byte i - 16
        q = (b[..., 2 + i % 16] >> (4 * (i // 16))) & 15
        return ((q.double() - 8) * f16(0)).flatten(-2)
    if type_ == "Q8_0":
        return (signed(b[..., 2 + i]) * f16(0)).flatten(-2)
    if type_ == "Q4_K":  # sub-block j = i / 32; its 6-bit scale and min
        j = i // 32
        q = (b[..., 16 + i // 2] >> (4 * (i % 2))) & 15
        sc = b[..., 4 + j] & 63
        mn = (b[..., 4 + j] >> 6) | (((b[..., 12 + j % 4] >> (4 * (j // 4))) & 15) << 2)
        return (f16(0) * (sc * q).double() - f16(2) * mn.double()).flatten(-2)
    if type_ == "Q3_K":  # group j = i / 16; low nibbles in bytes 96.., two high bits in bytes 104..
        j = i // 16
        q = ((b[..., 32 + i // 4] >> (2 * (i % 4))) & 3) + 4 * ((b[..., i // 8] >> (i % 8)) & 1) - 4
        low = (b[..., 96 + j % 8] >> (4 * (j // 8))) & 15
        high = (b[..., 104 + (j % 8) // 2] >> (4 * (j % 2) + 2 * (j // 8))) & 3
        return (f16(108) * ((low + 16 * high - 32) * q).double()).flatten(-2)
    q = ((b[..., i // 2] >> (4 * (i % 2))) & 15) + 16 * ((b[..., 128 + i // 4] >> (2 * (i % 4))) & 3) - 32
    return (f16(208) * signed(b[..., 192 + i // 16]) * q.double()).flatten(-2)


def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    op = case["op"]
    if op == "embedding":
        return _decode64(case["type"], s["table"].index_select(0, s["ids"])) * math.sqrt(case["K"])
    if op == "route":
        l = s["logits"].double()
        w = torch.zeros((case["T"], case["k"]), dtype=torch.float64, device="cuda")
        rest, total = l.clone(), torch.zeros(case["T"], dtype=torch.float64, device="cuda")
        peak = l.max(dim=1)[0]
        peak = torch.where(torch.isinf(peak), torch.zeros_like(peak), peak)
        for j in range(case["k"]):
            w[:, j] = torch.exp(rest.max(dim=1)[0] - peak)
            rest.scatter_(1, rest.argmax(dim=1, keepdim=True), -math.inf)
        total = w.sum(1) if case["norm"] else torch.exp(l - peak[:, None]).sum(1)
        w = torch.where(total[:, None] > 0, w / total[:, None], w)
        return {"ids": None, "weights": w, "offsets": None, "rows": None, "slots": None}
    if op == "combine":
        y = s["res"].double()
        for j in range(case["k"]):
            at = s["slots"][:, j].long()
            have = at >= 0
            y[have] += s["w"][have, j].double()[:, None] * s["h"][at[have]].double()
        return y
    y = [torch.zeros((case["T"] * case["k"], case["N"]), dtype=torch.float64, device="cuda") for _ in s["blocks"]]
    edges = s["offsets"].tolist()
    for e, (a, z) in enumerate(zip(edges, edges[1:])):
        if a < z:
            x = (s["x"][a:z] if s["rows"] is None else s["x"].index_select(0, s["rows"][a:z])).double()
            for out, b in zip(y, s["blocks"]):
                out[a:z] = x @ _decode64(case["type"], b[e]).T
    return y[0] if op == "ragged" else y[0] * torch.sigmoid(y[0]) * y[1]
