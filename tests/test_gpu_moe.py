"""GPU: embedding lookup, top-k routing, ragged expert products and their
combination against plain 64-bit computations.

Weights are decoded with nxq_dequant, whose values are pinned bit for bit
elsewhere.  Bounds, with u = 2^-11 (half a step of f16, relative):
  product kernels that round weights to f16 form w as one f16 rounding of
  q s + o with f16 s and o, so |dw| <= u(|q s| + |o|) + u|w| <= 2u(|w| + |o|);
  fp32 activations are rounded to f16 too (u|x|); f16 subnormals add at most
  2^-25 per weight; fp32 accumulation adds K 2^-24 sum|w x|.  The exact kernel
  has only the last term.  An output of type t adds eps(t)/2 of its value.
"""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from nxq import synth

pytestmark = pytest.mark.gpu

U = 2.0 ** -11
TYPE_NAMES = {"Q4_0": 2, "Q4_1": 3, "Q8_0": 8, "Q2_K": 10, "Q3_K": 11, "Q4_K": 12, "Q5_K": 13, "Q6_K": 14,
              "I4G32": 101, "I4G64": 102, "I4G128": 104, "I4G256": 108, "NXF_I8": 120, "NXF_F16": 121, "NXF_F32": 122}
# The largest offset |o| of a weight with the distributions of synth.make_blocks.
OFFSET = {2: 8 * 0.02, 3: 1e-3, 10: 15e-3, 12: 63e-3, 13: 63e-3, 101: 75e-3, 102: 75e-3, 104: 75e-3, 108: 75e-3}
EXACT = (121, 122)  # block types only the exact kernel multiplies
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def make_weights(gpu, t, E, N, K, seed):
    """E registered weights and their decoded values [E][N][K] in 64 bits."""
    ws = [gpu.Weight.register(synth.make_blocks(t, N, K, seed=seed + e), t, N, K) for e in range(E)]
    return ws, torch.stack([w.dequant().double() for w in ws])


def make_offsets(counts, first=0):
    return torch.tensor(np.concatenate([[first], first + np.cumsum(counts)]), dtype=torch.int32, device="cuda")


def products(W, t, x, counts, src, first=0):
    """(y, bound) of every slot in 64 bits."""
    R, N = len(src), W.shape[1]
    xs = x[src].double()
    y = torch.zeros((R, N), dtype=torch.float64, device="cuda")
    b = torch.zeros_like(y)
    x_round = U if x.dtype == torch.float32 and t not in EXACT else 0.0
    at = first
    for e, n in enumerate(counts):
        s = slice(at, at + n)
        at += n
        y[s] = xs[s] @ W[e].T
        mag = xs[s].abs() @ W[e].abs().T
        k = W.shape[2]
        b[s] = (k * 2.0 ** -24 + x_round) * mag
        if t not in EXACT:
            b[s] += 2 * U * 1.01 * (mag + OFFSET.get(t, 0.0) * xs[s].abs().sum(1, keepdim=True))
            b[s] += 2.0 ** -24 * xs[s].abs().sum(1, keepdim=True)
    return y, b


def check(got, want, bound):
    half = HALF_STEP[got.dtype]
    err = (got.double() - want).abs()
    tol = bound * (1 + half) + half * want.abs() + 2.0 ** -25
    assert bool((err <= tol).all()), f"max err/tol {(err / tol).max().item():.3g}"


def swiglu(g, bg, u, bu):
    s = g * torch.sigmoid(g)
    # |silu'| <= 1.1; expf and the division add at most 8 half steps of fp32.
    return s * u, 1.1 * bg * (u.abs() + bu) + s.abs() * bu + 2.0 ** -21 * (s * u).abs()


# ---- embedding ------------------------------------------------------------------

@pytest.mark.parametrize("t", TYPE_NAMES.values(), ids=TYPE_NAMES.keys())
@pytest.mark.parametrize("scale", [1.0, 0.37])
def test_embedding_types(gpu, t, scale):
    qk = synth.GEOMETRY[t][0]
    N, K = 301, qk * max(1, 544 // qk)  # rows over three tiles, an odd number of blocks
    w = gpu.Weight.register(synth.make_blocks(t, N, K, seed=t), t, N, K)
    try:
        W = w.dequant()
        ids = torch.from_numpy(synth.rng(3).integers(0, N, size=77)).cuda()
        ids[:4] = torch.tensor([0, N - 1, N - 1, 128])
        for dt in DT.values():
            want = (W[ids] * torch.tensor(scale, dtype=torch.float32, device="cuda")).to(dt)
            for i in (ids, ids.to(torch.int32), ids.view(7, 11)):
                got = gpu.embedding(w, i, scale=scale, out_dtype=dt)
                assert got.shape == (*i.shape, K)
                assert torch.equal(got.view(-1, K), want)
        gpu.stream_sync()
    finally:
        w.release()


def test_embedding_edges(gpu):
    t, N, K = 12, 130, 256
    w = gpu.Weight.register(synth.make_blocks(t, N, K, seed=9), t, N, K)
    try:
        W = w.dequant()
        assert gpu.embedding(w, torch.empty(0, dtype=torch.int64, device="cuda")).shape == (0, K)
        # Ids outside the table: zeros there, an error at the sync, the rest right.
        for bad in (-1, N, 2**40, -2**62):
            ids = torch.tensor([5, bad, 129], device="cuda")
            y = gpu.embedding(w, ids)
            with pytest.raises(gpu.NxqError) as e:
                gpu.stream_sync()
            assert e.value.name == "ERR_INDEX" and "token id" in str(e.value)
            assert torch.equal(y[0], W[5]) and torch.equal(y[2], W[129]) and not y[1].any()
            gpu.stream_sync()  # reported once
        with pytest.raises(gpu.NxqError):
            gpu.embedding(w, torch.arange(8, device="cuda")[::2])  # strided ids
        with pytest.raises(gpu.NxqError):  # unaligned output
            gpu.embedding(w, torch.zeros(1, dtype=torch.int32, device="cuda"),
                          out=torch.empty(K + 1, device="cuda")[1:].view(1, K))
    finally:
        w.release()


def test_embedding_table_beyond_32_bits(gpu):
    # Row offsets past 2^32 bytes in the packed table and past 2^31 elements.
    t, K = 8, 4096
    N = (2 ** 32 // (K // 32 * 34)) + 3000
    blocks = torch.randint(0, 120, (N, K // 32, 34), dtype=torch.uint8, device="cuda")
    blocks[:, :, 1] = 0x20  # scales about 2^-7
    w = gpu.Weight.register_device(blocks, t, N, K)
    try:
        ids = torch.tensor([0, N - 1, N // 2, N - 129], device="cuda")
        b = blocks[ids]
        want = b[:, :, 2:].view(torch.int8).float() * b[:, :, :2].contiguous().view(torch.float16).float()
        assert torch.equal(gpu.embedding(w, ids), want.reshape(4, K))
    finally:
        w.release()


# ---- routing ----------------------------------------------------------------------

def route_plain(logits, k, normalize):
    l = logits.double().cpu().numpy()
    T, E = l.shape
    l = np.where(np.isnan(l), -np.inf, l)
    ids, w = np.full((T, k), -1, np.int32), np.zeros((T, k))
    for t in range(T):
        order = np.argsort(-l[t], kind="stable")[:k]
        order = order[l[t][order] > -np.inf]
        if order.size == 0:
            continue
        m = l[t][order[0]]
        share = (l[t] == np.inf).astype(float) if m == np.inf else np.exp(l[t] - m)
        ids[t, :order.size] = order
        w[t, :order.size] = share[order] / (share[order].sum() if normalize else share.sum())
    flat = ids.reshape(-1)
    taken = np.nonzero(flat >= 0)[0]
    by = taken[np.argsort(flat[taken], kind="stable")]
    rows, slots = np.full(T * k, -1, np.int32), np.full(T * k, -1, np.int32)
    rows[:by.size] = by // k
    slots[by] = np.arange(by.size)
    offsets = np.concatenate([[0], np.cumsum(np.bincount(flat[taken], minlength=E))]).astype(np.int32)
    return ids, w, offsets, rows, slots.reshape(T, k)


def route_check(gpu, logits, k, normalize):
    got = [v.cpu().numpy() for v in gpu.moe_route(logits, k, normalize=normalize)]
    want = route_plain(logits, k, normalize)
    for n, a, b in zip(("ids", "weights", "offsets", "rows", "slots"), got, want):
        if n == "weights":
            # expf and its argument, the sum, the division: each within (|l - m| + 2) half steps
            # of fp32 and E - 1 additions at most.
            assert np.all(np.abs(a - b) <= b * (E_STEPS + logits.shape[1]) * 2.0 ** -24 + 1e-38), n
        else:
            assert np.array_equal(a, b), n


E_STEPS = 256  # covers |l - m| of the values used, doubled for the numerator and the sum


@pytest.mark.parametrize("T", [1, 2, 31, 128, 129, 700, 3001])
@pytest.mark.parametrize("E,k", [(1, 1), (2, 2), (8, 2), (60, 4), (128, 8), (257, 6), (1024, 32), (64, 32)])
def test_route(gpu, T, E, k):
    g = torch.Generator(device="cuda").manual_seed(T * 1000 + E)
    for dt in DT.values():
        logits = (2 * torch.randn((T, E), device="cuda", generator=g)).to(dt)
        logits[torch.rand((T, E), device="cuda", generator=g) < 0.2] = -math.inf
        logits[::3, : E // 2] = 0.5  # ties
        if T > 1:
            logits[1] = -math.inf    # a padded token
        for normalize in (True, False):
            route_check(gpu, logits, k, normalize)


@pytest.mark.parametrize("T", [9, 200])
def test_route_special_values(gpu, T):
    E, k = 40, 5
    logits = torch.zeros((T, E), device="cuda")  # every logit equal: the lowest indices
    logits[0, 7] = math.nan
    logits[1] = math.nan
    logits[2, 3], logits[2, 9] = math.inf, math.inf
    logits[3, ::2] = -0.0
    logits[4] = torch.finfo(torch.float32).min  # finite, so it is taken
    logits[5, 1:] = -math.inf
    logits[6] = torch.linspace(-3e38, 3e38, E, device="cuda")
    logits[7] = torch.linspace(-1e-45, 1e-45, E, device="cuda")
    logits[8, 5], logits[8, 6:] = math.inf, math.nan
    for normalize in (True, False):
        route_check(gpu, logits, k, normalize)


def test_route_no_tokens(gpu):
    ids, w, offsets, rows, slots = gpu.moe_route(torch.empty((0, 16), device="cuda"), 4)
    assert ids.shape == (0, 4) and rows.numel() == 0
    assert offsets.tolist() == [0] * 17


def test_route_many_tokens_repeats(gpu):
    logits = torch.randn((70001, 96), device="cuda").bfloat16()
    first = gpu.moe_route(logits, 3)
    route_check(gpu, logits, 3, True)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, gpu.moe_route(logits, 3)))


# ---- ragged products ----------------------------------------------------------------

COUNTS = [
    [0, 0, 0, 1],              # a single row
    [1, 1, 1, 1],
    [0, 3, 0, 9],
    [17, 0, 1, 40],
    [8, 16, 32, 33],
    [130, 0, 257, 5],
]


def run_ragged(gpu, t, N, K, counts, xdt, ydt, gather, pair, seed=0, first=0, behind=0):
    E, n = len(counts), sum(counts)
    ws, W = make_weights(gpu, t, E, N, K, seed + 10)
    us, Wu = make_weights(gpu, t, E, N, K, seed + 50) if pair else (None, None)
    g = torch.Generator(device="cuda").manual_seed(seed)
    R = first + n + behind
    X = max(1, n // 2) if gather else R
    scale = 0.05 if pair else 1.0  # keeps the gate's sigmoid away from 0 and 1
    x = (scale * torch.randn((X, K), device="cuda", generator=g)).to(xdt)
    rows = torch.randint(0, X, (R,), device="cuda", generator=g, dtype=torch.int32) if gather else None
    src = rows.long() if gather else torch.arange(R, device="cuda")
    off = make_offsets(counts, first)
    out = torch.full((R, N), -7.0, device="cuda", dtype=ydt)
    G = gpu.Experts(ws)
    Up = gpu.Experts(us) if pair else None
    try:
        if pair:
            gpu.qmatmul_ragged_swiglu(G, Up, x, off, rows=rows, out=out)
        else:
            gpu.qmatmul_ragged(G, x, off, rows=rows, out=out)
        gpu.stream_sync()
        y, b = products(W, t, x, counts, src, first)
        if pair:
            y, b = swiglu(y, b, *products(Wu, t, x, counts, src, first))
        s = slice(first, first + n)
        check(out[s], y[s], b[s])
        assert bool((out[:first] == -7).all()) and bool((out[first + n:] == -7).all())
        if n * N >= 64 and not pair:
            rel = ((out[s].double() - y[s]).norm() / y[s].norm()).item()
            assert rel < 1e-3 + 2 * HALF_STEP[ydt], rel
        return out
    finally:
        G.release()
        if pair:
            Up.release()
        for w in ws + (us or []):
            w.release()


@pytest.mark.parametrize("pair", [False, True], ids=["plain", "swiglu"])
@pytest.mark.parametrize("counts", COUNTS, ids=str)
@pytest.mark.parametrize("t", [2, 8, 11, 12], ids=["Q4_0", "Q8_0", "Q3_K", "Q4_K"])
def test_ragged_sizes(gpu, t, counts, pair):
    run_ragged(gpu, t, 200, 768, counts, torch.float16, torch.float32, True, pair, seed=t)


@pytest.mark.parametrize("pair", [False, True], ids=["plain", "swiglu"])
@pytest.mark.parametrize("counts", [[2, 0, 5], [70, 200, 3]], ids=str)
@pytest.mark.parametrize("t", TYPE_NAMES.values(), ids=TYPE_NAMES.keys())
def test_ragged_types(gpu, t, counts, pair):
    K = 512 if synth.GEOMETRY[t][0] == 256 else 256 + synth.GEOMETRY[t][0]  # a chunk that is not full
    run_ragged(gpu, t, 129, K, counts, torch.float16, torch.bfloat16, False, pair, seed=t)


@pytest.mark.parametrize("xdt", DT.keys())
@pytest.mark.parametrize("ydt", DT.keys())
@pytest.mark.parametrize("gather", [False, True], ids=["rows", "gather"])
@pytest.mark.parametrize("counts", [[1, 0, 2], [5, 20, 0], [300, 1, 90]], ids=str)
def test_ragged_dtypes(gpu, xdt, ydt, gather, counts):
    run_ragged(gpu, 12, 256, 512, counts, DT[xdt], DT[ydt], gather, False, seed=3)
    run_ragged(gpu, 12, 256, 512, counts, DT[xdt], DT[ydt], gather, True, seed=4)


@pytest.mark.parametrize("N", [1, 7, 128, 384, 1000])
@pytest.mark.parametrize("counts", [[0, 1], [11, 4], [100, 31], [513, 256]], ids=str)
def test_ragged_rows_left_alone(gpu, N, counts):
    """Odd row counts; slots before the first offset and behind the last keep their values."""
    run_ragged(gpu, 2, N, 96, counts, torch.float16, torch.float32, True, False, seed=N, first=3, behind=70)


@pytest.mark.parametrize("t", [2, 8, 10, 11, 12, 13, 14, 101],
                         ids=["Q4_0", "Q8_0", "Q2_K", "Q3_K", "Q4_K", "Q5_K", "Q6_K", "I4G32"])
def test_ragged_repeats(gpu, t):
    """Many calls in a row, of every ring depth the block types lead to, give the same bits."""
    counts = [20, 3, 31, 16, 9, 40, 1, 24]
    N, K = 1024, 2048
    ws, W = make_weights(gpu, t, len(counts), N, K, 7)
    E = gpu.Experts(ws)
    try:
        src = torch.arange(sum(counts), device="cuda")
        x = torch.randn((len(src), K), device="cuda").half()
        off = make_offsets(counts)
        first = gpu.qmatmul_ragged(E, x, off)
        check(first, *products(W, t, x, counts, src))
        outs = [gpu.qmatmul_ragged(E, x, off) for _ in range(300)]
        gpu.stream_sync()
        assert all(torch.equal(o, first) for o in outs)
    finally:
        E.release()
        for w in ws:
            w.release()


def test_ragged_large_shared_tiles(gpu):
    """More work tiles than SMs and tiles cut between CTAs: right, and the same bits on every call."""
    for counts in ([2, 0, 1, 3], [40, 25, 0, 90], [300, 0, 700, 20]):
        ws, W = make_weights(gpu, 12, 4, 4000, 1280, 70)
        E = gpu.Experts(ws)
        try:
            n = sum(counts)
            x = torch.randn((n, 1280), device="cuda").half()
            off = make_offsets(counts)
            first = gpu.qmatmul_ragged(E, x, off)
            pair = gpu.qmatmul_ragged_swiglu(E, E, x, off)
            y, b = products(W, 12, x, counts, torch.arange(n, device="cuda"))
            check(first, y, b)
            check(pair, *swiglu(y, b, y, b))
            for _ in range(4):
                assert torch.equal(first, gpu.qmatmul_ragged(E, x, off))
                assert torch.equal(pair, gpu.qmatmul_ragged_swiglu(E, E, x, off))
            gpu.stream_sync()
        finally:
            E.release()
            for w in ws:
                w.release()


def test_ragged_many_experts(gpu):
    rng = synth.rng(5)
    for E in (33, 1024):
        ws = [gpu.Weight.register(synth.make_blocks(2, 32, 64, seed=e), 2, 32, 64) for e in range(8)]
        ws = [ws[e % 8] for e in range(E)]  # one weight may serve several experts
        W = torch.stack([w.dequant().double() for w in ws])
        T = gpu.Experts(ws)
        try:
            for total in (1, 40, 3000):
                counts = np.bincount(rng.integers(0, E, size=total), minlength=E).tolist()
                x = torch.randn((total, 64), device="cuda").half()
                out = gpu.qmatmul_ragged(T, x, make_offsets(counts))
                y, b = products(W, 2, x, counts, torch.arange(total, device="cuda"))
                check(out, y, b)
        finally:
            T.release()
            for w in ws[:8]:
                w.release()


def test_ragged_unaligned_activations(gpu):
    ws, W = make_weights(gpu, 12, 2, 128, 256, 5)
    E = gpu.Experts(ws)
    try:
        for counts in ([3, 2], [50, 80]):
            n = sum(counts)
            for dt in DT.values():
                x = torch.randn(n * 256 + 1, device="cuda").to(dt)[1:].view(n, 256)
                out = torch.empty(n * 128 + 1, device="cuda")[1:].view(n, 128)
                gpu.qmatmul_ragged(E, x, make_offsets(counts), out=out)
                y, b = products(W, 12, x, counts, torch.arange(n, device="cuda"))
                check(out, y, b)
    finally:
        E.release()
        for w in ws:
            w.release()


@pytest.mark.parametrize("n", [6, 90])
def test_ragged_bad_indices(gpu, n):
    """Offsets and row indices outside their ranges are skipped and reported; nothing else is touched."""
    ws, W = make_weights(gpu, 12, 4, 128, 256, 5)
    E = gpu.Experts(ws)
    x = torch.randn((n, 256), device="cuda").half()
    h = n // 3

    def call(off, rows=None):
        out = torch.full((n, 128), -7.0, device="cuda")
        gpu.qmatmul_ragged(E, x, torch.tensor(off, dtype=torch.int32, device="cuda"), rows=rows, out=out)
        with pytest.raises(gpu.NxqError) as e:
            gpu.stream_sync()
        assert e.value.name == "ERR_INDEX"
        return out

    try:
        dense = [(x.double() @ W[e].T).float() for e in range(4)]

        def near(a, b):
            return bool(((a - b).norm() <= 2e-3 * b.norm()).item())

        out = call([0, h, h, 2 * h, n + 1])  # the last expert ends behind the rows
        assert near(out[:h], dense[0][:h]) and near(out[h:2 * h], dense[2][h:2 * h]) and bool((out[2 * h:] == -7).all())
        out = call([-1, h, h, 2 * h, n])     # the first starts before them
        assert bool((out[:h] == -7).all()) and near(out[2 * h:], dense[3][2 * h:])
        out = call([0, 2 * h, h, n, n])      # descending: experts 1 and 2 are left out
        assert near(out[:2 * h], dense[0][:2 * h]) and bool((out[2 * h:] == -7).all())
        call([2**31 - 1, -2**31, 2**31 - 1, -2**31, 2**31 - 1])
        rows = torch.arange(n, device="cuda", dtype=torch.int32)
        rows[1], rows[n - 1] = n, -5
        out = call([0, h, h, 2 * h, n], rows)
        assert not out[1].any() and not out[n - 1].any()
        assert near(out[2:h], dense[0][2:h]) if h > 2 else True
        assert near(out[2 * h:n - 1], dense[3][2 * h:n - 1])
    finally:
        E.release()
        for w in ws:
            w.release()


@pytest.mark.parametrize("xdt", DT.keys())
@pytest.mark.parametrize("n", [6, 90])
def test_ragged_bad_last_offset(gpu, n, xdt):
    """A last offset that descends leaves out the last expert only: the others' rows are there, whatever x's type."""
    ws, W = make_weights(gpu, 12, 3, 128, 256, 6)
    E = gpu.Experts(ws)
    x = torch.randn((n, 256), device="cuda").to(DT[xdt])
    h = n // 3
    try:
        out = torch.full((n, 128), -7.0, device="cuda")
        gpu.qmatmul_ragged(E, x, torch.tensor([0, h, 2 * h, 1], dtype=torch.int32, device="cuda"), out=out)
        with pytest.raises(gpu.NxqError) as e:
            gpu.stream_sync()
        assert e.value.name == "ERR_INDEX"
        for i in range(2):
            got, want = out[i * h:(i + 1) * h], (x[i * h:(i + 1) * h].double() @ W[i].T).float()
            assert bool(((got - want).norm() <= 2e-3 * want.norm()).item())
        assert bool((out[2 * h:] == -7).all())
    finally:
        E.release()
        for w in ws:
            w.release()


def test_ragged_infinite_values_stay_in_their_rows(gpu):
    """inf and NaN in a row, or in rows no slot reads, reach no other row."""
    ws, W = make_weights(gpu, 12, 2, 256, 512, 5)
    E = gpu.Experts(ws)
    try:
        for counts in ([3, 4], [60, 150]):
            n = sum(counts)
            x = torch.randn((n + 40, 512), device="cuda").half()
            x[1, 5], x[n - 1, 500] = math.inf, math.nan
            x[n:] = math.nan
            out = gpu.qmatmul_ragged(E, x, make_offsets(counts))[:n]
            y, b = products(W, 12, x[:n].nan_to_num(0, 0, 0), counts, torch.arange(n, device="cuda"))
            keep = torch.ones(n, dtype=torch.bool, device="cuda")
            keep[1] = keep[n - 1] = False
            check(out[keep], y[keep], b[keep])
            assert not torch.isfinite(out[1]).any() and torch.isnan(out[n - 1]).all()
    finally:
        E.release()
        for w in ws:
            w.release()


@pytest.mark.parametrize("n", [2, 200])
def test_ragged_range_error(gpu, n):
    ws, _ = make_weights(gpu, 12, 2, 128, 256, 5)
    E = gpu.Experts(ws)
    try:
        x = torch.zeros((n, 256), device="cuda")
        x[n - 1, 3] = 6.6e4
        gpu.qmatmul_ragged(E, x, make_offsets([1, n - 1]))
        with pytest.raises(gpu.NxqError) as e:
            gpu.stream_sync()
        assert e.value.name == "ERR_RANGE"
        x[n - 1, 3] = 65519.0
        gpu.qmatmul_ragged(E, x, make_offsets([1, n - 1]))
        gpu.stream_sync()
    finally:
        E.release()
        for w in ws:
            w.release()


def test_ragged_lost_arrival_times_out(gpu):
    """A partial sum that is never counted in: the bounded wait of the worker that needs it ends the call
    with an error, and the next call is right."""
    ws, W = make_weights(gpu, 12, 2, 1024, 2048, 5)
    E = gpu.Experts(ws)
    try:
        x = torch.randn((6, 2048), device="cuda").half()
        off = make_offsets([2, 4])
        y, b = products(W, 12, x, [2, 4], torch.arange(6, device="cuda"))
        check(gpu.qmatmul_ragged(E, x, off), y, b)
        gpu.stream_sync()
        gpu.set_wait_limit(2000)
        gpu.test_hook(gpu.HOOK_STREAMK_SKIP_COUNT, True)
        try:
            gpu.qmatmul_ragged(E, x, off)
            with pytest.raises(gpu.NxqError) as e:
                gpu.stream_sync()
            assert e.value.name == "ERR_TIMEOUT"
        finally:
            gpu.test_hook(gpu.HOOK_STREAMK_SKIP_COUNT, False)
            gpu.set_wait_limit(0)
        check(gpu.qmatmul_ragged(E, x, off), y, b)
        gpu.stream_sync()
    finally:
        E.release()
        for w in ws:
            w.release()


def test_ragged_crowded_expert(gpu):
    """Every slot with one expert of many: far from the average that the kernel is chosen by."""
    ws, W = make_weights(gpu, 2, 40, 130, 256, 5)
    E = gpu.Experts(ws)
    try:
        for n in (200, 300, 4000):
            counts = [0] * 40
            counts[17] = n
            x = torch.randn((n, 256), device="cuda").half()
            y, b = products(W, 2, x, counts, torch.arange(n, device="cuda"))
            check(gpu.qmatmul_ragged(E, x, make_offsets(counts)), y, b)
    finally:
        E.release()
        for w in ws:
            w.release()


def test_ragged_no_slots(gpu):
    ws, _ = make_weights(gpu, 12, 2, 128, 256, 5)
    E = gpu.Experts(ws)
    try:
        assert gpu.qmatmul_ragged(E, torch.empty((0, 256), device="cuda"), make_offsets([0, 0])).shape == (0, 128)
        for R in (5, 60):  # room for slots, none of them used
            out = torch.full((R, 128), 3.0, device="cuda")
            gpu.qmatmul_ragged(E, torch.full((R, 256), math.nan, device="cuda"), make_offsets([0, 0]), out=out)
            gpu.qmatmul_ragged_swiglu(E, E, torch.full((R, 256), math.nan, device="cuda"), make_offsets([0, 0], R), out=out)
            gpu.stream_sync()
            assert bool((out == 3).all())
    finally:
        E.release()
        for w in ws:
            w.release()


def test_expert_table_lifetime(gpu):
    ws, _ = make_weights(gpu, 12, 2, 128, 256, 5)
    other = gpu.Weight.register(synth.make_blocks(12, 128, 512, seed=1), 12, 128, 512)
    wrong = gpu.Weight.register(synth.make_blocks(13, 128, 256, seed=1), 13, 128, 256)
    E = gpu.Experts([ws[0], ws[1], ws[0]])
    for bad in (other, wrong):
        with pytest.raises(gpu.NxqError) as e:
            gpu.Experts([ws[0], bad])
        assert e.value.name == "ERR_SHAPE"
    with pytest.raises(gpu.NxqError) as e:
        ws[0].release()
    assert e.value.name == "ERR_STATE"
    with pytest.raises(gpu.NxqError) as e:
        two = gpu.Experts([ws[0], ws[1]])
        try:
            gpu.qmatmul_ragged_swiglu(E, two, torch.zeros((1, 256), device="cuda"), make_offsets([1, 0, 0]))
        finally:
            two.release()
    assert e.value.name == "ERR_SHAPE"
    with pytest.raises(gpu.NxqError):
        gpu.qmatmul_ragged(E, torch.zeros((1, 256), device="cuda"), make_offsets([1, 0]))  # offsets for two experts
    E.release()
    with pytest.raises(gpu.NxqError):
        E.handle
    for w in ws + [other, wrong]:
        w.release()


# ---- combine ------------------------------------------------------------------------

@pytest.mark.parametrize("N", [1, 8, 33, 1000, 1002, 4096])
@pytest.mark.parametrize("T,k", [(1, 1), (3, 8), (130, 3), (17, 32), (601, 32), (2000, 8)])
@pytest.mark.parametrize("hdt", DT.keys())
def test_combine(gpu, N, T, k, hdt):
    g = torch.Generator(device="cuda").manual_seed(N + T)
    R = T * k + 5
    h = torch.randn((R, N), device="cuda", generator=g).to(DT[hdt])
    h[R - 5:] = math.nan  # rows no slot names
    slots = torch.randperm(T * k, device="cuda", generator=g).to(torch.int32).view(T, k)
    w = torch.rand((T, k), device="cuda", generator=g)
    drop = torch.rand((T, k), device="cuda", generator=g) < 0.3
    drop[T // 2] = True  # a token without experts
    slots[drop] = -1
    w[drop] = math.nan   # weights of skipped choices are not used
    res = torch.randn((T, N), device="cuda", generator=g)
    hh = torch.where(drop[:, :, None], 0.0, h[slots.clamp(min=0).long()].double() * w.double()[:, :, None])
    for r in (None, res):
        want = hh.sum(1) + (0 if r is None else r.double())
        bound = (k + 2) * 2.0 ** -24 * (hh.abs().sum(1) + (0 if r is None else r.double().abs()))
        for dt in DT.values():
            check(gpu.moe_combine(h, slots, w, res=r, out_dtype=dt), want, bound)
    y = res.clone()
    assert gpu.moe_combine(h, slots, w, res=y, out=y) is y
    check(y, hh.sum(1) + res.double(), (k + 2) * 2.0 ** -24 * (hh.abs().sum(1) + res.double().abs()))
    gpu.stream_sync()


def test_combine_edges(gpu):
    h = torch.randn((4, 16), device="cuda").half()
    w = torch.ones((3, 2), device="cuda")
    slots = torch.tensor([[0, 4], [1, 2], [2**31 - 1, 3]], dtype=torch.int32, device="cuda")
    y = gpu.moe_combine(h, slots, w)
    with pytest.raises(gpu.NxqError) as e:
        gpu.stream_sync()
    assert e.value.name == "ERR_INDEX" and "slot" in str(e.value)
    assert torch.equal(y[0], h[0].float()) and torch.equal(y[2], h[3].float())
    assert gpu.moe_combine(h, torch.empty((0, 2), dtype=torch.int32, device="cuda"), torch.empty((0, 2), device="cuda")).shape == (0, 16)
    # No experts' outputs at all: the residual.
    none = torch.full((2, 2), -1, dtype=torch.int32, device="cuda")
    res = torch.randn((2, 16), device="cuda")
    assert torch.equal(gpu.moe_combine(h[:0], none, w[:2], res=res), res)


# ---- together -------------------------------------------------------------------------

class Layer:
    """A mixture-of-experts block behind an embedding, as a decode or prefill step uses it."""

    V, D, F, E, k = 500, 512, 384, 12, 3

    def __init__(self, gpu, t=12):
        self.gpu, self.t = gpu, t
        self.table = gpu.Weight.register(synth.make_blocks(14, self.V, self.D, seed=1), 14, self.V, self.D)
        self.router = gpu.Weight.register(synth.make_blocks(8, self.E, self.D, seed=2), 8, self.E, self.D)
        self.gw, self.Wg = make_weights(gpu, t, self.E, self.F, self.D, 100)
        self.uw, self.Wu = make_weights(gpu, t, self.E, self.F, self.D, 200)
        self.dw, self.Wd = make_weights(gpu, 2, self.E, self.D, 384, 300)
        self.gate, self.up, self.down = gpu.Experts(self.gw), gpu.Experts(self.uw), gpu.Experts(self.dw)

    def step(self, ids):
        g = self.gpu
        x = g.embedding(self.table, ids, scale=0.02)
        logits = g.qmatmul(self.router, x)
        choice, w, off, rows, slots = g.moe_route(logits, self.k)
        h = g.qmatmul_ragged_swiglu(self.gate, self.up, x, off, rows=rows, out_dtype=torch.float16)
        o = g.qmatmul_ragged(self.down, h, off, out_dtype=torch.float32)
        return g.moe_combine(o, slots, w, res=x), choice, w

    def plain(self, ids, choice, w):
        x = (self.table.dequant()[ids].double() * 0.02)
        y = x.clone()
        for j in range(self.k):
            e = choice[:, j].long()
            gt, u = torch.einsum("tk,tnk->tn", x, self.Wg[e]), torch.einsum("tk,tnk->tn", x, self.Wu[e])
            y += w[:, j, None].double() * torch.einsum("tn,tkn->tk", gt * torch.sigmoid(gt) * u, self.Wd[e])
        return y

    def release(self):
        for e in (self.gate, self.up, self.down):
            e.release()
        for w in [self.table, self.router, *self.gw, *self.uw, *self.dw]:
            w.release()


@pytest.fixture(scope="module")
def layer(gpu):
    l = Layer(gpu)
    yield l
    l.release()


# The block rounds x, h and three sets of weights to f16 (rel. u each, adding at
# most linearly through the products): 8 u.
BLOCK_TOL = 8 * U


@pytest.mark.parametrize("T", [1, 3, 50, 400])
def test_block(gpu, layer, T):
    ids = torch.randint(0, layer.V, (T,), device="cuda")
    y, choice, w = layer.step(ids)
    gpu.stream_sync()
    want = layer.plain(ids, choice, w)
    assert ((y.double() - want).norm() / want.norm()).item() < BLOCK_TOL


@pytest.mark.parametrize("T", [2, 150])
def test_block_captured(gpu, layer, T):
    """Two captured graphs and eager calls, replayed on two streams at once: every one has its own workspaces."""
    graphs = []
    for i in range(2):
        ids = torch.randint(0, layer.V, (T,), device="cuda")
        warm = torch.cuda.Stream()  # the router's product keeps its scratch by stream
        torch.cuda.synchronize()
        with torch.cuda.stream(warm):
            for _ in range(2):
                layer.step(ids)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=warm):
            y, choice, w = layer.step(ids)
        graphs.append((graph, ids, y, choice, w))
    streams = [torch.cuda.Stream() for _ in range(3)]
    for turn in range(4):
        for _, ids, *_ in graphs:
            ids.copy_(torch.randint(0, layer.V, (T,), device="cuda"))
        eager_ids = torch.randint(0, layer.V, (T,), device="cuda")
        torch.cuda.synchronize()
        for (graph, *_), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                for _ in range(3):
                    graph.replay()
        with torch.cuda.stream(streams[2]):
            eager = [layer.step(eager_ids) for _ in range(3)][-1]
        torch.cuda.synchronize()
        for ids, (y, choice, w) in [(eager_ids, eager)] + [(g[1], g[2:]) for g in graphs]:
            want = layer.plain(ids, choice, w)
            assert ((y.double() - want).norm() / want.norm()).item() < BLOCK_TOL
    gpu.stream_sync()


def test_block_on_threads(gpu, layer):
    """Calls from several host threads, each on its own stream."""
    import threading

    bad = []

    def work(i):
        try:
            s = torch.cuda.Stream()
            with torch.cuda.stream(s):
                for n in range(6):
                    ids = torch.randint(0, layer.V, (1 + 37 * n,), device="cuda")
                    y, choice, w = layer.step(ids)
                    want = layer.plain(ids, choice, w)
                    if not ((y.double() - want).norm() / want.norm()).item() < BLOCK_TOL:
                        bad.append((i, n))
        except Exception as e:  # noqa: BLE001
            bad.append((i, repr(e)))

    ts = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    [t.start() for t in ts]
    [t.join() for t in ts]
    assert not bad, bad
