"""GPU: norm and position rotation of heads, and their append to a paged cache, against
the plain formulas in 64 bits.

Bounds: a norm's factor is off by (D + 8) 2^-24 of itself (a sum of D squares, a root
and a division); a sine or cosine by 2^-21 (the angle's fraction, 2^-32 of a turn and its
rounding, and the functions' last places), of the pair's magnitude; products and sums 4 2^-24 of it;
one rounding of the output.
"""
from __future__ import annotations

import math
import random

import numpy as np
import pytest
import torch

from attention_cases import DT, HALF_STEP, Paged

pytestmark = pytest.mark.gpu


def turned(x, norm, eps, rope, inv, positions):
    """(y, bound) of x [T][H][D] in 64 bits."""
    x = x.double()
    D = x.shape[-1]
    if norm is not None:
        x = x / ((x * x).mean(-1, keepdim=True) + eps).sqrt() * norm.double()
    b = x.abs() * (D + 8) * 2.0 ** -24 if norm is not None else torch.zeros_like(x)
    if rope is None:
        return x, b
    n, dims = rope.dims // 2, rope.dims
    i = torch.arange(n, device=x.device)
    lo, hi = (i, i + n) if rope.layout == "half" else (2 * i, 2 * i + 1)
    pos = np.array(positions.tolist(), dtype=np.longdouble)
    a = np.asarray(inv, dtype=np.longdouble)[None, :] * pos[:, None]
    two_pi = np.longdouble("6.283185307179586476925286766559")
    a = a - np.rint(a / two_pi) * two_pi
    a = torch.from_numpy(a.astype(np.float64)).to(x.device)[:, None]
    c, s = torch.cos(a), torch.sin(a)
    y, bb = x.clone(), b.clone()
    u, v = x[..., lo], x[..., hi]
    m = abs(rope.scale)
    y[..., lo], y[..., hi] = rope.scale * (u * c - v * s), rope.scale * (u * s + v * c)
    both = m * ((u.abs() + v.abs()) * (2.0 ** -21 + 4 * 2.0 ** -24) + b[..., lo] + b[..., hi])
    bb[..., lo], bb[..., hi] = both, both
    return y, bb


def check(got, want, bound):
    half = HALF_STEP[got.dtype]
    tol = bound * (1 + half) + half * want.abs() + 2.0 ** -25
    err = (got.double() - want).abs()
    assert bool((err <= tol).all()), f"max err/tol {(err / tol).max().item():.3g}"


def make_rope(gpu, dims, layout, scaling="plain"):
    kw = {"plain": {}, "yarn": dict(factor=8.0, trained=4096.0), "blend": dict(factor=8.0, trained=8192.0),
          "linear": dict(factor=4.0), "ntk": dict(factor=4.0)}[scaling]
    inv, scale = gpu.rope_frequencies(dims, 10000.0, scaling, **kw)
    return gpu.Rope(inv, layout, scale), inv


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("D,dims", [(64, 64), (128, 128), (128, 64), (128, 96), (80, 80), (80, 32), (72, 16), (256, 64), (512, 512),
                                    (96, 40), (2, 2), (7, 4), (33, 32), (200, 100)])
@pytest.mark.parametrize("norm", [False, True])
def test_shapes(gpu, D, dims, layout, norm):
    g = torch.Generator(device="cuda").manual_seed(D + dims)
    r, inv = make_rope(gpu, dims, layout, "yarn")
    w = 1 + 0.2 * torch.randn(D, device="cuda", generator=g) if norm else None
    for T, Hq, Hk in ((1, 3, 1), (5, 8, 2), (650, 5, 3)):
        q = torch.randn((T, Hq, D), device="cuda", generator=g)
        k = torch.randn((T, Hk, D), device="cuda", generator=g)
        pos = torch.randint(0, 100000, (T,), device="cuda", generator=g)
        for x in (torch.float32, torch.bfloat16):
            qo, ko = gpu.rope(r, pos, q.to(x), k.to(x), q_norm=w, k_norm=w, eps=1e-5, out_dtype=torch.float32)
            check(qo, *turned(q.to(x), w, 1e-5, r, inv, pos))
            check(ko, *turned(k.to(x), w, 1e-5, r, inv, pos))
    gpu.stream_sync()
    r.release()


@pytest.mark.parametrize("x", DT.keys())
@pytest.mark.parametrize("y", DT.keys())
@pytest.mark.parametrize("scaling", ["plain", "linear", "ntk", "blend"])
def test_types(gpu, x, y, scaling):
    g = torch.Generator(device="cuda").manual_seed(3)
    r, inv = make_rope(gpu, 64, "half", scaling)
    q = torch.randn((77, 6, 128), device="cuda", generator=g).to(DT[x])
    w = 1 + 0.2 * torch.randn(128, device="cuda", generator=g)
    pos = torch.randint(0, 10**6, (77,), device="cuda", generator=g)
    for p in (pos, pos.to(torch.int32)):
        check(gpu.rope(r, p, q, q_norm=w, out_dtype=DT[y]), *turned(q, w, 1e-6, r, inv, pos))
    # Norms without a rotation, a rotation without norms, and neither (a conversion).
    check(gpu.rope(None, None, q, q_norm=w, out_dtype=DT[y]), *turned(q, w, 1e-6, None, inv, pos))
    check(gpu.rope(r, pos, q, out_dtype=DT[y]), *turned(q, None, 0, r, inv, pos))
    assert torch.equal(gpu.rope(None, None, q, out_dtype=DT[y]), q.to(DT[y]))
    r.release()


def test_far_positions(gpu):
    r, inv = make_rope(gpu, 128, "half")
    pos = torch.tensor([0, 1, 2**20, 2**31 - 1, 2**31, 2**40, -1, -2**31], device="cuda")
    q = torch.randn((8, 2, 128), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    # (The expected angles, in extended precision, are good to 2^-24 up to positions of 2^40.)
    check(gpu.rope(r, pos, q), *turned(q, None, 0, r, inv, pos))
    # A position and the same plus whole turns of a pair are one angle: frequency 2 pi / 1024.
    t = gpu.Rope([2 * math.pi / 1024] * 64)
    a = gpu.rope(t, torch.full((8,), 5, device="cuda"), q)
    b = gpu.rope(t, torch.full((8,), 5 + 1024 * 2**20, device="cuda"), q)
    assert bool(((a - b).abs() <= 2.0 ** -20).all())
    r.release()
    t.release()


def test_strides_and_in_place(gpu):
    g = torch.Generator(device="cuda").manual_seed(5)
    for D, pad, x in ((128, 0, torch.bfloat16), (128, 8, torch.float32), (64, 3, torch.float16)):
        r, inv = make_rope(gpu, 64, "interleaved")
        qkv = torch.randn((9, 12, D + pad), device="cuda", generator=g).to(x)
        pos = torch.arange(9, device="cuda") * 1000
        was = qkv.clone()
        q, k = qkv[:, :8, :D], qkv[:, 8:10, :D]
        want_q, want_k = gpu.rope(r, pos, q.contiguous(), k.contiguous(), out_dtype=x)
        out = gpu.rope(r, pos, q, k, q_out=q, k_out=k)
        assert out[0] is q and torch.equal(q, want_q) and torch.equal(k, want_k)
        assert torch.equal(qkv[:, 10:], was[:, 10:]) and torch.equal(qkv[..., D:], was[..., D:])
        turned_round = was[:, :8, :D].transpose(0, 1).contiguous().transpose(0, 1)
        assert torch.equal(gpu.rope(r, pos, turned_round, out_dtype=x), want_q)
        r.release()


def test_f16_overflow_is_reported(gpu):
    q = torch.full((3, 2, 64), 70000.0, device="cuda")
    gpu.rope(None, None, q, out_dtype=torch.bfloat16)
    gpu.stream_sync()
    gpu.rope(None, None, q, out_dtype=torch.float16)
    with pytest.raises(gpu.NxqError) as e:
        gpu.stream_sync()
    assert e.value.name == "ERR_RANGE"


def test_no_tokens(gpu):
    q = torch.empty((0, 2, 64), device="cuda")
    assert gpu.rope(None, None, q).shape == (0, 2, 64)


# ---- append ---------------------------------------------------------------------------

def batch(gpu, new, total, Hq, Hk, D, page, x, c, order="heads", seed=0):
    """A cache that holds the sequences' tokens but the new ones (fives elsewhere), and new q, k, v."""
    p = Paged(gpu, new, total, Hq, Hk, D, page, c, order=order, seed=seed, fill=5.0)
    for i, (n, t) in enumerate(zip(new, total)):
        pages, slots = p.places(i)
        for z in (p.keys, p.values):
            p.view(z)[pages[t - n:], slots[t - n:]] = 5.0
    g = torch.Generator(device="cuda").manual_seed(seed + 100)
    qkv = torch.randn((p.T, Hq + 2 * Hk, D), device="cuda", generator=g).to(x)
    p.q, p.newk, p.newv = qkv[:, :Hq], qkv[:, Hq:Hq + Hk], qkv[:, Hq + Hk:]
    return p


def positions(p):
    return torch.cat([torch.arange(t - n, t, device="cuda") for n, t in zip(p.new, p.total)] or [torch.empty(0)])


@pytest.mark.parametrize("order", ["heads", "tokens"])
@pytest.mark.parametrize("page", [1, 5, 16, 64])
@pytest.mark.parametrize("D,dims", [(128, 128), (64, 32), (72, 20), (256, 256)])
def test_append(gpu, D, dims, page, order):
    new, total = [1, 0, 3, 170, 1, 900], [10, 20, 3, 200, 64, 1000]
    for x, c, layout in ((torch.float32, torch.bfloat16, "half"), (torch.float16, torch.float16, "interleaved"),
                         (torch.bfloat16, torch.float16, "half")):
        r, inv = make_rope(gpu, dims, layout, "blend")
        p = batch(gpu, new, total, 4, 2, D, page, x, c, order=order, seed=page)
        wq, wk = 1 + torch.rand(D, device="cuda"), 1 + torch.rand(D, device="cuda")
        keys, values = p.keys.clone(), p.values.clone()
        q = gpu.kv_append(p.cache, p.newk, p.newv, p.q_offsets, p.kv_lens, p.table, rope=r, q=p.q, q_norm=wq, k_norm=wk, out_dtype=c)
        gpu.stream_sync()
        pos = positions(p)
        check(q, *turned(p.q, wq, 1e-6, r, inv, pos))
        want_k, bound = turned(p.newk, wk, 1e-6, r, inv, pos)
        at, touched = 0, torch.zeros(p.keys.shape[0], page, dtype=torch.bool, device="cuda")
        for i, (n, t) in enumerate(zip(new, total)):
            pages, slots = (z[t - n:] for z in p.places(i))
            check(p.view(p.keys)[pages, slots], want_k[at:at + n], bound[at:at + n])
            assert torch.equal(p.view(p.values)[pages, slots], p.newv[at:at + n].to(c))
            touched[pages, slots] = True
            at += n
        for now, was in ((p.keys, keys), (p.values, values)):
            assert torch.equal(p.view(now)[~touched], p.view(was)[~touched])
        r.release()


def test_append_keys_only(gpu):
    # Neither rotation nor norms nor queries: what was given, rounded.
    p = batch(gpu, [4, 1], [9, 40], 4, 2, 64, 16, torch.float32, torch.float16)
    assert gpu.kv_append(p.cache, p.newk, p.newv, p.q_offsets, p.kv_lens, p.table) is None
    gpu.stream_sync()
    at = 0
    for i, (n, t) in enumerate(zip(p.new, p.total)):
        pages, slots = (z[t - n:] for z in p.places(i))
        assert torch.equal(p.view(p.keys)[pages, slots], p.newk[at:at + n].half())
        assert torch.equal(p.view(p.values)[pages, slots], p.newv[at:at + n].half())
        at += n


def test_append_many_sequences(gpu):
    rng = random.Random(0)
    new = [rng.choice([0, 1, 1, 2, 5]) for _ in range(2500)]
    total = [n + rng.randrange(60) for n in new]
    p = batch(gpu, new, total, 2, 1, 64, 16, torch.float16, torch.float16, seed=1)
    q = gpu.kv_append(p.cache, p.newk, p.newv, p.q_offsets, p.kv_lens, p.table, q=p.q, out_dtype=torch.float16)
    gpu.stream_sync()
    assert torch.equal(q, p.q)
    at = 0
    for i in (0, 1, 31, 32, 33, 1023, 1024, 1025, 2499):
        n, t, at = new[i], total[i], sum(new[:i])
        pages, slots = (z[t - n:] for z in p.places(i))
        assert torch.equal(p.view(p.keys)[pages, slots], p.newk[at:at + n])


def test_append_leaves_out_what_is_wrong(gpu):
    def call(change, what, first=True):
        p = batch(gpu, [2, 3, 1], [20, 30, 40], 4, 2, 64, 16, torch.float16, torch.float16, seed=2)
        change(p)
        was = p.keys.clone()
        q = torch.full((p.T, 4, 64), 7.0, dtype=torch.float16, device="cuda")
        gpu.kv_append(p.cache, p.newk, p.newv, p.q_offsets, p.kv_lens, p.table, q=p.q, q_out=q)
        with pytest.raises(gpu.NxqError) as e:
            gpu.stream_sync()
        assert e.value.name == "ERR_INDEX" and what in str(e.value)
        gpu.stream_sync()
        pages, slots = p.places(0)
        if first:  # the first sequence is right
            assert torch.equal(p.view(p.keys)[pages, slots][18:], p.newk[:2])
        return p, q, was

    for bad in (-1, 10**6):
        p, q, was = call(lambda p: p.table.__setitem__((1, 1), bad), "page")
        assert bool((q[2:5] == 7.0).all()) and torch.equal(q[5], p.q[5])
    for bad in (-3, 10**6, 2**31 - 1):
        p, q, was = call(lambda p: p.kv_lens.__setitem__(1, bad), "sequence")
        assert bool((q[2:5] == 7.0).all())
    # More new tokens than the sequence has: the first have no position.
    p, q, was = call(lambda p: p.kv_lens.__setitem__(1, 1), "position")
    assert bool((q[2:4] == 7.0).all()) and torch.equal(q[4], p.q[4])
    # Offsets that descend, or leave the rows.
    call(lambda p: p.q_offsets.__setitem__(3, 10**6), "sequence")
    call(lambda p: p.q_offsets.__setitem__(2, 1), "sequence", first=False)  # (row 1 is of two sequences then)


def test_rows_outside_the_sequences(gpu):
    p = batch(gpu, [2, 3], [20, 30], 4, 2, 64, 16, torch.float16, torch.float16, seed=3)
    rows = lambda t: torch.cat([t.new_full((4, *t.shape[1:]), math.nan), t, t.new_full((6, *t.shape[1:]), math.nan)])  # noqa: E731
    q = torch.full((15, 4, 64), 7.0, dtype=torch.float16, device="cuda")
    gpu.kv_append(p.cache, rows(p.newk), rows(p.newv), p.q_offsets + 4, p.kv_lens, p.table, q=rows(p.q), q_out=q)
    gpu.stream_sync()
    assert torch.equal(q[4:9], p.q) and bool((q[:4] == 7.0).all()) and bool((q[9:] == 7.0).all())
    assert torch.isfinite(p.keys).all()


def test_captured(gpu):
    r, inv = make_rope(gpu, 64, "half")
    p = batch(gpu, [1, 1], [20, 30], 4, 2, 64, 16, torch.float16, torch.float16, seed=4)
    q = torch.zeros((2, 4, 64), dtype=torch.float16, device="cuda")
    call = lambda: gpu.kv_append(p.cache, p.newk, p.newv, p.q_offsets, p.kv_lens, p.table, rope=r, q=p.q, q_out=q)  # noqa: E731
    call()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call()
    for lens in ([20, 30], [3, 17]):
        p.kv_lens.copy_(torch.tensor(lens, dtype=torch.int32))
        g.replay()
        gpu.stream_sync()
        check(q, *turned(p.q, None, 0, r, inv, p.kv_lens.long() - 1))
    del g
    r.release()
