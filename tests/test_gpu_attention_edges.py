"""GPU: attention over a paged cache at its edges, against a plain 64-bit computation."""
from __future__ import annotations

import math
import random

import pytest
import torch

from attention_cases import DT, Paged

pytestmark = pytest.mark.gpu


# ---- rows that are not a call's -------------------------------------------------

@pytest.mark.parametrize("dt,D,y", [("bf16", 128, "bf16"), ("f16", 64, "f16"), ("bf16", 64, "f32")])
@pytest.mark.parametrize("n,G", [(33, 4), (9, 4), (70, 8)])
def test_rows_behind_a_sequence_do_not_matter(gpu, n, G, dt, D, y):
    # The last tile of the sequence is filled up with the rows of q that follow; bits may not depend on them (and
    # every run has several units, over which a row's maximum may be raised).
    Hk = 8
    p = Paged(gpu, [n], [n + 20000], G * Hk, Hk, D, 16, DT[dt], seed=n)
    outs = []
    for behind in (0.0, 100.0, math.nan):
        q = torch.full((n + 64, G * Hk, D), behind, dtype=DT[dt], device="cuda")
        if behind == 100.0:
            q.mul_(torch.randn(q.shape, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").to(DT[dt]))
        q[:n] = p.q
        outs.append(gpu.paged_attention(q, p.cache, p.q_offsets, p.kv_lens, p.table, out_dtype=DT[y])[:n])
    gpu.stream_sync()
    p.check(outs[0])
    assert torch.equal(outs[1], outs[0]) and torch.equal(outs[2], outs[0])


# ---- long sums ------------------------------------------------------------------

def long_items(gpu, D, new, dt, y):
    """(got, want) of 16 sequences of 131072 keys whose values have a mean: as many sequences (of the same pages) as
    the kernel has runs, so that a run sums a whole history."""
    t, page, G, Hk = 131072, 64, 4, 1
    runs = torch.cuda.get_device_properties(0).multi_processor_count * (1 if D > 128 else 2)
    g = torch.Generator(device="cuda").manual_seed(D)
    keys = torch.randn((t // page, Hk, page, D), generator=g, device="cuda").to(DT[dt])
    values = (1 + torch.randn((t // page, Hk, page, D), generator=g, device="cuda")).to(DT[dt])
    q = torch.randn((runs * new, G, D), generator=g, device="cuda").to(DT[dt])
    offsets = torch.arange(runs + 1, dtype=torch.int32, device="cuda") * new
    lens = torch.full((runs,), t, dtype=torch.int32, device="cuda")
    table = torch.arange(t // page, dtype=torch.int32, device="cuda").expand(runs, -1)
    got = gpu.paged_attention(q, gpu.KVCache(keys, values), offsets, lens, table, max_new=new, out_dtype=DT[y])
    gpu.stream_sync()
    k, v = keys.view(t, D).double(), values.view(t, D).double()
    see = torch.arange(t, device="cuda") <= torch.arange(t - new, t, device="cuda")[:, None]
    pick = [s * new + i for s in range(0, 16 * (runs // 16), runs // 16) for i in range(new)]
    want = []
    for r in pick:
        a = (q[r].double() @ k.T * D ** -0.5).masked_fill(~see[r % new], -math.inf)
        want.append(torch.softmax(a, dim=-1) @ v)
    return got[pick].double(), torch.stack(want)


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("D,new", [(64, 1), (128, 1), (128, 6), (256, 1), (256, 6)])
def test_long_items_with_fp32_outputs(gpu, D, new, dt):
    # Relative 2-norm: a weight as two numbers of the type is off by at most 2^-17 of itself.  A unit's
    # 16 or 32 keys are 2 or 4 sums of the tensor cores from zero on, each short by at most 2^-23 of itself: 2^-21.
    # The units' sums and those of the weights are up to 4096 roundings to nearest, half a step each at most and of
    # either sign, 2^6 2^-24 together, and scores (8 at most) are off by some 2^-23 of themselves, 2^-20.
    # 2^-17 + 2^-21 + 2 2^-18 + 2^-20 at the very most; together in square far below 2^-16.
    got, want = long_items(gpu, D, new, dt, "f32")
    err = float((got - want).norm() / want.norm())
    assert err <= 2.0 ** -16, f"{err:.3g}"


@pytest.mark.parametrize("D,new", [(64, 6), (128, 1), (128, 6), (256, 1)])
def test_long_items_are_not_short(gpu, D, new):
    # Roundings to nearest have no preferred sign: over 8192 outputs or more, each off by half a step (2^-11) at most, their
    # mean has a deviation of 2^-11 / 3^0.5 / 8192^0.5 = 3.1e-6, a fifth of 2^-16.  (2048 sums toward zero fell
    # short by 1.5e-4.)
    got, want = long_items(gpu, D, new, "f16", "f16")
    assert abs(float((got.sum() - want.sum()) / want.sum())) <= 2.0 ** -16


# ---- f16 outputs that a finite value does not fit ----------------------------------

@pytest.mark.parametrize("Hk,new,total", [(2, [1, 1, 1], [20, 5, 9]), (1, [1], [20000]), (1, [60], [60]), (1, [200], [3000])],
                         ids=["whole", "joined", "whole-chunk", "joined-chunk"])
def test_f16_outputs_out_of_range_are_reported(gpu, new, total, Hk):
    p = Paged(gpu, new, total, 4 * Hk, Hk, 64, 16, torch.bfloat16, seed=1)
    for v in p.v:
        v.fill_(70144.0)
    p.store()
    for y in (torch.float32, torch.bfloat16):  # (weights and output off by half a step each: 70144 (1 - 2^-8)^2 = 69597)
        assert bool((p.attend(gpu, out_dtype=y) > 69500).all())
        gpu.stream_sync()
    assert bool((p.attend(gpu, out_dtype=torch.float16) == math.inf).all())
    with pytest.raises(gpu.NxqError) as e:
        gpu.stream_sync()
    assert e.value.name == "ERR_RANGE" and "attention" in str(e.value)
    # 65024 (1 + 2^-8) = 65278 has an f16 form still, and an output of infinite values is no error.
    for v in (65024.0, math.inf):
        for x in p.v:
            x.fill_(v)
        p.store()
        got = p.attend(gpu, out_dtype=torch.float16)
        gpu.stream_sync()
        if v == math.inf:
            assert not torch.isfinite(got).any()
        else:  # half a step of the weights, half a step of the output (16)
            assert float((got.double() - v).abs().max()) <= v * 2.0 ** -8 + 16


@pytest.mark.parametrize("S,new,total", [(100, 1, 1280), (100, 8, 1280), (40, 64, 4000)])
def test_largest_f16_values(gpu, S, new, total):
    # The average of f16 values lies among them.  Here one key has almost all weight, 2^5 to 2^7 times that of the key which
    # sets the maximum in use, and its weight rounded to f16 may be up to 2^-11 of itself too large: 65536 of
    # 65504, which has no f16 form.
    p = Paged(gpu, [new] * S, [total] * S, 8, 2, 64, 16, torch.float16, seed=1)
    p.q.zero_()
    p.q[..., 0] = 28 + 12 * torch.rand(p.q.shape[:2], generator=torch.Generator(device="cuda").manual_seed(2), device="cuda")
    for k, v in zip(p.k, p.v):
        k.zero_()
        k[..., 0] = -4
        k[::128, :, 0] = 1
        k[7 * 128 + 5, :, 0] = 2
        v.fill_(65504.0)
        v[:, 1] = -65504.0
    p.store()
    got = p.attend(gpu, out_dtype=torch.float16)
    gpu.stream_sync()
    top = got.abs().double()
    assert bool((top <= 65504).all()) and bool((top >= 65504 * (1 - 2.0 ** -11) - 16).all())
    assert bool((got[:, :4] > 0).all()) and bool((got[:, 4:] < 0).all())


# ---- what unused slots hold -----------------------------------------------------

def fastest(call):
    """Least device time of 10 calls, of 7 tries."""
    best = math.inf
    for _ in range(7):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        for _ in range(10):
            call()
        b.record()
        torch.cuda.synchronize()
        best = min(best, a.elapsed_time(b))
    return best


@pytest.mark.parametrize("window,sinks", [(0, 0), (100, 4)])
@pytest.mark.parametrize("dt,D", [("bf16", 128), ("f16", 64)])
def test_unused_slots_cost_nothing(gpu, dt, D, window, sinks):
    # Values that no query sees may be NaN without a look at each of them: neither bits nor time change.
    n, total = 130, 1985
    p = Paged(gpu, [n], [total], 32, 8, D, 64, DT[dt], seed=3, fill=0.0)
    kw = dict(window=window, sinks=sinks, out_dtype=DT[dt])
    out = torch.empty_like(p.q)
    want = p.attend(gpu, **kw).clone()
    clean = fastest(lambda: p.attend(gpu, **kw, out=out))
    pages, slots = p.places(0)
    for x in (p.keys, p.values):
        seen = p.view(x)[pages, slots].clone()
        x.fill_(math.nan)
        if window:
            seen[sinks:total - n - window + 1] = math.nan
        p.view(x)[pages, slots] = seen
    full = fastest(lambda: p.attend(gpu, **kw, out=out))
    gpu.stream_sync()
    assert torch.equal(out, want)
    assert full <= 2 * clean, f"{full * 100:.0f} us, {clean * 100:.0f} with zeros in unused slots"


@pytest.mark.parametrize("dt,D", [("bf16", 128), ("f16", 64)])
def test_one_infinite_value_costs_little(gpu, dt, D):
    # One that some queries see and others do not: it is added where it is seen, without a look at each other element by all.
    p = Paged(gpu, [130], [1985], 32, 8, D, 64, DT[dt], seed=3, fill=0.0)
    out = torch.empty_like(p.q)
    call = lambda: p.attend(gpu, out_dtype=DT[dt], out=out)  # noqa: E731
    call()
    want, clean = out.clone(), fastest(call)
    p.v[0][1980, 0, 3] = math.inf
    p.store()
    one = fastest(call)
    gpu.stream_sync()
    seen = torch.zeros_like(out, dtype=torch.bool)
    seen[1980 - 1855:, :4, 3] = True  # positions from 1980 on, the query heads of key head 0
    assert bool((out[seen] == math.inf).all()) and torch.equal(out[~seen], want[~seen])
    assert one <= 2 * clean, f"{one * 100:.0f} us, {clean * 100:.0f} without"


@pytest.mark.parametrize("new", [1, 130])
@pytest.mark.parametrize("sinks", [2**30, 2**40])
def test_everything_is_a_sink(gpu, sinks, new):
    p = Paged(gpu, [new], [new + 700], 8, 2, 64, 32, torch.bfloat16, seed=4)
    want = p.attend(gpu)
    assert torch.equal(p.attend(gpu, window=50, sinks=sinks), want)
    gpu.stream_sync()


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("new", [1, 6, 140])
def test_infinite_values_of_no_weight(gpu, new, dt):
    # exp(-200) is zero in every type: zero times infinity is NaN.  Whatever it is, it is not finite, and other elements are.
    p = Paged(gpu, [new], [new + 300], 8, 2, 64, 32, DT[dt], seed=5)
    p.q[..., 0] = 40
    p.k[0][3, :, 0] = -40
    p.v[0][3, :, 7] = math.inf
    p.store()
    for y in (DT[dt], torch.float32):
        got = p.attend(gpu, out_dtype=y)
        gpu.stream_sync()
        assert not torch.isfinite(got[..., 7]).any()
        got[..., 7] = 0
        assert torch.isfinite(got).all()


# ---- many sequences -----------------------------------------------------------------

@pytest.mark.parametrize("S,lengths", [(700, [0, 1, 40, 70]), (1500, [1, 1, 1, 1, 1, 1, 2, 40]), (257, [33, 65])])
def test_chunks_of_many_sequences(gpu, S, lengths):
    # More than one chunk of the plan (256), all for the kernel of many rows, or for both.
    rng = random.Random(S)
    new = [rng.choice(lengths) for _ in range(S)]
    p = Paged(gpu, new, [n + rng.randrange(0, 90) for n in new], 8, 2, 64, 16, torch.float16, seed=3)
    got, lse = p.attend(gpu, return_lse=True)
    gpu.stream_sync()
    p.check(got, lse)


def test_most_sequences(gpu):
    # 65536 sequences over the same page, the last of them a chunk.
    S, n, t, Hk, G, D = 65536, 40, 50, 1, 2, 64
    g = torch.Generator(device="cuda").manual_seed(1)
    keys, values = (torch.randn((1, Hk, 64, D), generator=g, device="cuda").half() for _ in range(2))
    q = torch.randn((S - 1 + n, G, D), generator=g, device="cuda").half()
    offsets = torch.arange(S + 1, dtype=torch.int32, device="cuda")
    offsets[S] = S - 1 + n
    lens = torch.full((S,), t, dtype=torch.int32, device="cuda")
    table = torch.zeros((S, 1), dtype=torch.int32, device="cuda")
    k, v = keys[0, 0, :t].double(), values[0, 0, :t].double()
    pos = torch.full((S - 1 + n,), t - 1, device="cuda")
    pos[S - 1:] = torch.arange(t - n, t, device="cuda")
    a = q.double() @ k.T * D ** -0.5
    a.masked_fill_(torch.arange(t, device="cuda") > pos[:, None, None], -math.inf)
    want = torch.softmax(a, dim=-1) @ v
    for max_new in (0, n):
        got = gpu.paged_attention(q, gpu.KVCache(keys, values), offsets, lens, table, max_new=max_new, out_dtype=torch.float32)
        gpu.stream_sync()
        # Weights as two f16 numbers (2^-22), scores and sums of 64 in fp32: well below 2^-16 of the values' magnitude.
        assert float((got.double() - want).abs().max()) <= 2.0 ** -16 * float(v.abs().max())
