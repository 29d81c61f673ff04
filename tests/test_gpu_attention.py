"""GPU: attention over a paged cache against a plain 64-bit computation.

The bound of each output (attention_cases.Paged.expected) counts the roundings: scores
in fp32, weights rounded to the cache's type (half a step each), sums in fp32, one
rounding of the output.  Unused slots and pages hold NaN throughout.
"""
from __future__ import annotations

import math
import random

import pytest
import torch

from attention_cases import DT, HALF_STEP, Paged

pytestmark = pytest.mark.gpu


def run(gpu, p, y="f32", **kw):
    got, lse = p.attend(gpu, out_dtype=DT[y], return_lse=True, **kw)
    kw.pop("max_new", None)
    gpu.stream_sync()
    p.check(got, lse, **kw)
    return got, lse


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("D", [8, 64, 72, 96, 128, 200, 256])
@pytest.mark.parametrize("G", [1, 3, 4, 16])
def test_single_tokens(gpu, G, D, dt):
    # Lengths of one token, around a unit of 64 keys, around a page, and long.
    total = [1, 2, 63, 64, 65, 700, 16, 17, 129]
    p = Paged(gpu, [1] * len(total), total, 2 * G, 2, D, 16, DT[dt], seed=D + G)
    run(gpu, p, max_new=1)


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("order", ["heads", "tokens"])
@pytest.mark.parametrize("page", [1, 3, 8, 16, 24, 64, 100, 256])
def test_pages(gpu, page, order, dt):
    # Pages that end inside a unit, larger than a unit, no power of two.
    p = Paged(gpu, [1, 3, 1, 40, 150], [300, 77, 5, 515, 1000], 8, 2, 64, page, DT[dt], order=order, seed=page)
    run(gpu, p, y=dt)


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("D", [64, 80, 128, 256])
@pytest.mark.parametrize("G", [1, 4, 5, 7, 8])
def test_chunks(gpu, G, D, dt):
    # Drafted tokens, chunks, whole prompts; a sequence without new tokens, one without a history.
    new, ctx = [5, 1, 0, 33, 129, 300, 2], [100, 0, 50, 0, 1000, 70, 2000]
    p = Paged(gpu, new, [n + c for n, c in zip(new, ctx)], 2 * G, 2, D, 32, DT[dt], seed=G)
    run(gpu, p, y="f32")


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (7, 4), (64, 0), (64, 64), (100, 4), (128, 130), (1000, 4), (300, 700), (10**6, 3)])
def test_windows(gpu, window, sinks, D):
    new, ctx = [1, 1, 4, 70, 400, 1], [600, 20, 900, 130, 0, 3000]
    p = Paged(gpu, new, [n + c for n, c in zip(new, ctx)], 8, 2, D, 16, torch.bfloat16, seed=window)
    # What no query sees may be anything: pages gone from the table, NaN in the slots.
    for i, (n, t) in enumerate(zip(p.new, p.total)):
        low = t - n - window + 1  # the first query's first key
        for j0 in range(0, t, p.page):
            if j0 >= sinks and j0 + p.page <= low:
                p.table[i, j0 // p.page] = random.choice([-1, 10**9, -2**31])
    run(gpu, p, window=window, sinks=sinks)


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("S,new,total", [(40, 1, 8000), (2, 700, 20000), (1, 3000, 3000)])
def test_fp32_outputs_are_exact_enough(gpu, S, new, total, dt):
    # Relative 2-norm.  A weight as two numbers of the type is off by at most 2^-17 of itself (bf16; half a step of
    # what half a step leaves); the tensor cores sum toward zero, up to 2^-23 of the sum each, on average an eighth of
    # that, 128 times before the sums move on (tcgen05) or once per 64 keys (250 times here): 2^-18.
    p = Paged(gpu, [new] * S, [total] * S, 8, 2, 128, 32, DT[dt], seed=S)
    got = p.attend(gpu, out_dtype=torch.float32)
    want, _, _ = p.expected(y=torch.float32)
    assert float((got.double() - want).norm() / want.norm()) <= 2.0 ** -17 + 2.0 ** -18


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("S,total", [(1, 20000), (2, 33333), (40, 900)])
def test_split_histories(gpu, S, total, dt):
    # Few sequences: every item is cut between many runs and joined.
    rng = random.Random(S)
    totals = [total - rng.randrange(total // 2) for _ in range(S)]
    p = Paged(gpu, [1] * S, totals, 8, 1, 128, 64, DT[dt], seed=S)
    run(gpu, p, y=dt)


@pytest.mark.parametrize("dt,D,y", [("bf16", 128, "bf16"), ("f16", 64, "f32"), ("f16", 80, "f16")])
@pytest.mark.parametrize("window", [0, 300])
def test_long_runs(gpu, dt, D, y, window):
    # Many items and key blocks for each run: rings go round many times, items of one and two tiles alternate.
    new, ctx = [2200, 31, 700, 100, 17, 900], [500, 4000, 0, 1000, 300, 0]
    p = Paged(gpu, new, [n + c for n, c in zip(new, ctx)], 32, 8, D, 32, DT[dt], seed=D)
    for max_new in (0, 2200):
        run(gpu, p, y=y, window=window, sinks=4, max_new=max_new)


def test_many_sequences(gpu):
    # More than one chunk of the plan (256), with some that have nothing to do.
    rng = random.Random(1)
    new = [rng.choice([0, 1, 1, 1, 2]) for _ in range(1500)]
    p = Paged(gpu, new, [n + rng.randrange(0, 90) for n in new], 4, 2, 64, 16, torch.float16, seed=3)
    run(gpu, p)


def test_queries_without_keys(gpu):
    # More new tokens than cached ones: the first have negative positions and see nothing.
    p = Paged(gpu, [3, 40, 1], [3, 40, 1], 4, 1, 64, 16, torch.bfloat16, seed=5)
    p.kv_lens[0], p.kv_lens[1], p.kv_lens[2] = 1, 33, 0
    got, lse = p.attend(gpu, return_lse=True)
    gpu.stream_sync()
    assert not got[:2].any() and bool((lse[:2] == -math.inf).all())
    assert not got[3:10].any() and bool((lse[3:10] == -math.inf).all())
    assert not got[43].any() and bool((lse[43] == -math.inf).all())
    assert torch.isfinite(got).all()
    # The last query of the first sequence sees its one key.
    assert torch.allclose(got[2], p.v[0][0].float().repeat_interleave(4, dim=0), rtol=2.0 ** -20)


@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("new", [[1, 1], [4, 3], [200, 130]])
def test_values_that_only_some_queries_see(gpu, new, bad):
    # Causality is strict: a value that is not finite reaches the queries that see it and no other.
    D, ctx = 64, 70
    for dt in (torch.float16, torch.bfloat16):
        p = Paged(gpu, new, [n + ctx for n in new], 4, 2, D, 16, dt, seed=2)
        clean = {y: p.attend(gpu, window=50, out_dtype=y) for y in (dt, torch.float32)}
        at = [ctx + new[0] - 1, 30]  # the last token of sequence 0; one that leaves the window in sequence 1
        p.v[0][at[0], 1, 5] = bad
        p.v[1][at[1], 0, 7] = bad
        p.store()
        hit = torch.zeros((p.T, 4, D), dtype=torch.bool, device="cuda")
        hit[new[0] - 1, 2:, 5] = True  # query heads 2, 3 read key head 1
        for i in range(new[1]):
            if at[1] > ctx + i - 50:
                hit[new[0] + i, :2, 7] = True
        for y in (dt, torch.float32):
            got = p.attend(gpu, window=50, out_dtype=y)
            gpu.stream_sync()
            assert torch.equal(got[~hit], clean[y][~hit])
            assert not torch.isfinite(got[hit]).any()
            if y is dt and not math.isnan(bad):  # (an fp32 output may be NaN there)
                assert bool((got[hit] == bad).all())


def test_keys_that_only_some_queries_see(gpu):
    p = Paged(gpu, [3], [103], 2, 1, 64, 16, torch.bfloat16, seed=4)
    clean = p.attend(gpu)
    p.k[0][102] = math.nan
    p.store()
    got = p.attend(gpu)
    assert torch.equal(got[:2], clean[:2]) and torch.isnan(got[2]).all()


@pytest.mark.parametrize("peak", [30.0, 0.0])
def test_large_and_flat_scores(gpu, peak):
    # Scores of several hundred, whose maximum keeps rising; scores of zero.
    p = Paged(gpu, [1, 6, 64], [500, 700, 300], 8, 2, 128, 32, torch.float16, seed=6, peak=peak)
    run(gpu, p)
    run(gpu, p, scale=1.5)


def test_rising_scores(gpu):
    # Every key's score above the one before: the maximum in use is raised in every unit.
    for dt in (torch.float16, torch.bfloat16):
        p = Paged(gpu, [1, 40], [1500, 1500], 4, 1, 64, 16, dt, seed=7)
        p.q[:] = 1.0
        for i in range(2):
            p.k[i][:] = (torch.arange(1500, device="cuda") / 64).to(dt)[:, None, None]
        p.store()
        run(gpu, p)


def test_strides(gpu):
    # Queries inside a packed projection, outputs likewise; odd strides; a cache inside a larger one.
    new, total = [1, 7, 50], [90, 80, 200]
    for D, pad in ((64, 0), (64, 3), (72, 1)):
        p = Paged(gpu, new, total, 6, 2, D, 16, torch.float16, seed=8)
        want = p.attend(gpu)
        qkv = torch.full((p.T, 11, D + pad), 9.0, dtype=torch.float16, device="cuda")
        q = qkv[:, 1:7, :D]
        q.copy_(p.q)
        big = torch.full((p.T, 9, D + pad), -5.0, device="cuda")
        out = big[:, 2:8, :D]
        got = gpu.paged_attention(q, p.cache, p.q_offsets, p.kv_lens, p.table, out=out)
        assert got is out and torch.equal(out, want)
        out.fill_(-5.0)
        assert bool((big == -5.0).all())
        # Heads first: [Hq][T][D] seen as [T][Hq][D].
        q2 = p.q.transpose(0, 1).contiguous().transpose(0, 1)
        assert torch.equal(gpu.paged_attention(q2, p.cache, p.q_offsets, p.kv_lens, p.table), want)
        both = torch.full((p.keys.shape[0], 2, 3, p.page, D + 8), math.nan, dtype=torch.float16, device="cuda")
        both[:, 0, :2, :, :D], both[:, 1, :2, :, :D] = p.keys, p.values
        c = gpu.KVCache(both[:, 0, :2, :, :D], both[:, 1, :2, :, :D])
        assert torch.equal(gpu.paged_attention(p.q, c, p.q_offsets, p.kv_lens, p.table), want)
    gpu.stream_sync()


def test_rows_outside_the_sequences(gpu):
    p = Paged(gpu, [2, 30], [40, 60], 4, 2, 64, 16, torch.float16, seed=9)
    q = torch.cat([p.q.new_full((3, 4, 64), math.nan), p.q, p.q.new_full((5, 4, 64), math.nan)])
    out = torch.full((40, 4, 64), 3.0, device="cuda")
    gpu.paged_attention(q, p.cache, p.q_offsets + 3, p.kv_lens, p.table, out=out)
    gpu.stream_sync()
    p.check(out[3:35])
    assert bool((out[:3] == 3.0).all()) and bool((out[35:] == 3.0).all())


def test_no_rows(gpu):
    p = Paged(gpu, [1], [5], 4, 2, 64, 16, torch.float16)
    none = p.q[:0]
    assert gpu.paged_attention(none, p.cache, p.q_offsets * 0, p.kv_lens, p.table).shape == (0, 4, 64)


BROKEN = {
    "offset beyond the rows": lambda p: p.q_offsets.__setitem__(2, 10**6),
    "offsets that descend": lambda p: p.q_offsets.__setitem__(2, 0),
    "negative length": lambda p: p.kv_lens.__setitem__(1, -1),
    "length beyond the table": lambda p: p.kv_lens.__setitem__(1, 10**6),
}


@pytest.mark.parametrize("case", BROKEN.keys())
@pytest.mark.parametrize("new", [[1, 1, 1], [40, 3, 50]])
def test_broken_sequences_are_left_out(gpu, new, case):
    p = Paged(gpu, new, [n + 100 for n in new], 4, 2, 64, 16, torch.float16, seed=10)
    want = p.attend(gpu)
    BROKEN[case](p)
    out = torch.full_like(want, 3.0)
    p.attend(gpu, out=out)
    with pytest.raises(gpu.NxqError) as e:
        gpu.stream_sync()
    assert e.value.name == "ERR_INDEX" and "sequence" in str(e.value)
    a = new[0]
    if "descend" not in case:  # (the third sequence then starts at row 0: rows of two sequences hold the output of either)
        assert torch.equal(out[:a], want[:a])
    if "length" in case:
        assert bool((out[a:a + new[1]] == 3.0).all()) and torch.equal(out[a + new[1]:], want[a + new[1]:])
    gpu.stream_sync()  # reported once


def test_too_many_new_tokens(gpu):
    p = Paged(gpu, [1, 3, 1], [50, 60, 70], 4, 2, 64, 16, torch.float16, seed=11)
    want = p.attend(gpu)
    out = torch.full_like(want, 3.0)
    p.attend(gpu, out=out, max_new=1)
    with pytest.raises(gpu.NxqError):
        gpu.stream_sync()
    assert torch.equal(out[0], want[0]) and torch.equal(out[4], want[4]) and bool((out[1:4] == 3.0).all())


@pytest.mark.parametrize("new", [[1, 1], [30, 100]])
def test_bad_pages(gpu, new):
    # Reported; the page counts as zeros, the other sequence is right.
    p = Paged(gpu, new, [n + 60 for n in new], 4, 2, 64, 16, torch.bfloat16, seed=12)
    want = p.attend(gpu)
    for bad in (-1, p.keys.shape[0], 2**31 - 1):
        p.table[0, 1] = bad
        got = p.attend(gpu)
        with pytest.raises(gpu.NxqError) as e:
            gpu.stream_sync()
        assert "page" in str(e.value)
        assert torch.equal(got[new[0]:], want[new[0]:]) and torch.isfinite(got).all()
    p.k[0][16:32], p.v[0][16:32] = 0, 0
    p.check(got)


def test_same_bits(gpu):
    p = Paged(gpu, [1, 1, 90], [9000, 333, 5000], 8, 2, 128, 16, torch.bfloat16, seed=13)
    want = p.attend(gpu)
    for _ in range(20):
        assert torch.equal(p.attend(gpu), want)


def test_cache_beyond_32_bits(gpu):
    # Element offsets past 2^31 in the cache: a page far out.
    D, page, Hk = 128, 64, 8
    pages = 2**31 // (D * page * Hk) + 40
    keys = torch.zeros((pages, Hk, page, D), dtype=torch.bfloat16, device="cuda")
    values = torch.zeros_like(keys)
    p = Paged(gpu, [1, 70], [200, 300], 8, Hk, D, page, torch.bfloat16, seed=14)
    want = p.attend(gpu)
    n = p.keys.shape[0]
    keys[-n:], values[-n:] = p.keys, p.values
    table = torch.where(p.table >= 0, p.table + (pages - n), p.table)
    got = gpu.paged_attention(p.q, gpu.KVCache(keys, values), p.q_offsets, p.kv_lens, table)
    gpu.stream_sync()
    assert torch.equal(got, want)


@pytest.mark.parametrize("D,dt", [(128, "bf16"), (64, "f16"), (192, "bf16")])
@pytest.mark.parametrize("new,total", [([1, 1, 1], [4000, 3, 700]), ([5, 3, 6], [900, 3, 700]), ([300, 1, 129], [2100, 50, 129])])
def test_in_place(gpu, new, total, D, dt):
    b = Paged(gpu, new, total, 10, 2, D, 16, DT[dt], seed=D)
    want = b.attend(gpu, out_dtype=DT[dt])
    q = b.q.clone()
    for _ in range(3):
        b.q.copy_(q)
        assert torch.equal(b.attend(gpu, out=b.q), want)


@pytest.mark.parametrize("page", [1, 3, 8, 200, 4096])
@pytest.mark.parametrize("new", [1, 140])
def test_odd_pages(gpu, new, page):
    b = Paged(gpu, [new, new], [new + 333, new], 4, 2, 64, page, torch.float16, seed=page)
    b.check(b.attend(gpu, out_dtype=torch.float16))
    b.check(b.attend(gpu, out_dtype=torch.float16, window=100, sinks=3), window=100, sinks=3)


def test_another_stream_and_graphs(gpu):
    # Calls on two streams at once, and two captured graphs replayed in turn and at once.
    a = Paged(gpu, [1] * 8, [3000] * 8, 8, 2, 128, 16, torch.bfloat16, seed=15)
    b = Paged(gpu, [20, 150], [4000, 700], 8, 2, 64, 32, torch.float16, seed=16)
    want = [a.attend(gpu), b.attend(gpu)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    outs = [[torch.zeros_like(w) for w in want] for _ in range(2)]
    for _ in range(10):
        for s, p, o in zip(streams, (a, b), outs[0]):
            p.attend(gpu, out=o, stream=s)
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for o, w in zip(outs[0], want))
    graphs = []
    for s, p, o in zip(streams, (a, b), outs[1]):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            p.attend(gpu, out=o)
        graphs.append(g)
    for _ in range(5):
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        for p, o in zip((a, b), outs[0]):
            p.attend(gpu, out=o)
    torch.cuda.synchronize()
    gpu.stream_sync()
    for o in outs:
        assert all(torch.equal(x, w) for x, w in zip(o, want))
    del graphs


def test_lengths_change_between_replays(gpu):
    # A captured call takes the lengths that are on the device when it runs.
    p = Paged(gpu, [1, 1, 1], [500, 40, 3000], 4, 2, 64, 16, torch.float16, seed=17)
    out = torch.zeros((3, 4, 64), device="cuda")
    g = torch.cuda.CUDAGraph()
    p.attend(gpu, out=out, max_new=1)
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        p.attend(gpu, out=out, max_new=1)
    for lens in ([500, 40, 3000], [1, 40, 2], [444, 39, 2999]):
        p.kv_lens.copy_(torch.tensor(lens, dtype=torch.int32))
        g.replay()
        got = out.clone()
        assert torch.equal(got, p.attend(gpu, max_new=1))
    gpu.stream_sync()
    del g


@pytest.mark.parametrize("seed", range(12))
def test_random_batches(gpu, seed):
    rng = random.Random(seed)
    Hk, G, D = rng.choice([1, 2, 8]), rng.choice([1, 2, 5, 8, 12]), rng.choice([64, 96, 128])
    S = rng.randint(1, 12)
    new = [rng.choice([1, 1, 1, rng.randint(0, 9), rng.randint(1, 400)]) for _ in range(S)]
    total = [n + rng.choice([0, rng.randint(0, 3000)]) for n in new]
    page, order = rng.choice([8, 16, 40, 128]), rng.choice(["heads", "tokens"])
    kw = dict(window=rng.choice([0, rng.randint(1, 500)]), sinks=rng.choice([0, 2, 70]))
    dt = rng.choice(["f16", "bf16"])
    p = Paged(gpu, new, total, Hk * G, Hk, D, page, DT[dt], order=order, seed=seed)
    if p.T:
        run(gpu, p, y=rng.choice(["f32", dt]), **kw)
