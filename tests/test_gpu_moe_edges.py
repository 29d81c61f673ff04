"""GPU: the mixture-of-experts and embedding calls at the edges of what they take.

Bounds as in test_gpu_moe.py, whose helpers are used here.
"""
from __future__ import annotations

import os
import subprocess
import sys

import numpy as np
import pytest
import torch

from conftest import PKG, ROOT

from nxq import synth
from test_gpu_moe import DT, EXACT, TYPE_NAMES, check, make_offsets, make_weights, products, swiglu

pytestmark = pytest.mark.gpu

# Block type and slots per expert that lead to each product kernel.
KERNELS = {"warp": (12, 3), "tcgen05": (12, 40), "exact": (121, 40)}


def release(tables, weights):
    for t in tables:
        t.release()
    for w in weights:
        w.release()


@pytest.mark.parametrize("xdt", DT.keys())
@pytest.mark.parametrize("kernel", KERNELS.keys())
@pytest.mark.parametrize("bad", [[1], [0], [2], [1, 2], [0, 3]], ids=str)
@pytest.mark.parametrize("value", [10**6, 2**31 - 1, -1, -2**31])
def test_offset_out_of_range_costs_its_neighbours_only(gpu, value, bad, kernel, xdt):
    """An offset outside [0, R] leaves out the two experts it bounds; every other expert's rows are there."""
    t, m = KERNELS[kernel]
    E, N, K = 5, 128, 256
    ws, W = make_weights(gpu, t, E, N, K, 6)
    T = gpu.Experts(ws)
    try:
        R = E * m
        x = torch.randn((R, K), device="cuda").to(DT[xdt])
        good = [m * e for e in range(E + 1)]
        off = [value if e in bad else o for e, o in enumerate(good)]
        out = torch.full((R, N), -7.0, device="cuda")
        gpu.qmatmul_ragged(T, x, torch.tensor(off, dtype=torch.int32, device="cuda"), out=out)
        with pytest.raises(gpu.NxqError) as e:
            gpu.stream_sync()
        assert e.value.name == "ERR_INDEX"
        y, b = products(W, t, x, [m] * E, torch.arange(R, device="cuda"))
        for e in range(E):
            s = slice(good[e], good[e + 1])
            if e in bad or e + 1 in bad:
                assert bool((out[s] == -7).all()), e
            else:
                assert bool(((out[s].double() - y[s]).abs() <= b[s] + 2.0 ** -24 * y[s].abs() + 2.0 ** -25).all()), e
    finally:
        release([T], ws)


def test_most_slots(gpu):
    """2^31 - 1 slots, all but five of them with one expert."""
    t, K, R = 122, 32, 2**31 - 1
    ws, W = make_weights(gpu, t, 2, 1, K, 3)
    T = gpu.Experts(ws)
    try:
        x = torch.randn((2, K), device="cuda")
        rows = torch.zeros(R, dtype=torch.int32, device="cuda")
        rows[1::2] = 1
        out = torch.full((R, 1), -7.0, dtype=torch.bfloat16, device="cuda")
        gpu.qmatmul_ragged(T, x, torch.tensor([0, 5, R], dtype=torch.int32, device="cuda"), rows=rows, out=out)
        gpu.stream_sync()
        for odd in (0, 1):
            for e, got in enumerate((out[odd:5:2, 0], out[5:][1 - odd::2, 0])):
                want = (x[odd].double() @ W[e, 0]).item()
                bound = K * 2.0 ** -24 * (x[odd].double() * W[e, 0]).abs().sum().item()
                lo, hi = got.min().double().item(), got.max().double().item()
                assert lo == hi and abs(lo - want) <= bound + 2.0 ** -8 * (abs(want) + bound), (odd, e)
    finally:
        release([T], ws)
        del rows, out, got
        torch.cuda.empty_cache()


def test_most_tokens(gpu):
    """2^31 - 1 choices: token t takes expert t % 2."""
    T, step = 2**31 - 1, 2**28
    logits = torch.zeros((T, 2), dtype=torch.bfloat16, device="cuda")
    logits[1::2, 1] = 1
    ids, w, offsets, rows, slots = gpu.moe_route(logits, 1)
    gpu.stream_sync()
    del logits
    even = (T + 1) // 2
    assert offsets.tolist() == [0, even, T]
    for a in range(0, T, step):
        z = min(a + step, T)
        t = torch.arange(a, z, device="cuda")  # as a token, then as a slot
        assert torch.equal(ids[a:z, 0], (t % 2).int()) and bool((w[a:z] == 1).all())
        assert torch.equal(slots[a:z, 0], (t // 2 + (t % 2) * even).int())
        assert torch.equal(rows[a:z], torch.where(t < even, 2 * t, 2 * (t - even) + 1).int())
    del ids, w, rows, slots, t
    torch.cuda.empty_cache()


def stream_calls(gpu):
    """name -> call(stream) -> its new outputs; each large enough to take a freed tensor's place."""
    N, K, T, E, k = 1024, 256, 640, 4, 2
    w = gpu.Weight.register(synth.make_blocks(12, N, K, seed=1), 12, N, K)
    ws, _ = make_weights(gpu, 12, E, N, K, 6)
    X = gpu.Experts(ws)
    x = torch.randn((T, K), device="cuda").half()
    off = make_offsets([T // E] * E)
    res = torch.randn((T, N), device="cuda")
    h = torch.randn((T, N), device="cuda")
    logits = torch.randn((70000, 64), device="cuda")
    ids = torch.randint(0, N, (4096,), device="cuda")
    slots = torch.zeros((T, k), dtype=torch.int32, device="cuda")
    share = torch.ones((T, k), device="cuda")
    norm = torch.ones(K, device="cuda")
    calls = {
        "embedding": lambda s: [gpu.embedding(w, ids, stream=s)],
        "moe_route": lambda s: list(gpu.moe_route(logits, 8, stream=s)),
        "qmatmul_ragged": lambda s: [gpu.qmatmul_ragged(X, x, off, stream=s)],
        "qmatmul_ragged_swiglu": lambda s: [gpu.qmatmul_ragged_swiglu(X, X, x, off, stream=s)],
        "moe_combine": lambda s: [gpu.moe_combine(h, slots, share, res=res, stream=s)],
        "dequant": lambda s: [w.dequant(stream=s)],
        "qmatmul": lambda s: [gpu.qmatmul(w, x, stream=s)],
        "qmatmul_grouped": lambda s: gpu.qmatmul_grouped([w, w], [x, x], stream=s),
        "qmatmul_swiglu": lambda s: [gpu.qmatmul_swiglu(w, w, x, stream=s)],
        "qmatmul_residual": lambda s: [gpu.qmatmul_residual(w, x, res, stream=s)],
        "rmsnorm_qmatmul": lambda s: gpu.rmsnorm_qmatmul([w, w], x, norm, 1e-5, stream=s),
    }
    return calls, [X], [w, *ws]


@pytest.mark.parametrize("handle", [False, True], ids=["stream", "handle"])
def test_outputs_on_another_stream(gpu, handle):
    """A call on another stream writes no memory that the current stream still reads, and its outputs
    outlive the work that the current stream does on them."""
    calls, tables, weights = stream_calls(gpu)
    side = torch.cuda.Stream()
    s = side.cuda_stream if handle else side
    try:
        for name, call in calls.items():
            want = call(None)
            for _ in range(2):  # sizes the stream's scratch
                call(s)
            torch.cuda.synchronize()
            old = [torch.full_like(o, 3) for o in want]
            kept = [torch.empty_like(o) for o in want]
            torch.cuda.synchronize()
            torch.cuda._sleep(40_000_000)  # some 20 ms before the current stream reads them
            for a, b in zip(kept, old):
                a.copy_(b)
            del old, b
            got = call(s)
            torch.cuda.current_stream().wait_stream(side)
            copies = [torch.empty_like(o) for o in got]
            torch.cuda._sleep(40_000_000)
            for a, b in zip(copies, got):
                a.copy_(b)
            shapes = [(o.shape, o.dtype) for o in got]
            del got, b
            with torch.cuda.stream(side):
                junk = [torch.full(shape, 5, dtype=dtype, device="cuda") for shape, dtype in shapes]
            torch.cuda.synchronize()
            for a, c, o in zip(kept, copies, want):
                assert bool((a == 3).all()), f"{name}: wrote a tensor that was still read"
                assert torch.equal(c, o), f"{name}: its outputs were reused while they were read"
            del junk
        gpu.stream_sync()
    finally:
        torch.cuda.synchronize()
        release(tables, weights)


@pytest.mark.parametrize("pair", [False, True], ids=["plain", "swiglu"])
def test_unaligned_arrays_are_refused(gpu, pair):
    """Arrays off their element type's boundary never reach a kernel."""
    ws, _ = make_weights(gpu, 12, 2, 128, 256, 5)
    T = gpu.Experts(ws)
    L, buf = gpu.lib(), torch.zeros(1 << 16, dtype=torch.uint8, device="cuda")
    size = {gpu.F32: 4, gpu.F16: 2, gpu.BF16: 2}
    try:
        for xd in size:
            for yd in size:
                for bad, n in enumerate((size[xd], 4, size[yd], 4)):  # x, rows, y, offsets
                    for by in range(1, n):
                        x, rows, y, off = (buf.data_ptr() + 16384 * i + (by if i == bad else 0) for i in range(4))
                        before = gpu.launch_count()
                        if pair:
                            rc = L.nxq_qmatmul_ragged_swiglu(T.handle, T.handle, x, xd, 4, rows, y, yd, 4, off, None)
                        else:
                            rc = L.nxq_qmatmul_ragged(T.handle, x, xd, 4, rows, y, yd, 4, off, None)
                        assert rc == -1 and "aligned" in gpu.last_error() and gpu.launch_count() == before
        gpu.stream_sync()
    finally:
        release([T], ws)


def test_tables_while_weights_are_released(gpu):
    """A table holds the weights it was made from, whatever another thread releases meanwhile."""
    import threading
    import time

    t, N, K, E = 12, 128, 256, 64
    blocks = synth.make_blocks(t, N, K, seed=1)
    ws = [gpu.Weight.register(blocks, t, N, K) for _ in range(E)]
    x = torch.randn((E, K), device="cuda").half()
    off = make_offsets([1] * E)
    W = ws[0].dequant().double()
    want = (x.double() @ W.T).float()
    rng = synth.rng(8)
    bad, counts = [], {"made": 0, "gone": 0, "kept": 0}
    stop = threading.Event()

    def renew():
        try:
            while not stop.is_set():
                for i in (E - 1, E // 2):
                    try:
                        ws[i].release()
                    except gpu.NxqError as e:
                        if e.name != "ERR_STATE":
                            bad.append(repr(e))
                        counts["kept"] += 1
                        time.sleep(1e-4)
                        continue
                    ws[i] = gpu.Weight.register(blocks, t, N, K)
                    time.sleep(2e-3 * rng.random())  # a while in which tables can be made
        except Exception as e:  # noqa: BLE001
            bad.append(repr(e))

    thread = threading.Thread(target=renew)
    thread.start()
    try:
        end = time.time() + 3
        while time.time() < end and not bad:
            try:
                T = gpu.Experts(ws)
            except gpu.NxqError as e:  # a weight was gone
                if e.code != -1:
                    bad.append(repr(e))
                counts["gone"] += 1
                time.sleep(1e-4)
                continue
            counts["made"] += 1
            y = gpu.qmatmul_ragged(T, x, off)
            if not ((y - want).norm() <= 2e-3 * want.norm()).item():
                bad.append("wrong product")
            T.release()
        gpu.stream_sync()
    finally:
        stop.set()
        thread.join()
    assert not bad, bad[:3]
    assert counts["made"] > 0, counts
    for w in ws:
        w.release()  # no reference was left behind


def test_weight_released_from_two_threads(gpu):
    """Of several threads that release a weight at once, one does and the others are told."""
    import threading

    blocks = synth.make_blocks(12, 128, 256, seed=1)
    threads = 4
    barrier = threading.Barrier(threads)
    for _ in range(100):
        w = gpu.Weight.register(blocks, 12, 128, 256)
        rcs = []

        def release_it(h=w.handle):
            barrier.wait()
            rcs.append(gpu.lib().nxq_weight_release(h))

        ts = [threading.Thread(target=release_it) for _ in range(threads)]
        [t.start() for t in ts]
        [t.join() for t in ts]
        assert sorted(rcs) == [-1] * (threads - 1) + [0]
        w._h = None


MANY = {"tcgen05": [16, 3, 131, 0, 40, 17, 1, 64] * 4, "warp": [3, 0, 5, 1, 8, 9, 2, 4] * 4}
TENSOR_TYPES = {n: t for n, t in TYPE_NAMES.items() if t not in EXACT}


@pytest.mark.parametrize("ydt", ["f32", "bf16"])
@pytest.mark.parametrize("pair", [False, True], ids=["plain", "swiglu"])
@pytest.mark.parametrize("kernel", MANY.keys())
@pytest.mark.parametrize("t", TENSOR_TYPES.values(), ids=TENSOR_TYPES.keys())
def test_many_work_tiles(gpu, t, kernel, pair, ydt):
    """Every CTA walks several work tiles: what its rings, accumulators and staging carry from one to the
    next (an odd number of chunks and of weight tiles, row blocks of every size) gives the right product, and
    the same bits on every call."""
    counts, N, K, distinct = MANY[kernel], 3900, 1280, 4
    E, n = len(counts), sum(counts)
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    weight_tiles = -(-N // 128)
    per_block, blk = ((weight_tiles if pair else -(-weight_tiles // 2)), 128) if kernel == "tcgen05" else (weight_tiles, 8)
    assert (n > 6 * E) == (kernel == "tcgen05")  # the kernel that such a call takes
    assert sum(-(-c // blk) for c in counts) * per_block >= 3 * sms
    tables, weights, W = [], [], []
    try:
        for seed in ((10, 50) if pair else (10,)):
            ws, dec = make_weights(gpu, t, distinct, N, K, seed)
            weights += ws
            W.append(dec[torch.arange(E) % distinct])
            tables.append(gpu.Experts([ws[e % distinct] for e in range(E)]))
        g = torch.Generator(device="cuda").manual_seed(t)
        off = make_offsets(counts)
        if pair:  # gathered rows; small ones keep the gate's sigmoid away from 0 and 1
            x = (0.05 * torch.randn((n // 2, K), device="cuda", generator=g)).bfloat16()
            rows = torch.randint(0, n // 2, (n,), device="cuda", generator=g, dtype=torch.int32)
            src = rows.long()
        else:
            x, rows, src = torch.randn((n, K), device="cuda", generator=g).half(), None, torch.arange(n, device="cuda")

        def call():
            f = gpu.qmatmul_ragged_swiglu if pair else gpu.qmatmul_ragged
            return f(*tables, x, off, rows=rows, out_dtype=DT[ydt])

        first = call()
        y, b = products(W[0], t, x, counts, src)
        if pair:
            y, b = swiglu(y, b, *products(W[1], t, x, counts, src))
        check(first, y, b)
        again = [call() for _ in range(12)]
        gpu.stream_sync()
        assert all(torch.equal(a, first) for a in again)
    finally:
        release(tables, weights)


GATES = [0.0, -0.0, 1e-3, -1e-3, 1.0, -1.0, 60.0, -60.0, 88.0, -86.5, -87.25, -87.5, -88.0, -88.5, -88.6875, -89.0,
         -100.0, -120.0, 1000.0, -1000.0]


@pytest.mark.parametrize("u", [1.0, -3.0, 96.0])
@pytest.mark.parametrize("kernel", KERNELS.keys())
def test_swiglu_of_far_gates(gpu, kernel, u):
    """silu over the whole range of its exponential, in every product kernel.

    Weights are 0 and 1, so the gate and up values are the activations, exactly.  In half steps of fp32
    (2^-24): expf is within 2 units in the last place (4), the sum within half of one (1), the quotient within 2
    in the tcgen05 kernel's fast division (4), the product within half of one (1).  Where exp(-g) passes the
    fp32 range the quotient is 0: off by at most |g| 2^-128.
    """
    N, K = 128, 32
    def blocks(k):  # w[n][k] = 1, all else 0
        if kernel == "exact":
            b = np.zeros((N, 1, K), np.float16)
            b[:, :, k] = 1
            return b.view(np.uint8)
        b = np.zeros((N, 1, 18), np.uint8)  # Q4_0: a half scale, then 16 bytes of codes, (code - 8) * scale
        b[:, :, :2] = np.array([1], np.float16).view(np.uint8)
        b[:, :, 2:] = 0x88
        b[:, :, 2 + k] = 0x89
        return b

    t = 121 if kernel == "exact" else 2
    per = 4 if kernel == "warp" else len(GATES)  # slots per expert
    E = len(GATES) // per
    gate, up = (gpu.Weight.register(blocks(k), t, N, K) for k in (0, 1))
    G, Up = gpu.Experts([gate] * E), gpu.Experts([up] * E)
    try:
        x = torch.zeros((len(GATES), K), device="cuda", dtype=torch.float16)
        x[:, 0], x[:, 1] = torch.tensor(GATES), u
        got = gpu.qmatmul_ragged_swiglu(G, Up, x, make_offsets([per] * E)).double()
        gpu.stream_sync()
        g = x[:, :1].double()
        want = g / (1 + torch.exp(-g)) * u
        lost = torch.where(g < -88.7, g.abs() * abs(u) * 2.0 ** -128, 0.0)
        err = (got - want).abs()
        bad = (err > 10 * 2.0 ** -24 * want.abs() + lost).any(1)
        assert not bool(bad.any()), [(a.item(), b[0].item()) for a, b in zip(g[bad][:, 0], got[bad])]
    finally:
        release([G, Up], [gate, up])


@pytest.mark.parametrize("hdt", DT.keys())
@pytest.mark.parametrize("k,N", [(1, 64), (1, 4096), (2, 1536), (2, 2560), (8, 64), (8, 1024), (8, 1536), (8, 1544),
                                 (8, 2048), (16, 1344), (16, 1352), (32, 128), (32, 1248)])
def test_combine_of_many_tokens(gpu, k, N, hdt):
    """Rows on both sides of the size from which many tokens are combined by bulk copies."""
    T = 5 * torch.cuda.get_device_properties(0).multi_processor_count + 3
    g = torch.Generator(device="cuda").manual_seed(N + k)
    h = torch.randn((T * k, N), device="cuda", generator=g).to(DT[hdt])
    slots = torch.randperm(T * k, device="cuda", generator=g).to(torch.int32).view(T, k)
    w = torch.rand((T, k), device="cuda", generator=g)
    slots[torch.rand((T, k), device="cuda", generator=g) < 0.2] = -1
    res = torch.randn((T, N), device="cuda", generator=g)
    parts = h[slots.clamp(min=0).long()].double() * (w * (slots >= 0)).double()[:, :, None]
    bound = (k + 2) * 2.0 ** -24 * (parts.abs().sum(1) + res.double().abs())
    for dt in DT.values():
        check(gpu.moe_combine(h, slots, w, res=res, out_dtype=dt), parts.sum(1) + res.double(), bound)
    gpu.stream_sync()


@pytest.mark.parametrize("power", [-12, -16, -20, -24])
@pytest.mark.parametrize("xdt", DT.keys())
@pytest.mark.parametrize("kernel", KERNELS.keys())
def test_small_activations(gpu, kernel, xdt, power):
    """fp32 and bf16 activations below 2^-14 are rounded to multiples of 2^-24 where products run in f16: each
    is off by at most 2^-25 (and by 2^-11 of itself above), which the weights carry into the sum.  f16
    activations, and the exact kernel, lose nothing."""
    t, m = KERNELS[kernel]
    E, N, K = 3, 128, 256
    ws, W = make_weights(gpu, t, E, N, K, 6)
    T = gpu.Experts(ws)
    try:
        x = (2.0 ** power * torch.randn((E * m, K), device="cuda")).to(DT[xdt])
        y, b = products(W, t, x, [m] * E, torch.arange(E * m, device="cuda"))
        if xdt != "f16" and t not in EXACT:
            b = b + 2.0 ** -25 * 1.01 * W.abs().sum(2).repeat_interleave(m, 0)
        got = gpu.qmatmul_ragged(T, x, make_offsets([m] * E)).double()
        gpu.stream_sync()
        # Sums of f16 products are multiples of 2^-48, far above the smallest fp32.
        assert bool(((got - y).abs() <= b + 2.0 ** -24 * (y.abs() + b)).all())
    finally:
        release([T], ws)


CHOICE = """
import sys, torch
sys.path[:0] = [{tests!r}, {pkg!r}, {root!r}]
import nxq
from test_gpu_moe import make_offsets, make_weights, products, swiglu
nxq.init(0)
decode, prefill = {decode}, {prefill}  # whether each is the exact kernel
for counts in ([2, 0, 3, 1], [40, 3, 0, 130]):
    n = sum(counts)
    exact = decode and prefill
    ws, W = make_weights(nxq, 12, 4, 200, 512, 6)
    T = nxq.Experts(ws)
    x = 0.05 * torch.randn((n, 512), device="cuda")
    x[0, 0] = 1e-9  # zero in f16
    x[n - 1, 1] = 1e5 if exact else 1.0  # beyond f16
    off = make_offsets(counts)
    got, pair = nxq.qmatmul_ragged(T, x, off), nxq.qmatmul_ragged_swiglu(T, T, x, off)
    nxq.stream_sync()
    y, b = products(W, 121 if exact else 12, x, counts, torch.arange(n, device="cuda"))
    if not exact:
        b = b + 2.0 ** -25 * 1.01 * W.abs().sum(2).max()
    assert bool(((got.double() - y).abs() <= b + 2.0 ** -24 * y.abs()).all()), counts
    h, hb = swiglu(y, b, y, b)
    assert bool(((pair.double() - h).abs() <= hb + 2.0 ** -24 * h.abs()).all()), counts
"""


@pytest.mark.parametrize("decode", [False, True], ids=["", "decode-simt"])
@pytest.mark.parametrize("prefill", [False, True], ids=["", "prefill-simt"])
def test_kernel_choice_by_environment(gpu, decode, prefill):
    """NXQ_DECODE_KERNEL / NXQ_PREFILL_KERNEL = simt: with both, the exact kernel takes every call and f16's
    range does not apply; with one, the other tensor-core kernel takes the calls or the exact one does."""
    env = {k: v for k, v in os.environ.items() if k not in ("NXQ_DECODE_KERNEL", "NXQ_PREFILL_KERNEL")}
    env.update({"NXQ_DECODE_KERNEL": "simt"} if decode else {}, **({"NXQ_PREFILL_KERNEL": "simt"} if prefill else {}))
    code = CHOICE.format(tests=str(ROOT / "tests"), pkg=str(PKG), root=str(ROOT), decode=decode, prefill=prefill)
    r = subprocess.run([sys.executable, "-c", code], env=env, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
