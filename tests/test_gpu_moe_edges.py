"""GPU: the mixture-of-experts and embedding calls at the edges of what they take.

Bounds as in test_gpu_moe.py, whose helpers are used here.
"""
from __future__ import annotations

import pytest
import torch

from test_gpu_moe import DT, make_weights, products

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
