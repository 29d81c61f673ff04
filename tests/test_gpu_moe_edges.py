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
