"""CPU: mixture-of-experts calls refuse arrays that are not aligned to their element type
(an access across that boundary would be a fault on the GPU; nothing is launched here)."""
from __future__ import annotations

import ctypes

import pytest

import nxq

ARG = -1
P = 256  # a non-null, aligned address that is never followed
SIZE = {nxq.F32: 4, nxq.F16: 2, nxq.BF16: 2}
TYPES = sorted(SIZE)


def refused(rc):
    return rc == ARG and "aligned" in nxq.last_error()


def pointers(n, bad, by):
    return [ctypes.c_void_p(P + (by if i == bad else 0)) for i in range(n)]


@pytest.mark.parametrize("T", [1, 4, 1000])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bad", range(6))
def test_route(bad, dtype, T):
    for by in range(1, SIZE[dtype] if bad == 0 else 4):
        logits, *outs = pointers(6, bad, by)
        assert refused(nxq.lib().nxq_moe_route(logits, dtype, T, 8, 2, 1, *outs, None)), by


def test_route_no_tokens():
    none = ctypes.c_void_p()
    assert refused(nxq.lib().nxq_moe_route(none, nxq.F32, 0, 8, 2, 1, none, none, ctypes.c_void_p(P + 2), none, none, None))


@pytest.mark.parametrize("hd", TYPES)
@pytest.mark.parametrize("yd", TYPES)
@pytest.mark.parametrize("bad", range(5))
def test_combine(bad, yd, hd):
    for by in range(1, {0: SIZE[hd], 4: SIZE[yd]}.get(bad, 4)):
        h, slots, w, res, y = pointers(5, bad, by)
        y = ctypes.c_void_p(y.value + 4096)  # not the residual itself
        assert refused(nxq.lib().nxq_moe_combine(h, hd, 8, 16, slots, w, 4, 2, res, y, yd, None)), by
