"""CPU: the embedding and mixture-of-experts entry points refuse bad arguments
before they touch a GPU (no device is needed, nothing is launched)."""
from __future__ import annotations

import ctypes

import pytest
import torch

import nxq

ARG, SHAPE, STATE, UNSUPPORTED = -1, -3, -7, -9
P = ctypes.c_void_p(256)  # a non-null pointer that is never followed


def route(T=4, E=8, k=2, dtype=nxq.F32, arrays=(P, P, P, P, P, P)):
    logits, ids, weights, offsets, rows, slots = arrays
    return nxq.lib().nxq_moe_route(logits, dtype, T, E, k, 1, ids, weights, offsets, rows, slots, None)


@pytest.mark.parametrize("kw", [dict(E=0), dict(E=1025), dict(k=0), dict(k=9), dict(E=64, k=33), dict(T=-1),
                                dict(T=2**30, k=2), dict(dtype=3), dict(dtype=-1)])
def test_route_refuses(kw):
    assert route(**kw) == ARG


@pytest.mark.parametrize("i", range(6))
def test_route_refuses_null_arrays(i):
    arrays = [P] * 6
    arrays[i] = None
    assert route(arrays=arrays) == ARG


def combine(R=8, N=16, T=4, k=2, h_dtype=nxq.F16, y_dtype=nxq.F32, h=P, slots=P, w=P, res=None, y=P):
    return nxq.lib().nxq_moe_combine(h, h_dtype, R, N, slots, w, T, k, res, y, y_dtype, None)


@pytest.mark.parametrize("kw", [dict(R=-1), dict(R=2**31), dict(N=-1), dict(T=-1), dict(k=0), dict(k=33), dict(h_dtype=7),
                                dict(y_dtype=7), dict(h=None), dict(slots=None), dict(w=None), dict(y=None),
                                dict(res=P, y_dtype=nxq.BF16)])
def test_combine_refuses(kw):
    assert combine(**kw) == ARG


def test_nothing_to_do_is_no_error_without_a_gpu():
    assert combine(T=0) == 0
    assert combine(N=0) == 0


def test_handles_are_checked():
    L = nxq.lib()
    h = ctypes.c_void_p()
    null = (ctypes.c_void_p * 1)(None)
    assert L.nxq_experts_create(None, 1, ctypes.byref(h)) == ARG
    assert L.nxq_experts_create(null, 0, ctypes.byref(h)) == ARG
    assert L.nxq_experts_create(null, 1025, ctypes.byref(h)) == ARG
    assert L.nxq_experts_create(null, 1, None) == ARG
    assert L.nxq_experts_create(null, 1, ctypes.byref(h)) == ARG  # null weight
    for bad in (None, P):  # null and foreign tables
        assert L.nxq_experts_release(bad) == ARG
        assert L.nxq_experts_info(bad, None, None, None, None) == ARG
        assert L.nxq_qmatmul_ragged(bad, P, nxq.F16, 1, None, P, nxq.F32, 1, P, None) == ARG
        assert L.nxq_qmatmul_ragged_swiglu(bad, bad, P, nxq.F16, 1, None, P, nxq.F32, 1, P, None) == ARG
    assert L.nxq_embedding(None, P, nxq.I32, 1, 1.0, P, nxq.F32, None) == ARG


def test_route_before_init():
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    assert route() in (STATE, UNSUPPORTED)


class _Fake:
    """Stands in for a table of experts: the binding reads its shape only."""

    N, K, count, type = 128, 256, 2, 12

    @property
    def handle(self):
        raise AssertionError("the call was not refused")


class _FakeWeight(_Fake):
    pass


@pytest.mark.parametrize("call", [
    lambda: nxq.embedding(_FakeWeight(), torch.zeros(3)),                                       # ids not integers
    lambda: nxq.embedding(_FakeWeight(), torch.zeros(3, dtype=torch.int64)),                    # not on the GPU
    lambda: nxq.moe_route(torch.zeros(4, 8, dtype=torch.float64), 2),                           # logits' type
    lambda: nxq.moe_route(torch.zeros(8), 2),                                                   # one dimension
    lambda: nxq.moe_route(torch.zeros(4, 8), 2),                                                # not on the GPU
    lambda: nxq.qmatmul_ragged(_Fake(), torch.zeros(4, 128), torch.zeros(3, dtype=torch.int32)),  # K
    lambda: nxq.qmatmul_ragged(_Fake(), torch.zeros(4, 256), torch.zeros(3)),                   # offsets' type
    lambda: nxq.qmatmul_ragged(_Fake(), torch.zeros(4, 256), torch.zeros(3, dtype=torch.int32)),  # not on the GPU
    lambda: nxq.moe_combine(torch.zeros(8, 16), torch.zeros(4, 2), torch.zeros(4, 2)),          # slots' type
    lambda: nxq.moe_combine(torch.zeros(8, 16), torch.zeros(4, 2, dtype=torch.int32), torch.zeros(4, 3)),  # weights' shape
    lambda: nxq.moe_combine(torch.zeros(8, 16), torch.zeros(4, 2, dtype=torch.int32), torch.zeros(4, 2),
                            res=torch.zeros(4, 15)),                                            # residual's shape
    lambda: nxq.Experts([]),
])
def test_binding_refuses(call):
    with pytest.raises(nxq.NxqError) as e:
        call()
    assert e.value.code == ARG
