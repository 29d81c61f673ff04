"""CPU: the rotation and attention entry points refuse bad arguments before they touch
a GPU (nothing is launched), and the frequencies of the rotations are the formulas'."""
from __future__ import annotations

import ctypes
import math
import struct

import numpy as np
import pytest
import torch

import nxq

ARG, SHAPE, STATE, UNSUPPORTED = -1, -3, -7, -9
P = 4096  # a non-null, aligned address that is never followed


def heads(dev=P, n=4, token=256, head=64):
    return nxq._HEADS(dev, n, token, head)


def cache(k=P, v=P, dtype=nxq.F16, pages=8, page=16, n=2, D=64, page_stride=2048, head_stride=1024, slot_stride=64):
    return nxq._CACHE(k, v, dtype, pages, page, n, D, page_stride, head_stride, slot_stride)


def batch(S=2, q=P, lens=P, table=P, stride=4, pages=4):
    return nxq._BATCH(S, q, lens, table, stride, pages)


def rope(r=None, positions=P, ptype=nxq.I32, T=3, D=64, q=heads(), q_norm=None, k=None, k_norm=None, x=nxq.F16, q_out=heads(),
         k_out=None, y=nxq.F16):
    return nxq.lib().nxq_rope(r, positions, ptype, T, D, q, q_norm, k, k_norm, 1e-6, x, q_out, k_out, y, None)


def append(c=cache(), b=batch(), T=3, k=heads(n=2), v=heads(n=2), k_norm=None, r=None, q=None, q_norm=None, x=nxq.F16, q_out=None,
           y=nxq.F16):
    return nxq.lib().nxq_kv_append(c, b, T, k, v, k_norm, r, q, q_norm, 1e-6, x, q_out, y, None)


def attention(c=cache(), b=batch(), q=heads(), T=3, scale=0.125, window=0, sinks=0, max_new=0, out=heads(), y=nxq.F16, lse=None):
    return nxq.lib().nxq_paged_attention(c, b, q, T, scale, window, sinks, max_new, out, y, lse, None)


@pytest.mark.parametrize("kw", [
    dict(q=None), dict(q_out=None), dict(q=heads(dev=0)), dict(q=heads(n=0)), dict(q=heads(token=-1)), dict(q=heads(head=-8)),
    dict(q=heads(dev=P + 1)), dict(q_out=heads(dev=P + 2), y=nxq.F32), dict(T=-1), dict(T=2**31), dict(D=0), dict(D=513),
    dict(x=3), dict(y=-1), dict(k=heads()), dict(k_out=heads()), dict(q_norm=P + 2), dict(ptype=2), dict(r=P), dict(r=P, positions=None)])
def test_rope_refuses(kw):
    assert rope(**kw) == ARG


def test_rope_refuses_shapes():
    assert rope(q_out=heads(n=5)) == SHAPE
    assert rope(k=heads(n=2), k_out=heads(n=3)) == SHAPE


CACHES = [cache(k=0), cache(v=0), cache(dtype=nxq.F32), cache(pages=-1), cache(pages=0), cache(page=0), cache(n=0), cache(k=P + 8), cache(v=P + 2),
          cache(page_stride=0), cache(head_stride=4), cache(slot_stride=-64), None]
BATCHES = [batch(S=0), batch(S=65537), batch(q=0), batch(lens=0), batch(table=0), batch(stride=-1), batch(pages=-1), batch(q=P + 2),
           batch(lens=P + 1), batch(table=P + 3), None]


@pytest.mark.parametrize("c", CACHES)
def test_bad_caches(c):
    assert append(c=c) == ARG and attention(c=c) == ARG


@pytest.mark.parametrize("D", [0, 4, 60, 264, 512])
def test_bad_head_sizes(D):
    assert append(c=cache(D=D)) == SHAPE and attention(c=cache(D=D)) == SHAPE


@pytest.mark.parametrize("b", BATCHES)
def test_bad_batches(b):
    assert append(b=b) == ARG and attention(b=b) == ARG


@pytest.mark.parametrize("kw,code", [
    (dict(k=None), ARG), (dict(v=None), ARG), (dict(k=heads(n=4)), SHAPE), (dict(v=heads(n=1)), SHAPE), (dict(T=-1), ARG),
    (dict(T=2**30 + 1), ARG), (dict(q=heads()), ARG), (dict(q_out=heads()), ARG), (dict(x=9), ARG), (dict(r=P), ARG),
    (dict(q=heads(), q_out=heads(n=3)), SHAPE), (dict(k_norm=P + 1), ARG), (dict(k=heads(n=2, dev=P + 1)), ARG)])
def test_append_refuses(kw, code):
    assert append(**kw) == code


@pytest.mark.parametrize("kw,code", [
    (dict(q=None), ARG), (dict(out=None), ARG), (dict(q=heads(n=3), out=heads(n=3)), SHAPE), (dict(out=heads(n=2)), SHAPE),
    (dict(T=-1), ARG), (dict(T=2**30 + 1), ARG), (dict(scale=0.0), ARG), (dict(scale=-1.0), ARG), (dict(scale=math.inf), ARG),
    (dict(scale=math.nan), ARG), (dict(window=-1), ARG), (dict(sinks=-1), ARG), (dict(max_new=-1), ARG), (dict(y=3), ARG),
    (dict(lse=P + 2), ARG), (dict(q=heads(dev=P + 1)), ARG), (dict(out=heads(dev=P + 2), y=nxq.F32), ARG),
    (dict(q=heads(n=16), out=heads(n=16), T=2**29), SHAPE)])
def test_attention_refuses(kw, code):
    assert attention(**kw) == code


Q2 = P + 4096


@pytest.mark.parametrize("y,other", [(nxq.F32, {}), (nxq.BF16, {}), (nxq.F16, dict(token=512)), (nxq.F16, dict(head=128))])
def test_in_place_only_where_each_head_lay(y, other):
    assert rope(q_out=heads(**other), y=y) == ARG
    assert rope(q_out=heads(dev=Q2), k=heads(), k_out=heads(**other), y=y) == ARG
    assert append(q=heads(), q_out=heads(**other), y=y) == ARG
    assert attention(out=heads(**other), y=y) == ARG
    # Strides that no address depends on may differ.
    if not torch.cuda.is_available():
        assert attention(T=1, out=heads(token=512)) in (STATE, UNSUPPORTED)
        assert rope(T=1, q_out=heads(token=512)) in (STATE, UNSUPPORTED)


def test_scale_beyond_fp32_with_its_logarithm():
    assert attention(scale=3e38) == ARG


def test_nothing_to_do_is_no_error_without_a_gpu():
    assert rope(T=0) == 0 and append(T=0) == 0 and attention(T=0) == 0


def test_good_arguments_before_init():
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    for rc in (rope(), append(), attention()):
        assert rc in (STATE, UNSUPPORTED)
    with pytest.raises(nxq.NxqError) as e:
        nxq.Rope([1.0, 0.5])
    assert e.value.code in (STATE, UNSUPPORTED)


def test_rope_handles():
    h = ctypes.c_void_p()
    f = np.array([1.0, 0.1])
    create = nxq.lib().nxq_rope_create
    assert create(None, 4, 0, 1.0, ctypes.byref(h)) == ARG
    assert create(f.ctypes.data, 4, 0, 1.0, None) == ARG
    for dims in (0, 3, 514, -2):
        assert create(f.ctypes.data, dims, 0, 1.0, ctypes.byref(h)) == ARG
    assert create(f.ctypes.data, 4, 2, 1.0, ctypes.byref(h)) == ARG
    assert create(f.ctypes.data, 4, 0, math.nan, ctypes.byref(h)) == ARG
    f[1] = math.inf
    assert create(f.ctypes.data, 4, 0, 1.0, ctypes.byref(h)) == ARG
    for bad in (None, P):
        assert nxq.lib().nxq_rope_release(bad) == ARG


# ---- frequencies ----------------------------------------------------------------------

@pytest.mark.parametrize("dims,base", [(128, 10000.0), (64, 500000.0), (2, 10000.0), (96, 1e6)])
def test_frequencies(dims, base):
    i = np.arange(dims // 2)
    plain = base ** (-2.0 * i / dims)
    inv, scale = nxq.rope_frequencies(dims, base)
    assert scale == 1.0 and np.allclose(inv, plain, rtol=1e-14)
    inv, scale = nxq.rope_frequencies(dims, base, "linear", factor=4.0)
    assert scale == 1.0 and np.allclose(inv, plain / 4, rtol=1e-14)
    if dims > 2:
        inv, _ = nxq.rope_frequencies(dims, base, "ntk", factor=4.0)
        assert np.allclose(inv, (base * 4.0 ** (dims / (dims - 2))) ** (-2.0 * i / dims), rtol=1e-13)
        # The slowest pair is slowed by the factor, the fastest kept.
        assert inv[0] == 1.0 and math.isclose(inv[-1], plain[-1] / 4, rel_tol=1e-12)
    # By wavelength: long ones divided, short ones kept, the share of turns between them.
    inv, scale = nxq.rope_frequencies(dims, base, "blend", factor=8.0, trained=8192.0)
    turns = 8192.0 * plain / (2 * math.pi)
    share = np.clip((turns - 1.0) / 3.0, 0.0, 1.0)
    assert scale == 1.0 and np.allclose(inv, (1 - share) * plain / 8 + share * plain, rtol=1e-13)
    assert np.allclose(inv[turns > 4], plain[turns > 4], rtol=1e-14) and np.allclose(inv[turns < 1], plain[turns < 1] / 8, rtol=1e-14)


def test_yarn():
    dims, base, factor, trained = 128, 10000.0, 16.0, 4096.0
    inv, scale = nxq.rope_frequencies(dims, base, "yarn", factor=factor, trained=trained)
    assert math.isclose(scale, 0.1 * math.log(factor) + 1, rel_tol=1e-6)
    plain = base ** (-2.0 * np.arange(64) / dims)
    index = lambda turns: dims * math.log(trained / (turns * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
    lo, hi = math.floor(index(32)), math.ceil(index(1))
    assert np.allclose(inv[:lo + 1], plain[:lo + 1], rtol=1e-14) and np.allclose(inv[hi:], plain[hi:] / factor, rtol=1e-14)
    mid = np.arange(lo, hi + 1)
    ramp = (mid - lo) / (hi - lo)
    assert np.allclose(inv[mid], plain[mid] / factor * ramp + plain[mid] * (1 - ramp), rtol=1e-13)
    assert nxq.rope_frequencies(dims, base, "yarn", factor=1.0, trained=trained)[1] == 1.0


@pytest.mark.parametrize("kw", [dict(dims=3), dict(dims=0), dict(dims=514), dict(base=1.0), dict(base=math.nan), dict(scaling="other"),
                                dict(scaling="linear", factor=0.5), dict(scaling="yarn", factor=4.0),
                                dict(scaling="blend", factor=4.0, trained=8192.0, low=4.0, high=1.0), dict(scaling="ntk", dims=2, factor=2.0)])
def test_frequencies_refuse(kw):
    with pytest.raises(nxq.NxqError) as e:
        nxq.rope_frequencies(**{"dims": 64, **kw})
    assert e.value.code == ARG


# ---- the binding ------------------------------------------------------------------------

def test_structures_are_the_header_s():
    # Their sizes and the offsets of their last fields, as a C compiler lays them out on this ABI.
    assert struct.calcsize("Pi4xqq") == 32 and struct.calcsize("PPi4xqiii4xqqq") == 72 and struct.calcsize("i4xPPPqq") == 48


Z = torch.zeros
I32 = torch.int32


@pytest.mark.parametrize("call", [
    lambda: nxq.rope(None, None, Z(3, 4)),                                              # two dimensions
    lambda: nxq.rope(None, None, Z(3, 4, 64)),                                          # not on the GPU
    lambda: nxq.KVCache(Z(2, 2, 16, 64), Z(2, 2, 16, 64), order="other"),
    lambda: nxq.KVCache(Z(2, 2, 16, 64), Z(2, 2, 16, 64)),                              # fp32
    lambda: nxq.KVCache(Z(2, 2, 16, 64).half(), Z(2, 2, 16, 32).half()),                # unlike
    lambda: nxq.KVCache(Z(2, 2, 16, 64).half(), Z(2, 2, 16, 64).bfloat16()),
    lambda: nxq.KVCache(Z(2, 16, 64).half(), Z(2, 16, 64).half()),
    lambda: nxq.KVCache(Z(2, 2, 16, 64).half(), Z(2, 2, 16, 64).half()),                # not on the GPU
    lambda: nxq.Rope([[1.0]]),
    lambda: nxq.Rope([1.0], layout="other"),
])
def test_binding_refuses(call):
    with pytest.raises(nxq.NxqError) as e:
        call()
    assert e.value.code == ARG
