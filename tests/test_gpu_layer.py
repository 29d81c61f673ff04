"""GPU: a layer's attention half from projections to residual, through the library's calls.

Every stage is held to its own bound on what the stage before gave: products to the
library's bar of 1e-3 (relative 2-norm), rotations and attention to the bounds of
their own tests, so nothing hides behind anything.
"""
from __future__ import annotations

import pytest
import torch

from attention_cases import Paged
from nxq import synth
from test_gpu_rope import check, turned

pytestmark = pytest.mark.gpu

HIDDEN, HQ, HK, D, PAGE = 512, 8, 2, 64, 16


class Layer:
    def __init__(self, nxq):
        t = nxq.TYPES["Q4_K"]
        shapes = {"q": (HQ * D, HIDDEN), "k": (HK * D, HIDDEN), "v": (HK * D, HIDDEN), "o": (HIDDEN, HQ * D)}
        self.w = {n: nxq.Weight.register(synth.make_blocks(t, *s, seed=i), t, *s) for i, (n, s) in enumerate(shapes.items())}
        self.norm = 1 + 0.1 * torch.rand(HIDDEN, device="cuda")
        self.q_norm, self.k_norm = 1 + 0.1 * torch.rand(D, device="cuda"), 1 + 0.1 * torch.rand(D, device="cuda")
        self.inv, scale = nxq.rope_frequencies(D, 10000.0, "blend", factor=8.0, trained=8192.0)
        self.rope = nxq.Rope(self.inv, "half", scale)

    def __call__(self, nxq, p, x, out=None):
        """The residual stream after attention, and what lay between."""
        T = x.shape[0]
        q, k, v = nxq.rmsnorm_qmatmul([self.w[n] for n in "qkv"], x, self.norm, 1e-5, out_dtype=torch.float16)
        q, k, v = q.view(T, HQ, D), k.view(T, HK, D), v.view(T, HK, D)
        r = nxq.kv_append(p.cache, k, v, p.q_offsets, p.kv_lens, p.table, rope=self.rope, q=q, q_norm=self.q_norm, k_norm=self.k_norm,
                          out_dtype=torch.float16)
        a = nxq.paged_attention(r, p.cache, p.q_offsets, p.kv_lens, p.table, out_dtype=torch.float16)
        y = nxq.qmatmul_residual(self.w["o"], a.view(T, HQ * D), x, out=out)
        return q, k, v, r, a, y

    def release(self):
        self.rope.release()
        for w in self.w.values():
            w.release()


def bar(got, want):
    assert float((got.double() - want).norm() / want.norm()) <= 1e-3


def verify(layer, p, x, stages):
    q, k, v, r, a, y = stages
    W = {n: w.dequant().double() for n, w in layer.w.items()}
    xn = x.double() / ((x.double() ** 2).mean(-1, keepdim=True) + 1e-5).sqrt() * layer.norm.double()
    for n, got in (("q", q), ("k", k), ("v", v)):
        bar(got.reshape(len(x), -1), xn @ W[n].T)
    pos = torch.cat([torch.arange(t - n, t, device="cuda") for n, t in zip(p.new, p.total)])
    check(r, *turned(q, layer.q_norm, 1e-6, layer.rope, layer.inv, pos))
    want_k, bound = turned(k, layer.k_norm, 1e-6, layer.rope, layer.inv, pos)
    at = 0
    for i, (n, t) in enumerate(zip(p.new, p.total)):
        pages, slots = p.places(i)
        p.k[i], p.v[i] = p.view(p.keys)[pages, slots], p.view(p.values)[pages, slots]
        check(p.k[i][t - n:], want_k[at:at + n], bound[at:at + n])
        assert torch.equal(p.v[i][t - n:], v[at:at + n])
        at += n
    p.q, p.T = r, len(x)
    p.check(a)
    bar(y, a.reshape(len(x), -1).double() @ W["o"].T + x.double())


def test_prompt_then_single_tokens(gpu):
    layer = Layer(gpu)
    steps, prompts = 4, [70, 33, 200]
    # Room for the tokens to come; lengths as of the prompt.
    p = Paged(gpu, prompts, [n + steps for n in prompts], HQ, HK, D, PAGE, torch.float16, seed=1)
    p.keys.fill_(float("nan")), p.values.fill_(float("nan"))
    p.total = list(prompts)
    p.kv_lens.copy_(torch.tensor(prompts, dtype=torch.int32))
    x = torch.randn((sum(prompts), HIDDEN), device="cuda")
    stages = layer(gpu, p, x)
    gpu.stream_sync()
    verify(layer, p, x, stages)

    # Single tokens: the step is captured once and replayed with the lengths on the device.
    S = len(prompts)
    p.new = [1] * S
    p.q_offsets = torch.arange(S + 1, dtype=torch.int32, device="cuda")
    x = torch.zeros((S, HIDDEN), device="cuda")
    p.kv_lens += 1
    layer(gpu, p, x)  # (workspaces of the products)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        layer(gpu, p, x)
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=s):
        stages = layer(gpu, p, x)
    for step in range(steps):
        p.total = [n + step + 1 for n in prompts]
        p.kv_lens.copy_(torch.tensor(p.total, dtype=torch.int32))
        x.copy_(torch.randn((S, HIDDEN), device="cuda"))
        g.replay()
        gpu.stream_sync()
        torch.cuda.synchronize()
        verify(layer, p, x, stages)
    del g
    layer.release()
