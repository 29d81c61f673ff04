"""GPU: attention over a paged cache at its edges, against a plain 64-bit computation."""
from __future__ import annotations

import math

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
