"""What INTEGRATION.md shows of attention runs as it stands there."""
from __future__ import annotations

import re
from pathlib import Path

import pytest
import torch

import nxq

DOC = (Path(__file__).resolve().parents[1] / "INTEGRATION.md").read_text()
SECTION = DOC[DOC.index("## Attention over a paged cache"):].split("\n## ", 1)[0]
BLOCKS = re.findall(r"```python\n(.*?)```", SECTION, re.S)
INLINE = re.findall(r"`(nxq\.Rope\([^`]*\))`", SECTION)


def rope_lines():
    """The Python that makes a rotation, one piece of code each."""
    code = [c.replace("...", "64") for c in INLINE]
    for b in BLOCKS:
        code.append("\n".join(x for x in b.splitlines() if "rope_frequencies(" in x or "nxq.Rope(" in x))
    return [c for c in code if "Rope(" in c]


def test_rotations_are_made_as_documented():
    assert rope_lines()
    for code in rope_lines():
        try:
            exec(code, {"nxq": nxq})
        except nxq.NxqError as e:  # (nothing but the GPU may be missing)
            assert e.name in ("ERR_STATE", "ERR_UNSUPPORTED"), f"{code}: {e}"


@pytest.mark.gpu
def test_a_step_runs_as_documented(gpu):
    assert len(BLOCKS) == 1
    g = torch.Generator(device="cuda").manual_seed(1)
    rand = lambda *s: torch.randn(s, generator=g, device="cuda").bfloat16()  # noqa: E731
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    names = dict(nxq=gpu, torch=torch, keys=rand(9, 2, 16, 128), values=rand(9, 2, 16, 128), q=rand(5, 8, 128), k=rand(5, 2, 128),
                 v=rand(5, 2, 128), q_offsets=i32([0, 1, 5]), kv_lens=i32([30, 50]), block_table=i32([[3, 1, 0, 0], [8, 2, 7, 5]]))
    exec(BLOCKS[0], names)
    gpu.stream_sync()
    assert names["a"].shape == (5, 8, 128) and torch.isfinite(names["a"]).all()
    names["rope"].release()
