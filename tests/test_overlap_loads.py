"""CPU: kernels that start while the one before them drains promise the compiler
nothing about memory which that one may still be writing.

A load by the non-coherent path (__ldg, const __restrict__) needs its memory
unchanged for the whole life of the kernel, and such a kernel's life begins
before its inputs are complete.  Only registered weights (`tiled`) are.
"""
from __future__ import annotations

import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "nexus-inference-engine-_b200" / "csrc"


def overlapped_kernels():
    for path in sorted(CSRC.glob("*.cu")):
        text = re.sub(r"//[^\n]*", "", path.read_text())
        for body in text.split("__global__")[1:]:
            body = body.split("\n}\n")[0]
            if "overlap_begin()" in body:
                name = re.search(r"\b(\w+_kernel)\b", body).group(1)
                yield pytest.param(body, id=f"{path.stem}:{name}")


KERNELS = list(overlapped_kernels())


def test_kernels_are_found():
    assert len(KERNELS) >= 9


@pytest.mark.parametrize("body", KERNELS)
def test_no_read_only_loads(body):
    assert "__ldg" not in body and "ld.global.nc" not in body
    restricted = re.findall(r"__restrict__\s+(\w+)", body)
    assert set(restricted) <= {"tiled"}, restricted


def test_no_read_only_loads_in_their_helpers():
    for path in CSRC.glob("*.cu"):
        if "overlap_begin()" in path.read_text():
            assert "__ldg(" not in path.read_text(), path.name
