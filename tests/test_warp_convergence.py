"""CPU: warps are whole where the attention kernel touches tensor memory.

tcgen05.ld, .st and their waits are .sync.aligned: all lanes of a warp run them
together.  After a branch that only some lanes take (rows behind an item's end, one
lane's arrival) the source says where they meet again, instead of leaving that to
the compiler.  The scan walks the kernel's text in order, loop bodies twice, so that a
branch at the end of a body is followed by the body's start.
"""
from __future__ import annotations

import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "nexus-inference-engine-_b200" / "csrc"
# Conditions that differ between the lanes of a warp.
PARTS = re.compile(r"\bif\s*(?:constexpr\s*)?\((?P<cond>(?:[^()]|\((?:[^()]|\([^()]*\))*\))*)\)")
LANE = re.compile(r"\b(mine|lane|row|threadIdx|sees)\b")
MEETS = re.compile(r"__syncwarp|__syncthreads|warp_mbar_wait|\b__\w+_sync\(")
WHOLE = re.compile(r"\btmem_(?:ld|st|wait|alloc|dealloc)\w*\(")


def block_end(text, i):
    """Index behind the block or statement that starts at i."""
    depth = 0
    while True:
        c = text[i]
        if c in "({":
            depth += 1
        elif c in ")}":
            depth -= 1
            if depth == 0 and c == "}":
                return i + 1
        elif c == ";" and depth == 0:
            return i + 1
        i += 1


def unrolled(text):
    """The text with every loop body that touches tensor memory written twice."""
    out, i = "", 0
    while True:
        m = re.compile(r"\b(?:for|while)\s*\(").search(text, i)
        if not m:
            return out + text[i:]
        depth, k = 0, m.end() - 1
        while True:  # the loop's head
            depth += {"(": 1, ")": -1}.get(text[k], 0)
            k += 1
            if depth == 0:
                break
        end = block_end(text, k)
        body = unrolled(text[k:end])
        out += text[i:k] + body + (body if WHOLE.search(body) else "")
        i = end


def faults(text):
    """Places where lanes that parted touch tensor memory before they have met."""
    text = re.sub(r"//[^\n]*", "", text)
    text = unrolled(text)
    marks = [(m.start(), "part") for m in PARTS.finditer(text) if LANE.search(m["cond"])]
    marks += [(m.start(), "meet") for m in MEETS.finditer(text)] + [(m.start(), "whole") for m in WHOLE.finditer(text)]
    parted, bad = None, []
    for at, what in sorted(marks):
        if what == "part":
            parted = at
        elif what == "meet":
            parted = None
        elif parted is not None:
            bad.append(text[parted:at + 20].strip())
            parted = None
    return bad


def softmax_warps():
    text = (CSRC / "attn_tc.cu").read_text()
    start = text.index("} else if (warp >= kWarpSoft0) {")
    return text[start:text.index("    __syncthreads();", start)]


def test_the_scan_finds_them():
    assert faults("for (int d = 0; d < 4; ++d) { ptx::tmem_ld8(a, o); if (!mine) continue; x[d] = o; }")
    assert not faults("for (int d = 0; d < 4; ++d) { ptx::tmem_ld8(a, o); if (mine) x[d] = o; __syncwarp(); }")
    assert not faults("for (int d = 0; d < 4; ++d) { ptx::tmem_ld8(a, o); if (whole) x[d] = o; }")
    assert faults("if (lane == 0) ptx::mbar_arrive(b); if (half) ptx::tmem_ld32(a, s);")


@pytest.mark.parametrize("text", [pytest.param(softmax_warps(), id="attn_tc")])
def test_lanes_meet_before_they_touch_tensor_memory(text):
    assert len(WHOLE.findall(text)) >= 20
    assert not faults(text), "\n---\n".join(faults(text))
