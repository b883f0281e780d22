"""Rules that the kernels' sources keep and that no run on a GPU would show reliably.

Kernels launched with programmatic dependent launch may be running while their predecessor
still writes what they read. Their loads stay behind ``griddepcontrol.wait`` because its
``memory`` clobber orders them; a ``const T* __restrict__`` parameter tells the compiler that
the data is read-only for the grid's whole life, and such a load may move ahead of the wait.

Where one lane arrives on a barrier for its warp, the other lanes' reads are ordered before
the arrival by a ``__syncwarp()`` only.
"""

from __future__ import annotations

import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "aios_b200" / "csrc"
FILES = sorted(p.name for p in CSRC.glob("*.cu") if "griddepcontrol" in p.read_text() or "pdl_" in p.read_text())
CONSTANTS = {"w", "wq", "norm_w"}  # weights: written when the model was loaded


def _kernels(text: str) -> list[tuple[str, str, str]]:
    """(name, parameters, body) of every __global__ function."""
    out = []
    for m in re.finditer(r"__global__\s+void\s+(?:__launch_bounds__\s*\((?:[^()]|\([^()]*\))*\)\s*)?(\w+)\s*\(", text):
        depth, at = 1, m.end()
        while depth:
            depth += {"(": 1, ")": -1}.get(text[at], 0)
            at += 1
        start = text.index("{", at)
        depth, end = 1, start + 1
        while depth:
            depth += {"{": 1, "}": -1}.get(text[end], 0)
            end += 1
        out.append((m.group(1), text[m.end() : at - 1], text[start:end]))
    return out


@pytest.mark.parametrize("name", FILES)
def test_inputs_of_dependent_launches_are_not_declared_read_only(name: str) -> None:
    kernels = _kernels((CSRC / name).read_text())
    assert kernels and any("pdl_wait()" in body or "pdl_enter()" in body for _, _, body in kernels)
    for kernel, parameters, body in kernels:
        if "pdl_wait()" in body or "pdl_enter()" in body:
            bad = set(re.findall(r"const\s+[\w:]+\s*\*\s*__restrict__\s+(\w+)", parameters)) - CONSTANTS
            assert not bad, f"{kernel}: {bad}"


def test_the_sources_are_found() -> None:
    assert {"fp8_rows.cu", "fp8_linear.cu", "elementwise.cu", "attnres.cu", "sampler.cu", "attention.cu"} <= set(FILES)


@pytest.mark.parametrize("name", sorted(p.name for p in CSRC.glob("*.cu")))
def test_a_lane_that_arrives_for_its_warp_follows_the_others(name: str) -> None:
    lines = [line.strip() for line in (CSRC / name).read_text().splitlines()]
    for i, line in enumerate(lines):
        if re.match(r"if \(lane == 0\) mbar_arrive\w*\(", line):
            assert lines[i - 1] == "__syncwarp();", f"line {i + 1}: {line}"
