"""Kernels that begin while the one before them on the stream still runs (launch.cuh) read what
that one writes: none of their loads may promise that the data is read-only."""
from __future__ import annotations

import re

import pytest

from freemoe_b200.build import CSRC

INCLUDE = re.compile(r'^#include "([\w.]+)"', re.M)


def code(name: str) -> str:
    """A source without its comments."""
    text = (CSRC / name).read_text()
    return re.sub(r"//[^\n]*|/\*.*?\*/", "", text, flags=re.S)


def files_of(name: str, seen: set) -> set:
    if name not in seen and (CSRC / name).exists():
        seen.add(name)
        for other in INCLUDE.findall((CSRC / name).read_text()):
            files_of(other, seen)
    return seen


UNITS = sorted(p.name for p in CSRC.glob("*.cu") if "launch.cuh" in files_of(p.name, set()))


def test_the_units_are_found():
    assert {"attention.cu", "attention_sinks.cu", "logprobs.cu", "norm.cu", "norm_pair.cu", "rope.cu"} <= set(UNITS)


@pytest.mark.parametrize("unit", UNITS)
def test_no_read_only_loads(unit):
    for name in files_of(unit, set()):
        text = code(name)
        if name == "common.cuh":  # load_x reads activations for kernels that begin when others have ended
            before, found, after = text.partition("template <> __device__ __forceinline__ float load_x<float>")
            assert found
            text = before + after.partition("\n")[2]
        else:
            assert not re.search(r"\bload_x\b", text), name
        assert not re.search(r"__ldg\b|\bld\.global[\w.:]*\.nc\b", text), name
