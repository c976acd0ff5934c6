"""Kernels that begin before their predecessor has ended: read in the sources, since what goes wrong would be a race."""
from __future__ import annotations

import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "molt_b200" / "csrc"
SOURCES = [p for p in sorted(CSRC.glob("*.cu")) if "wait_for_previous()" in p.read_text()]


def _functions(text):
    """(name, parameter list, body) of every function whose body is written out."""
    for match in re.finditer(r"(\w+)\(([^;{}]*?)\)\s*(?:const\s*)?\{", text):
        depth, end = 1, match.end()
        while depth and end < len(text):
            depth += {"{": 1, "}": -1}.get(text[end], 0)
            end += 1
        yield match.group(1), match.group(2), text[match.end():end]


def _code(path):
    return re.sub(r"__launch_bounds__\([^)]*\)", "", re.sub(r"//[^\n]*", "", path.read_text()))


def test_the_kernels_are_found():
    found = {name for path in SOURCES for name, _, body in _functions(_code(path)) if "wait_for_previous()" in body}
    assert found == {"norm_finish_kernel", "scale_kernel", "policy_finish_kernel", "policy_rows_finish_kernel",
                     "preference_finish_kernel"}


@pytest.mark.parametrize("path", SOURCES, ids=lambda p: p.name)
def test_partial_sums_are_not_promised_to_be_constant(path):
    """``const T* __restrict__`` says that nobody writes the values while the kernel lives; its predecessor does, until the
    wait.  Neither such a kernel nor a function it hands the partial sums to may make that promise."""
    for name, parameters, body in _functions(_code(path)):
        for parameter in parameters.split(","):
            promised = re.search(r"const\s[^*]*\*\s*__restrict__", parameter)
            if "wait_for_previous()" in body or re.search(r"\bpart$", parameter.strip()):
                assert not promised, f"{path.name}: {name}({parameter.strip()})"


@pytest.mark.parametrize("path", SOURCES, ids=lambda p: p.name)
def test_partial_sums_are_read_by_loads_that_stay_behind_the_wait(path):
    """A dependent kernel hands its partial sums on as ``Written``, whose loads are volatile like the wait."""
    for name, parameters, body in _functions(_code(path)):
        if "wait_for_previous()" in body:
            assert "const Written part" in parameters, f"{path.name}: {name}"
            before = body.split("wait_for_previous()")[0]
            assert "part[" not in before and "finish" not in before, f"{path.name}: {name} reads before it waits"
