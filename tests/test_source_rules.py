"""CPU: rules of the CUDA sources that no run can show reliably, read from the sources."""

from __future__ import annotations

import re

import pytest

from conftest import PKG

SOURCES = sorted((PKG / "csrc").glob("*.cu"))


def _kernels(text):
    """(name, parameters, body) of every __global__ function."""
    for m in re.finditer(r"__global__ void\s+(?:__launch_bounds__\([^{;]*?\)\s+)?(\w+)\(", text):
        at, depth = m.end(), 1
        while depth:
            depth += {"(": 1, ")": -1}.get(text[at], 0)
            at += 1
        params, begin = text[m.end():at - 1], text.index("{", at)
        end, depth = begin + 1, 1
        while depth:
            depth += {"{": 1, "}": -1}.get(text[end], 0)
            end += 1
        yield m.group(1), params, text[begin:end]


def _code(path):
    return re.sub(r"//[^\n]*|/\*.*?\*/", "", path.read_text(), flags=re.S)


def test_kernels_are_found():
    found = {name for path in SOURCES for name, _, _ in _kernels(_code(path))}
    assert {"dequantize_int8_kernel", "int8_rows_kernel", "linear_int8_kernel", "rmsnorm_warp_kernel",
            "linear_int8_few_kernel"} <= found


@pytest.mark.parametrize("path", SOURCES, ids=lambda p: p.name)
def test_early_starters_do_not_promise_unaliased_inputs(path):
    """A kernel that may start while its predecessor runs reads what that one writes: __restrict__ would let the
    compiler load it before, or without regard to, the wait for the predecessor."""
    bad = [name for name, params, body in _kernels(_code(path)) if "grid_dep_wait" in body and "__restrict__" in params]
    assert not bad, bad


@pytest.mark.parametrize("path", [p for p in SOURCES if p.name.startswith("int8")], ids=lambda p: p.name)
def test_state_between_calls_is_shared_safely(path):
    """Calls from several threads run at once (ctypes releases the interpreter's lock): what a function keeps
    between calls is atomic or constant."""
    kept = re.findall(r"^ +static (?!const(?:expr)?\b|_)([^;(]*?)[;={[]", _code(path), flags=re.M)
    bad = [k for k in kept if not k.startswith("std::atomic<")]
    assert kept and not bad, bad
