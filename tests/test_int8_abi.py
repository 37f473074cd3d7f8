"""CPU: the 8-bit entry points refuse bad host arguments before touching the device."""

from __future__ import annotations

import ctypes

import pytest
import torch

P = 0x1000  # never dereferenced: the call is refused, or has no rows


def _msg(lib):
    return lib.specdec_last_error().decode()


def _quantize(lib, x=P, xs=64, c=P, cs=64, s=P, dtype=1, rows=4, width=64):
    return lib.specdec_quantize_int8(x, xs, c, cs, s, dtype, rows, width, None)


@pytest.mark.parametrize("kw,msg", [
    (dict(rows=-1), "row count out of range"),
    (dict(rows=1 << 31), "row count out of range"),
    (dict(width=0), "empty row"),
    (dict(width=(1 << 24) + 1, xs=1 << 25, cs=1 << 25), "row longer than"),
    (dict(dtype=2), "supports float32 and bfloat16"),
    (dict(x=None), "must be CUDA"),
    (dict(c=None), "must be CUDA"),
    (dict(s=None), "must be CUDA"),
    (dict(xs=63), "row stride is smaller"),
    (dict(cs=63), "row stride is smaller"),
])
def test_quantize_refuses(lib, kw, msg):
    assert _quantize(lib, **kw) == 1 and msg in _msg(lib)


def test_swiglu_needs_both_halves_in_a_row(lib):
    assert lib.specdec_swiglu_int8(P, 127, P, 64, P, 1, 4, 64, None) == 1 and "row stride is smaller" in _msg(lib)


@pytest.mark.parametrize("residual,summed,weight,stride,msg", [
    (P, None, P, 64, "residual and summed come together"),
    (None, P, P, 64, "residual and summed come together"),
    (None, None, None, 64, "must be CUDA"),
    (P, P, P, 63, "row stride is smaller"),
])
def test_rmsnorm_refuses(lib, residual, summed, weight, stride, msg):
    rc = lib.specdec_rmsnorm_int8(P, 64, residual, stride, weight, 1e-6, summed, stride, P, 64, P, 1, 4, 64, None)
    assert rc == 1 and msg in _msg(lib)


def _linear(lib, a=P, a_st=64, sa=P, w=P, w_st=64, sw=P, out=P, o_st=32, dtype=1, rows=4, width=64, n=32):
    return lib.specdec_linear_int8(a, a_st, sa, w, w_st, sw, None, out, o_st, dtype, rows, width, n, 0, None, None)


@pytest.mark.parametrize("kw,msg", [
    (dict(rows=-1), "row count out of range"),
    (dict(rows=(1 << 21) + 1), "row count out of range"),
    (dict(width=0), "width must be in 1 .. 131072"),
    (dict(width=131073, a_st=131088, w_st=131088), "width must be in 1 .. 131072"),
    (dict(n=0), "out_features out of range"),
    (dict(dtype=2), "writes float32 or bfloat16"),
    (dict(a=None), "must be CUDA"),
    (dict(sw=None), "must be CUDA"),
    (dict(a_st=48), "row stride is smaller"),
    (dict(o_st=31), "row stride is smaller"),
    (dict(a_st=72), "multiples of 16"),
    (dict(w_st=72), "multiples of 16"),
    (dict(a=P + 8), "16-byte aligned"),
    (dict(w=P + 4), "16-byte aligned"),
])
def test_linear_refuses(lib, kw, msg):
    assert _linear(lib, **kw) == 1 and msg in _msg(lib)


def test_no_rows_launch_nothing(lib):
    before = lib.specdec_launch_count()
    assert _quantize(lib, rows=0) == 0 and _linear(lib, rows=0) == 0
    assert lib.specdec_rmsnorm_int8(P, 64, None, 64, P, 1e-6, None, 64, P, 64, P, 1, 0, 64, None) == 0
    assert lib.specdec_swiglu_int8(P, 128, P, 64, P, 0, 0, 64, None) == 0
    assert lib.specdec_dequantize_int8(P, 64, P, P, 64, 1, 0, 64, None) == 0
    assert lib.specdec_launch_count() == before


def test_ops_refuse_host_tensors():
    from specdec_b200.kernels import ops

    x = torch.zeros(2, 64)
    c = torch.zeros(2, 64, dtype=torch.int8)
    for call in (lambda: ops.quantize_int8(x), lambda: ops.swiglu_int8(x), lambda: ops.rmsnorm_int8(x, x[0]),
                 lambda: ops.dequantize_int8(c, x[:, 0]), lambda: ops.linear_int8(c, x[:, 0], c, x[:, 0])):
        with pytest.raises(RuntimeError, match="must be CUDA"):
            call()


def test_struct_free_signatures_match_the_header():
    """Every pointer argument of the 8-bit entry points is bound as a pointer (argument counts of the header)."""
    from specdec_b200 import _lib

    counts = {"quantize": 9, "rmsnorm": 15, "swiglu": 9, "dequantize": 9, "linear": 16}
    for name, n in counts.items():
        res, args = _lib.SIGNATURES[f"specdec_{name}_int8"]
        assert res is ctypes.c_int and len(args) == n


def test_wait_limit_refuses_what_is_out_of_range(lib):
    for ns in (-1, 1_000_000_001):
        assert lib.specdec_wait_limit_selftest(ns) == 1 and "wait limit must be" in _msg(lib)
    assert lib.specdec_wait_limit_selftest(1_000_000_000) == 0


@pytest.mark.parametrize("call", [
    lambda lib: _quantize(lib, x=P + 1), lambda lib: _quantize(lib, x=P + 2, dtype=0), lambda lib: _quantize(lib, s=P + 2),
    lambda lib: lib.specdec_swiglu_int8(P + 1, 128, P, 64, P, 1, 4, 64, None),
    lambda lib: lib.specdec_dequantize_int8(P, 64, P, P + 2, 64, 0, 4, 64, None),
    lambda lib: lib.specdec_rmsnorm_int8(P, 64, P, 64, P + 1, 1e-6, P, 64, P, 64, P, 1, 4, 64, None),
    lambda lib: lib.specdec_rmsnorm_int8(P, 64, P + 2, 64, P, 1e-6, P, 64, P, 64, P, 0, 4, 64, None),
    lambda lib: lib.specdec_rmsnorm_int8(P, 64, P, 64, P, 1e-6, P + 1, 64, P, 64, P, 1, 4, 64, None),
    lambda lib: _linear(lib, sa=P + 2), lambda lib: _linear(lib, sw=P + 1), lambda lib: _linear(lib, out=P + 1),
    lambda lib: _linear(lib, out=P + 2, dtype=0),
    lambda lib: lib.specdec_linear_int8(P, 64, P, P, 64, P, P + 2, P, 32, 1, 4, 64, 32, 0, None, None),
])
def test_elements_have_to_be_aligned(lib, call):
    """An address between two elements would fault on the device."""
    assert call(lib) == 1 and "not aligned to its elements" in _msg(lib)
