"""Oracle of the 8-bit linear path (test infrastructure): the operators' definitions in 64 bits, and the
quantiser's fp32 steps bit for bit.  No counterpart in the reference, whose linear layers are bf16."""

from __future__ import annotations

import numpy as np
import torch

FLOOR = 2.0 ** -100


def quantize_rows_f32(x: np.ndarray):
    """(codes int8, scale f32) of fp32 rows, every step rounded to fp32 (IEEE), NaN / infinity rows marked."""
    x = x.astype(np.float32)
    m = np.abs(x).max(axis=1)
    ok = np.isfinite(m)
    m = np.maximum(np.where(ok, m, np.float32(1)), np.float32(FLOOR)).astype(np.float32)
    inv = (np.float32(127) / m).astype(np.float32)
    with np.errstate(invalid="ignore"):
        q = np.rint((x * inv[:, None]).astype(np.float32))
    codes = np.where(ok[:, None], q, 0).astype(np.int8)
    return codes, np.where(ok, m / np.float32(127), np.float32("nan")).astype(np.float32)


def quotients(v: torch.Tensor):
    """(v / scale, scale) in 64 bits of rows v: a code is right when it is next to its quotient."""
    v = v.double()
    scale = v.abs().amax(dim=1).clamp(min=FLOOR) / 127.0
    return v / scale[:, None], scale


def rmsnorm_rows(x, weight, eps, residual=None):
    """(normalised rows, sum) in 64 bits."""
    s = x.double() if residual is None else x.double() + residual.double()
    return s / (s.square().mean(dim=1, keepdim=True) + eps).sqrt() * weight.double(), s


def swiglu_rows(gate_up):
    gate, up = gate_up.double().chunk(2, dim=1)
    return gate / (1.0 + (-gate).exp()) * up


def linear(codes, scale, weight_codes, weight_scale, bias=None):
    """(product, product + bias) in 64 bits."""
    p = (codes.double() @ weight_codes.double().t()) * scale.double()[:, None] * weight_scale.double()
    return p, p if bias is None else p + bias.double()
