"""The 8-bit linear path of the decoder, as a list of measurable cases.

Four operators that a decoder layer strings together:

  rmsnorm_int8   s = x + residual;  y = s / sqrt(mean(s^2) + eps) * weight;  int8(y) with one scale a row
  quantize_int8  int8(x) with one scale a row (the attention output before its projection)
  swiglu_int8    h = silu(gate) * up of a fused gate|up projection;  int8(h) with one scale a row
  linear_int8    y[r, n] = sum_k a[r, k] w[n, k] * a_scale[r] * w_scale[n] + bias[n]

int8(v) of a row: m = max(max |v|, 2^-100), scale = m / 127, code = round(v * (127 / m)), ties to even.
What is held in 8 bits is returned as the values it stands for, code * scale in bfloat16.

``own = False`` runs elementary torch operations in 32 bits; ``own = True`` calls specdec_b200.kernels.ops.
"""

from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

own = False

_PACKAGE = str(Path(__file__).resolve().parents[1] / "specdec-context-scaling_b200")
_ops = None


def _own_ops():
    global _ops
    if _ops is None:
        if _PACKAGE not in sys.path:
            sys.path.insert(0, _PACKAGE)
        from specdec_b200.kernels import ops

        _ops = ops
    return _ops


# ------------------------------------------------------------------------------------ cases
def _norm(name, rows, hidden, dtype="bf16", residual=True, pad=0):
    return {"name": name, "op": "rmsnorm", "rows": rows, "width": hidden, "dtype": dtype, "residual": residual,
            "pad": pad}


def _quant(name, rows, width, dtype="bf16", pad=0):
    return {"name": name, "op": "quantize", "rows": rows, "width": width, "dtype": dtype, "pad": pad}


def _swiglu(name, rows, inter, dtype="bf16", pad=0):
    return {"name": name, "op": "swiglu", "rows": rows, "width": inter, "dtype": dtype, "pad": pad}


def _linear(name, rows, width, out, bias=False, out_dtype="bf16"):
    return {"name": name, "op": "linear", "rows": rows, "width": width, "out": out, "bias": bias,
            "out_dtype": out_dtype}


def listed():
    return [
        # one sequence's verify block (pending token + 4 candidates) entering a target layer
        _norm("norm_verify_1", 5, 1536),
        # four 8192-token prompts entering a target layer
        _norm("norm_prompt", 32768, 1536),
        # fp32 hidden states of an odd width, no residual (a model outside the named ones)
        _norm("norm_ragged_f32", 777, 1001, dtype="f32", residual=False),
        # attention output of one decode step of 256 draft sequences, before o_proj
        _quant("quant_decode_256", 256, 896),
        # attention output of two 8192-token target prompts
        _quant("quant_prompt", 16384, 1536),
        # MLP activation of one verify block, target width
        _swiglu("swiglu_verify_1", 5, 8960),
        # MLP activation of one 8192-token prompt, target width
        _swiglu("swiglu_prompt", 8192, 8960),
        # fused QKV projection (with its bias) of one verify block: the latency end
        _linear("linear_qkv_verify_1", 5, 1536, 2048, bias=True),
        # down projection of a decode step of 64 sequences: few tokens, long rows
        _linear("linear_down_decode_64", 64, 8960, 1536),
        # fused gate|up projection of a verify step of 256 sequences
        _linear("linear_gate_up_verify_256", 1280, 1536, 17920),
        # the same projection over four 8192-token prompts: the compute end
        _linear("linear_gate_up_prompt", 32768, 1536, 17920),
        # odd everything, fp32 output (logits-like rows of a small head)
        _linear("linear_ragged_f32", 333, 1001, 777, bias=True, out_dtype="f32"),
    ]


_MOST_VALUES = 32768 * 1536
_MOST_MACS = 32768 * 1536 * 17920
_MOST_OUT = 32768 * 17920


def _size(rng, low, high, step=1):
    """Log-uniform over [low, high], a multiple of ``step``; the target's own hidden size (a
    listed case) and its double are passed over."""
    n = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    n = min(high, max(low, -(-n // step) * step))
    return n + step if n in (1536, 2 * 1536) else n


def draw(rng):
    op = rng.choice(["rmsnorm", "quantize", "swiglu", "linear", "linear"])
    odd = rng.random() < 0.3
    if op == "linear":
        width = _size(rng, 64, 9000, 1 if odd else 64)
        out = _size(rng, 64, 17920, 1 if odd else 16)
        most = min(32768, _MOST_MACS // (width * out), _MOST_OUT // out)
        c = _linear("", _size(rng, 1, most), width, out, bias=rng.random() < 0.5,
                    out_dtype=rng.choice(["bf16", "bf16", "bf16", "f32"]))
    else:
        width = _size(rng, 64, 17920, 1 if odd else 32)
        rows = _size(rng, 1, min(32768, max(1, _MOST_VALUES // (width * (2 if op == "swiglu" else 1)))))
        dtype = rng.choice(["bf16", "bf16", "bf16", "f32"])
        pad = rng.choice([0, 0, 0, 8, 3])
        if dtype == "f32":
            rows = max(1, rows // 2)
        if op == "rmsnorm":
            c = _norm("", rows, width, dtype, rng.random() < 0.6, pad)
        elif op == "quantize":
            c = _quant("", rows, width, dtype, pad)
        else:
            c = _swiglu("", rows, width, dtype, pad)
    del c["name"]
    return c


# ------------------------------------------------------------------------------------ inputs
_DTYPE = {"bf16": torch.bfloat16, "f32": torch.float32}
_EPS = 1e-6


def _rows(g, rows, width, pad, dtype, spread):
    """(rows, width) of hidden-state-like values, rows ``width + pad`` apart: unit normal, the level of a
    channel varying (1 % of the channels at ``spread`` times the others)."""
    level = torch.ones(width + pad, device="cuda")
    level[torch.rand(width + pad, device="cuda", generator=g) < 0.01] = spread
    x = torch.randn(rows, width + pad, device="cuda", generator=g)
    return x.mul_(level).to(dtype)[:, :width]


def _codes(g, rows, width):
    """int8 rows on 16-byte strides, as the quantising operators lay them out."""
    stride = -(-width // 16) * 16
    c = torch.zeros(rows, stride, dtype=torch.int8, device="cuda")
    step = max(1, (1 << 28) // max(1, width))
    for r in range(0, rows, step):
        n = min(step, rows - r)
        v = torch.randn(n, width, device="cuda", generator=g).mul_(32.0).round_().clamp_(-127, 127)
        c[r:r + n, :width] = v.to(torch.int8)
    return c[:, :width]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    rows, width = case["rows"], case["width"]
    s = dict(case)
    if case["op"] == "linear":
        n = case["out"]
        s["a"], s["w"] = _codes(g, rows, width), _codes(g, n, width)
        s["a_scale"] = torch.rand(rows, device="cuda", generator=g).add_(0.5).mul_(4.0 / 127)
        s["w_scale"] = torch.rand(n, device="cuda", generator=g).add_(0.5).mul_(0.08 / 127)
        s["b"] = torch.randn(n, device="cuda", generator=g) if case["bias"] else None
        return s
    dtype = _DTYPE[case["dtype"]]
    if case["op"] == "rmsnorm":
        s["x"] = _rows(g, rows, width, case["pad"], dtype, 4.0)
        s["r"] = _rows(g, rows, width, case["pad"], dtype, 4.0) if case["residual"] else None
        s["weight"] = torch.rand(width, device="cuda", generator=g).add_(0.5).to(dtype)
    elif case["op"] == "quantize":
        s["x"] = _rows(g, rows, width, case["pad"], dtype, 4.0)
    else:
        s["x"] = _rows(g, rows, 2 * width, case["pad"], dtype, 1.0)
    return s


# ------------------------------------------------------------------------------------ one pass
def _plain_int8(v):
    """Codes' values and scales of fp32 rows ``v``."""
    m = v.abs().amax(dim=1, keepdim=True).clamp(min=2.0 ** -100)
    scale = m / 127.0
    return (torch.round(v * (127.0 / m)) * scale).to(torch.bfloat16), scale[:, 0]


def _run_plain(s):
    op = s["op"]
    if op == "linear":
        y = torch.matmul(s["a"].float(), s["w"].float().t())
        y = y * s["a_scale"][:, None] * s["w_scale"]
        if s["b"] is not None:
            y = y + s["b"]
        return y.to(_DTYPE[s["out_dtype"]])
    x = s["x"].float()
    if op == "quantize":
        return _plain_int8(x)
    if op == "swiglu":
        gate, up = x[:, :s["width"]], x[:, s["width"]:]
        return _plain_int8(gate / (1.0 + torch.exp(-gate)) * up)
    total = x if s["r"] is None else x + s["r"].float()
    y = total * torch.rsqrt((total * total).mean(dim=1, keepdim=True) + _EPS) * s["weight"].float()
    values, scale = _plain_int8(y)
    return (values, scale) if s["r"] is None else (values, scale, total.to(s["x"].dtype))


def _run_own(s):
    ops = _own_ops()
    op = s["op"]
    if op == "linear":
        return ops.linear_int8(s["a"], s["a_scale"], s["w"], s["w_scale"], bias=s["b"],
                               out_dtype=_DTYPE[s["out_dtype"]], weight_ready=True)
    if op == "quantize":
        codes, scale = ops.quantize_int8(s["x"])
        return ops.dequantize_int8(codes, scale), scale
    if op == "swiglu":
        codes, scale = ops.swiglu_int8(s["x"])
        return ops.dequantize_int8(codes, scale), scale
    codes, scale, total = ops.rmsnorm_int8(s["x"], s["weight"], _EPS, residual=s["r"])
    values = ops.dequantize_int8(codes, scale)
    return (values, scale) if total is None else (values, scale, total)


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ------------------------------------------------------------------------------------ accounting
def work(case):
    rows, width = case["rows"], case["width"]
    if case["op"] == "linear":
        n = case["out"]
        esize = 2 if case["out_dtype"] == "bf16" else 4
        read = rows * width + n * width + 4 * rows + (8 if case["bias"] else 4) * n
        return {"bytes": read + esize * rows * n, "flops": 2 * rows * width * n}
    esize = 2 if case["dtype"] == "bf16" else 4
    values = rows * width
    out = 2 * values + 4 * rows
    if case["op"] == "quantize":
        return {"bytes": esize * values + out, "flops": 4 * values}
    if case["op"] == "swiglu":
        return {"bytes": 2 * esize * values + out, "flops": 9 * values}
    tensors = 3 if case["residual"] else 1  # x; the residual and the sum
    return {"bytes": esize * (tensors * values + width) + out, "flops": 9 * values}


# ------------------------------------------------------------------------------------ 64 bits
def _exact_int8(v):
    top = torch.maximum(v.max(dim=1).values, -v.min(dim=1).values)
    scale = torch.where(top < 2.0 ** -100, torch.full_like(top, 2.0 ** -100), top) / 127
    q = torch.div(v, scale.unsqueeze(1)).round_()
    return q.mul_(scale.unsqueeze(1)), scale


def exact(case, seed):
    """The definitions in 64 bits. The values are those of codes taken in 64 bits: a code whose quotient lies
    on a rounding boundary may be its neighbour in 32 bits, one step of the row's scale away."""
    s = prepare(case, seed)
    if case["op"] == "linear":
        a = s["a"].double() * s["a_scale"].double().unsqueeze(1)
        w = s["w"].double() * s["w_scale"].double().unsqueeze(1)
        y = a @ w.t()
        return y if s["b"] is None else y.add_(s["b"].double())
    x = s["x"].double()
    if case["op"] == "quantize":
        return _exact_int8(x)
    if case["op"] == "swiglu":
        gate, up = x.split(case["width"], dim=1)
        return _exact_int8(gate * torch.sigmoid(gate) * up)
    if s["r"] is not None:
        x = x + s["r"].double()
    norm = torch.sqrt(torch.linalg.vector_norm(x, dim=1, keepdim=True).square() / case["width"] + _EPS)
    values, scale = _exact_int8(x / norm * s["weight"].double())
    return (values, scale) if s["r"] is None else (values, scale, x)
