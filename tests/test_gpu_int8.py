"""GPU: the 8-bit linear path against its definitions in 64 bits (oracle/int8.py).

Bars, from the arithmetic (u = 2^-24, the fp32 unit roundoff):
* quantize_int8, dequantize_int8: the fp32 steps are IEEE operations, so codes and values are bit-exact.
* rmsnorm_int8: the sum of squares of K values adds at most K / 32 + 16 terms in a row in any order a warp or
  a block takes, so it is off by (K / 32 + 16) u and its root by half of that; division, root and products
  add 8 u.  That bounds the scale; a code lies within 1/2 of its quotient v / scale, plus 127 times the
  relative error of value and scale together (twice the bound).
* swiglu_int8: the hardware exponential is within 2 + 1.2 |g| ulps, |g| <= 12 here: 2^-19 covers silu, the
  product and the scale.
* linear_int8: the integer sum is exact; its conversion and the two scales are three roundings of the product
  and the bias one of the result: within 4 u |product| + u |y| of it, then rounded to the output type."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import int8 as o8

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def _ops():
    from specdec_b200.kernels import ops

    return ops


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _hidden(rows, width, dtype, seed, pad=0):
    """Activations with 2 % of the channels at eight times the others; rows width + pad apart."""
    g = _gen(seed)
    x = torch.randn(rows, width + pad, generator=g)
    x[:, torch.rand(width + pad, generator=g) < 0.02] *= 8
    return x.to(dtype).cuda()[:, :width]


def _codes(rows, width, seed, extra=0):
    """int8 rows 16-byte strided; the bytes past a row's end are not zero."""
    stride = -(-width // 16) * 16 + extra
    c = torch.randint(-127, 128, (rows, stride), generator=_gen(seed), dtype=torch.int64).to(torch.int8)
    return c.cuda()[:, :width]


def _scales(n, seed):
    return (torch.rand(n, generator=_gen(seed)) + 0.5).cuda() / 127


def _assert_codes(codes, scale, exact, rtol):
    q, s = o8.quotients(exact)
    assert ((scale.double() - s).abs() <= rtol * s).all(), "scale"
    off = (codes.double() - q).abs().max().item() if codes.numel() else 0.0
    assert off <= 0.5 + 127 * 2 * rtol, f"a code is {off} from its quotient"


# ---------------------------------------------------------------------------- rows to 8 bits
ROWS_WIDTHS = [(1, 1), (3, 7), (2, 8), (1, 31), (5, 33), (7, 64), (17, 127), (4, 896), (5, 1536), (33, 1001), (3, 2056),
               (2, 4864), (5, 8960), (300, 256), (2, 17921), (3, 40000)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("pad", [0, 3, 8])
@pytest.mark.parametrize("rows,width", ROWS_WIDTHS)
def test_quantize_is_bit_exact(rows, width, pad, dtype):
    ops = _ops()
    x = _hidden(rows, width, dtype, rows + width, pad)
    codes, scale = ops.quantize_int8(x)
    assert codes.shape == (rows, width) and codes.stride(0) % 16 == 0
    want_codes, want_scale = o8.quantize_rows_f32(x.float().cpu().numpy())
    assert np.array_equal(codes.cpu().numpy(), want_codes)
    assert np.array_equal(scale.cpu().numpy(), want_scale)
    for out_dtype in (torch.bfloat16, torch.float32):
        values = ops.dequantize_int8(codes, scale, dtype=out_dtype)
        assert torch.equal(values, (codes.float() * scale[:, None]).to(out_dtype))


# enough rows for the kernels that take a warp or more a row, and for the ring in shared memory
MANY = [(1300, 500), (1300, 896), (1300, 1536), (1200, 2048), (1200, 2500), (1200, 4864), (1200, 6000), (1200, 8960),
        (1300, 101), (1300, 1001), (300, 1537), (1200, 1792), (400, 2501), (200, 6001), (160, 11003), (1190, 12000),
        (4, 16001), (4, 26001)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("op", ["quantize", "rmsnorm", "rmsnorm_add", "rmsnorm_add_in_place", "swiglu"])
@pytest.mark.parametrize("rows,width", MANY)
def test_many_rows(rows, width, op, dtype):
    """Every operator at sizes that other kernels take than the few rows above; rows are padded by 0 to 9
    values, so that those of the two inputs start at every alignment."""
    ops = _ops()
    g = _gen(rows + width)
    pad = [int(torch.randint(0, 10, (1,), generator=g)) * (width % 2) for _ in range(2)]
    if op == "swiglu":
        x = (torch.randn(rows, 2 * width + pad[0], generator=g) * 2).clamp(-12, 12).to(dtype).cuda()[:, :2 * width]
        codes, scale = ops.swiglu_int8(x)
        return _assert_codes(codes, scale, o8.swiglu_rows(x), 2.0 ** -19)
    x = _hidden(rows, width, dtype, 2 * rows + width, pad[0])
    x[rows // 2, width - 1] = float("nan")
    x[rows // 3] = 0
    keep = torch.arange(rows, device="cuda") != rows // 2
    if op == "quantize":
        codes, scale = ops.quantize_int8(x)
        want_codes, want_scale = o8.quantize_rows_f32(x.float().cpu().numpy())
        assert np.array_equal(codes.cpu().numpy(), want_codes)
        assert np.array_equal(scale.cpu().numpy(), want_scale, equal_nan=True)
        values = ops.dequantize_int8(codes, scale, dtype=dtype)
        assert torch.equal(values[keep], (codes.float() * scale[:, None]).to(dtype)[keep])
        return
    r = _hidden(rows, width, dtype, 3 * rows + width, pad[1]) if "add" in op else None
    w = (torch.rand(width, generator=g) + 0.5).to(dtype).cuda()
    y, _ = o8.rmsnorm_rows(x, w, 1e-6, r)
    want = None if r is None else (x.float() + r.float()).to(dtype)
    codes, scale, summed = ops.rmsnorm_int8(x, w, 1e-6, residual=r, summed=r if "place" in op else None)
    assert torch.isnan(scale[rows // 2]) and (codes[rows // 2] == 0).all()
    if r is not None:
        assert torch.equal(summed[keep], want[keep])
    _assert_codes(codes[keep], scale[keep], y[keep], ((width / 32 + 16) / 2 + 8) * U)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("width", [8, 100, 1536, 20000])
def test_quantize_special_rows(width, dtype):
    """Zero, subnormal, tiny, huge, NaN and infinite rows; a bad row leaves its neighbours alone."""
    x = _hidden(9, width, dtype, 5).clone()
    x[0] = 0
    x[1] = 1e-40
    x[2] = x[2] * 2.0 ** -99
    x[3] = torch.finfo(dtype).max
    x[4, width - 1] = float("nan")
    x[5, width // 2] = float("inf")
    x[6, 0] = -float("inf")
    x[7] = 0
    x[7, width // 3] = -3.0
    codes, scale = _ops().quantize_int8(x)
    want_codes, want_scale = o8.quantize_rows_f32(x.float().cpu().numpy())
    assert np.array_equal(codes.cpu().numpy(), want_codes)
    assert np.array_equal(scale.cpu().numpy(), want_scale, equal_nan=True)
    assert torch.isnan(scale).tolist() == [False] * 4 + [True] * 3 + [False] * 2
    values = _ops().dequantize_int8(codes, scale)
    good = [0, 1, 2, 7, 8]  # row 3: 127 * (max / 127) rounds past the largest number
    assert torch.isnan(values[4:7]).all() and torch.isfinite(values[good]).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("rows,width", ROWS_WIDTHS)
def test_rmsnorm(rows, width, residual, dtype):
    ops = _ops()
    pad = (rows + width) % 3 * 4
    x = _hidden(rows, width, dtype, 2 * rows + width, pad)
    r = _hidden(rows, width, dtype, 3 * rows + width, 8 - pad) if residual else None
    w = (torch.rand(width, generator=_gen(width)) + 0.5).to(dtype).cuda()
    codes, scale, summed = ops.rmsnorm_int8(x, w, 1e-6, residual=r)
    y, s = o8.rmsnorm_rows(x, w, 1e-6, r)
    _assert_codes(codes, scale, y, ((width / 32 + 16) / 2 + 8) * U)
    if residual:
        assert torch.equal(summed, (x.float() + r.float()).to(dtype))
    else:
        assert summed is None


@pytest.mark.parametrize("width", [64, 1001, 1536, 40000])
@pytest.mark.parametrize("target", ["x", "residual"])
def test_rmsnorm_updates_in_place(width, target):
    ops = _ops()
    x, r = (_hidden(6, width, torch.bfloat16, s) for s in (1, 2))
    w = (torch.rand(width, generator=_gen(3)) + 0.5).to(torch.bfloat16).cuda()
    want = ops.rmsnorm_int8(x, w, residual=r)
    x2, r2 = x.clone(), r.clone()
    got = ops.rmsnorm_int8(x2, w, residual=r2, summed=x2 if target == "x" else r2)
    assert got[2] is (x2 if target == "x" else r2)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_rmsnorm_special_rows():
    ops = _ops()
    x = _hidden(5, 1536, torch.bfloat16, 4).clone()
    x[0] = 0
    x[1, 7] = float("nan")
    x[2, 9] = float("inf")
    x[3] = 1e-30
    w = torch.ones(1536, dtype=torch.bfloat16, device="cuda")
    codes, scale, _ = ops.rmsnorm_int8(x, w)
    assert (codes[:3] == 0).all() and torch.isnan(scale).tolist() == [False, True, True, False, False]
    y, _ = o8.rmsnorm_rows(x[[0, 3, 4]], w, 1e-6)
    _assert_codes(codes[[0, 3, 4]], scale[[0, 3, 4]], y, ((1536 / 32 + 16) / 2 + 8) * U)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("pad", [0, 3, 8])
@pytest.mark.parametrize("rows,inter", ROWS_WIDTHS)
def test_swiglu(rows, inter, pad, dtype):
    g = _gen(rows * 7 + inter)
    x = (torch.randn(rows, 2 * inter + pad, generator=g) * 2).clamp(-12, 12).to(dtype).cuda()[:, :2 * inter]
    codes, scale = _ops().swiglu_int8(x)
    _assert_codes(codes, scale, o8.swiglu_rows(x), 2.0 ** -19)


def test_swiglu_extreme_gates():
    """exp overflows for very negative gates: silu is -0 there, not NaN."""
    x = torch.zeros(2, 64)
    x[:, :32] = torch.linspace(-3e4, 60, 32)
    x[:, 32:] = 1.0
    x[1, 3] = float("nan")
    codes, scale = _ops().swiglu_int8(x.cuda())
    assert codes[0].tolist() == [0] * 31 + [127] and abs(scale[0].item() - 60 / 127) < 1e-6
    assert torch.isnan(scale[1]) and (codes[1] == 0).all()


def test_rows_into_given_buffers():
    """Codes in a slice of a wider buffer: the bytes around it stay."""
    ops = _ops()
    x = _hidden(9, 100, torch.bfloat16, 8)
    buf = torch.full((9, 160), 77, dtype=torch.int8, device="cuda")
    scale = torch.empty(9, device="cuda")
    codes, s = ops.quantize_int8(x, codes=buf[:, 16:116], scale=scale)
    want, ws = ops.quantize_int8(x)
    assert torch.equal(codes, want) and s is scale and torch.equal(scale, ws)
    assert (buf[:, :16] == 77).all() and (buf[:, 116:] == 77).all()


# ---------------------------------------------------------------------------- linear
def _check_linear(codes, scale, w, ws, bias, got):
    p, y = o8.linear(codes, scale, w, ws, bias)
    tol = 4 * U * p.abs() + U * y.abs()
    # rounding is monotone: a bf16 result lies between the roundings of the ends of the fp32 interval
    low, high = ((y - tol).to(got.dtype), (y + tol).to(got.dtype)) if got.dtype == torch.bfloat16 else (y - tol, y + tol)
    bad = (got < low) | (got > high) if got.dtype == torch.bfloat16 else (got.double() < low) | (got.double() > high)
    assert not bad.any(), f"{int(bad.sum())} outputs beyond the bound"


@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("rows,width,n", [
    (1, 1, 1), (1, 16, 128), (2, 17, 7), (5, 1536, 2048), (5, 1001, 333), (8, 8960, 1536), (16, 128, 129), (17, 127, 127),
    (33, 896, 1152), (64, 129, 257), (65, 4864, 896), (127, 64, 500), (128, 256, 128), (129, 255, 256), (200, 8960, 100),
    (256, 1536, 1536), (257, 384, 384), (300, 100, 4000), (512, 1536, 2048), (777, 1001, 333), (1280, 1536, 2048),
    (2100, 896, 1153), (4099, 72, 130),
])
def test_linear(rows, width, n, bias, out_dtype):
    a, w = _codes(rows, width, rows + n), _codes(n, width, width + n, extra=16 * (n % 3))
    sa, sw = _scales(rows, 1), _scales(n, 2)
    b = torch.randn(n, generator=_gen(3)).cuda() if bias else None
    got = _ops().linear_int8(a, sa, w, sw, bias=b, out_dtype=out_dtype)
    _check_linear(a, sa, w, sw, b, got)


@pytest.mark.parametrize("rows", [1, 40, 300])
def test_linear_largest_sums(rows):
    """Every product 127^2 of one sign over the largest width: the sum still fits 32 bits, and is exact."""
    width = 131072
    a = torch.full((rows, width), 127, dtype=torch.int8, device="cuda")
    w = torch.full((130, width), -127, dtype=torch.int8, device="cuda")
    w[1] = 127
    one = torch.ones(rows, device="cuda")
    got = _ops().linear_int8(a, one, w, torch.ones(130, device="cuda"), out_dtype=torch.float32)
    want = torch.full((rows, 130), -float(width * 127 * 127))
    want[:, 1] *= -1
    assert torch.equal(got.cpu(), want)  # 2^17 * 127^2 is a 24-bit number times a power of two


@pytest.mark.parametrize("rows,width,n", [(5, 1536, 1536), (200, 500, 300), (1500, 1536, 1000)])
def test_linear_nan_rows_strides_and_ready_weights(rows, width, n):
    """A row of scale NaN gives a NaN row and nothing else; strided output; weights promised final; the same
    call twice gives the same bits."""
    ops = _ops()
    a, w = _codes(rows, width, 1, extra=32), _codes(n, width, 2)
    sa, sw = _scales(rows, 1), _scales(n, 2)
    sa[rows // 2] = float("nan")
    buf = torch.full((rows, n + 5), 7.0, dtype=torch.bfloat16, device="cuda")
    torch.cuda.synchronize()
    got = ops.linear_int8(a, sa, w, sw, out=buf[:, 2:n + 2], weight_ready=True)
    again = ops.linear_int8(a, sa, w, sw)
    keep = torch.arange(rows) != rows // 2
    assert torch.isnan(got[rows // 2].float()).all()
    assert torch.equal(got[keep.cuda()], again[keep.cuda()])
    _check_linear(a[keep.cuda()], sa[keep.cuda()], w, sw, None, got[keep.cuda()])
    assert (buf[:, :2] == 7).all() and (buf[:, n + 2:] == 7).all()


def test_linear_outputs_past_2_31():
    """131072 x 16448 outputs (2.16e9): offsets need 64 bits.  First, middle and last rows are checked."""
    rows, width, n = 131072, 32, 16448
    a, w = _codes(rows, width, 1), _codes(n, width, 2)
    sa, sw = _scales(rows, 1), _scales(n, 2)
    got = _ops().linear_int8(a, sa, w, sw)
    pick = torch.tensor([0, 1, 65535, 65536, 130000, rows - 1], device="cuda")
    _check_linear(a[pick], sa[pick], w, sw, None, got[pick])
    # and as the packed gate|up input of swiglu
    codes, scale = _ops().swiglu_int8(got)
    want, ws = _ops().swiglu_int8(got[pick].contiguous())
    assert torch.equal(codes[pick], want) and torch.equal(scale[pick], ws)


def test_empty_batches():
    ops = _ops()
    x = torch.empty(0, 64, dtype=torch.bfloat16, device="cuda")
    codes, scale = ops.quantize_int8(x)
    assert codes.shape == (0, 64) and scale.shape == (0,)
    assert ops.swiglu_int8(x)[0].shape == (0, 32)
    assert ops.rmsnorm_int8(x, torch.ones(64, dtype=torch.bfloat16, device="cuda"), residual=x)[2].shape == (0, 64)
    assert ops.dequantize_int8(codes, scale).shape == (0, 64)
    w = _codes(96, 64, 1)
    assert ops.linear_int8(codes, scale, w, _scales(96, 1)).shape == (0, 96)


def test_other_stream_and_graph():
    """The path on a side stream, eagerly and captured in a graph that replays on new inputs."""
    ops = _ops()
    w, ws = ops.quantize_int8(_hidden(700, 1536, torch.bfloat16, 1))
    x = _hidden(37, 1536, torch.bfloat16, 2).clone()
    ln = torch.ones(1536, dtype=torch.bfloat16, device="cuda")

    def path():
        codes, scale, _ = ops.rmsnorm_int8(x, ln)
        return ops.linear_int8(codes, scale, w, ws, weight_ready=True)

    want = path()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = path()
    side.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            out = path()
    torch.cuda.synchronize()
    x.copy_(_hidden(37, 1536, torch.bfloat16, 9))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, path())


def test_fresh_weights_without_the_promise():
    """Weights quantised on the stream right before the product that reads them (no promise given)."""
    ops = _ops()
    a, sa = ops.quantize_int8(_hidden(64, 896, torch.bfloat16, 3))
    for seed in range(4, 12):
        src = _hidden(4000, 896, torch.bfloat16, seed)
        torch.cuda.synchronize()
        w, sw = ops.quantize_int8(src)
        got = ops.linear_int8(a, sa, w, sw)
        _check_linear(a, sa, w, sw, None, got)


# ---------------------------------------------------------------------------- refusals
def test_ops_refuse():
    ops = _ops()
    x = _hidden(4, 64, torch.bfloat16, 1)
    codes, scale = ops.quantize_int8(x)
    w, ws = _codes(32, 64, 2), _scales(32, 1)
    with pytest.raises(ValueError, match="float32 or bfloat16"):
        ops.quantize_int8(x.half())
    with pytest.raises(ValueError, match="contiguous columns"):
        ops.quantize_int8(x.t())
    with pytest.raises(ValueError, match="codes must be int8"):
        ops.quantize_int8(x, codes=torch.empty(4, 65, dtype=torch.int8, device="cuda"))
    with pytest.raises(ValueError, match="scale must be"):
        ops.quantize_int8(x, scale=torch.empty(5, device="cuda"))
    with pytest.raises(ValueError, match="weight must be"):
        ops.rmsnorm_int8(x, torch.ones(64, device="cuda"))
    with pytest.raises(ValueError, match="residual and summed"):
        ops.rmsnorm_int8(x, torch.ones(64, dtype=x.dtype, device="cuda"), residual=x[:2])
    with pytest.raises(ValueError, match="only with a residual"):
        ops.rmsnorm_int8(x, torch.ones(64, dtype=x.dtype, device="cuda"), summed=x)
    with pytest.raises(ValueError, match="2 inter"):
        ops.swiglu_int8(x[:, :63])
    with pytest.raises(ValueError, match="share a contiguous width"):
        ops.linear_int8(codes, scale, w[:, :48], ws)
    with pytest.raises(ValueError, match="scale must be"):
        ops.linear_int8(codes, scale[:3], w, ws)
    with pytest.raises(ValueError, match="weight_scale must be"):
        ops.linear_int8(codes, scale, w, ws.double())
    with pytest.raises(ValueError, match="bias must be"):
        ops.linear_int8(codes, scale, w, ws, bias=torch.zeros(31, device="cuda"))
    with pytest.raises(ValueError, match="out must be"):
        ops.linear_int8(codes, scale, w, ws, out_dtype=torch.float16)
    with pytest.raises(RuntimeError, match="multiples of 16"):
        ops.linear_int8(torch.zeros(4, 65, dtype=torch.int8, device="cuda")[:, :64], scale, w, ws)
    with pytest.raises(RuntimeError, match="16-byte aligned"):
        ops.linear_int8(torch.zeros(4, 80, dtype=torch.int8, device="cuda")[:, 8:72], scale, w, ws)
    with pytest.raises(RuntimeError, match="must be CUDA"):
        ops.linear_int8(codes, scale.cpu(), w, ws)
    with pytest.raises(RuntimeError, match="must be CUDA"):
        ops.quantize_int8(x.cpu())
