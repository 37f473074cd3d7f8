"""GPU: the 8-bit linear path at the edges of its definitions."""

from __future__ import annotations

import pytest
import torch

from oracle import int8 as o8
from test_gpu_int8 import _assert_codes, _codes, _gen, _hidden, _ops, _scales, U

pytestmark = pytest.mark.gpu


# registers (aligned, then a few unaligned rows), the ring (aligned, unaligned), rows read twice
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("rows,width", [(5, 1536), (1300, 896), (5, 1001), (6, 6001), (1200, 12000), (1300, 1001),
                                        (5, 60000)])
def test_rmsnorm_sum_of_squares_past_fp32(rows, width, residual, dtype):
    """Finite values whose squares sum past fp32's largest number: scale NaN and codes 0, like a row that is not
    finite; the rows beside it, one of them just below the limit, are untouched."""
    x = _hidden(rows, width, dtype, rows + width).clone()
    x[1] = 1e20            # a square alone passes
    x[2] = 0
    x[2, :5] = 1.8e19      # each square (3.24e38) fits, their sum does not
    x[3] = 0
    x[3, width // 2] = 1e19  # one square of 1e38: fits
    r = torch.zeros_like(x) if residual else None
    w = (torch.rand(width, generator=_gen(3)) + 0.5).to(dtype).cuda()
    codes, scale, _ = _ops().rmsnorm_int8(x, w, residual=r)
    assert torch.isnan(scale).nonzero().flatten().tolist() == [1, 2]
    assert (codes[1:3] == 0).all()
    keep = torch.tensor([i for i in range(rows) if i not in (1, 2)], device="cuda")
    y, _ = o8.rmsnorm_rows(x[keep], w, 1e-6)
    _assert_codes(codes[keep], scale[keep], y, ((width / 32 + 16) / 2 + 8) * U)


@pytest.mark.parametrize("rows,width,dtype", [(1300, 1001, torch.bfloat16), (777, 1001, torch.float32),
                                              (1200, 2501, torch.bfloat16), (300, 6001, torch.float32)])
def test_rmsnorm_without_residual_is_that_of_a_zero_residual(rows, width, dtype):
    """The same rows take the same kernel, and so the same order of summation, whether or not there is a residual:
    equal bits."""
    ops = _ops()
    x = _hidden(rows, width, dtype, rows + width)
    w = (torch.rand(width, generator=_gen(3)) + 0.5).to(dtype).cuda()
    codes, scale, _ = ops.rmsnorm_int8(x, w)
    codes0, scale0, _ = ops.rmsnorm_int8(x, w, residual=torch.zeros_like(x))
    assert torch.equal(scale, scale0) and torch.equal(codes, codes0)


@pytest.fixture
def wait_limit():
    """Sets the limit of the 8-bit kernels' device waits for a test; one second again after it."""
    from specdec_b200 import _lib

    lib = _lib.load_library()
    yield lambda ns: _lib.check(lib.specdec_wait_limit_selftest(ns), "wait_limit_selftest")
    torch.cuda.synchronize()
    lib.specdec_wait_limit_selftest(1_000_000_000)


# a tile for each CTA, more tiles than CTAs (pairs), a split of K, a split over few rows
@pytest.mark.parametrize("rows,width,n", [(333, 1001, 777), (1280, 1536, 17920), (64, 8960, 1536), (40, 4864, 896)])
@pytest.mark.parametrize("weight_ready", [False, True])
def test_linear_behind_a_long_predecessor(rows, width, n, weight_ready, wait_limit):
    """A kernel that lets its successor start and then runs on for four times the limit of a wait: that time is
    the predecessor's, and no wait of the product gives up."""
    from specdec_b200 import _lib

    lib = _lib.load_library()
    ops = _ops()
    a, w = _codes(rows, width, 1), _codes(n, width, 2)
    sa, sw = _scales(rows, 1), _scales(n, 2)
    want = ops.linear_int8(a, sa, w, sw)
    status, other = (torch.zeros(1, dtype=torch.int32, device="cuda") for _ in range(2))
    out = torch.full_like(want, 7.0)
    torch.cuda.synchronize()
    wait_limit(25_000_000)
    stream = torch.cuda.current_stream().cuda_stream
    _lib.check(lib.specdec_wait_selftest(3, None, 1, 1, 100_000_000, other.data_ptr(), None, stream), "wait_selftest")
    ops.linear_int8(a, sa, w, sw, out=out, weight_ready=weight_ready, status=status)
    torch.cuda.synchronize()
    assert int(status.item()) == 0 and torch.equal(out, want)
    assert int(other.item()) == _lib.STATUS_TIMEOUT  # the predecessor did run that long


# a tile for each CTA, several tiles a CTA (pairs, single CTAs, f32), a split of K, unaligned outputs
@pytest.mark.parametrize("rows,width,n,out_dtype", [(333, 1001, 777, torch.float32), (1280, 1536, 17920, torch.bfloat16),
                                                    (1280, 1536, 17920, torch.float32), (4099, 384, 1153, torch.bfloat16),
                                                    (64, 8960, 1536, torch.bfloat16), (40, 4864, 897, torch.float32)])
def test_linear_marks_what_its_waits_gave_up_on(rows, width, n, out_dtype, wait_limit):
    """Waits that give up without looking: the status bit is raised, no output keeps what the buffer held before,
    nothing beside the output is written, and the next call is right."""
    from specdec_b200 import _lib

    ops = _ops()
    a, w = _codes(rows, width, 1), _codes(n, width, 2)
    sa, sw = _scales(rows, 1), _scales(n, 2)
    want = ops.linear_int8(a, sa, w, sw, out_dtype=out_dtype)
    buf = torch.full((rows + 2, n), 7.0, dtype=out_dtype, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    wait_limit(0)
    out = ops.linear_int8(a, sa, w, sw, out=buf[1:-1], status=status)
    torch.cuda.synchronize()
    assert int(status.item()) == _lib.STATUS_TIMEOUT and torch.isnan(out).all()
    assert (buf[0] == 7).all() and (buf[-1] == 7).all()
    wait_limit(1_000_000_000)
    status.zero_()
    assert torch.equal(ops.linear_int8(a, sa, w, sw, out_dtype=out_dtype, status=status), want)
    assert int(status.item()) == 0


# the ring with a warp, 4, 8 and 16 warps a row; unaligned and aligned rows (a second each: the limit of a wait)
@pytest.mark.parametrize("rows,width,dtype", [(1300, 501, torch.bfloat16), (1200, 2501, torch.float32),
                                              (1200, 6001, torch.bfloat16), (1200, 12000, torch.bfloat16)])
@pytest.mark.parametrize("op", ["swiglu", "rmsnorm_add", "rmsnorm_add_in_place"])
def test_rows_mark_what_their_waits_gave_up_on(rows, width, dtype, op, wait_limit):
    """Rows whose copies never come: every row has scale NaN and (with a residual) a sum of NaN, nothing
    beside the outputs is written, and the next call is right."""
    ops = _ops()
    x = _hidden(rows, width * 2 if op == "swiglu" else width, dtype, 1)
    r = _hidden(rows, width, dtype, 2) if "add" in op else None
    w = torch.ones(width, dtype=dtype, device="cuda")
    stride = -(-width // 16) * 16

    def call(x, summed=None):
        codes = torch.full((rows, stride), 7, dtype=torch.int8, device="cuda")
        if op == "swiglu":
            return codes, ops.swiglu_int8(x, codes=codes[:, :width])[1], None
        return codes, *ops.rmsnorm_int8(x, w, residual=r, summed=summed, codes=codes[:, :width])[1:]

    want = call(x)
    buf = torch.full((rows, stride), 7.0, dtype=dtype, device="cuda")
    summed = None if r is None else buf[:, :width]
    y = x
    if "place" in op:  # a padded row stride, so that the outputs are aligned
        y = summed.copy_(x)
    torch.cuda.synchronize()
    wait_limit(0)
    codes, scale, s = call(y, summed)
    torch.cuda.synchronize()
    assert torch.isnan(scale).all() and (codes[:, width:] == 7).all() and (buf[:, width:] == 7).all()
    assert r is None or torch.isnan(s).all()
    wait_limit(1_000_000_000)
    for got, ref in zip(call(x), want):
        assert got is None or torch.equal(got, ref)


@pytest.mark.parametrize("rows", [1, 12, 24, 40, 300, 3000])
@pytest.mark.parametrize("width", [131071, 131072])
def test_linear_sums_of_the_lowest_code(rows, width):
    """Codes of -128 on both sides: at the largest width the sum is 2^31, one past the largest int32."""
    a = torch.full((rows, 131072), -128, dtype=torch.int8, device="cuda")[:, :width]
    w = torch.full((130, 131072), -128, dtype=torch.int8, device="cuda")[:, :width]
    w[1] = 127
    w[2] = 0
    one = torch.ones(rows, device="cuda")
    for out_dtype in (torch.float32, torch.bfloat16):
        got = _ops().linear_int8(a, one, w, torch.ones(130, device="cuda"), out_dtype=out_dtype)
        want = torch.full((rows, 130), float(width * 128 * 128))
        want[:, 1] = -float(width * 128 * 127)
        want[:, 2] = 0
        assert torch.equal(got.cpu(), want.to(out_dtype))  # width * 2^14 and width * 2^7 * 127: exact in fp32


def test_first_calls_from_several_threads():
    """Eight threads of a fresh process make their first calls of the path together, each on a stream of its own."""
    import subprocess
    import sys

    from conftest import PKG, ROOT

    code = f"""
import sys, threading
sys.path[:0] = [{str(PKG)!r}, {str(ROOT / 'tests')!r}, {str(ROOT)!r}]
import torch
from specdec_b200.kernels import ops
from test_gpu_int8 import _check_linear, _codes, _hidden, _scales
shapes = [(64, 8960, 300), (40, 4864, 897), (1280, 1536, 600), (333, 1001, 777)]
data = [(_codes(r, k, 1), _scales(r, 1), _codes(n, k, 2), _scales(n, 2), _hidden(1300, k | 1, torch.bfloat16, 3))
        for r, k, n in shapes]
torch.cuda.synchronize()
start, got = threading.Barrier(8), [None] * 8
def call(i):
    a, sa, w, sw, x = data[i % 4]
    with torch.cuda.stream(torch.cuda.Stream()):
        start.wait()
        y = ops.linear_int8(a, sa, w, sw)
        got[i] = y, ops.quantize_int8(x)
        torch.cuda.current_stream().synchronize()
threads = [threading.Thread(target=call, args=(i,)) for i in range(8)]
[t.start() for t in threads]; [t.join() for t in threads]
for i, (y, (codes, scale)) in enumerate(got):
    a, sa, w, sw, x = data[i % 4]
    _check_linear(a, sa, w, sw, None, y)
    want = ops.quantize_int8(x)
    assert torch.equal(codes, want[0]) and torch.equal(scale, want[1])
print("all right")
"""
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "all right" in r.stdout, r.stderr[-2000:]


def test_linear_refuses_a_status_the_device_cannot_write():
    ops = _ops()
    a, w = _codes(4, 64, 1), _codes(32, 64, 2)
    sa, sw = _scales(4, 1), _scales(32, 2)
    with pytest.raises(RuntimeError, match="must be CUDA"):
        ops.linear_int8(a, sa, w, sw, status=torch.zeros(1, dtype=torch.int32))
    for status in (torch.zeros(1, device="cuda"), torch.zeros(0, dtype=torch.int32, device="cuda")):
        with pytest.raises(ValueError, match="status must be int32"):
            ops.linear_int8(a, sa, w, sw, status=status)
