"""GPU: attention of packed prompts against a plain 64-bit form (tolerance: rows_helpers)."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

from rows_helpers import assert_rows, check_packed, i32, make_batch, packed_case, plain_attention

pytestmark = pytest.mark.gpu
FILL = 7.0


def _ops():
    from specdec_b200.kernels import ops

    return ops


def _run(case, lens, *, q_max=None, **kw):
    q, k, v, row0, kv0, ctx = case
    out = torch.full(q.shape, FILL, dtype=q.dtype, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    batch = make_batch(row0, lens, ctx, q.shape[0], q_max)
    _ops().prompt_attention(q, k, v, batch, kv_row0=i32(kv0), out=out, status=status, **kw)
    assert int(status) == 0
    return out


HEADS = [(12, 2, 128), (14, 2, 64), (5, 5, 128), (33, 1, 64), (128, 1, 128), (6, 1, 64), (80, 2, 128), (4, 4, 64)]
LENS = [[1], [2], [16], [127], [128], [129], [255, 257], [1, 0, 64, 65, 63], [0, 0], [0, 3], [700, 5, 130]]


@pytest.mark.parametrize("H,KV,D", HEADS)
@pytest.mark.parametrize("lens", LENS, ids=lambda x: "-".join(map(str, x)))
def test_whole_prompts(H, KV, D, lens):
    case = packed_case(lens, H, KV, D, sum(lens) + H)
    out = _run(case, lens)
    check_packed(out, FILL, *case[:5], lens, case[5])


@pytest.mark.parametrize("H,KV,D", [(12, 2, 128), (14, 2, 64), (7, 7, 64), (64, 1, 128)])
@pytest.mark.parametrize("lens,extra", [
    ([1], [0]), ([1], [1]), ([1], [127]), ([1], [128]), ([5], [8192]), ([1, 1, 1], [0, 5000, 64]),
    ([64, 1, 0, 17], [3, 1000, 50, 127]), ([512], [1024]), ([33, 200], [4096, 0]),
])
def test_next_pieces_of_prompts(H, KV, D, lens, extra):
    """More keys than rows; nobody's rows between the sequences stay as they were."""
    case = packed_case(lens, H, KV, D, sum(lens) + sum(extra) + H, gap=3, extra=extra)
    out = _run(case, lens)
    check_packed(out, FILL, *case[:5], lens, case[5])


@pytest.mark.parametrize("H,KV,D", [(12, 2, 128), (14, 2, 64)])
def test_many_sequences(H, KV, D):
    """Several items a CTA, more sequences than threads, and the largest number of sequences of a call."""
    g = torch.Generator().manual_seed(3)
    for n, most in ((300, 40), (2048, 3)):
        lens = torch.randint(0, most, (n,), generator=g).tolist()
        extra = torch.randint(0, most, (n,), generator=g).tolist()
        case = packed_case(lens, H, KV, D, n, extra=extra, gap=1)
        out = _run(case, lens)
        some = set(range(n)) - set(torch.randperm(n, generator=g)[:60].tolist())
        q, k, v, row0, kv0, ctx = case
        for b in set(range(n)) - some:
            if lens[b]:
                r, c = row0[b], kv0[b]
                want, tol = plain_attention(q[r:r + lens[b]], k[c:c + ctx[b]], v[c:c + ctx[b]],
                                            torch.arange(lens[b]) + extra[b] + 1, 1 / math.sqrt(D))
                assert_rows(out[r:r + lens[b]], want, tol, f"sequence {b}")
        assert (out[row0[0] - 1] == FILL).all() and (out[-1] == FILL).all()


@pytest.mark.parametrize("H,KV,D", [(12, 2, 128), (14, 2, 64), (5, 5, 128)])
def test_second_tiles_after_items_without_them(H, KV, D):
    """Items with rows for one tile only, then one whose second tile sees more keys than the first and washes the first
    block: its warps wait for nobody in the items before."""
    per = 128 // (H // KV)
    unit = [min(5, per)] * 6 + [2 * per]
    lens = unit * (2048 // 7 if per < 100 else 40)
    extra = [62 - per] * len(lens) if per < 62 else [0] * len(lens)
    case = packed_case(lens, H, KV, D, 17, extra=extra)
    q, k, v, row0, kv0, ctx = case
    first = _run(case, lens)
    for _ in range(20):
        assert torch.equal(_run(case, lens), first)
    for b in range(6, len(lens), 21):
        r, c = row0[b], kv0[b]
        want, tol = plain_attention(q[r:r + lens[b]], k[c:c + ctx[b]], v[c:c + ctx[b]],
                                    torch.arange(lens[b]) + extra[b] + 1, 1 / math.sqrt(D))
        assert_rows(first[r:r + lens[b]], want, tol, f"sequence {b}")


@pytest.mark.parametrize("KV,D", [(1, 128), (1, 64)])
def test_last_blocks_of_second_tiles(KV, D):
    """Two tokens a unit, the second of which sees one key past a block's end: the first tile is done with the item before
    that block is washed."""
    lens, extra = [2] * 1500, [127, 255, 127] * 500
    case = packed_case(lens, 128, KV, D, 23, extra=extra)
    q, k, v, row0, kv0, ctx = case
    first = _run(case, lens)
    for _ in range(20):
        assert torch.equal(_run(case, lens), first)
    for b in range(0, 1500, 97):
        r, c = row0[b], kv0[b]
        want, tol = plain_attention(q[r:r + 2], k[c:c + ctx[b]], v[c:c + ctx[b]], torch.arange(2) + extra[b] + 1,
                                    1 / math.sqrt(D))
        assert_rows(first[r:r + 2], want, tol, f"sequence {b}")


def test_long_prompts_of_mixed_lengths():
    """Units that CTA boundaries cut, at both head sizes."""
    for H, KV, D in ((12, 2, 128), (14, 2, 64)):
        lens = [2500, 1, 900, 40, 1700]
        case = packed_case(lens, H, KV, D, D)
        out = _run(case, lens)
        check_packed(out, FILL, *case[:5], lens, case[5])


@pytest.mark.parametrize("D", [64, 128])
def test_views_of_a_fused_projection(D):
    """q, k and v as columns of one matrix, head-major q, out inside a larger tensor."""
    H, KV, lens = 6, 2, [37, 0, 150]
    rows = sum(lens)
    g = torch.Generator().manual_seed(D)
    qkv = torch.randn(rows, (H + 2 * KV) * D, generator=g).to(torch.bfloat16).cuda()
    q = qkv[:, :H * D].view(rows, H, D)
    k = qkv[:, H * D:(H + KV) * D].view(rows, KV, D)
    v = qkv[:, (H + KV) * D:].view(rows, KV, D)
    batch = make_batch([0, 37, 37], lens, lens, rows)
    big = torch.full((rows, H + 3, D + 24), FILL, dtype=torch.bfloat16, device="cuda")
    _ops().prompt_attention(q, k, v, batch, out=big[:, 1:1 + H, 8:8 + D])
    check_packed(big[:, 1:1 + H, 8:8 + D].contiguous(), FILL, q, k, v, [0, 37, 37], [0, 37, 37], lens, lens)
    big[:, 1:1 + H, 8:8 + D] = FILL
    assert (big == FILL).all()  # and nothing beside it was written
    heads_first = q.transpose(0, 1).contiguous().transpose(0, 1)
    same = _ops().prompt_attention(heads_first, k, v, batch)
    assert torch.equal(same, _ops().prompt_attention(q, k, v, batch))


@pytest.mark.parametrize("H,KV,D", [(12, 2, 128), (14, 2, 64)])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf, 3.38e38])
def test_nothing_of_others_reaches_a_row(H, KV, D, bad):
    """Whatever the rows before, between and behind the sequences hold, their answers keep their bits."""
    lens, extra = [130, 1, 0, 65], [0, 200, 9, 31]
    case = packed_case(lens, H, KV, D, 5, gap=20, extra=extra)
    want = _run(case, lens)
    q, k, v, row0, kv0, ctx = case
    mine = torch.zeros(k.shape[0], dtype=torch.bool)
    for c, t, n in zip(kv0, ctx, lens):
        if n:
            mine[c:c + t] = True
    k, v, q = k.clone(), v.clone(), q.clone()
    k[~mine.cuda()] = bad
    v[~mine.cuda()] = bad
    used = torch.zeros(q.shape[0], dtype=torch.bool)
    for r, n in zip(row0, lens):
        used[r:r + n] = True
    q[~used.cuda()] = bad
    assert torch.equal(_run((q, k, v, row0, kv0, ctx), lens), want)


@pytest.mark.parametrize("H,KV,D", [(12, 2, 128), (14, 2, 64)])
@pytest.mark.parametrize("at", [0, 1, 63, 64, 100, 128, 191, 298])
def test_infinities_and_nans_of_later_tokens(H, KV, D, at):
    """V of token `at` holds infinities and NaNs: rows before it are as if it were zero, rows from it on have them."""
    lens = [299]
    case = packed_case(lens, H, KV, D, at)
    q, k, v, row0, kv0, ctx = case
    v = v.clone()
    v[at, 0, 3], v[at, 0, 7], v[at, KV - 1, D - 1] = math.inf, math.nan, -math.inf
    out = _run((q, k, v, row0, kv0, ctx), lens)
    check_packed(out, FILL, q, k, v, row0, kv0, lens, ctx)
    # a NaN key: rows before it do not notice, the others are NaN
    k = k.clone()
    k[at] = math.nan
    out = _run((q, k, case[2], row0, kv0, ctx), lens)
    want, tol = plain_attention(q[:at], k[:at], case[2][:at], torch.arange(at) + 1, 1 / math.sqrt(D)) if at else (None, None)
    if at:
        assert_rows(out[:at], want, tol)
    assert out[at:].isnan().all()


@pytest.mark.parametrize("D", [64, 128])
def test_every_value_of_later_tokens_is_strange(D):
    """All of V from some token on is NaN or infinite, in a batch of several sequences."""
    lens, extra = [90, 300, 40], [70, 0, 500]
    case = packed_case(lens, 6, 2, D, 11, extra=extra)
    q, k, v, row0, kv0, ctx = case
    v = v.clone()
    for b, t in enumerate((100, 200, 530)):
        v[kv0[b] + t:kv0[b] + ctx[b]] = math.nan if b != 1 else math.inf
    out = _run((q, k, v, row0, kv0, ctx), lens)
    check_packed(out, FILL, q, k, v, row0, kv0, lens, ctx)


@pytest.mark.parametrize("D", [64, 128])
def test_scores_that_grow_and_shrink(D):
    """The reference maximum of the first keys is passed by factors of 2^30 to 2^3000 and by steps, or never reached."""
    n, H, KV = 400, 4, 2
    q, k, v, row0, kv0, ctx = packed_case([n], H, KV, D, 9)
    k = torch.zeros_like(k)
    q = torch.zeros_like(q)
    q[..., 0] = 1.0
    for steps in (lambda t: 0.25 * t, lambda t: -0.25 * t, lambda t: 40.0 * (t // 64), lambda t: 3000.0 * (t == 200),
                  lambda t: -2000.0 + 10 * (t % 7), lambda t: 1e30 * (t % 2), lambda t: -1e30 * (t < 150)):
        k[:, 0] = 0.0
        k[:, :, 0] = torch.tensor([steps(t) for t in range(n)]).to(torch.bfloat16).cuda()[:, None]
        out = _run((q, k, v, row0, kv0, ctx), [n], sm_scale=1.0)
        # one product a score, exact as q is 1 (the others are zeros)
        check_packed(out, FILL, q, k, v, row0, kv0, [n], ctx, scale=1.0, exact=True)


@pytest.mark.parametrize("D", [64, 128])
def test_minus_infinity_scores(D):
    """Keys whose scores are -inf weigh nothing, also where they are all that a row's first 64 keys are and the later
    scores lie far below zero; a row that sees no other key has no answer to give and is zero."""
    n, H, KV = 300, 2, 1
    q, k, v, row0, kv0, ctx = packed_case([n], H, KV, D, 21)
    q = q.abs()
    k = -k.abs() - 3.0  # scores around -400
    k[:130] = -math.inf
    out = _run((q, k, v, row0, kv0, ctx), [n], sm_scale=1.0)
    k1 = k.clone()
    k1[:130] = 0
    want, tol = plain_attention(q[130:], k1[130:], v[130:], torch.arange(n - 130) + 1, 1.0)
    assert_rows(out[130:], want, tol)
    assert (out[:130] == 0).all()


def test_bad_lengths_skip_the_sequence():
    from specdec_b200 import _lib

    H, KV, D = 6, 2, 64
    lens = [20, 30, 40]
    for field, value in (("q_len", -1), ("q_len", 41), ("ctx", 29), ("row0", -1), ("row0", 61), ("kv0", -1), ("kv0", 61),
                         ("q_len", 2**31 - 1), ("row0", 2**31 - 1), ("kv0", 2**31 - 1), ("ctx", 2**31 - 1)):
        q, k, v, row0, kv0, ctx = packed_case(lens, H, KV, D, 2)
        a = dict(row0=list(row0), kv0=list(kv0), ctx=list(ctx), q_len=list(lens))
        a[field][1] = value
        out = torch.full(q.shape, FILL, dtype=q.dtype, device="cuda")
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        batch = _ops().RaggedBatch(i32(a["row0"]), i32(a["q_len"]), i32(a["ctx"]), 3, 40, 90, 0)
        _ops().prompt_attention(q, k, v, batch, kv_row0=i32(a["kv0"]), out=out, status=status)
        assert int(status) == _lib.STATUS_BAD_LENGTH, (field, value)
        check_packed(out, FILL, q, k, v, row0, kv0, lens, ctx, what=f"{field}={value}", skip=(1,))
        # no status word: the same, silently
        _ops().prompt_attention(q, k, v, batch, kv_row0=i32(a["kv0"]), out=out)
        check_packed(out, FILL, q, k, v, row0, kv0, lens, ctx, skip=(1,))


def test_plan_of_an_earlier_call():
    from specdec_b200 import _lib

    ops, (H, KV, D) = _ops(), (12, 2, 128)
    lens, extra = [513, 2, 90], [40, 700, 0]
    layers = [packed_case(lens, H, KV, D, s, extra=extra) for s in (1, 2, 3)]
    batch = make_batch(layers[0][3], lens, layers[0][5], layers[0][0].shape[0])
    kv0 = i32(layers[0][4])
    ws = ops.prompt_workspace(batch, H, KV, D)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    for i, c in enumerate(layers):
        out = ops.prompt_attention(*c[:3], batch, kv_row0=kv0, workspace=ws, reuse_plan=i > 0, status=status)
        assert torch.equal(out, ops.prompt_attention(*c[:3], batch, kv_row0=kv0))
    assert int(status) == 0
    # a workspace without a plan, or with one for other shapes, is refused and nothing is written
    c = layers[0]
    for other in (torch.zeros_like(ws), torch.randint(0, 256, ws.shape, dtype=torch.uint8, device="cuda"), ws):
        status.zero_()
        if other is ws:
            small = make_batch(c[3][:2], lens[:2], c[5][:2], c[0].shape[0])
            ops.prompt_attention(*c[:3], small, kv_row0=kv0[:2].contiguous(), workspace=ws)
        out = torch.full_like(c[0], FILL)
        ops.prompt_attention(*c[:3], batch, kv_row0=kv0, workspace=other, reuse_plan=True, status=status, out=out)
        assert int(status) == _lib.STATUS_PLAN_MISMATCH and (out == FILL).all()
    with pytest.raises(ValueError):
        ops.prompt_attention(*c[:3], batch, kv_row0=kv0, reuse_plan=True)


def test_graph_with_changing_lengths_and_another_stream():
    """One captured call replayed over other lengths and values; a second stream with its own workspace beside it."""
    ops, (H, KV, D) = _ops(), (14, 2, 64)
    q, k, v, row0, kv0, ctx = packed_case([200, 200, 200], H, KV, D, 4)
    lens_d, ctx_d, row_d, kv_d = i32([200, 200, 200]), i32([200, 200, 200]), i32(row0), i32(kv0)
    batch = ops.RaggedBatch(row_d, lens_d, ctx_d, 3, 200, 600, 200)
    ws = ops.prompt_workspace(batch, H, KV, D)
    out = torch.full_like(q, FILL)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.prompt_attention(q, k, v, batch, kv_row0=kv_d, out=out, workspace=ws)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.prompt_attention(q, k, v, batch, kv_row0=kv_d, out=out, workspace=ws)
    for lens in ([200, 200, 200], [1, 0, 199], [0, 0, 0], [64, 128, 3]):
        lens_d.copy_(i32(lens))
        ctx_d.copy_(i32(lens))
        out.fill_(FILL)
        side.wait_stream(torch.cuda.current_stream())
        graph.replay()
        with torch.cuda.stream(side):
            beside = ops.prompt_attention(q, k, v, batch, kv_row0=kv_d)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        check_packed(out, FILL, q, k, v, row0, kv0, lens, lens)
        for r, n in zip(row0, lens):
            assert torch.equal(out[r:r + n], beside[r:r + n])


@pytest.mark.parametrize("H,KV,D", [(12, 2, 128), (14, 2, 64)])
def test_a_strange_query_is_its_row_s_own(H, KV, D):
    lens = [200, 70]
    case = packed_case(lens, H, KV, D, 13)
    want = _run(case, lens)
    q = case[0].clone()
    for r, h in ((0, 0), (77, 3), (128, H - 1), (230, 1)):
        q[r, h, 5] = math.nan
        q[r, (h + 1) % H, 9] = math.inf
    got = _run((q, *case[1:]), lens)
    hit = torch.zeros(q.shape[:2], dtype=torch.bool)
    for r, h in ((0, 0), (77, 3), (128, H - 1), (230, 1)):
        hit[r, h] = hit[r, (h + 1) % H] = True
    hit = hit.cuda()
    assert torch.equal(got[~hit], want[~hit])
    # the rows themselves: the formula's NaNs (a row whose only score is -inf has no weight at all and is zero)
    check_packed(got, FILL, q, *case[1:5], lens, case[5])


def test_same_bits_every_time():
    for D in (64, 128):
        lens = [700, 30, 1200]
        case = packed_case(lens, 12, 2, D, 8)
        first = _run(case, lens)
        assert all(torch.equal(first, _run(case, lens)) for _ in range(5))


@pytest.mark.parametrize("sms", [1, 3, 100, 10000])
def test_few_sms(sms):
    """The C entry point with an SM budget (its workspace follows it), and a max_q_len above what is there."""
    from specdec_b200 import _lib

    lib = _lib.load_library()
    H, KV, D, lens, extra = 12, 2, 128, [300, 1, 77], [10, 600, 0]
    q, k, v, row0, kv0, ctx = packed_case(lens, H, KV, D, 6, extra=extra)
    arrays = [i32(x) for x in (row0, lens, ctx, kv0)]
    out = torch.full_like(q, FILL)
    n = lib.specdec_prompt_workspace_bytes(3, H, KV, D, 1000, sms)
    ws = torch.empty(n, dtype=torch.uint8, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    batch = _lib.Batch(q_row0=arrays[0].data_ptr(), q_len=arrays[1].data_ptr(), ctx_len=arrays[2].data_ptr(), num_seqs=3,
                       num_q_heads=H, max_q_len=1000, max_ctx_len=0)
    args = _lib.PromptArgs(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), H * D, D, KV * D, D, KV * D, D, H * D,
                           D, batch, arrays[3].data_ptr(), q.shape[0], k.shape[0], KV, D, 1 / math.sqrt(D), ws.data_ptr(),
                           n, status.data_ptr(), 0, sms)
    _lib.check(lib.specdec_prompt_attention(ctypes.byref(args), torch.cuda.current_stream().cuda_stream), "prompt")
    assert int(status) == 0
    check_packed(out, FILL, q, k, v, row0, kv0, lens, ctx)


def test_refusals_on_the_device():
    ops = _ops()
    q, k, v, row0, kv0, ctx = packed_case([8], 4, 2, 64, 1)
    batch = make_batch(row0, [8], ctx, 8)
    for bad in (dict(out=torch.empty(7, 4, 64, dtype=torch.bfloat16, device="cuda")),
                dict(status=torch.zeros(1, device="cuda")),
                dict(workspace=torch.zeros(64, device="cuda")),
                dict(kv_row0=torch.zeros(1, dtype=torch.int64, device="cuda")),
                dict(sm_scale=0.0), dict(sm_scale=math.nan),
                dict(workspace=torch.zeros(64, dtype=torch.uint8, device="cuda"))):
        with pytest.raises((ValueError, RuntimeError)):
            ops.prompt_attention(q, k, v, batch, **bad)
    for bad in ((q.float(), k, v), (q, k[:, :, :32], v), (q, k, v[:4]), (q, k.cpu(), v.cpu()), (q[:, :3], k, v)):
        with pytest.raises((ValueError, RuntimeError)):
            ops.prompt_attention(*bad, batch)
    assert ops.prompt_attention(q[:0], k, v, batch).shape == (0, 4, 64)
