"""GPU: attention over cache pages that groups of sequences share, against a plain 64-bit form over each sequence's own
page table (tolerance: rows_helpers; E4M3 V as the unrounded products of codes and scales)."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

from rows_helpers import Pages, assert_rows, check_pages, i32, make_batch, plain_attention

pytestmark = pytest.mark.gpu
FILL = 7.0


def _ops():
    from specdec_b200.kernels import ops

    return ops


def _rows(lens, H, D, seed, gap=0, order=None):
    """q and the first row of every sequence, sequences' rows in ``order``, ``gap`` rows of nobody's between."""
    row0, r = [0] * len(lens), gap
    for b in order or range(len(lens)):
        row0[b] = r
        r += lens[b] + gap
    q = torch.randn(max(r, 1), H, D, generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16).cuda()
    return q, row0


def _run(q, row0, lens, ctx, pages, groups, *, q_max=None, layer=0, want_status=0, **kw):
    prefix = groups if not isinstance(groups, list) else _ops().SharedPrefix.from_groups(groups)
    out = torch.full(q.shape, FILL, dtype=q.dtype, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    batch = make_batch(row0, lens, ctx, q.shape[0], q_max)
    _ops().shared_prefix_attention(q, pages.cache, layer, batch, prefix, out=out, status=status, **kw)
    assert int(status) == want_status
    return out


FORMS = [(12, 2, 128, False), (12, 2, 128, True), (14, 2, 64, False), (7, 7, 64, False), (33, 1, 128, True),
         (128, 1, 128, False), (80, 2, 64, False)]
CASES = {  # name: (new tokens, context, groups)
    "one_alone": ([1], [1], []),
    "nobody_shares": ([1, 1, 5], [40, 700, 5], []),
    "decode": ([1] * 4, [300, 301, 290, 272], [([0, 1, 2, 3], 272)]),
    "decode_ends": ([1] * 6, [257, 258, 259, 272, 273, 512], [([0, 1, 2, 3, 4, 5], 256)]),
    "verify": ([5] * 7, [150, 145, 133, 160, 149, 700, 133], [(list(range(7)), 128)]),
    "ragged": ([5, 1, 0, 3, 2, 5], [90, 81, 300, 84, 85, 400], [([0, 1, 2, 3], 80), ([4, 5], 64)]),
    "groups_and_others": ([2, 1, 4, 1, 3], [600, 50, 604, 70, 603], [([4, 0, 2], 590)]),
    "not_whole_pages": ([1, 1, 1], [100, 90, 80], [([0, 1, 2], 79)]),
    "longer_than_seen": ([3, 3], [67, 100], [([0, 1], 96)]),  # sequence 0 sees 64 .. 66 keys
    "short_prefix": ([1, 2], [40, 30], [([0, 1], 15)]),
    "no_prefix": ([1, 2], [40, 30], [([0, 1], 0)]),
    "empty_groups": ([1, 2], [40, 30], [([], 16), ([0, 1], 16), ([], 0)]),
    "one_member": ([2, 2], [200, 200], [([1], 160)]),
    "all_of_it": ([1, 1], [65, 65], [([0, 1], 64)]),
    "first_has_no_rows": ([0, 2, 2], [20, 100, 130], [([0, 1, 2], 96)]),
    "nobody_has_rows": ([0, 0], [30, 30], [([0, 1], 16)]),
    "long": ([5, 5, 5], [8200, 8300, 8192], [([0, 1, 2], 8176)]),
    "blocks": ([140, 30], [300, 260], [([0, 1], 128)]),
    "many": ([3] * 70, [200 + i for i in range(70)], [(list(range(0, 70, 2)), 192), (list(range(1, 70, 2)), 160)]),
}


@pytest.mark.parametrize("H,KV,D,v8", FORMS)
@pytest.mark.parametrize("case", CASES)
def test_groups(H, KV, D, v8, case):
    lens, ctx, groups = CASES[case]
    pages = Pages(ctx, groups, KV, D, v8, len(case) + H)
    q, row0 = _rows(lens, H, D, H + D)
    out = _run(q, row0, lens, ctx, pages, groups)
    check_pages(out, FILL, q, pages, row0, lens, ctx, what=case)


@pytest.mark.parametrize("H,KV,D,v8", FORMS[:3])
@pytest.mark.parametrize("case", ["ragged", "groups_and_others", "verify", "many"])
def test_rows_anywhere(H, KV, D, v8, case):
    """The members' rows in another order, with rows of nobody's between them; a larger max_q_len than there is."""
    lens, ctx, groups = CASES[case]
    pages = Pages(ctx, groups, KV, D, v8, 2)
    order = torch.randperm(len(lens), generator=torch.Generator().manual_seed(4)).tolist()
    q, row0 = _rows(lens, H, D, 1, gap=2, order=order)
    for q_max in (None, max(lens) + 4):
        out = _run(q, row0, lens, ctx, pages, groups, q_max=q_max)
        check_pages(out, FILL, q, pages, row0, lens, ctx, what=case)


@pytest.mark.parametrize("H,KV,D,v8", FORMS[:3])
def test_the_answer_of_paged_attention(H, KV, D, v8):
    ops = _ops()
    lens, ctx, groups = CASES["verify"]
    pages = Pages(ctx, groups, KV, D, v8, 9)
    q, row0 = _rows(lens, H, D, 9)
    got = _run(q, row0, lens, ctx, pages, groups, sm_scale=0.05)
    check_pages(got, FILL, q, pages, row0, lens, ctx, scale=0.05)
    batch = make_batch(row0, lens, ctx, q.shape[0])
    want = ops.paged_attention(q, pages.cache, 0, batch)
    got = _run(q, row0, lens, ctx, pages, groups)
    # both within their own bounds of the same formula: this one's, and one output rounding and P's twice for the other
    for b, (r, n, t) in enumerate(zip(row0, lens, ctx)):
        k, v = pages.kv(b)
        _, tol = plain_attention(q[r:r + n], k, v, torch.arange(n) + (t - n + 1), 1 / math.sqrt(D))
        assert ((got[r:r + n].double() - want[r:r + n].double()).abs() <= 4 * tol).all(), b


@pytest.mark.parametrize("H,KV,D,v8", FORMS[:3])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_nothing_behind_a_sequence_reaches_it(H, KV, D, v8, bad):
    """NaN and infinite values in pages that are nobody's, and behind the last key of every sequence's last page."""
    lens, ctx, groups = CASES["ragged"]
    pages = Pages(ctx, groups, KV, D, v8, 3)
    q, row0 = _rows(lens, H, D, 3)
    want = _run(q, row0, lens, ctx, pages, groups)
    pool, pt = pages.cache.pools[0], pages.cache.page_table.cpu()
    unused = torch.ones(pages.cache.num_pages, dtype=torch.bool)
    unused[pt[pt >= 0].long()] = False
    from specdec_b200.engine.paged_cache import kblock_index

    idx = kblock_index(D, "cuda").view(16, D)
    pool.k[unused.cuda()] = bad
    if v8:
        pool.v[unused.cuda()] = 0x7f  # NaN codes
        pool.v_scale[unused.cuda()] = bad
    else:
        pool.v[unused.cuda()] = bad
    for b, t in enumerate(ctx):
        if t % 16 == 0:
            continue
        page, tail = int(pt[b, t // 16]), idx[t % 16:].reshape(-1)
        pool.k[page][:, tail] = bad
        if v8:
            pool.v[page].view(KV, 16, D)[:, t % 16:] = 0x7f
            pool.v_scale[page][:, t % 16:] = bad
        else:
            pool.v[page][:, tail] = bad
    assert torch.equal(_run(q, row0, lens, ctx, pages, groups), want)


@pytest.mark.parametrize("H,KV,D,v8", FORMS[:3])
def test_strange_values_of_the_last_tokens(H, KV, D, v8):
    """In a verify block V of its second-last token is infinite: the rows before it do not notice."""
    lens, ctx = [5, 5, 4], [150, 133, 170]
    groups = [([0, 1, 2], 128)]
    pages = Pages(ctx, groups, KV, D, v8, 5)
    q, row0 = _rows(lens, H, D, 5)
    clean = _run(q, row0, lens, ctx, pages, groups)
    pool, pt = pages.cache.pools[0], pages.cache.page_table.cpu()
    from specdec_b200.engine.paged_cache import kblock_index

    for b, t in enumerate(ctx):
        page, at = int(pt[b, (t - 2) // 16]), (t - 2) % 16
        if v8:
            pool.v_scale[page, 0, at] = math.nan
        else:
            pool.v[page, 0, kblock_index(D, "cuda").view(16, D)[at, 5:7]] = math.inf
    out = _run(q, row0, lens, ctx, pages, groups)
    check_pages(out, FILL, q, pages, row0, lens, ctx)
    for r, n in zip(row0, lens):
        assert torch.equal(out[r:r + n - 2], clean[r:r + n - 2])
        assert not out[r + n - 2:r + n, 0].isfinite().all()


def test_bad_groups():
    """A bad group is reported; what the rest of the call says stands, and every row has its answer."""
    from specdec_b200 import _lib

    ops, (H, KV, D) = _ops(), (12, 2, 128)
    lens, ctx, groups = CASES["verify"]
    pages = Pages(ctx, groups, KV, D, False, 6)
    q, row0 = _rows(lens, H, D, 6)
    for start, members, length in [
        ([0, 8], [0, 1, 2, 3, 3, 4, 5, 6], [128]),       # listed twice
        ([0, 3, 6], [0, 1, 2, 2, 1, 3], [128, 128]),      # in two groups: the first counts
        ([0, 4], [0, -1, 2, 7], [128]),                   # no sequences
        ([0, 4], [2**31 - 1, -2**31, 0, 1], [128]),
        ([0, 3], [0, 1, 2], [-16]),                       # a negative prefix
        ([0, 4], [0, 1, 2], [128]),                       # starts past the members
        ([-1, 3], [0, 1, 2], [128]),
        ([2, 1], [0, 1, 2], [128]),
        ([0, 3, 2], [0, 1, 2], [128, 128]),
        ([2**31 - 1, -2**31], [0, 1, 2], [128]),
    ]:
        prefix = ops.SharedPrefix(i32(start), i32(members), i32(length), len(length), len(members))
        out = _run(q, row0, lens, ctx, pages, prefix, want_status=_lib.STATUS_BAD_GROUP)
        check_pages(out, FILL, q, pages, row0, lens, ctx, what=str((start, members, length)))
    # lists that leave members out, and a prefix far past everything, are fine
    for start, members, length in [([1, 3], [0, 1, 2, 3], [128]), ([0, 2], [0, 6], [2**31 - 1])]:
        short = Pages(ctx, [([0, 6], 128)], KV, D, False, 6) if length[0] > 128 else pages
        prefix = ops.SharedPrefix(i32(start), i32(members), i32(length), 1, len(members))
        out = _run(q, row0, lens, ctx, short, prefix)
        check_pages(out, FILL, q, short, row0, lens, ctx)


def test_bad_lengths_and_pages():
    from specdec_b200 import _lib

    H, KV, D = 12, 2, 128
    lens, ctx, groups = CASES["verify"]
    for v8 in (False, True):
        pages = Pages(ctx, groups, KV, D, v8, 7)
        q, row0 = _rows(lens, H, D, 7)
        cap = pages.cache.capacity
        for b, field, value, want in [(2, "lens", -3, _lib.STATUS_BAD_LENGTH), (2, "ctx", 4, _lib.STATUS_BAD_LENGTH),
                                      (0, "row0", -1, _lib.STATUS_BAD_LENGTH), (6, "row0", 31, _lib.STATUS_BAD_LENGTH),
                                      (1, "ctx", cap + 1, _lib.STATUS_PAGE_OVERFLOW),
                                      (1, "ctx", 2**31 - 1, _lib.STATUS_PAGE_OVERFLOW)]:
            a = dict(lens=list(lens), ctx=list(ctx), row0=list(row0))
            a[field][b] = value
            out = _run(q, a["row0"], a["lens"], a["ctx"], pages, groups, q_max=5, want_status=want)
            check_pages(out, FILL, q, pages, row0, lens, ctx, what=f"{field}[{b}]={value}", skip=(b,))
        # a page id outside the pool is reported and never followed
        for value in (-1, pages.cache.num_pages, 2**31 - 1, -2**31):
            pages.cache.page_table[3, 9] = value
            out = _run(q, row0, lens, ctx, pages, groups, want_status=_lib.STATUS_BAD_PAGE)
            for b in (0, 1, 2, 4, 5, 6):
                k, v = pages.kv(b)
                r, n, t = row0[b], lens[b], ctx[b]
                want, tol = plain_attention(q[r:r + n], k, v, torch.arange(n) + (t - n + 1), 1 / math.sqrt(D))
                assert_rows(out[r:r + n], want, tol, f"sequence {b}")


def test_layers_reuse_the_plan():
    from specdec_b200 import _lib

    ops, (H, KV, D) = _ops(), (12, 2, 128)
    lens, ctx, groups = CASES["ragged"]
    pages = Pages(ctx, groups, KV, D, True, 8, layers=3)
    prefix = ops.SharedPrefix.from_groups(groups)
    q, row0 = _rows(lens, H, D, 8)
    batch = make_batch(row0, lens, ctx, q.shape[0])
    ws = ops.shared_prefix_workspace(batch, prefix, H, pages.cache)
    for layer in range(3):
        out = torch.full_like(q, FILL)
        ops.shared_prefix_attention(q, pages.cache, layer, batch, prefix, out=out, workspace=ws, reuse_plan=layer > 0)
        check_pages(out, FILL, q, pages, row0, lens, ctx, layer=layer)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    for other in (torch.zeros_like(ws), torch.randint(0, 256, ws.shape, dtype=torch.uint8, device="cuda")):
        out = torch.full_like(q, FILL)
        status.zero_()
        ops.shared_prefix_attention(q, pages.cache, 0, batch, prefix, out=out, workspace=other, reuse_plan=True,
                                    status=status)
        assert int(status) == _lib.STATUS_PLAN_MISMATCH and (out == FILL).all()


@pytest.mark.parametrize("v8", [False, True])
def test_graph_with_changing_lengths(v8):
    """Lengths, groups' prefixes and page tables change between replays; a call on another stream runs beside."""
    ops, (H, KV, D) = _ops(), (12, 2, 128)
    ctx = [400, 380, 390, 300]
    groups = [([0, 1, 2], 368)]
    pages = Pages(ctx, groups, KV, D, v8, 10)
    lens = [3, 3, 3, 3]
    q, row0 = _rows(lens, H, D, 10)
    prefix = ops.SharedPrefix.from_groups(groups)
    batch = make_batch(row0, lens, ctx, q.shape[0])
    ws = ops.shared_prefix_workspace(batch, prefix, H, pages.cache)
    out = torch.full_like(q, FILL)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.shared_prefix_attention(q, pages.cache, 0, batch, prefix, out=out, workspace=ws)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.shared_prefix_attention(q, pages.cache, 0, batch, prefix, out=out, workspace=ws)
    for new, now, shared in [(lens, ctx, 368), ([1, 0, 3, 2], [370, 380, 390, 2], 160), ([3, 3, 3, 3], [3, 3, 3, 3], 368),
                             ([0, 0, 0, 1], ctx, 0)]:
        batch.q_len.copy_(i32(new))
        batch.ctx_len.copy_(i32(now))
        prefix.prefix_len.fill_(shared)
        out.fill_(FILL)
        side.wait_stream(torch.cuda.current_stream())
        graph.replay()
        with torch.cuda.stream(side):
            beside = ops.shared_prefix_attention(q, pages.cache, 0, batch, prefix)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        check_pages(out, FILL, q, pages, row0, new, now)
        for r, n in zip(row0, new):
            assert torch.equal(out[r:r + n], beside[r:r + n])


def test_most_sequences():
    ops, (H, KV, D), B = _ops(), (14, 2, 64), 2048
    g = torch.Generator().manual_seed(12)
    ctx = torch.randint(33, 80, (B,), generator=g).tolist()
    groups = [(list(range(i, B, 16)), 32) for i in range(16)]
    pages = Pages(ctx, groups, KV, D, False, 12)
    q, row0 = _rows([1] * B, H, D, 12)
    out = _run(q, row0, [1] * B, ctx, pages, groups)
    for b in torch.randperm(B, generator=g)[:80].tolist():
        k, v = pages.kv(b)
        want, tol = plain_attention(q[b:b + 1], k, v, torch.tensor([ctx[b]]), 1 / math.sqrt(D))
        assert_rows(out[b:b + 1], want, tol, f"sequence {b}")
    # as many groups as sequences
    groups = [([b], 32) for b in range(B)]
    assert torch.equal(_run(q, row0, [1] * B, ctx, pages, groups)[::37], _run(q, row0, [1] * B, ctx, pages, groups)[::37])
    with pytest.raises(ValueError):
        batch = make_batch([0] * 2049, [0] * 2049, [0] * 2049, q.shape[0])
        ops.shared_prefix_attention(q, pages.cache, 0, batch, ops.SharedPrefix.from_groups([]))


def test_same_bits_every_time():
    for v8 in (False, True):
        lens, ctx, groups = CASES["many"]
        pages = Pages(ctx, groups, 2, 128, v8, 14)
        q, row0 = _rows(lens, 12, 128, 14)
        first = _run(q, row0, lens, ctx, pages, groups)
        assert all(torch.equal(first, _run(q, row0, lens, ctx, pages, groups)) for _ in range(5))


def test_offsets_past_32_bits():
    """A pool whose V lies more than 2^32 bytes behind its start."""
    H, KV, D = 12, 2, 128
    pages = Pages([100, 90], [([0, 1], 64)], KV, D, False, 15, spare=600_000)  # 4.9 GB a pool
    c = pages.cache
    last = c.num_pages - 7
    table = c.page_table.clone()
    for e, (b, j) in enumerate([(0, 6), (1, 5)]):
        for t in (c.pools[0].k, c.pools[0].v):
            t[last + e] = t[int(table[b, j])]
        table[b, j] = last + e
    c.page_table.copy_(table)
    assert last * KV * 16 * D * 2 > 2**32
    q, row0 = _rows([2, 2], H, D, 15)
    out = _run(q, row0, [2, 2], [100, 90], pages, [([0, 1], 64)])
    check_pages(out, FILL, q, pages, row0, [2, 2], [100, 90])


@pytest.mark.parametrize("sms", [1, 5, 1000])
def test_few_sms(sms):
    from specdec_b200 import _lib

    ops, lib = _ops(), _lib.load_library()
    H, KV, D = 12, 2, 128
    lens, ctx, groups = CASES["groups_and_others"]
    pages = Pages(ctx, groups, KV, D, True, 16)
    q, row0 = _rows(lens, H, D, 16)
    p = ops.SharedPrefix.from_groups(groups)
    batch = make_batch(row0, lens, ctx, q.shape[0])
    n = lib.specdec_shared_prefix_workspace_bytes(len(lens), H, KV, D, batch.max_q_len, 1, 3, sms)
    ws = torch.empty(n, dtype=torch.uint8, device="cuda")
    out, status = torch.full_like(q, FILL), torch.zeros(1, dtype=torch.int32, device="cuda")
    args = _lib.SharedPrefixArgs(q.data_ptr(), out.data_ptr(), H * D, D, H * D, D,
                                 _lib.Batch(*ops._batch_fields(batch, H, q.get_device())), ops._paged_kv(pages.cache, 0),
                                 p.group_start.data_ptr(), p.members.data_ptr(), p.prefix_len.data_ptr(), 1, 3, q.shape[0],
                                 1 / math.sqrt(D), ws.data_ptr(), n, status.data_ptr(), 0, sms)
    _lib.check(lib.specdec_shared_prefix_attention(ctypes.byref(args), torch.cuda.current_stream().cuda_stream), "shared")
    assert int(status) == 0
    check_pages(out, FILL, q, pages, row0, lens, ctx)


def test_refusals_on_the_device():
    ops = _ops()
    lens, ctx, groups = CASES["decode"]
    pages = Pages(ctx, groups, 2, 64, False, 1)
    q, row0 = _rows(lens, 14, 64, 1)
    batch, prefix = make_batch(row0, lens, ctx, 4), ops.SharedPrefix.from_groups(groups)
    for bad in (dict(out=q.float()), dict(status=torch.zeros(1, device="cuda")), dict(reuse_plan=True),
                dict(workspace=torch.zeros(8, dtype=torch.uint8, device="cuda")), dict(sm_scale=-1.0)):
        with pytest.raises((ValueError, RuntimeError)):
            ops.shared_prefix_attention(q, pages.cache, 0, batch, prefix, **bad)
    wide = torch.zeros(4, 14, 128, dtype=torch.bfloat16, device="cuda")
    more = make_batch(row0 + [0], lens + [0], ctx + [0], 4)
    cpu = ops.SharedPrefix.from_groups(groups, device="cpu")
    for args in ((wide, pages.cache, 0, batch, prefix), (q, pages.cache, 0, more, prefix), (q, pages.cache, 0, batch, cpu),
                 (q[:, :13], pages.cache, 0, batch, prefix)):
        with pytest.raises((ValueError, RuntimeError)):
            ops.shared_prefix_attention(*args)
