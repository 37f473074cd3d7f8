"""GPU: prompt_attention and shared_prefix_attention at the edges of what they promise: waits that give up."""

from __future__ import annotations

import pytest
import torch

from rows_helpers import Pages, check_packed, check_pages, i32, make_batch, packed_case

pytestmark = pytest.mark.gpu
FILL = 7.0


def _ops():
    from specdec_b200.kernels import ops

    return ops


@pytest.fixture
def wait_limit():
    """Sets the limit of the attention's device waits for a test; one second again after it."""
    from specdec_b200 import _lib

    lib = _lib.load_library()
    yield lambda ns: _lib.check(lib.specdec_wait_limit_selftest(ns), "wait_limit_selftest")
    torch.cuda.synchronize()
    lib.specdec_wait_limit_selftest(1_000_000_000)


# prompts of one item, of several items a CTA, cut into pieces, with rows of nobody's between; (key rows before each)
PROMPTS = {
    "one": (12, 2, 128, [37], [0]),
    "chunk": (12, 2, 128, [100], [3000]),
    "packed": (12, 2, 128, [300, 1, 0, 700, 129], [0, 40, 0, 0, 500]),
    "packed_64": (14, 2, 64, [300, 1, 0, 700, 129], [0, 40, 0, 0, 500]),
    "many_items": (2, 2, 128, [3] * 1500, [0] * 1500),
    "many_items_64": (5, 5, 64, [3] * 900, [1] * 900),
}
# (heads, KV heads, head_dim, E4M3, new rows, contexts, groups)
SHARED = {
    "alone": (12, 2, 128, False, [1], [300], []),
    "verify": (12, 2, 128, False, [5] * 7, [750, 745, 733, 760, 749, 900, 733], [(list(range(7)), 720)]),
    "verify_e4m3": (12, 2, 128, True, [5] * 7, [750, 745, 733, 760, 749, 900, 733], [(list(range(7)), 720)]),
    "rows_anywhere": (14, 2, 64, False, [5, 1, 0, 3], [90, 181, 300, 84], [([2, 0, 3], 80)]),
    "many_e4m3": (12, 2, 128, True, [3] * 400, [40 + i % 50 for i in range(400)], [(list(range(400)), 32)]),
}


def _prompt_call(name):
    H, KV, D, lens, extra = PROMPTS[name]
    q, k, v, row0, kv0, ctx = packed_case(lens, H, KV, D, 3, gap=1, extra=extra)
    batch = make_batch(row0, lens, ctx, q.shape[0])
    buf = torch.full((q.shape[0] + 2, H, D), FILL, dtype=q.dtype, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    rows = [i for r, n in zip(row0, lens) for i in range(r, r + n)]

    def call():
        return _ops().prompt_attention(q, k, v, batch, kv_row0=i32(kv0), out=buf[1:-1], status=status)

    return call, buf, status, rows, lambda: check_packed(buf[1:-1], FILL, q, k, v, row0, kv0, lens, ctx, what=name)


def _shared_call(name):
    H, KV, D, v8, lens, ctx, groups = SHARED[name]
    pages = Pages(ctx, groups, KV, D, v8, 4)
    row0 = [sum(lens[:b]) + b for b in range(len(lens))]
    g = torch.Generator().manual_seed(6)
    q = torch.randn(sum(lens) + len(lens), H, D, generator=g).to(torch.bfloat16).cuda()
    batch, prefix = make_batch(row0, lens, ctx, q.shape[0]), _ops().SharedPrefix.from_groups(groups)
    buf = torch.full((q.shape[0] + 2, H, D), FILL, dtype=q.dtype, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    rows = [i for r, n in zip(row0, lens) for i in range(r, r + n)]

    def call():
        return _ops().shared_prefix_attention(q, pages.cache, 0, batch, prefix, out=buf[1:-1], status=status)

    return call, buf, status, rows, lambda: check_pages(buf[1:-1], FILL, q, pages, row0, lens, ctx, what=name)


CALLS = [(_prompt_call, name) for name in PROMPTS] + [(_shared_call, name) for name in SHARED]


@pytest.mark.parametrize("make,name", CALLS, ids=[n for _, n in CALLS])
def test_waits_that_give_up_end_the_call(make, name, wait_limit):
    """The softmax warps give up on their first item, with copies and products of it under way: the call ends and says
    so, nothing beside its rows is written, and the next call is right."""
    from specdec_b200 import _lib

    call, buf, status, rows, check = make(name)
    torch.cuda.synchronize()
    for _ in range(3):
        wait_limit(0)
        call()
        torch.cuda.synchronize()
        assert int(status) == _lib.STATUS_TIMEOUT
        assert (buf[0] == FILL).all() and (buf[-1] == FILL).all()
        wait_limit(1_000_000_000)
        status.zero_()
        buf.fill_(FILL)
        call()
        assert int(status) == 0
        check()


@pytest.mark.parametrize("make,name", CALLS, ids=[n for _, n in CALLS])
def test_what_waits_gave_up_on_is_nan(make, name, wait_limit):
    """No row keeps what the output or the workspace held before: all are NaN where every first wait gives up, and each
    is NaN or right where only some run out."""
    from specdec_b200 import _lib

    call, buf, status, rows, check = make(name)
    call()
    torch.cuda.synchronize()
    good = buf.clone()
    for limit in (0, 0, 1, 1000, 5000, 20_000, 50_000):
        buf.fill_(FILL)
        status.zero_()
        wait_limit(limit)
        call()
        torch.cuda.synchronize()
        wait_limit(1_000_000_000)
        out = buf[1:-1]
        here, want = out[rows], good[1:-1][rows]
        nan = here.isnan().all(-1)
        assert torch.equal(here[~nan], want[~nan])
        assert nan.all() or limit > 0
        assert int(status) == (_lib.STATUS_TIMEOUT if nan.any() else int(status) & _lib.STATUS_TIMEOUT)
        left = torch.ones(buf.shape[0], dtype=torch.bool)
        left[[r + 1 for r in rows]] = False
        assert (buf[left.cuda()] == FILL).all()
