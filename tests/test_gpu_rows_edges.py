"""GPU: prompt_attention and shared_prefix_attention at the edges of what they promise: waits that give up, values that
are not finite under weights of zero."""

from __future__ import annotations

import math

import pytest
import torch

from rows_helpers import Pages, assert_rows, check_packed, check_pages, i32, make_batch, packed_case, plain_attention

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


def _weightless(how, q, k, strong, key):
    """Gives ``key`` no weight in any row: ``strong`` past it by more than fp32's range, or its own score -inf."""
    q[..., 0] = 64.0
    k[..., 0] = 0.0
    if how == "underflow":
        k[strong, :, 0] = 64.0  # 4096 of scale 1 / sqrt(D) and log2 e: 522 (D 64: 738)
    else:
        k[key, :, 0] = -math.inf


def _check_weightless(out, q, k, v, limit, key, dim, what):
    """Rows that see ``key``: the value at ``dim`` of its KV head is not finite, the rest is as without it."""
    fine = torch.where(v.isfinite(), v, 0.0)
    want, tol = plain_attention(q, torch.where(k.isfinite(), k, -1e4), fine, limit, 1 / math.sqrt(q.shape[-1]))
    rep = q.shape[1] // k.shape[1]
    sees = (limit > key).cuda()
    assert not out[sees][:, :rep, dim].isfinite().any(), what
    got = out.clone()
    got[sees, :rep, dim] = want[sees][:, :rep, dim].to(out.dtype)
    assert_rows(got, want, tol, what)


# a key in front of everything, in a middle piece of a cut unit, before and behind the first key that some row does not see
@pytest.mark.parametrize("how", ["underflow", "minus_infinity"])
@pytest.mark.parametrize("H,KV,D", [(12, 2, 128), (14, 2, 64)])
def test_infinite_values_without_weight_packed(H, KV, D, how):
    for n, e in ((300, 2500), (40, 5000), (200, 0)):
        for key in (0, e // 2, e - 1, e, e + n // 2, e + n - 1):
            if key < 0:
                continue
            for strong in {key + 1, max(key - 1, 0), 0, e // 3} - {key}:
                if strong >= e + 1:  # (every row sees it)
                    continue
                q, k, v, row0, kv0, ctx = packed_case([n], H, KV, D, 11, extra=[e])
                _weightless(how, q, k, strong, key)
                v[key, 0, 5] = math.inf
                out = _ops().prompt_attention(q, k, v, make_batch(row0, [n], ctx, n), kv_row0=i32(kv0))
                _check_weightless(out, q, k, v, torch.arange(n) + e + 1, key, 5, f"{n} after {e}, key {key}, {strong} strong")


@pytest.mark.parametrize("how", ["underflow", "minus_infinity"])
@pytest.mark.parametrize("H,KV,D", [(12, 2, 128), (14, 2, 64)])
def test_infinite_values_without_weight_pages(H, KV, D, how):
    """The key in the shared prefix, the strong one among the sequence's own keys, and the other way round."""
    from specdec_b200.engine.paged_cache import kblock_index

    lens, ctx, groups = [5] * 4, [2100, 2110, 2095, 2400], [([0, 1, 2, 3], 2080)]
    idx = kblock_index(D, "cuda").view(16, D)
    for key, strong in ((17, 2085), (2079, 2085), (2085, 17), (2092, 2079), (900, 17)):
        pages = Pages(ctx, groups, KV, D, False, 12)
        pool, pt = pages.cache.pools[0], pages.cache.page_table.cpu()
        q = torch.randn(20, H, D, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).cuda()
        q[..., 0] = 64.0
        pool.k[..., idx[:, 0]] = 0.0
        for b in range(4):
            at = {j: (int(pt[b, j // 16]), j % 16) for j in (key, strong)}
            if how == "underflow":
                pool.k[at[strong][0], :, idx[at[strong][1], 0]] = 64.0
            else:
                pool.k[at[key][0], :, idx[at[key][1], 0]] = -math.inf
            pool.v[at[key][0], 0, idx[at[key][1], 5]] = math.inf
        out = _ops().shared_prefix_attention(q, pages.cache, 0, make_batch([0, 5, 10, 15], lens, ctx, 20),
                                             _ops().SharedPrefix.from_groups(groups))
        for b in range(4):
            k, v = pages.kv(b)
            _check_weightless(out[5 * b:5 * b + 5], q[5 * b:5 * b + 5], k, v, torch.arange(5) + ctx[b] - 4, key, 5,
                              f"sequence {b}, key {key}, {strong} strong")
