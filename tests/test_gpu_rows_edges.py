"""GPU: prompt_attention and shared_prefix_attention at the edges of what they promise: waits that give up, values that
are not finite under weights of zero, E4M3 scales."""

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


def _f16_tolerance(q, k, v, limit, scale):
    """As rows_helpers' tolerance with weights that are rounded to f16: 2^-11 A in the place of 2^-8 A, where none of them
    is below f16's normal range."""
    want, tol = plain_attention(q, k, v, limit, scale)
    A, _ = plain_attention(q, k, v.abs(), limit, scale)
    return want, tol - A * (2.0**-8 - 2.0**-11)


def _e4m3_pages(ctx, groups, scales, seed, zero=()):
    """E4M3 pages, scales[b](n) the scales of sequence b's tokens; the codes of the tokens in ``zero`` are 0."""
    pages = Pages(ctx, groups, 2, 128, True, seed)
    pool, pt = pages.cache.pools[0], pages.cache.page_table.cpu()
    for b, n in enumerate(ctx):
        s = scales[b](n).cuda()
        for j in range(n):
            page, at = int(pt[b, j // 16]), j % 16
            pool.v_scale[page, :, at] = s[j]
            if j in zero:
                pool.v[page].view(2, 16, 128)[:, at] = 0
    return pages, pool, pt


def test_e4m3_weights_keep_eleven_bits():
    """Two keys of equal weight and opposite codes: what is left is the difference of their scales, and the rounding of
    weight times scale shows at its full size."""
    B = 60
    g = torch.Generator().manual_seed(1)
    pages = Pages([2] * B, [], 2, 128, True, 21)
    pool, pt = pages.cache.pools[0], pages.cache.page_table.cpu()
    for b in range(B):
        codes = pool.v[int(pt[b, 0])].view(2, 16, 128)
        codes[:, 1] = codes[:, 0] ^ 0x80
    q = torch.zeros(B, 12, 128, dtype=torch.bfloat16, device="cuda")
    for groups in ([], [(list(range(B)), 0)]):
        out = _ops().shared_prefix_attention(q, pages.cache, 0, make_batch(list(range(B)), [1] * B, [2] * B, B),
                                             _ops().SharedPrefix.from_groups(groups))
        for b in range(B):
            k, v = pages.kv(b)
            assert_rows(out[b:b + 1], *_f16_tolerance(q[b:b + 1], k, v, torch.tensor([2]), 0.1), f"sequence {b}")


# scales of a sequence's tokens; with queries of zero every weight is 1, and times its scale and the unit (2^-b where
# the reference moves by b) stays between 2^-14 and 2^15
SCALES = {
    "mixed": lambda n: torch.exp2(torch.rand(n, generator=torch.Generator().manual_seed(n)) * 12 - 6),
    "zero_tokens": lambda n: torch.where(torch.arange(n) % 100 == 3, 1.0, 2.0**-22 * 1.3),
    "growing": lambda n: torch.where(torch.arange(n) < 128, 2.0**-20, 1.1),
    "falling": lambda n: torch.where(torch.arange(n) < 128, 1.7, 2.0**-9),
    "first_zero": lambda n: torch.where(torch.arange(n) == 0, 1.0, 2.0**-12 * 1.9),
    "tiny": lambda n: torch.full((n,), 2.0**-90),
    "huge": lambda n: torch.full((n,), 2.0**90),
}


@pytest.mark.parametrize("name", SCALES)
def test_e4m3_scales_of_any_size(name):
    lens, ctx, groups = [1, 5, 3], [1500, 700, 90], [([0, 1], 640)]
    zero = [j for j in range(1500) if j % 100 == 3] if name == "zero_tokens" else [0] if name == "first_zero" else []
    pages, _, _ = _e4m3_pages(ctx, groups, [SCALES[name]] * 3, 22, zero)
    q = torch.zeros(9, 12, 128, dtype=torch.bfloat16, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    for members in ([], groups):
        out = _ops().shared_prefix_attention(q, pages.cache, 0, make_batch([0, 1, 6], lens, ctx, 9),
                                             _ops().SharedPrefix.from_groups(members), status=status)
        for b, r in enumerate((0, 1, 6)):
            k, v = pages.kv(b)
            limit = torch.arange(lens[b]) + (ctx[b] - lens[b] + 1)
            assert_rows(out[r:r + lens[b]], *_f16_tolerance(q[r:r + lens[b]], k, v, limit, 0.1), f"sequence {b}")
    assert int(status) == 0


@pytest.mark.parametrize("below", [10, 16, 18, 20])
def test_e4m3_scales_far_below_the_mean_lose_bits_only(below):
    """The first 128 tokens are zeros (scale 1), the others' scales are 2^-below: their weights count as 1.3 2^(2 - below),
    below 2^-14 a number of f16's subnormal range, off by half of its step, 2^-25, and not by all of it."""
    n = 600
    pages, _, _ = _e4m3_pages([n], [], [lambda n: torch.where(torch.arange(n) < 128, 1.0, 1.3 * 2.0**-below)], 24, range(128))
    q = torch.zeros(1, 12, 128, dtype=torch.bfloat16, device="cuda")
    out = _ops().shared_prefix_attention(q, pages.cache, 0, make_batch([0], [1], [n], 1), _ops().SharedPrefix.from_groups([]))
    k, v = pages.kv(0)
    want, tol = _f16_tolerance(q, k, v, torch.tensor([n]), 0.1)
    A, _ = plain_attention(q, k, v.abs(), torch.tensor([n]), 0.1)
    assert_rows(out, want, tol + A * (2.0**-25 / (1.3 * 2.0**(2 - below))), f"2^-{below}")


@pytest.mark.parametrize("scale", [1e30, 1e-30, 0.0, math.inf, math.nan])
def test_e4m3_scale_of_a_later_token_reaches_no_bit(scale):
    """The last new token's scale is anything: the rows before it keep their bits, and its own are that token's."""
    lens, ctx = [5] * 4, [20, 131, 300, 645]
    pages, pool, pt = _e4m3_pages(ctx, [], [lambda n: torch.rand(n, generator=torch.Generator().manual_seed(n)) + 0.5] * 4, 23)
    q = torch.randn(20, 12, 128, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16).cuda()
    q[:, ::3] *= 8  # (a reference that moves, too)

    def run(groups):
        return _ops().shared_prefix_attention(q, pages.cache, 0, make_batch([0, 5, 10, 15], lens, ctx, 20),
                                              _ops().SharedPrefix.from_groups(groups))

    for groups in ([], [([0, 1, 2, 3], 16)]):
        clean = run(groups)
        kept = []
        for b, t in enumerate(ctx):
            page, at = int(pt[b, (t - 1) // 16]), (t - 1) % 16
            kept.append((page, at, pool.v_scale[page, :, at].clone()))
            pool.v_scale[page, :, at] = scale
        out = run(groups)
        for b in range(4):
            assert torch.equal(out[5 * b:5 * b + 4], clean[5 * b:5 * b + 4]), b
            k, v = pages.kv(b)
            if math.isfinite(scale):
                want, tol = plain_attention(q[5 * b + 4:5 * b + 5], k, v, torch.tensor([ctx[b]]), 1 / math.sqrt(128))
                assert_rows(out[5 * b + 4:5 * b + 5], want, tol, f"sequence {b}")
            else:
                assert not out[5 * b + 4].isfinite().any()
        for page, at, s in kept:
            pool.v_scale[page, :, at] = s


def test_as_many_groups_as_sequences():
    """2048 groups of one sequence each, the most of a call: values, against the 64-bit form."""
    B, H, KV, D = 2048, 14, 2, 64
    g = torch.Generator().manual_seed(12)
    ctx = torch.randint(33, 80, (B,), generator=g).tolist()
    pages = Pages(ctx, [], KV, D, False, 12)
    q = torch.randn(B, H, D, generator=g).to(torch.bfloat16).cuda()
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    order = torch.randperm(B, generator=g).tolist()
    for groups in ([([b], 32) for b in order], [([b], 16 * (b % 3)) for b in range(B)]):
        out = _ops().shared_prefix_attention(q, pages.cache, 0, make_batch(list(range(B)), [1] * B, ctx, B),
                                             _ops().SharedPrefix.from_groups(groups), status=status)
        for b in [0, 1, B - 2, B - 1, *torch.randperm(B, generator=g)[:150].tolist()]:
            k, v = pages.kv(b)
            assert_rows(out[b:b + 1], *plain_attention(q[b:b + 1], k, v, torch.tensor([ctx[b]]), 1 / math.sqrt(D)), f"{b}")
    assert int(status) == 0


def test_groups_without_members():
    """Groups that list nobody, and no member at all: every sequence is attended to alone."""
    ops, (H, KV, D) = _ops(), (12, 2, 128)
    lens, ctx = [5, 1, 0, 140], [300, 17, 9, 2000]
    pages = Pages(ctx, [], KV, D, True, 31)
    row0 = [0, 5, 6, 6]
    q = torch.randn(146, H, D, generator=torch.Generator().manual_seed(8)).to(torch.bfloat16).cuda()
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    for groups in ([([], 16)], [([], 0), ([], 1000)], []):
        out = torch.full_like(q, FILL)
        ops.shared_prefix_attention(q, pages.cache, 0, make_batch(row0, lens, ctx, 146), ops.SharedPrefix.from_groups(groups),
                                    out=out, status=status)
        check_pages(out, FILL, q, pages, row0, lens, ctx, what=str(groups))
    assert int(status) == 0
