"""CPU: prompt attention, shared-prefix attention and the page operators refuse bad host arguments before touching
the device, and their Python side checks what it is given."""

from __future__ import annotations

import ctypes

import pytest
import torch

P = 0x10000  # never dereferenced: the call is refused, or has nothing to do


def _msg(lib):
    return lib.specdec_last_error().decode()


def _batch(**kw):
    from specdec_b200 import _lib

    return _lib.Batch(**{**dict(q_row0=P, q_len=P, ctx_len=P, num_seqs=4, num_q_heads=12, max_q_len=9, max_ctx_len=0),
                         **kw})


def _prompt_args(batch=None, **kw):
    from specdec_b200 import _lib

    base = dict(q=P, k=P, v=P, out=P, q_stride_tok=12 * 128, q_stride_head=128, k_stride_tok=256, k_stride_head=128,
                v_stride_tok=256, v_stride_head=128, o_stride_tok=12 * 128, o_stride_head=128, kv_row0=P, q_rows=36,
                kv_rows=36, num_kv_heads=2, head_dim=128, sm_scale=0.1, workspace=P, workspace_bytes=1 << 40)
    return _lib.PromptArgs(batch=_batch(**(batch or {})), **{**base, **kw})


def _shared_args(batch=None, kv=None, **kw):
    from specdec_b200 import _lib

    pool = _lib.PagedKV(**{**dict(k_pool=P, v_pool=P, v_scale=None, page_table=P, num_pages=64, max_pages_per_seq=8,
                                  num_kv_heads=2, head_dim=128, v_dtype=_lib.BF16), **(kv or {})})
    base = dict(q=P, out=P, q_stride_tok=12 * 128, q_stride_head=128, o_stride_tok=12 * 128, o_stride_head=128,
                group_start=P, members=P, prefix_len=P, num_groups=1, num_members=4, q_rows=36, sm_scale=0.1,
                workspace=P, workspace_bytes=1 << 40)
    return _lib.SharedPrefixArgs(batch=_batch(**(batch or {})), kv=pool, **{**base, **kw})


# ---------------------------------------------------------------- attention
ROWS = [  # of both entry points: (batch fields, argument fields, result, message)
    (dict(num_seqs=0), {}, 1, "must be positive"),
    (dict(num_q_heads=0), {}, 1, "must be positive"),
    (dict(num_q_heads=13), {}, 1, "divide KV heads"),
    (dict(num_q_heads=258), {}, 2, "at most 128 query heads"),
    (dict(max_q_len=0), {}, 1, "max_q_len must be positive"),
    (dict(num_seqs=2049), {}, 2, "at most 2048"),
    (dict(max_q_len=(1 << 30) + 1), {}, 2, "too large for one call"),
    (dict(num_seqs=2048, max_q_len=1 << 28), {}, 2, "too large for one call"),
    (dict(q_row0=None), {}, 1, "batch arrays"),
    (dict(q_len=None), {}, 1, "batch arrays"),
    (dict(ctx_len=None), {}, 1, "batch arrays"),
    ({}, dict(q=None), 1, "q and out must be device pointers"),
    ({}, dict(out=None), 1, "q and out must be device pointers"),
    ({}, dict(q=P + 8), 1, "q/out must be 16-byte aligned"),
    ({}, dict(out=P + 2), 1, "q/out must be 16-byte aligned"),
    ({}, dict(q_stride_tok=12 * 128 + 4), 1, "q/out strides"),
    ({}, dict(q_stride_head=0), 1, "q/out strides"),
    ({}, dict(o_stride_head=-128 + 4), 1, "q/out strides"),
    ({}, dict(q_rows=0), 1, "row counts"),
    ({}, dict(q_rows=1 << 31), 1, "row counts"),
    ({}, dict(sm_scale=0.0), 1, "sm_scale"),
    ({}, dict(sm_scale=float("nan")), 1, "sm_scale"),
    ({}, dict(sm_scale=float("inf")), 1, "sm_scale"),
    ({}, dict(workspace=None), 4, "workspace"),
    ({}, dict(workspace_bytes=256), 4, "workspace of 256 bytes"),
    ({}, dict(workspace=P + 128), 1, "256-byte aligned"),
]


@pytest.mark.parametrize("batch,kw,rc,msg", ROWS + [
    ({}, dict(num_kv_heads=0), 1, "must be positive"),
    ({}, dict(head_dim=96), 2, "head_dim must be 64 or 128"),
    ({}, dict(k=None), 1, "k and v must be device pointers"),
    ({}, dict(v=None), 1, "k and v must be device pointers"),
    ({}, dict(k=P + 8), 1, "k/v must be 16-byte aligned"),
    ({}, dict(k_stride_head=0), 1, "k/v strides"),
    ({}, dict(v_stride_tok=257), 1, "k/v strides"),
    ({}, dict(kv_row0=None), 1, "batch arrays"),
    ({}, dict(kv_rows=0), 1, "row counts"),
])
def test_prompt_attention_refuses(lib, batch, kw, rc, msg):
    from specdec_b200 import _lib

    want = {1: _lib.ERR_INVALID, 2: _lib.ERR_UNSUPPORTED, 4: _lib.ERR_WORKSPACE}[rc]
    got = lib.specdec_prompt_attention(ctypes.byref(_prompt_args(batch, **kw)), None)
    assert got == want and msg in _msg(lib), (got, _msg(lib))


@pytest.mark.parametrize("batch,kw,rc,msg", ROWS + [
    ({}, dict(kv=dict(num_kv_heads=0)), 1, "must be positive"),
    ({}, dict(kv=dict(head_dim=32)), 2, "head_dim must be 64 or 128"),
    ({}, dict(kv=dict(k_pool=None)), 1, "kv pool pointers"),
    ({}, dict(kv=dict(v_pool=None)), 1, "kv pool pointers"),
    ({}, dict(kv=dict(page_table=None)), 1, "kv pool pointers"),
    ({}, dict(kv=dict(v_pool=P + 8)), 1, "pool pointers must be 16-byte"),
    ({}, dict(kv=dict(num_pages=0)), 1, "empty page pool"),
    ({}, dict(kv=dict(max_pages_per_seq=0)), 1, "empty page pool"),
    ({}, dict(kv=dict(v_dtype=0)), 2, "v_dtype"),
    ({}, dict(kv=dict(v_dtype=2, v_scale=None)), 1, "v_scale"),
    ({}, dict(kv=dict(v_dtype=2, v_scale=P, head_dim=64)), 2, "E4M3 V needs head_dim 128"),
    ({}, dict(kv=dict(num_pages=1 << 30)), 2, "page pool too large"),
    ({}, dict(kv=dict(max_pages_per_seq=(1 << 26) + 1)), 2, "page pool too large"),
    ({}, dict(num_groups=-1), 1, "group or member count"),
    ({}, dict(num_members=-1), 1, "group or member count"),
    ({}, dict(num_groups=0), 1, "group or member count"),
    ({}, dict(num_groups=2049), 2, "at most 2048"),
    ({}, dict(num_members=2049), 2, "at most 2048"),
    ({}, dict(group_start=None), 1, "group arrays"),
    ({}, dict(members=None), 1, "group arrays"),
    ({}, dict(prefix_len=None), 1, "group arrays"),
])
def test_shared_prefix_attention_refuses(lib, batch, kw, rc, msg):
    from specdec_b200 import _lib

    assert _lib.E4M3 == 2
    want = {1: _lib.ERR_INVALID, 2: _lib.ERR_UNSUPPORTED, 4: _lib.ERR_WORKSPACE}[rc]
    got = lib.specdec_shared_prefix_attention(ctypes.byref(_shared_args(batch, **kw)), None)
    assert got == want and msg in _msg(lib), (got, _msg(lib))


def test_null_arguments(lib):
    from specdec_b200 import _lib

    assert lib.specdec_prompt_attention(None, None) == _lib.ERR_INVALID
    assert lib.specdec_shared_prefix_attention(None, None) == _lib.ERR_INVALID


def test_workspace_bytes(lib):
    small, large = (lib.specdec_prompt_workspace_bytes(n, 12, 2, 128, 64, 0) for n in (1, 64))
    assert 0 < small <= large and small % 256 == 0
    for bad in ((0, 12, 2, 128, 64), (1, 12, 5, 128, 64), (1, 12, 2, 96, 64), (1, 12, 2, 128, 0), (2049, 12, 2, 128, 64),
                (1, 129, 1, 128, 64)):
        assert lib.specdec_prompt_workspace_bytes(*bad, 0) == 0
    none = lib.specdec_shared_prefix_workspace_bytes(64, 12, 2, 128, 5, 0, 0, 0)
    assert 0 < none < lib.specdec_shared_prefix_workspace_bytes(64, 12, 2, 128, 5, 4, 64, 0)
    assert lib.specdec_shared_prefix_workspace_bytes(64, 12, 2, 128, 5, 2049, 64, 0) == 0
    assert lib.specdec_shared_prefix_workspace_bytes(64, 12, 2, 128, 5, -1, 64, 0) == 0


def test_struct_sizes_match_the_header():
    from specdec_b200 import _lib

    assert ctypes.sizeof(_lib.PromptArgs) == 8 * 4 + 8 * 8 + 40 + 8 + 16 + 8 + 8 + 8 + 8 + 8 + 8
    assert ctypes.sizeof(_lib.SharedPrefixArgs) == 16 + 32 + 40 + 56 + 24 + 8 + 8 + 8 + 8 + 8 + 8 + 8
    assert ctypes.sizeof(_lib.PagePool) == 3 * 8 + 5 * 4 + 4
    assert ctypes.sizeof(_lib.PageTable) == 3 * 8 + 8 + 8 + 8 + 8


def test_status_names():
    from specdec_b200 import _lib

    assert "group" in _lib.status_message(_lib.STATUS_BAD_GROUP)
    assert "page request" in _lib.status_message(_lib.STATUS_BAD_SEQUENCE)
    assert "no free page" in _lib.status_message(_lib.STATUS_NO_PAGES)


# ---------------------------------------------------------------- pages
def _pool(**kw):
    from specdec_b200 import _lib

    arrays = (ctypes.c_void_p * 2)(P, P)
    base = dict(k_pools=ctypes.addressof(arrays), v_pools=ctypes.addressof(arrays), v_scales=None, num_layers=2,
                num_pages=16, num_kv_heads=2, head_dim=128, v_dtype=_lib.BF16)
    pool = _lib.PagePool(**{**base, **kw})
    pool.keep = arrays
    return pool


def _table(**kw):
    from specdec_b200 import _lib

    return _lib.PageTable(**{**dict(page_table=P, page_refs=P, lengths=P, num_seqs=4, max_pages_per_seq=8, workspace=P,
                                    workspace_bytes=1 << 30, status=None), **kw})


def _calls(lib, pool, table, n=2, ptr=P):
    pool, table = pool and ctypes.byref(pool), table and ctypes.byref(table)
    return {
        "copy": lambda: lib.specdec_copy_pages(pool, ptr, ptr, n, None, None),
        "fork": lambda: lib.specdec_fork_sequences(pool, table, ptr, ptr, ptr, n, None),
        "reserve": lambda: lib.specdec_reserve_pages(pool, table, ptr, None),
        "free": lambda: lib.specdec_free_sequences(pool, table, ptr, n, None),
        "compact": lambda: lib.specdec_compact_pages(pool, table, ptr, None),
    }


NULLS = (ctypes.c_void_p * 2)(P, None)
ODD = (ctypes.c_void_p * 2)(P, P + 8)


@pytest.mark.parametrize("op", ["copy", "fork", "reserve", "free", "compact"])
@pytest.mark.parametrize("kw,msg", [
    (dict(num_layers=0), "empty page pool"),
    (dict(num_pages=0), "empty page pool"),
    (dict(num_kv_heads=0), "empty page pool"),
    (dict(num_kv_heads=(1 << 14) + 1), "at most 16384"),
    (dict(head_dim=80), "head_dim"),
    (dict(v_dtype=0), "v_dtype"),
    (dict(k_pools=None), "pool pointers must be set"),
    (dict(v_pools=None), "pool pointers must be set"),
    (dict(v_dtype=2), "pool pointers must be set"),
    (dict(k_pools=ctypes.addressof(NULLS)), "pool pointers must be set"),
    (dict(v_pools=ctypes.addressof(ODD)), "16-byte aligned"),
])
def test_page_operators_refuse_bad_pools(lib, op, kw, msg):
    assert _calls(lib, _pool(**kw), _table())[op]() != 0 and msg in _msg(lib), _msg(lib)


@pytest.mark.parametrize("op", ["fork", "reserve", "free", "compact"])
@pytest.mark.parametrize("kw,msg", [
    (dict(page_table=None), "device pointers"),
    (dict(page_refs=None), "device pointers"),
    (dict(lengths=None), "device pointers"),
    (dict(num_seqs=0), "page table shape"),
    (dict(max_pages_per_seq=0), "page table shape"),
    (dict(max_pages_per_seq=(1 << 26) + 1), "page table shape"),
    (dict(workspace=None), "workspace of 0 bytes"),
    (dict(workspace_bytes=64), "workspace of 64 bytes"),
    (dict(workspace=P + 4), "16-byte aligned"),
])
def test_page_operators_refuse_bad_tables(lib, op, kw, msg):
    assert _calls(lib, _pool(), _table(**kw))[op]() != 0 and msg in _msg(lib), _msg(lib)


def test_page_operators_refuse_bad_requests(lib):
    for op in ("copy", "fork", "free"):
        assert _calls(lib, _pool(), _table(), n=-1)[op]() != 0 and "out of range" in _msg(lib)
        assert _calls(lib, _pool(), _table(), n=0)[op]() == 0
    for op, call in _calls(lib, _pool(), _table(), ptr=None).items():
        assert call() != 0 and "must be" in _msg(lib), op
    for op, call in _calls(lib, None, None).items():
        assert call() != 0 and "pool is NULL" in _msg(lib), op
    for op, call in _calls(lib, _pool(), None).items():
        if op != "copy":
            assert call() != 0 and "table is NULL" in _msg(lib), op


def test_page_workspace_bytes(lib):
    assert lib.specdec_page_workspace_bytes(4, 64, 0) < lib.specdec_page_workspace_bytes(4, 64, 100)
    for bad in ((0, 64, 0), (4, 0, 0), (4, 64, -1)):
        assert lib.specdec_page_workspace_bytes(*bad) == 0


# ---------------------------------------------------------------- the Python side
def test_shared_prefix_groups():
    from specdec_b200.kernels import ops

    p = ops.SharedPrefix.from_groups([([0, 2], 33), ([], 5), ([3], 0)], device="cpu")
    assert (p.num_groups, p.num_members) == (3, 3)
    assert p.group_start.tolist() == [0, 2, 2, 3] and p.members.tolist() == [0, 2, 3]
    assert p.prefix_len.tolist() == [33, 5, 0]
    none = ops.SharedPrefix.from_groups([], device="cpu")
    assert (none.num_groups, none.num_members) == (0, 0) and none.group_start.tolist() == [0]
    for bad in ([([0, 0], 5)], [([0], 5), ([0], 5)], [([-1], 5)], [([0], -1)]):
        with pytest.raises(ValueError):
            ops.SharedPrefix.from_groups(bad, device="cpu")


def test_row_shapes():
    from specdec_b200.kernels import ops

    x = torch.zeros(6, 4, 64, dtype=torch.bfloat16)
    assert ops._head_rows(x, "x") == (6, 4, 64, 256, 64, x.data_ptr())
    assert ops._head_rows(x.transpose(0, 1), "x")[:5] == (4, 6, 64, 64, 256)
    # strides that are never taken: one row, one head
    assert ops._head_rows(x[:, :1].as_strided((6, 1, 64), (256, 3, 1)), "x")[:5] == (6, 1, 64, 256, 64)
    assert ops._head_rows(x.as_strided((1, 4, 64), (5, 64, 1)), "x")[:5] == (1, 4, 64, 256, 64)
    bad = [x.float(), x[0], x[..., ::2], x[..., 4:], x.as_strided((6, 4, 64), (0, 64, 1)),
           x.as_strided((5, 4, 64), (260, 64, 1)), x.as_strided((6, 4, 64), (256, 0, 1))]
    for t in bad:
        with pytest.raises(ValueError):
            ops._head_rows(t, "x")
    with pytest.raises(ValueError):
        ops._head_rows(x, "x", D=128)
    with pytest.raises(RuntimeError):
        ops.prompt_attention(x, x, x, ops.RaggedBatch.from_lengths([6], [6], device="cpu"))


def test_on_demand_cache():
    from specdec_b200.engine.paged_cache import PagedKVCache
    from specdec_b200.kernels import ops

    c = PagedKVCache.allocate(2, 3, 2, 64, 40, device="cpu", num_pages=5, on_demand=True)
    assert c.num_pages == 5 and c.max_pages == 3 and (c.page_table == -1).all()
    assert c.page_refs.tolist() == [0] * 5 and c.with_lengths(c.lengths, None).page_refs is c.page_refs
    static = PagedKVCache.allocate(2, 3, 2, 64, 40, device="cpu")
    assert static.page_refs is None
    with pytest.raises(ValueError):
        PagedKVCache.allocate(2, 3, 2, 64, 40, device="cpu", num_pages=5)
    with pytest.raises(ValueError):
        PagedKVCache.allocate(2, 3, 2, 64, 40, device="cpu", num_pages=0, on_demand=True)
    with pytest.raises(ValueError):
        PagedKVCache.allocate(2, 3, 2, 64, 40, device="cpu", on_demand=True, page_order_seed=1)
    with pytest.raises(RuntimeError):  # device arrays only
        c.free([0])
    with pytest.raises(ValueError):
        ops._page_table(static, 0, None, None, None, -1)


def test_cache_from_pools():
    from specdec_b200.engine.paged_cache import PagedKVCache

    k = [torch.zeros(5, 2, 16 * 128, dtype=torch.bfloat16) for _ in range(2)]
    v8 = [torch.zeros(5, 2, 16 * 128, dtype=torch.uint8) for _ in range(2)]
    sc = [torch.zeros(5, 2, 16) for _ in range(2)]
    pt, ln = torch.zeros(3, 4, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    c = PagedKVCache.from_pools(k, k, None, pt, ln, 128)
    assert (c.num_layers, c.num_seqs, c.num_pages, c.max_pages, c.v_dtype) == (2, 3, 5, 4, "bf16")
    assert PagedKVCache.from_pools(k, v8, sc, pt, ln, 128).v_dtype == "e4m3"
    for args in [([], [], None, pt, ln, 128), (k, k[:1], None, pt, ln, 128), (k, v8, None, pt, ln, 128),
                 (k, k, sc, pt, ln, 128), (k, v8, sc[:1], pt, ln, 128), (k, k, None, pt.long(), ln, 128),
                 (k, k, None, pt, ln[:2], 128), (k, k, None, pt, ln, 96), (k, k, None, pt, ln, 64)]:
        with pytest.raises(ValueError):
            PagedKVCache.from_pools(*args)
    with pytest.raises(ValueError):
        PagedKVCache.from_pools(k, k, None, pt, ln, 128, page_refs=torch.zeros(4, dtype=torch.int32))


def test_piece_layout():
    from specdec_b200.engine.model import PieceLayout

    p = PieceLayout(5, 2, 2, 3, "cpu")
    assert p.rows == 6 and p.q_len.tolist() == [0, 0, 3, 3, 0] and p.q_row0.tolist() == [0, 0, 0, 3, 3]
    p.set(torch.tensor([7, 7, 10, 20, 7], dtype=torch.int32))
    assert p.batch.ctx_len.tolist()[2:4] == [13, 23]
    assert p.positions().tolist() == [10, 11, 12, 20, 21, 22] and p.last_rows().tolist() == [2, 5]
