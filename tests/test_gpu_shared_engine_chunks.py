"""GPU: the engine's prompts behind a shared prefix, a chunk of sequences a step."""

from __future__ import annotations

import pytest
import torch

from test_gpu_engine import _cfgs, _check_tokens, _oracle
from test_gpu_shared_engine import _prompts

pytestmark = pytest.mark.gpu


def _engine(B, P, N, shared, **kw):
    from specdec_b200.engine.model import PagedModel
    from specdec_b200.engine.specdec import SpecDecEngine

    tcfg, dcfg = _cfgs()
    return SpecDecEngine(PagedModel.random(tcfg, 31), PagedModel.random(dcfg, 32), B, P, N, k=4, shared_prefix=shared, **kw)


def test_a_chunks_workspace_does_not_grow_with_the_batch(monkeypatch):
    """The attention of a chunk works over the chunk's rows: as much workspace in a batch of 24 as in one of 3, taken
    once a model, and every call's batch and group are the chunk's."""
    from specdec_b200.engine import specdec

    taken, calls = [], []
    space, attend = specdec.ops.shared_prefix_workspace, specdec.ops.shared_prefix_attention

    def workspace(batch, prefix, *args):
        ws = space(batch, prefix, *args)
        taken.append(ws.numel())
        return ws

    def attention(q, cache, layer, batch, prefix, **kw):
        calls.append((batch.num_seqs, prefix.num_members, q.shape[0] // batch.max_q_len))
        return attend(q, cache, layer, batch, prefix, **kw)

    monkeypatch.setattr(specdec.ops, "shared_prefix_workspace", workspace)
    monkeypatch.setattr(specdec.ops, "shared_prefix_attention", attention)
    sizes = []
    for B in (3, 24):
        eng = _engine(B, 300, 8, 130, share_reads=False)
        prompts = _prompts(B, 300, 130, eng.target.cfg.vocab, 7)
        taken.clear(), calls.clear()
        eng.prefill(prompts, chunk=2)
        assert len(taken) == 2 and all(n == m == rows for n, m, rows in calls)
        assert max(n for n, _, _ in calls) == 2
        sizes.append(list(taken))
    assert sizes[0] == sizes[1]


@pytest.mark.parametrize("chunk", [1, 2, 3, 7, 50])
def test_chunks_of_any_size_emit_the_target_s_tokens(chunk):
    from specdec_b200.engine.model import PagedModel, random_state
    from specdec_b200.engine.specdec import SpecDecEngine

    tcfg, dcfg = _cfgs()
    state = random_state(tcfg, 21, "cuda", std=0.05)
    eng = SpecDecEngine(PagedModel(tcfg, state), PagedModel.random(dcfg, 22), 7, 90, 16, k=4, shared_prefix=50)
    prompts = _prompts(7, 90, 50, tcfg.vocab, 9)
    eng.prefill(prompts, chunk=chunk)
    assert eng.tc.lengths.tolist() == [90] * 7 and eng.dc.lengths.tolist() == [90] * 7
    eng.decode(use_graph=False)
    _check_tokens(eng.tokens().cpu(), prompts, _oracle(tcfg, state), 16)
    assert int(eng.status) == 0


def test_sequences_of_a_cache():
    """A view of some sequences is a cache over the same pages and lengths; pages are taken through the whole one."""
    from specdec_b200.engine.paged_cache import PagedKVCache
    from specdec_b200.kernels import ops

    c = PagedKVCache.allocate(2, 5, 2, 64, 40, num_pages=20, on_demand=True)
    c.reserve([40] * 5)
    some = c.sequences(1, 3)
    assert some.num_seqs == 3 and some.pools is c.pools and some.max_pages == c.max_pages
    assert torch.equal(some.page_table, c.page_table[1:4]) and some.page_table.is_contiguous()
    some.lengths.fill_(9)
    assert c.lengths.tolist() == [0, 9, 9, 9, 0]
    for call in (lambda: some.free([0]), lambda: some.reserve([40] * 3), lambda: some.compact()):
        with pytest.raises(ValueError):
            call()
    for bad in ((-1, 2), (0, 0), (3, 3), (5, 1), (0, 6)):
        with pytest.raises(ValueError):
            c.sequences(*bad)
    k = torch.ones(3, 2, 64, dtype=torch.bfloat16, device="cuda")
    one = torch.ones(3, dtype=torch.int32, device="cuda")
    ops.append_kv(k, k, some, 0, row0=torch.arange(3, dtype=torch.int32, device="cuda"), n_new=one, pos0=some.lengths,
                  max_new=1)
    assert all((c.gather_layer(0, b, 10)["k"][0][:, 9] == 1).all() for b in (1, 2, 3))
    assert not c.gather_layer(0, 0, 10)["k"].any() and not c.gather_layer(0, 4, 10)["k"].any()


@pytest.mark.parametrize("B,P,N,shared,want", [(64, 2304, 16, 2048, True), (64, 2544, 16, 2048, True),
                                               (64, 2545, 16, 2048, False), (64, 2304, 400, 2048, False),
                                               (63, 2304, 16, 2048, False), (64, 2100, 16, 2047, False)])
def test_rounds_share_reads_where_the_prefix_outweighs_the_rest(B, P, N, shared, want):
    """64 sequences, 2048 shared tokens and four times as many of them as a sequence has of its own; an argument decides
    otherwise."""
    assert (_engine(B, P, N, shared).step_prefix is not None) == want
    assert (_engine(B, P, N, shared, share_reads=not want).step_prefix is not None) == (not want)
