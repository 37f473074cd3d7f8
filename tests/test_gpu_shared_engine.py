"""GPU: prompts, shared first pages and page operators as the engine runs them together."""

from __future__ import annotations

import math

import pytest
import torch

from rows_helpers import assert_rows, i32, plain_attention
from test_gpu_engine import LOGIT_RTOL, _cfgs, _check_tokens, _close, _oracle

pytestmark = pytest.mark.gpu


def _prompts(B, P, shared, vocab, seed):
    p = torch.randint(0, vocab, (B, P), generator=torch.Generator().manual_seed(seed), dtype=torch.int32)
    p[:, :shared] = p[:1, :shared].clone()
    return p.cuda()


def test_prompts_of_different_lengths():
    """One pass over padded prompts gives each prompt's own logits and cache; the padding reaches neither."""
    from specdec_b200.engine.model import PagedModel, random_state

    cfg, _ = _cfgs()
    for v, weights in (("bf16", "bf16"), ("e4m3", "bf16"), ("bf16", "int8")):
        pm = PagedModel(cfg, random_state(cfg, 12, "cuda", std=0.05), weights=weights)
        lens, P = [37, 1, 64, 20], 64
        ids = _prompts(4, P, 0, cfg.vocab, 5)
        cache = pm.new_cache(5, 80, v)
        with torch.inference_mode():
            got = pm.prefill(ids, cache, 1, lengths=lens)
            assert cache.lengths.tolist() == [0] + lens
            for b, n in enumerate(lens):
                one = pm.new_cache(1, 80, v)
                want = pm.prefill(ids[b:b + 1, :n], one, 0)
                _close(got[b:b + 1], want, f"{v} {weights} prompt {b}", LOGIT_RTOL)
                for layer in range(cfg.layers):
                    x, y = cache.gather_layer(layer, b + 1, n), one.gather_layer(layer, 0, n)
                    _close(x["k"], y["k"], "keys", LOGIT_RTOL)
        # other padding, the same bits
        ids2 = ids.clone()
        for b, n in enumerate(lens):
            ids2[b, n:] = (ids2[b, n:] + 1) % cfg.vocab
        with torch.inference_mode():
            assert torch.equal(pm.prefill(ids2, pm.new_cache(5, 80, v), 1, lengths=lens), got)
        for bad in ([37, 1, 64], [0, 1, 2, 3], [65, 1, 1, 1]):
            with pytest.raises(ValueError):
                pm.prefill(ids, cache, 1, lengths=bad)


@pytest.mark.parametrize("target_v", ["bf16", "e4m3"])
@pytest.mark.parametrize("share_reads", [True, None])
@pytest.mark.parametrize("shared,P", [(32, 48), (40, 48), (47, 48), (5, 20), (1, 20), (130, 131)])
def test_shared_prompts_emit_the_same_tokens(target_v, shared, P, share_reads):
    from specdec_b200.engine.model import PagedModel, random_state
    from specdec_b200.engine.specdec import SpecDecEngine

    tcfg, dcfg = _cfgs()
    state = random_state(tcfg, 21, "cuda", std=0.05)
    target, draft = PagedModel(tcfg, state), PagedModel.random(dcfg, 22)
    ref = _oracle(tcfg, state)
    if target_v == "e4m3":
        ref.set_kv_format("v_fp8")
    B, N = 5, 16
    prompts = _prompts(B, P, shared, tcfg.vocab, 7)
    eng = SpecDecEngine(target, draft, B, P, N, k=4, target_v=target_v, shared_prefix=shared,
                        share_reads=share_reads)
    eng.capture()
    for again in range(2):  # a second batch takes the first one's pages over
        eng.prefill(prompts, chunk=2)
        for cache in (eng.tc, eng.dc):
            full, table = shared // 16, cache.page_table.cpu()
            assert (table[:, :full] == table[:1, :full]).all()
            own = table[:, full:].flatten()
            assert (own >= 0).all() and len(set(own.tolist())) == own.numel()
            refs = cache.page_refs.cpu()
            assert (refs[table[0, :full].long()] == B).all() and (refs[own.long()] == 1).all()
        eng.decode()
        _check_tokens(eng.tokens().cpu(), prompts, ref, N)
        prompts = _prompts(B, P, shared, tcfg.vocab, 8)


def test_shared_engine_replay_equals_eager_rounds():
    from specdec_b200.engine.model import PagedModel
    from specdec_b200.engine.specdec import SpecDecEngine

    tcfg, dcfg = _cfgs()
    target, draft = PagedModel.random(tcfg, 31, weights="int8"), PagedModel.random(dcfg, 32)
    prompts = _prompts(3, 40, 33, tcfg.vocab, 8)
    outs = []
    for use_graph in (True, False):
        eng = SpecDecEngine(target, draft, 3, 40, 16, k=4, shared_prefix=33, share_reads=True)
        if use_graph:
            eng.capture()
        eng.prefill(prompts)
        eng.decode(use_graph=use_graph)
        outs.append(eng.tokens().cpu())
    assert torch.equal(*outs)


def test_round_captured_after_the_prompts():
    """A round recorded when the sequences hold their pages already runs as one of the decode."""
    from specdec_b200.engine.model import PagedModel
    from specdec_b200.engine.specdec import SpecDecEngine

    tcfg, dcfg = _cfgs()
    target, draft = PagedModel.random(tcfg, 31), PagedModel.random(dcfg, 32)
    prompts = _prompts(3, 40, 33, tcfg.vocab, 8)
    outs = []
    for late in (False, True):
        eng = SpecDecEngine(target, draft, 3, 40, 16, k=4, shared_prefix=33)
        if not late:
            eng.capture()
        eng.prefill(prompts)
        if late:
            eng.capture()
        eng.decode()
        outs.append(eng.tokens().cpu())
    assert torch.equal(*outs)


def test_more_prompts_than_a_call_takes():
    from specdec_b200.engine.model import ModelConfig, PagedModel

    cfg = ModelConfig(vocab=100, hidden=128, heads=2, kv_heads=1, head_dim=64, intermediate=128, layers=2)
    pm = PagedModel.random(cfg, 3)
    n, P = 2500, 6
    ids = _prompts(n, P, 0, cfg.vocab, 4)
    lens = [1 + i % P for i in range(n)]
    with torch.inference_mode():
        cache = pm.new_cache(n, 16)
        got = pm.prefill(ids, cache, 0, lengths=lens)
        for s0 in (0, 1000, 2040, 2400):
            one = pm.prefill(ids[s0:s0 + 100], pm.new_cache(100, 16), 0, lengths=lens[s0:s0 + 100])
            _close(got[s0:s0 + 100], one, f"prompts {s0} ..", LOGIT_RTOL)


def test_job_with_a_shared_prefix():
    """The data-parallel job's tokens are the engine's over its prompts, the first of whose tokens are all alike."""
    from specdec_b200.engine.dp import run_specdec_dp, synthetic_prompts
    from specdec_b200.engine.model import PagedModel
    from specdec_b200.engine.specdec import SpecDecEngine

    tcfg, dcfg = _cfgs()
    job = dict(total_seqs=3, prompt_len=40, max_new=12, k=4, seed=5)
    res = run_specdec_dp(tcfg, dcfg, shared_prefix=24, **job)
    prompts = synthetic_prompts(3, 40, tcfg.vocab, 5)
    prompts[:, :24] = prompts[0, :24]
    eng = SpecDecEngine(PagedModel.random(tcfg, 6), PagedModel.random(dcfg, 7), 3, 40, 12, k=4, shared_prefix=24)
    eng.capture()
    eng.prefill(prompts.cuda())
    eng.decode()
    assert torch.equal(res.tokens, eng.tokens())
    for bad in (-1, 40):
        with pytest.raises(ValueError):
            run_specdec_dp(tcfg, dcfg, shared_prefix=bad, **job)


def test_engine_refusals():
    from specdec_b200.engine.model import PagedModel
    from specdec_b200.engine.specdec import SpecDecEngine

    tcfg, dcfg = _cfgs()
    target, draft = PagedModel.random(tcfg, 31), PagedModel.random(dcfg, 32)
    for bad in (-1, 40, 41):
        with pytest.raises(ValueError):
            SpecDecEngine(target, draft, 3, 40, 16, shared_prefix=bad)
    with pytest.raises(ValueError):
        SpecDecEngine(target, draft, 2049, 40, 16, shared_prefix=33)
    eng = SpecDecEngine(target, draft, 3, 40, 16, shared_prefix=33)
    other = _prompts(3, 40, 33, tcfg.vocab, 1)
    other[2, 20] = (other[2, 20] + 1) % tcfg.vocab
    with pytest.raises(ValueError):
        eng.prefill(other)


@pytest.mark.parametrize("v8,D,H", [(False, 128, 12), (True, 128, 12), (False, 64, 14)])
def test_operators_together(v8, D, H):
    """A prompt attended to and appended, forked to three sequences, each going on for itself (a page shared in the
    middle is replaced), one given up and the pools compacted: after each step every sequence's attention over its
    pages is that over its own keys, kept beside in plain tensors."""
    from specdec_b200.engine.paged_cache import PagedKVCache
    from specdec_b200.kernels import ops
    from oracle import fp8 as ofp8

    KV, P, B = 2, 77, 4
    g = torch.Generator().manual_seed(D + v8)
    c = PagedKVCache.allocate(1, B, KV, D, 160, v_dtype="e4m3" if v8 else "bf16", num_pages=30, on_demand=True)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    plain = [(torch.zeros(0, KV, D).cuda(), torch.zeros(0, KV, D).cuda()) for _ in range(B)]
    lens = [0] * B

    def append(new):
        """new[b] tokens of every sequence through append_kv and into the plain tensors"""
        total = sum(new)
        k = torch.randn(total, KV, D, generator=g).to(torch.bfloat16).cuda()
        v = torch.randn(total, KV, D, generator=g).to(torch.bfloat16).cuda()
        c.reserve([n + m for n, m in zip(lens, new)], status=status)
        row0 = [sum(new[:b]) for b in range(B)]
        ops.append_kv(k, v, c, 0, row0=i32(row0), n_new=i32(new), pos0=i32(lens), max_new=max(new), status=status)
        codes, scale = ofp8.quantize_v(v.float().cpu().transpose(0, 1).numpy()) if v8 else (None, None)
        # (float32: a product of a code and a scale has 4 + 24 bits, rounded by 2^-24 of it)
        kept = torch.from_numpy(ofp8.dequantize_v(codes, scale)).float().transpose(0, 1).cuda() if v8 else v
        for b in range(B):
            at = slice(row0[b], row0[b] + new[b])
            plain[b] = (torch.cat([plain[b][0], k[at]]), torch.cat([plain[b][1], kept[at]]))
            lens[b] += new[b]
        c.lengths.copy_(i32(lens))
        return k, v

    def attend(groups, rows):
        q = torch.randn(sum(rows), H, D, generator=g).to(torch.bfloat16).cuda()
        batch = ops.RaggedBatch.from_lengths(rows, lens)
        out = ops.shared_prefix_attention(q, c, 0, batch, ops.SharedPrefix.from_groups(groups), status=status)
        for b in range(B):
            r, n = sum(rows[:b]), rows[b]
            if n:
                k, v = plain[b]
                want, tol = plain_attention(q[r:r + n], k, v, torch.arange(n) + (lens[b] - n + 1), 1 / math.sqrt(D))
                assert_rows(out[r:r + n], want, tol, f"sequence {b}")

    k, v = append([P, 0, 0, 0])
    q = torch.randn(P, H, D, generator=g).to(torch.bfloat16).cuda()
    out = ops.prompt_attention(q, k, v, ops.RaggedBatch.from_lengths([P], [P]), status=status)
    want, tol = plain_attention(q, k, v, torch.arange(P) + 1, 1 / math.sqrt(D))
    assert_rows(out, want, tol, "prompt")
    c.fork([0, 0, 0], [1, 2, 3], [P, 64, 70], status=status)
    for b, n in ((1, P), (2, 64), (3, 70)):
        plain[b] = (plain[0][0][:n], plain[0][1][:n])
        lens[b] = n
    attend([([0, 1, 2, 3], 64)], [1, 1, 1, 1])
    append([5, 3, 5, 1])
    attend([([0, 1, 2, 3], 64)], [5, 3, 5, 1])
    # back into the shared pages, and on from there
    lens[1] = 50
    plain[1] = (plain[1][0][:50], plain[1][1][:50])
    c.lengths.copy_(i32(lens))
    append([1, 30, 0, 20])
    attend([([0, 2, 3], 64), ([1], 48)], [1, 5, 1, 3])
    attend([([0, 1, 2, 3], 48)], [1, 5, 1, 3])
    c.free([0], status=status)
    plain[0], lens[0] = (plain[0][0][:0], plain[0][1][:0]), 0
    live = c.compact(status=status)
    used = c.page_table[c.page_table >= 0].unique()
    assert int(live) == used.numel() and int(used.max()) == used.numel() - 1
    attend([([2, 3], 64), ([1], 16)], [0, 2, 4, 1])
    append([20, 1, 1, 1])
    attend([([2, 3], 64)], [20, 1, 1, 1])
    assert int(status) == 0
