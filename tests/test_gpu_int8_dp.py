"""GPU: the data-parallel SpecDec job with 8-bit projections (run_specdec_dp(weights="int8")), one rank."""

from __future__ import annotations

import pytest
import torch

from test_gpu_engine import _cfgs

pytestmark = pytest.mark.gpu

JOB = dict(total_seqs=3, prompt_len=40, max_new=12, k=4, seed=5)


def _tokens_by_hand(draft_is_target):
    from specdec_b200.engine.dp import synthetic_prompts
    from specdec_b200.engine.model import PagedModel
    from specdec_b200.engine.specdec import SpecDecEngine

    target_cfg, draft_cfg = _cfgs()
    target = PagedModel.random(target_cfg, JOB["seed"] + 1, weights="int8")
    draft = target if draft_is_target else PagedModel.random(draft_cfg, JOB["seed"] + 2, weights="int8")
    eng = SpecDecEngine(target, draft, JOB["total_seqs"], JOB["prompt_len"], JOB["max_new"], k=JOB["k"])
    eng.capture()
    eng.prefill(synthetic_prompts(JOB["total_seqs"], JOB["prompt_len"], target_cfg.vocab, JOB["seed"]).cuda())
    eng.decode()
    return eng.tokens()


@pytest.mark.parametrize("draft_is_target", [False, True])
def test_job_is_the_engine_with_int8_models(draft_is_target):
    """The job's tokens are those of the engine built from 8-bit models of the same seeds, and both of its models
    are 8-bit: a draft that is the target agrees with it."""
    from specdec_b200.engine.dp import run_specdec_dp

    target_cfg, draft_cfg = _cfgs()
    res = run_specdec_dp(target_cfg, draft_cfg, draft_is_target=draft_is_target, weights="int8", **JOB)
    assert torch.equal(res.tokens, _tokens_by_hand(draft_is_target))
    assert res.tokens.shape == (3, 12) and res.local_seqs == 3 and res.rounds >= 3 and res.decode_s > 0
    if draft_is_target:
        assert res.acceptance > 2.0


def test_job_refuses_other_weights():
    from specdec_b200.engine.dp import run_specdec_dp

    with pytest.raises(ValueError, match="'bf16' or 'int8'"):
        run_specdec_dp(*_cfgs(), weights="fp4", **JOB)
