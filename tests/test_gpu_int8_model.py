"""GPU: the decoder and the SpecDec engine with 8-bit projections (PagedModel(weights="int8")).

The expected values come from the model-level oracle with every projection replaced by its 8-bit definition (rows and
output channels quantised as in oracle/int8.py, products in fp32), fed like the kernels are: norms in fp32
from the unrounded sum of the residual and the last projection, SwiGLU in fp32.  What is left between the
two are fp32 orders of summation and the attention's bf16 roundings, so the logits are held to the bar that
the prompt pass of the bf16 tests has."""

from __future__ import annotations

import pytest
import torch
import torch.nn as nn

import oracle.engine as oeng
from test_gpu_engine import NEAR_TIE, PROMPT_LOGIT_RTOL, _cfgs, _close, _oracle

pytestmark = pytest.mark.gpu


class _Int8Linear(nn.Module):
    """nn.Linear by the 8-bit definition, applied to the fp32 rows ``exact`` that its bf16 input stands for."""

    def __init__(self, lin: nn.Linear):
        super().__init__()
        self.w, self.b, self.exact = self._values(lin.weight), lin.bias, None

    @staticmethod
    def _values(v):
        v = v.float()
        m = v.abs().amax(dim=-1, keepdim=True).clamp(min=2.0 ** -100)
        return torch.round(v * (127.0 / m)) * (m / 127.0)

    def forward(self, x):
        y = self._values(x if self.exact is None else self.exact) @ self.w.t()
        return (y if self.b is None else y + self.b.float()).to(torch.bfloat16)


def _int8_oracle(cfg, state):
    ref = _oracle(cfg, state)
    for layer in ref.layers:
        for owner in (layer.self_attn, layer.mlp):
            for name, child in list(owner.named_children()):
                if isinstance(child, nn.Linear):
                    setattr(owner, name, _Int8Linear(child))
    return ref


def _run(ref, ids, cache_list):
    """QwenLM._run with the residual stream held as (bf16 sum, last projection): logits and caches."""
    x, delta, new = ref.embed_tokens(ids), None, []
    start = 0 if cache_list is None else cache_list[0]["k"].shape[2]
    cos, sin = oeng.rope_cache(ref.head_dim, x.size(1), ref.rope_theta, x.device, x.dtype, start)

    def norm(ln, x, delta):
        s = x.float() if delta is None else x.float() + delta.float()
        return s * torch.rsqrt((s * s).mean(dim=-1, keepdim=True) + ln.eps) * ln.weight.float(), s.to(x.dtype)

    for i, layer in enumerate(ref.layers):
        att, mlp = layer.self_attn, layer.mlp
        h, x = norm(layer.input_layernorm, x, delta)
        for lin in (att.q_proj, att.k_proj, att.v_proj):
            lin.exact = h
        delta, c = att(h.to(x.dtype), cos, sin, None if cache_list is None else cache_list[i])
        new.append(c)
        h, x = norm(layer.post_attention_layernorm, x, delta)
        mlp.gate_proj.exact = mlp.up_proj.exact = h
        gate, up = mlp.gate_proj(x).float(), mlp.up_proj(x).float()
        delta = mlp.down_proj(gate / (1.0 + torch.exp(-gate)) * up)
    x = ref.norm(x + delta)
    return x @ ref.embed_tokens.weight.T, new


@pytest.mark.parametrize("fmt", ["fp16", "v_fp8"])
def test_int8_model_matches_oracle_logits(fmt):
    from specdec_b200.engine.model import PagedModel, StepLayout, random_state
    from specdec_b200.kernels import ops

    cfg, _ = _cfgs()
    state = random_state(cfg, 12, "cuda", std=0.05)
    ref = _int8_oracle(cfg, state)
    ref.set_kv_format(fmt)
    pm = PagedModel(cfg, state, weights="int8")
    g = torch.Generator().manual_seed(6)
    B, P = 3, 37
    prompts = torch.randint(0, cfg.vocab, (B, P), generator=g, dtype=torch.int32).cuda()
    cache = pm.new_cache(B, 128, "e4m3" if fmt == "v_fp8" else "bf16")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    with torch.inference_mode():
        lg = pm.prefill(prompts, cache, 0, status=status)
        lay = StepLayout(B, 5, "cuda")
        ws = ops.attn_workspace(lay.batch, cfg.heads, cache)
        toks = torch.randint(0, cfg.vocab, (B, 5), generator=g, dtype=torch.int32).cuda()
        lay.set(cache.lengths)
        got = pm.logits(pm.step(toks.reshape(-1), lay, cache, ws, status=status)).view(B, 5, -1)
        for b in range(B):
            want, c = _run(ref, prompts[b:b + 1].long(), None)
            _close(lg[b:b + 1], want[:, -1], f"prefill seq {b}", PROMPT_LOGIT_RTOL)
            want, _ = _run(ref, toks[b:b + 1].long(), c)
            _close(got[b], want[0], f"verify step seq {b}", PROMPT_LOGIT_RTOL)
    assert int(status.item()) == 0


def _greedy(pm, prompts, n):
    """Greedy tokens one step at a time, and the top-2 logit gap of each."""
    from specdec_b200.engine.model import StepLayout
    from specdec_b200.kernels import ops

    B, P = prompts.shape
    cache = pm.new_cache(B, P + n + 1)
    lay = StepLayout(B, 1, "cuda")
    ws = ops.attn_workspace(lay.batch, pm.cfg.heads, cache)
    toks, gaps = [], []
    with torch.inference_mode():
        lg = pm.prefill(prompts, cache, 0)
        for _ in range(n):
            top = lg.float().topk(2, dim=-1)
            gaps.append(top.values[:, 0] - top.values[:, 1])
            toks.append(lg.argmax(-1).int())
            lay.set(cache.lengths)
            lg = pm.logits(pm.step(toks[-1], lay, cache, ws))
            cache.lengths.add_(1)
    return torch.stack(toks, 1).cpu(), torch.stack(gaps, 1).cpu()


def test_int8_specdec_emits_its_targets_greedy_tokens():
    """SpecDec with 8-bit target and draft (round graph included) against the same target's greedy decoding,
    one token at a time.  Sums of norms and attention run in other orders: a divergence only at a near-tie."""
    from specdec_b200.engine.model import PagedModel, random_state
    from specdec_b200.engine.specdec import SpecDecEngine

    cfg, _ = _cfgs()
    state = random_state(cfg, 21, "cuda", std=0.05)
    target = PagedModel(cfg, state, weights="int8")
    B, P, N = 4, 48, 20
    prompts = torch.randint(0, cfg.vocab, (B, P), generator=torch.Generator().manual_seed(7),
                            dtype=torch.int32).cuda()
    want, gaps = _greedy(target, prompts, N)
    for draft in (target, PagedModel(cfg, state)):
        eng = SpecDecEngine(target, draft, B, P, N, k=4)
        eng.capture()
        eng.prefill(prompts)
        eng.decode()
        got = eng.tokens().cpu()
        for b in range(B):
            differ = (got[b] != want[b]).nonzero()
            if len(differ):
                j = int(differ[0])
                assert gaps[b, j] < NEAR_TIE, f"seq {b} diverges at {j} with top-2 gap {gaps[b, j]:.4f}"
        assert eng.acceptance() > 2.0  # the draft is the target, or its bf16 original


def test_weights_argument():
    from specdec_b200.engine.model import PagedModel

    cfg, _ = _cfgs()
    with pytest.raises(ValueError, match="'bf16' or 'int8'"):
        PagedModel(cfg, {}, weights="int4")
