"""How a draft model's decode attention is split, and its scratch, are the draft model's: its heads may be more than the target's (scratch of
the target's shape is then too small), and its cache may be held in another type. On the CPU, with a stand-in for the operators."""
import types

import pytest
import torch

from vllm_cpp_b200.config import EngineArgs, synthetic_config
from vllm_cpp_b200.engine import LLM, SamplingParams
from vllm_cpp_b200.spec_decode import SpeculativeConfig


def _engine(kv, draft_heads):
    cfg, draft = synthetic_config("tiny-dense"), synthetic_config("tiny-dense")
    cfg.head_dim = 64
    draft.head_dim, draft.num_heads, draft.num_kv_heads = 128, draft_heads, 1
    spec = SpeculativeConfig(method="draft_model", num_speculative_tokens=2, draft_model_config=draft)
    return LLM(EngineArgs(model_config=cfg, device="cpu", block_size=16, num_blocks=40, max_model_len=256, max_num_seqs=3,
                          max_num_batched_tokens=128, kv_cache_dtype=kv, speculative_config=spec))


@pytest.mark.parametrize("kv", ["auto", "fp4"])
def test_drafters_steps_are_split_by_the_drafters_shape(kv, monkeypatch):
    llm = _engine(kv, 16)
    r, draft = llm.runner, llm.runner.drafter.model
    # the runner's CUDA side on the CPU: splits by shape, scratch in host memory
    asked = []

    def splits(batch, hkv, group, D, max_len, block):
        asked.append((batch, hkv, group, D, max_len))
        return 3 if D == draft.D else 2
    monkeypatch.setattr(r, "ops", types.SimpleNamespace(attn_decode_splits=splits), raising=False)
    monkeypatch.setattr(r, "_decode_tmp", {}, raising=False)
    if kv == "fp4":
        monkeypatch.setattr(r.model, "decode_workspace", lambda *a: (1, torch.empty(10)))
    seen = []

    class Attended:                                            # contexts as the draft model's forward gets them
        def __init__(self, forward):
            self.forward = forward

        def __call__(self, ctx):
            if ctx.num_decodes:
                seen.append((ctx.num_decodes, ctx.decode_splits, ctx.extra.get("decode_tmp")))
            return self.forward(ctx)
    monkeypatch.setattr(draft, "forward", Attended(draft.forward))
    inner = r._decode_splits

    def as_on_a_gpu(*a, **kw):
        r.is_cuda = True
        try:
            return inner(*a, **kw)
        finally:
            r.is_cuda = False
    monkeypatch.setattr(r, "_decode_splits", as_on_a_gpu)
    g = torch.Generator().manual_seed(3)
    prompts = [torch.randint(0, llm.cfg.vocab_size, (n,), generator=g).tolist() for n in (30, 41)]
    llm.generate(prompts, SamplingParams(temperature=0.0, max_tokens=5, ignore_eos=True))
    assert seen
    for n, s, tmp in seen:
        assert s == 3
        assert [tuple(t.shape) for t in tmp] == [(n, draft.hq, 3, draft.D), (n, draft.hq, 3)]
    assert all(a[1:4] == ((draft.hkv, draft.hq // draft.hkv, draft.D) if a[3] == draft.D else (r.model.hkv, r.model.hq // r.model.hkv, r.model.D))
               for a in asked)
    if kv == "fp4":
        assert r._decode_splits(2)[0] == 1                     # the target's own
    else:
        assert r._decode_splits(2)[0] == 2


@pytest.mark.gpu
@pytest.mark.parametrize("kv", ["auto", "fp4"])
def test_drafts_of_a_model_with_more_heads(kv):
    """On the GPU, with parts enough that scratch of the target's shape would not hold them: the tokens are the target's own."""
    from vllm_cpp_b200 import ops
    cfg, draft = synthetic_config("tiny-dense"), synthetic_config("tiny-dense")
    cfg.head_dim = 64
    draft.head_dim, draft.num_heads, draft.num_kv_heads = 128, 32, 2
    g = torch.Generator().manual_seed(4)
    prompts = [torch.randint(0, cfg.vocab_size, (n,), generator=g).tolist() for n in (900, 450)]
    tokens, llm = [], None
    for spec in (None, SpeculativeConfig(method="draft_model", num_speculative_tokens=2, draft_model_config=draft)):
        llm = LLM(EngineArgs(model_config=cfg, device="cuda", block_size=32, num_blocks=100, max_model_len=1024, max_num_seqs=3, max_num_batched_tokens=512,
                             kv_cache_dtype=kv, speculative_config=spec))
        tokens.append([o.outputs[0].token_ids for o in llm.generate(prompts, SamplingParams(temperature=0.0, max_tokens=10, ignore_eos=True))])
    splits, tmp = llm.runner._decode_splits(2, llm.runner.drafter.model)
    assert splits > 1 and tuple(tmp[0].shape) == (2, 32, splits, 128)
    # (steps of several query rows add in another order: a near-tie may fall the other way, and what follows it)
    assert [t[0] for t in tokens[0]] == [t[0] for t in tokens[1]]
    assert ops.read_status() == 0
