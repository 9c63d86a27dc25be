"""Engines whose KV cache is held in 4 bits, on the CPU: token streams do not depend on how a prompt is cut, the cache's blocks move between
tiers and programs, and models that cannot hold it say so."""
import time

import pytest
import torch

from test_lmcache import MockServer
from vllm_cpp_b200.config import EngineArgs, synthetic_config
from vllm_cpp_b200.engine import LLM, SamplingParams
from vllm_cpp_b200.models import attention_backends
from vllm_cpp_b200.ops import fp4_cache

GREEDY = SamplingParams(temperature=0.0, max_tokens=6, ignore_eos=True)


def _cfg(name="tiny-dense"):
    c = synthetic_config(name)
    c.head_dim = 64
    return c


def _prompts(cfg, lens, seed=3):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, cfg.vocab_size, (n,), generator=g).tolist() for n in lens]


def _engine(cfg, budget=128, **kw):
    args = dict(model_config=cfg, device="cpu", block_size=16, num_blocks=40, max_model_len=256, max_num_seqs=3,
                max_num_batched_tokens=budget, kv_cache_dtype="fp4")
    return LLM(EngineArgs(**{**args, **kw}))


def _tokens(llm, prompts, sp=GREEDY):
    return [o.outputs[0].token_ids for o in llm.generate(prompts, sp)]


@pytest.mark.parametrize("name", ["tiny-dense", "tiny-qwen3", "tiny-moe"])
def test_a_prompt_cut_in_portions_gives_the_same_tokens(name):
    cfg = _cfg(name)
    prompts = _prompts(cfg, (90, 7, 33))
    llm = _engine(cfg)
    assert llm.model.kv_caches[0].dtype == torch.uint8
    want = _tokens(llm, prompts)
    assert _tokens(_engine(cfg, budget=24), prompts) == want
    assert _tokens(_engine(cfg, cpu_backend="native"), prompts)[0][:1] == want[0][:1]


def test_blocks_cost_nine_bits_for_two_bytes():
    cfg = _cfg()
    a, b = _engine(cfg), _engine(cfg, kv_cache_dtype="auto")
    assert a.model.kv_bytes_per_block(16) * 32 == b.model.kv_bytes_per_block(16) * 9
    for m, c in ((a.model, a.model.kv_caches), (b.model, b.model.kv_caches)):
        assert sum(x.numel() * x.element_size() for x in c) == 40 * m.kv_bytes_per_block(16)


def test_who_holds_it_and_who_does_not():
    with pytest.raises(ValueError, match="auto, not in fp4"):
        LLM(EngineArgs(model_config=synthetic_config("tiny-mla"), device="cpu", kv_cache_dtype="fp4", max_model_len=64))
    with pytest.raises(ValueError, match="auto, fp4, not in fp8"):
        _engine(_cfg(), kv_cache_dtype="fp8")
    with pytest.raises(ValueError, match="block_size in multiples of 16"):
        _engine(_cfg(), block_size=8)
    c = _cfg()
    c.head_dim = 32
    with pytest.raises(ValueError, match="head_dim 64, 128 or 256"):
        _engine(c)
    d = attention_backends.describe(_cfg(), 16, "fp4")
    assert d["fp4"]["decode"] and d["fp4"]["prefill"]


def test_drafts_are_verified_over_it():
    from vllm_cpp_b200.spec_decode import SpeculativeConfig
    cfg = _cfg()
    prompts = [p + p[:20] for p in _prompts(cfg, (30, 41))]
    sp = SamplingParams(temperature=0.0, max_tokens=16, ignore_eos=True)
    plain = _tokens(_engine(cfg), prompts, sp)
    llm = _engine(cfg, speculative_config=SpeculativeConfig(method="ngram", num_speculative_tokens=3))
    assert _tokens(llm, prompts, sp) == plain


def test_a_draft_model_keeps_a_cache_of_its_own_kind():
    from vllm_cpp_b200.spec_decode import SpeculativeConfig
    cfg = _cfg()
    prompts = _prompts(cfg, (30, 41))
    spec = SpeculativeConfig(method="draft_model", num_speculative_tokens=2, draft_model_config=synthetic_config("tiny-dense"))
    llm = _engine(cfg, speculative_config=spec)
    assert _tokens(llm, prompts) == _tokens(_engine(cfg), prompts)
    assert llm.runner.drafter.model.kv_caches[0].dtype == torch.bfloat16


def test_prefixes_come_back_from_the_host_tier():
    cfg = _cfg()
    shared = _prompts(cfg, (96,))[0]
    kw = dict(num_blocks=12, enable_prefix_caching=True, max_num_seqs=2)
    want = _tokens(_engine(cfg, **kw), [shared + [1, 2, 3]])
    llm = _engine(cfg, kv_transfer_config={"cpu_blocks": 64}, **kw)
    assert _tokens(llm, [shared + [1, 2, 3]]) == want
    for p in _prompts(cfg, (150, 150, 150), seed=8):
        llm.generate([p], GREEDY)
    assert llm.offload.stored_blocks > 0
    assert _tokens(llm, [shared + [1, 2, 3]]) == want and llm.offload.loaded_blocks > 0


def test_chunks_travel_as_bf16_and_come_back_as_the_same_codes():
    from vllm_cpp_b200.worker.lmcache import LMCacheStore
    srv = MockServer()
    srv.start()
    H, D, bs, chunk = 2, 64, 16, 32
    gen = torch.Generator().manual_seed(0)
    caches = [fp4_cache.alloc(8, H, bs, D, "cpu") for _ in range(2)]
    for c in caches:
        x = torch.randn((2, 8 * bs, H * D), generator=gen).to(torch.bfloat16)
        fp4_cache.ref_write(x[0], x[1], c, torch.arange(8 * bs))
    url = f"lm://127.0.0.1:{srv.port}"
    store = LMCacheStore(url, "tiny", caches, bs, chunk_size=chunk)
    tokens, blocks, others = list(range(70)), [5, 2, 7, 1, 3], [0, 1, 2, 3]
    assert store.store(tokens, blocks) == 2
    key = store.chunk_keys(tokens)[0]
    assert "+fp4kv@" in key                                   # (a bf16 engine of the model asks for other keys)
    deadline = time.monotonic() + 5.0
    while len(srv.store) < 2 and time.monotonic() < deadline:
        time.sleep(0.01)
    assert srv.store[key][3] == (2, 2, chunk, H * D) and len(srv.store[key][0]) == 2 * 2 * chunk * H * D * 2
    back = [torch.zeros_like(c) for c in caches]
    other = LMCacheStore(url, "tiny", back, bs, chunk_size=chunk, connect=False)
    other.client = store.client
    assert other.load(tokens, others, 64) == 64
    for a, b in zip(caches, back):
        for x, y in zip(blocks[:4], others):
            assert torch.equal(fp4_cache.ref_expand(a)[x], fp4_cache.ref_expand(b)[y])
    store.client.close()


def test_a_model_class_that_says_nothing_of_its_cache(monkeypatch):
    from vllm_cpp_b200.models import registry
    from vllm_cpp_b200.models.dense import DenseModel

    class Quiet:
        """What an engine asks of a model, from one that it is made of; no KV_CACHE_DTYPES."""
        DTYPES = ("bfloat16",)

        def __new__(cls, *a, **kw):
            return DenseModel(*a, **kw)
    monkeypatch.setattr(registry, "resolve", lambda architectures: ("Quiet", Quiet))
    cfg = _cfg()
    llm = LLM(EngineArgs(model_config=cfg, device="cpu", max_model_len=64, num_blocks=8))
    assert llm.model.kv_caches[0].dtype == torch.bfloat16
    with pytest.raises(ValueError, match="holds its KV cache in auto, not in fp4"):
        LLM(EngineArgs(model_config=cfg, device="cpu", kv_cache_dtype="fp4", max_model_len=64, num_blocks=8))
