"""Engines whose KV cache is held in 4 bits, on the GPU, against the same model through the CPU back end."""
import pytest
import torch

from test_engine_gpu import _agreement, _cfg, _prompts, _run
from vllm_cpp_b200 import ops
from vllm_cpp_b200.config import EngineArgs, synthetic_config
from vllm_cpp_b200.engine import LLM, SamplingParams
from vllm_cpp_b200.ops import fp4_cache

pytestmark = pytest.mark.gpu


def test_gpu_matches_the_cpu_back_end():
    cfg = _cfg()
    prompts = _prompts(cfg, (150, 9, 300, 40, 17, 64))
    gpu, llm = _run("cuda", cfg, prompts, kv_cache_dtype="fp4")
    assert llm.model.kv_caches[0].dtype == torch.uint8
    cpu, _ = _run("cpu", cfg, prompts, kv_cache_dtype="fp4")
    assert ops.read_status() == 0
    # (as for the bf16 cache: sums in another order, many near-ties in a random model)
    assert [g[0] for g in gpu] == [c[0] for c in cpu]
    assert _agreement(gpu, cpu) > 0.8


def test_graphs_eager_steps_and_asynchronous_scheduling_agree():
    cfg = _cfg()
    prompts = _prompts(cfg, (33, 200, 5, 77, 130, 18), seed=5)
    a, _ = _run("cuda", cfg, prompts, kv_cache_dtype="fp4")
    b, _ = _run("cuda", cfg, prompts, graphs=False, kv_cache_dtype="fp4")
    c, llm = _run("cuda", cfg, prompts, async_scheduling=True, kv_cache_dtype="fp4")
    assert a == b == c and llm.use_async
    d, _ = _run("cuda", cfg, prompts, budget=64, kv_cache_dtype="fp4")
    assert _agreement(a, d) > 0.9
    assert ops.read_status() == 0


@pytest.mark.parametrize("name", ["tiny-moe", "tiny-opt", "tiny-dense"])
def test_other_families(name):
    cfg = synthetic_config(name)
    if name == "tiny-dense":                                  # layers with a window beside full ones, capped scores
        cfg.sliding_window, cfg.layer_types, cfg.attn_logit_softcap = 24, ["sliding_attention", "full_attention"], 30.0
    prompts = _prompts(cfg, (40, 9, 100), seed=2)
    gpu, llm = _run("cuda", cfg, prompts, kv_cache_dtype="fp4")
    cpu, _ = _run("cpu", cfg, prompts, kv_cache_dtype="fp4")
    assert [g[0] for g in gpu] == [c[0] for c in cpu]
    assert ops.read_status() == 0


def test_drafts_are_verified_over_it():
    from vllm_cpp_b200.spec_decode import SpeculativeConfig
    cfg = _cfg()
    prompts = [p + p[:30] for p in _prompts(cfg, (60, 45))]
    plain, _ = _run("cuda", cfg, prompts, kv_cache_dtype="fp4")
    drafted, llm = _run("cuda", cfg, prompts, kv_cache_dtype="fp4",
                        speculative_config=SpeculativeConfig(method="ngram", num_speculative_tokens=3))
    assert _agreement(plain, drafted) > 0.9
    assert ops.read_status() == 0


def test_a_prefix_is_found_again():
    cfg = _cfg()
    p = _prompts(cfg, (128,))[0]
    llm = LLM(EngineArgs(model_config=cfg, device="cuda", block_size=32, num_blocks=100, max_model_len=640, max_num_seqs=4,
                         max_num_batched_tokens=256, kv_cache_dtype="fp4"))
    sp = SamplingParams(temperature=0.0, max_tokens=8, ignore_eos=True)
    first, second = (llm.generate([p + [1, 2, 3]], sp)[0] for _ in range(2))
    assert second.num_cached_tokens >= 96 and first.outputs[0].token_ids == second.outputs[0].token_ids


def test_chunks_of_a_gpu_cache_travel_as_bf16():
    from test_lmcache import MockServer
    from vllm_cpp_b200.worker.lmcache import LMCacheStore
    srv = MockServer()
    srv.start()
    H, D, bs, chunk = 2, 128, 16, 32
    caches = [fp4_cache.alloc(8, H, bs, D, "cuda") for _ in range(2)]
    for i, c in enumerate(caches):
        x = torch.randn((2, 8 * bs, H * D), generator=torch.Generator().manual_seed(i)).to(torch.bfloat16).cuda()
        fp4_cache.write(x[0], x[1], c, torch.arange(8 * bs, device="cuda"))
    url = f"lm://127.0.0.1:{srv.port}"
    store = LMCacheStore(url, "tiny", caches, bs, chunk_size=chunk)
    tokens, blocks, others = list(range(70)), [5, 2, 7, 1, 3], [0, 1, 2, 3]
    assert store.store(tokens, blocks) == 2
    back = [torch.zeros_like(c) for c in caches]
    other = LMCacheStore(url, "tiny", back, bs, chunk_size=chunk, connect=False)
    other.client = store.client
    assert other.load(tokens, others, 64) == 64
    for a, b in zip(caches, back):
        assert torch.equal(fp4_cache.ref_expand(a)[blocks[:4]], fp4_cache.ref_expand(b)[others])
    store.client.close()


def test_a_draft_model_with_a_cache_in_bf16():
    from vllm_cpp_b200.spec_decode import SpeculativeConfig
    cfg = _cfg()
    prompts = _prompts(cfg, (60, 45))
    plain, _ = _run("cuda", cfg, prompts, kv_cache_dtype="fp4")
    drafted, llm = _run("cuda", cfg, prompts, kv_cache_dtype="fp4", speculative_config=SpeculativeConfig(
        method="draft_model", num_speculative_tokens=2, draft_model_config=_cfg()))
    assert llm.runner.drafter.model.kv_caches[0].dtype == torch.bfloat16
    assert _agreement(plain, drafted) > 0.9
    assert ops.read_status() == 0
