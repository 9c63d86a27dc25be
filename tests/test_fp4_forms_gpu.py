"""Forms of the 4-bit cache's kernels that their size chooses, and its blocks in the host tier."""
import pytest
import torch

import fp4_reference as F
from vllm_cpp_b200 import ops
from vllm_cpp_b200.ops import fp4_cache as C

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("H,D", [(1, 64), (2, 64), (1, 128), (1, 256), (20, 128)])
@pytest.mark.parametrize("over", [-1, 0, 1, 12345])
def test_read_on_both_sides_of_two_lots_a_block(H, D, over):
    """A block reads two lots of tokens from so many tokens on that every SM has eight blocks then."""
    per = 2 * H * (D // 8)                                     # threads of a token
    tokens = 256 // per if per < 256 else 1
    n, bs, nb = 2 * tokens * 8 * ops.num_sms() + over, 16, 20
    gen = torch.Generator().manual_seed(n)
    cache = F.random_cache(nb, H, bs, D, gen)
    slots = torch.randint(-3, nb * bs + 3, (n,), generator=gen)
    k, v = C.read(cache.to(DEV), slots.to(DEV))
    rk, rv = C.ref_read(cache, slots)
    assert torch.equal(k.cpu(), rk) and torch.equal(v.cpu(), rv)


def test_prefixes_come_back_from_the_host_tier():
    from vllm_cpp_b200.config import EngineArgs, synthetic_config
    from vllm_cpp_b200.engine import LLM, SamplingParams
    cfg = synthetic_config("tiny-dense")
    cfg.head_dim = 64
    gen = torch.Generator().manual_seed(3)
    shared, others = (torch.randint(0, cfg.vocab_size, (n, m), generator=gen).tolist() for n, m in ((1, 96), (3, 150)))
    greedy = SamplingParams(temperature=0.0, max_tokens=6, ignore_eos=True)

    def engine(**kw):
        return LLM(EngineArgs(model_config=cfg, device="cuda", block_size=16, num_blocks=12, max_model_len=256, max_num_seqs=2, max_num_batched_tokens=128,
                              kv_cache_dtype="fp4", enable_prefix_caching=True, **kw))

    def tokens(llm):
        return llm.generate([shared[0] + [1, 2, 3]], greedy)[0].outputs[0].token_ids
    want, llm = tokens(engine()), engine(kv_transfer_config={"cpu_blocks": 64})
    assert tokens(llm) == want
    for p in others:
        llm.generate([p], greedy)
    assert llm.offload.stored_blocks > 0
    assert tokens(llm) == want and llm.offload.loaded_blocks > 0
    assert ops.read_status() == 0
