"""Which steps the attention over a 4-bit cache takes: by what its kernels count, and refused before an engine runs into one. Sizes are decided on the
host, without a GPU."""
import itertools

import pytest
import torch

from vllm_cpp_b200.config import EngineArgs, synthetic_config
from vllm_cpp_b200.engine import LLM
from vllm_cpp_b200.ops import _lib
from vllm_cpp_b200.ops import fp4_cache as C

MOST = 2 ** 31 - 1


def _takes(*, D=128, Hq=32, Hkv=8, block=32, positions, tokens, reqs=1, tiles=None, most=0, decode=False):
    C._declare()
    a = C.AttnArgs()
    a.D, a.Hq, a.Hkv, a.block_size, a.max_blocks, a.total_q, a.num_reqs, a.most_q = D, Hq, Hkv, block, -(-positions // block), tokens, reqs, most
    if not decode:
        a.q_start, a.num_tiles = 1, -(-tokens // 128) + reqs if tiles is None else tiles
    return _lib.lib().b200_fp4_attn_takes(a)


def test_long_tables_of_big_steps_are_taken():
    """Steps of models with long contexts, whose real lengths the table's width does not tell."""
    for D, reqs in itertools.product((64, 128, 256), (1, 2, 64, 256)):
        assert _takes(D=D, positions=1 << 20, tokens=8192, reqs=reqs) == 0
        assert _takes(D=D, Hq=64, positions=1 << 19, tokens=8192, reqs=reqs) == 0
        assert _takes(D=D, Hq=64, positions=1 << 18, tokens=16384, reqs=reqs) == 0
    assert _takes(Hq=64, positions=1 << 22, tokens=16384, reqs=1) == 0
    assert _takes(positions=1 << 22, tokens=256, reqs=256, decode=True) == 0


@pytest.mark.parametrize("D", [64, 128, 256])
def test_nothing_is_taken_whose_line_passes_31_bits(D):
    """The longest lines that ascending bounds allow, counted as the kernels do, against what is taken."""
    gen = torch.Generator().manual_seed(D)
    answers = set()
    for _ in range(4000):
        Hkv, G = (int(2 ** torch.randint(0, n, (1,), generator=gen)) for n in (6, 6))
        reqs = int(2 ** (13 * torch.rand(1, generator=gen)))
        tokens = reqs + int(2 ** (19 * torch.rand(1, generator=gen)))
        positions = int(2 ** (8 + 22 * torch.rand(1, generator=gen)))
        most = int(torch.randint(0, 3, (1,), generator=gen))
        tiles = -(-tokens // 128) + reqs
        got = _takes(D=D, Hq=G * Hkv, Hkv=Hkv, positions=positions, tokens=tokens, reqs=reqs, tiles=tiles, most=most)
        rows, R = tokens * G, 16 if D <= 128 and tokens * G > 8 * reqs else 8
        both = D <= 128 and (most or tokens) * G > 48
        # one sequence with all rows, all alike, or all but one with a single token
        shapes = [[tokens], [tokens // reqs] * (reqs - 1) + [tokens - tokens // reqs * (reqs - 1)], [1] * (reqs - 1) + [tokens - reqs + 1]]
        longest = 0
        for q in shapes:
            mine = [n * G for n in q if not both or n * G <= 48]
            if not (both and reqs == 1):
                longest = max(longest, sum(-(-n // R) for n in mine) * Hkv * (-(-positions // 32) + (28 if R == 16 else 20)))
            if both:
                longest = max(longest, sum(-(-min(128, n - at) * G // 256) for n in q for at in range(0, n, 128)) * Hkv * (-(-positions // 128) + 3))
        if got == 0:
            assert longest <= MOST and reqs <= 8192 and tiles <= 8000
        elif reqs <= 8192 and tiles <= 8000 and rows * G < 2 ** 32:
            # Refused is no less than what is said to be counted: of the rows a tile that is not full for every sequence (which the shapes above do not
            # all have, so they may come to half of it or less), of the tiles listed 128 tokens each (which may be one each, and listed twice).
            count = (tokens * G / R + reqs) * Hkv * (-(-positions // 32) + 28)
            if both:
                count = max(count if reqs > 1 else 0, tiles * -(-min(128, tokens) * G // 256) * Hkv * (-(-positions // 128) + 3))
            assert got == -4 and count > MOST
        answers.add(got)
    assert answers == {0, -4}


def test_other_limits():
    assert _takes(positions=2 ** 31 - 2 ** 12 + 1, tokens=1, Hq=1, Hkv=1, block=2 ** 12) == -4
    # cells of 16 times the cells of a block below 2^32: 2^30 / 16 * 32 = 2^31 is, * 64 is not
    assert _takes(positions=2 ** 30, tokens=1, Hq=1, Hkv=1, block=512) == 0
    assert _takes(positions=2 ** 30, tokens=1, Hq=1, Hkv=1, block=1024) == -4
    assert _takes(positions=64, tokens=8193, reqs=8193, tiles=10) == -4
    assert _takes(positions=64, tokens=8192, reqs=8192, decode=True) == 0
    assert _takes(positions=64, tokens=8192, tiles=8001) == -4
    assert _takes(D=96, positions=64, tokens=1) == -1 and _takes(Hq=31, positions=64, tokens=1) == -1


def test_an_engine_says_so_before_its_first_step():
    cfg = synthetic_config("tiny-dense")
    cfg.head_dim = 64
    llm = LLM(EngineArgs(model_config=cfg, device="cpu", block_size=16, num_blocks=40, max_model_len=256, max_num_seqs=3, max_num_batched_tokens=128,
                         kv_cache_dtype="fp4"))
    m = llm.model
    ok = dict(max_tokens=8192, max_reqs=256, max_tiles=64 + 256, max_blocks=(1 << 20) // 16 + 1, block_size=16)
    m.check_steps(**ok)
    for bad in (dict(max_reqs=8193), dict(max_tiles=8001), dict(max_blocks=1 << 27), dict(max_tokens=1 << 30)):
        with pytest.raises(ValueError, match="lower max_num_seqs"):
            m.check_steps(**{**ok, **bad})
    plain = LLM(EngineArgs(model_config=cfg, device="cpu", block_size=16, num_blocks=40, max_model_len=256, max_num_seqs=3))
    plain.model.check_steps(**{**ok, "max_reqs": 10 ** 6})      # (the bf16 cache has no such limits)


@pytest.mark.gpu
@pytest.mark.parametrize("D,Hq,Hkv", [(128, 32, 8), (64, 64, 8), (256, 16, 4)])
def test_wide_tables_change_nothing(D, Hq, Hkv):
    """A step of 8192 tokens over tables for more than a million: the same bits as over narrow ones."""
    import fp4_reference as F
    from vllm_cpp_b200.ops import reference as ref
    bs, new, lens = 16, [8000, 5, 187], [8000, 900, 187]
    wide, narrow = (1 << 20) // bs + 1, -(-max(lens) // bs)
    if D == 256:
        new, lens = [700, 5, 187], [8000, 900, 187]             # (many rows of 256 dims take long)
    gen = torch.Generator().manual_seed(D)
    cache = F.random_cache(600, Hkv, bs, D, gen, "cuda")
    table = torch.randint(0, 600, (3, wide), generator=gen, dtype=torch.int32).cuda()
    q = torch.randn((sum(new), Hq * D), generator=gen).to(torch.bfloat16).cuda()
    req, q0 = (torch.tensor(t, dtype=torch.int32, device="cuda") for t in ref.build_prefill_tiles(new))
    args = dict(seq_lens=torch.tensor(lens, dtype=torch.int32, device="cuda"), q_start=torch.tensor([0] + new, device="cuda").cumsum(0).int(), tile_req=req,
                tile_q0=q0, scale=D ** -0.5)
    want = C.prefill(q, cache, block_table=table[:, :narrow], **args)
    assert torch.equal(C.prefill(q, cache, block_table=table, **args), want)
    at = sum(new[:1])
    slots = (table[1].long()[:, None] * bs + torch.arange(bs, device="cuda")).flatten()[: lens[1]]
    k, v = C.read(cache, slots)
    F.check_attention(want[at: at + 5].view(5, Hq, D), *F.attention(q[at: at + 5].view(5, Hq, D), k, v, lens[1] - 5, D ** -0.5, 0.0, 0))
    from vllm_cpp_b200 import ops
    assert ops.read_status() == 0
