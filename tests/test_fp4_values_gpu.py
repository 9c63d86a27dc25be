"""Attention of many rows over the 4-bit cache with values that are hard for it: queries of every size and none at all, a maximum that rises."""
import math

import pytest
import torch

import fp4_reference as F
from vllm_cpp_b200 import ops
from vllm_cpp_b200.ops import fp4_cache as C
from vllm_cpp_b200.ops import reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("size", [1e-30, 1e-3, 1.0, 1e4, 1e30])
@pytest.mark.parametrize("cap", [0.0, 5.0])
def test_many_rows_of_values_of_every_size(D, size, cap):
    """Queries from 1e-30 to 1e30, keys that grow along the sequence, so that the running maximum is raised again and again, and values of
    very different sizes."""
    Hq, Hkv, bs, n, m = 4, 1, 32, 900, 300
    gen = torch.Generator().manual_seed(D)
    x = torch.randn((2, n, Hkv, D), generator=gen)
    x[0] *= torch.linspace(0.01, 30, n)[:, None, None]
    x[1] *= torch.exp(4 * torch.randn((n, 1, 1), generator=gen))
    x = x.to(torch.bfloat16).to(DEV)
    cache = C.alloc(n // bs + 1, Hkv, bs, D, DEV)
    C.write(x[0], x[1], cache, torch.arange(n, device=DEV))
    k, v = C.read(cache, torch.arange(n, device=DEV))
    q = (torch.randn((m, Hq * D), generator=gen) * size).to(torch.bfloat16).to(DEV)
    q[7] = 0
    scale = 0.02 / size * math.sqrt(128 / D)
    req, q0 = (torch.tensor(t, dtype=torch.int32, device=DEV) for t in ref.build_prefill_tiles([m]))
    out = C.prefill(q, cache, block_table=torch.arange(n // bs + 1, dtype=torch.int32, device=DEV)[None], softcap=cap, tile_req=req, tile_q0=q0, scale=scale,
                    seq_lens=torch.tensor([n], dtype=torch.int32, device=DEV), q_start=torch.tensor([0, m], dtype=torch.int32, device=DEV))
    F.check_attention(out.view(m, Hq, D), *F.attention(q.view(m, Hq, D), k, v, n - m, scale, cap, 0))
    assert ops.read_status() == 0


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("scale", [1e-45, 1e-38, 1e-30, 1e-8, 1.0])
@pytest.mark.parametrize("m", [4, 300])
def test_queries_of_zeros(D, scale, m):
    """All scores are 0, whatever the scale: the average of the values that a row sees."""
    Hq, Hkv, bs, n, window = 4, 2, 16, 500, 200
    gen = torch.Generator().manual_seed(m)
    cache = F.random_cache(40, Hkv, bs, D, gen, DEV)
    table = torch.randperm(40, generator=gen)[: n // bs + 1].int().to(DEV)[None]
    q = torch.zeros((m, Hq * D), dtype=torch.bfloat16, device=DEV)
    q[1] = 1e-30
    req, q0 = (torch.tensor(t, dtype=torch.int32, device=DEV) for t in ref.build_prefill_tiles([m]))
    out = C.prefill(q, cache, block_table=table, seq_lens=torch.tensor([n], dtype=torch.int32, device=DEV), window=window, tile_req=req, tile_q0=q0,
                    q_start=torch.tensor([0, m], dtype=torch.int32, device=DEV), scale=scale)
    slots = (table[0].long()[:, None] * bs + torch.arange(bs, device=DEV)).flatten()[:n]
    k, v = C.read(cache, slots)
    F.check_attention(out.view(m, Hq, D), *F.attention(q.view(m, Hq, D), k, v, n - m, scale, 0.0, window))
    assert ops.read_status() == 0


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("cap", [1e-45, 1e-30, 1e-9, 1000.0, 1e4, 1e6, 1e9, 1e30])
@pytest.mark.parametrize("m", [1, 5, 300])
def test_caps_of_every_size(D, cap, m):
    """Rows of zeros beside rows of up to 1e30: a score of 0 stays 0 under the smallest cap, and the largest ones leave scores as they are."""
    Hq, Hkv, bs, n = 4, 2, 16, 500
    gen = torch.Generator().manual_seed(m)
    cache = F.random_cache(40, Hkv, bs, D, gen, DEV)
    table = torch.randperm(40, generator=gen)[: n // bs + 1].int().to(DEV)[None]
    q = torch.randn((m, Hq, D), generator=gen)
    q[:, 0] = 0
    q[:, 1] *= 1e30
    q[:, 2] *= 0.01
    q = q.to(torch.bfloat16).to(DEV)
    args = dict(block_table=table, seq_lens=torch.tensor([n], dtype=torch.int32, device=DEV), scale=D ** -0.5, softcap=cap)
    if m == 1:
        out = C.decode(q.view(m, -1), cache, **args)
    else:
        req, q0 = (torch.tensor(t, dtype=torch.int32, device=DEV) for t in ref.build_prefill_tiles([m]))
        out = C.prefill(q.view(m, -1), cache, q_start=torch.tensor([0, m], dtype=torch.int32, device=DEV), tile_req=req, tile_q0=q0, **args)
    slots = (table[0].long()[:, None] * bs + torch.arange(bs, device=DEV)).flatten()[:n]
    k, v = C.read(cache, slots)
    if cap < 1:
        # scores of at most the cap are equal but for 2^-29
        want, size = F.attention(torch.zeros_like(q), k, v, n - m, 1.0, 0.0, 0)
        F.check_attention(out.view(m, Hq, D), want, size)
    else:
        # a cap far above every score but those of the second head, which is equal to it for many keys
        want, size = F.attention(q, k, v, n - m, D ** -0.5, cap, 0)
        keep = [0, 2, 3]
        F.check_attention(out.view(m, Hq, D)[:, keep], want[:, keep], size[:, keep])
        assert not out.isnan().any()
    assert ops.read_status() == 0


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("size", [2.0 ** -122, 2.0 ** -110, 2.0 ** 110, 2.0 ** 122])
@pytest.mark.parametrize("m", [1, 5, 300])
def test_queries_at_the_ends_of_their_type(D, size, m):
    """Queries that an f16 does not hold, with a scale that makes their scores ordinary ones."""
    Hq, Hkv, bs, n = 4, 2, 16, 500
    gen = torch.Generator().manual_seed(m)
    cache = F.random_cache(40, Hkv, bs, D, gen, DEV)
    table = torch.randperm(40, generator=gen)[: n // bs + 1].int().to(DEV)[None]
    q = (torch.randn((m, Hq, D), generator=gen) * size).to(torch.bfloat16).to(DEV)
    args = dict(block_table=table, seq_lens=torch.tensor([n], dtype=torch.int32, device=DEV), scale=0.25 / size)
    if m == 1:
        out = C.decode(q.view(m, -1), cache, **args)
    else:
        req, q0 = (torch.tensor(t, dtype=torch.int32, device=DEV) for t in ref.build_prefill_tiles([m]))
        out = C.prefill(q.view(m, -1), cache, q_start=torch.tensor([0, m], dtype=torch.int32, device=DEV), tile_req=req, tile_q0=q0, **args)
    slots = (table[0].long()[:, None] * bs + torch.arange(bs, device=DEV)).flatten()[:n]
    k, v = C.read(cache, slots)
    F.check_attention(out.view(m, Hq, D), *F.attention(q, k, v, n - m, 0.25 / size, 0.0, 0))
    assert ops.read_status() == 0
