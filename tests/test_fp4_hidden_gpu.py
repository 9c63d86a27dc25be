"""NaN among the keys and values that a query does not see, because they come later or lie before its window, does not reach its result, although
its row shares tiles with rows that see them; and it reaches the rows that do, in the 16 dims of its group."""
import math

import pytest
import torch

import fp4_reference as F
from vllm_cpp_b200.ops import fp4_cache as C
from vllm_cpp_b200.ops import reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"

CASES = [
    # lengths, new tokens, Hq, Hkv, D, block, window, causal
    ([40, 9], [5, 3], 8, 8, 128, 16, 0, True),            # few rows: tiles of 8 with several tokens,
    ([40, 9], [5, 3], 16, 2, 128, 16, 0, True),           # with one,
    ([300, 70], [6, 4], 24, 8, 128, 32, 0, True),         # of 16
    ([300, 70], [6, 4], 6, 2, 64, 32, 40, True),
    ([300, 70], [7, 2], 4, 2, 256, 16, 0, True),
    ([300, 70], [7, 2], 3, 1, 256, 48, -64, True),
    ([90, 33], [4, 33], 3, 1, 64, 16, 7, False),
    ([600, 200], [600, 130], 8, 2, 128, 32, 0, True),     # many rows
    ([600, 200], [300, 130], 3, 3, 64, 16, 0, True),
    ([900, 200], [640, 130], 4, 1, 128, 32, 100, True),
    ([900, 200], [640, 130], 4, 4, 64, 48, -128, True),
    ([700, 260], [200, 260], 8, 2, 128, 32, 60, False),
    ([5000], [70], 32, 8, 128, 32, 0, True),              # items that several CTAs share
    ([260, 3, 2000, 17], [130, 3, 5, 17], 24, 4, 128, 32, 0, True),      # both kernels
]


@pytest.mark.parametrize("lens,new,Hq,Hkv,D,bs,window,causal", CASES)
def test_nan_that_a_query_does_not_see(lens, new, Hq, Hkv, D, bs, window, causal):
    gen = torch.Generator().manual_seed(sum(lens) + D)
    pages = [-(-n // bs) for n in lens]
    perm = torch.randperm(sum(pages) + 2, generator=gen)
    table, at = torch.zeros((len(lens), max(pages)), dtype=torch.int32), 0
    for r, n in enumerate(pages):
        table[r, :n] = perm[at: at + n].int()
        at += n
    cache = C.alloc(sum(pages) + 2, Hkv, bs, D, DEV)
    held = []
    for r, (n, m) in enumerate(zip(lens, new)):
        x = torch.randn((2, n, Hkv, D), generator=gen).to(torch.bfloat16)
        # around the first and last queries, around their windows' beginnings, and in the middle of the queries
        for j, near in enumerate((n - 1, n - 2, n - m, n - m + 1, n - m // 2, n - m - abs(window), n - 1 - abs(window), n // 2)):
            if 0 <= near < n:
                x[1, near, j % Hkv, (5 * j + near) % D] = math.nan
        if causal:
            x[0, n - 1, 0, 3] = math.nan                  # a key that only the last query sees
        slots = (table[r].long()[:, None] * bs + torch.arange(bs)).flatten()[:n].to(DEV)
        C.write(x[0].to(DEV), x[1].to(DEV), cache, slots)
        held.append(C.read(cache, slots))
    q = torch.randn((sum(new), Hq * D), generator=gen).to(torch.bfloat16).to(DEV)
    req, q0 = (torch.tensor(t, dtype=torch.int32, device=DEV) for t in ref.build_prefill_tiles(new))
    out = C.prefill(q, cache, block_table=table.to(DEV), seq_lens=torch.tensor(lens, dtype=torch.int32, device=DEV),
                    q_start=torch.tensor([0] + new, device=DEV).cumsum(0).int(), tile_req=req, tile_q0=q0, scale=D ** -0.5, window=window, causal=causal)
    at = 0
    for (k, v), n, m in zip(held, lens, new):
        got, G = out[at: at + m].view(m, Hq, D), Hq // Hkv
        pos, key = torch.arange(n - m, n, device=DEV)[:, None], torch.arange(n, device=DEV)[None]
        seen = (key <= (pos if causal else n)).expand(m, n)
        if window > 0:
            seen = seen & (key > pos - window)
        elif window < 0:
            seen = seen & (key >= pos // -window * -window)
        # rows that see a NaN: by its key all of them, by its value those dims
        bad = torch.einsum("mn,nhd->mhd", seen.float(), v.isnan().float()) + torch.einsum("mn,nh->mh", seen.float(), k.isnan().any(-1).float())[..., None]
        bad = (bad > 0).repeat_interleave(G, 1)
        assert bool(bad.any()) and not bool(bad.all())
        assert torch.equal(got.isnan(), bad)
        want, size = F.attention(q[at: at + m].view(m, Hq, D), k.nan_to_num(), v.nan_to_num(), n - m, D ** -0.5, 0.0, window, causal)
        zero = torch.zeros((), dtype=torch.float64, device=DEV)
        F.check_attention(torch.where(bad, zero, got.double()), torch.where(bad, zero, want), size)
        at += m
    from vllm_cpp_b200 import ops
    assert ops.read_status() == 0
