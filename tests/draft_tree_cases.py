"""Inputs for the tests of drafted trees, and the attention's definition in 64 bits with its error bound."""
import math
import random

import torch


def tree_parents(n, rng, wide=4):
    """Parents of a random tree (chains for wide 1), parents before children."""
    return [-1 if j == 0 else j - 1 if wide == 1 else rng.randrange(max(0, j - 2 * wide), j) for j in range(n)]


def starts_of(sizes, device="cpu"):
    at = [0]
    for n in sizes:
        at.append(at[-1] + n)
    return torch.tensor(at, dtype=torch.int32, device=device)


def page_table(lengths, page, gen, spare=1):
    """A page table over pages in no order (page 0 is nobody's) -> table, pages."""
    counts = [max(1, -(-n // page)) for n in lengths]
    total = sum(counts) + spare
    order = (torch.randperm(total - 1, generator=gen) + 1).tolist()
    table = torch.zeros((len(lengths), max(counts)), dtype=torch.int32)
    at = 0
    for r, n in enumerate(counts):
        table[r, :n] = torch.tensor(order[at: at + n], dtype=torch.int32)
        at += n
    return table, total


def attention_case(sizes, contexts, *, hq, hkv, d, page, seed=0, wide=4, words=None, pad=0, spread=3.0, stride=0, device="cpu"):
    """Inputs of a call as a dict; ``pad`` rows behind the last request, ``stride`` columns behind q's in a row."""
    from vllm_cpp_b200.ops import draft_tree
    rng, gen = random.Random(seed), torch.Generator().manual_seed(seed)
    lengths = [a + b for a, b in zip(sizes, contexts)]
    rows = sum(sizes) + pad
    table, pages = page_table(lengths, page, gen)
    parents = torch.tensor([p for n in sizes for p in tree_parents(n, rng, wide)] + [-1] * pad, dtype=torch.int32)
    q_start, seq_lens = starts_of(sizes), torch.tensor(lengths, dtype=torch.int32)
    words = words or max(1, -(-max(sizes, default=1) // 64))
    bits, positions = draft_tree.ref_mask(parents, q_start=q_start, seq_lens=seq_lens, max_nodes=64 * words)
    q = torch.randn((rows, hq * d + stride), generator=gen).mul_(spread).to(torch.bfloat16)
    cache = torch.randn((pages, 2, page, hkv, d), generator=gen).to(torch.bfloat16)
    case = dict(q=q, kv_cache=cache, block_table=table, seq_lens=seq_lens, q_start=q_start, mask=bits, positions=positions)
    case = {k: v.to(device) for k, v in case.items()}
    case["q"] = case["q"][:, : hq * d]
    return case, d ** -0.5


def attention_bound(case, scale, softcap=0.0, window=0):
    """(outputs in 64 bits, bound of what bf16 outputs may be off). Weights are rounded to bf16, half a step 2^-8 of each, and the sum that
    divides is that of the rounded ones, so that an output moves by at most 2^-8 sum p |v - o| <= 2^-8 (sum p |v| + |o|). The output's own rounding
    is 2^-8 |o|. Scores are sums of D products in 32 bits: off by D 2^-23 of sum |q k| scale, which is what the weights are off by relatively (twice: the
    sum too); exponentials and soft cap add some 2^-20 of a score of at most 2^7, or of the cap."""
    from vllm_cpp_b200.ops import draft_tree
    c = {k: v.double() if v.dtype == torch.bfloat16 else v for k, v in case.items()}
    o = draft_tree.ref_attention(scale=scale, softcap=softcap, window=window, dtype=torch.float64, **c)
    size = dict(c, kv_cache=torch.stack([c["kv_cache"][:, 0], c["kv_cache"][:, 1].abs()], 1))
    a = draft_tree.ref_attention(scale=scale, softcap=softcap, window=window, dtype=torch.float64, **size)
    d = case["kv_cache"].shape[-1]
    finite = torch.where(torch.isfinite(c["kv_cache"]), c["kv_cache"], torch.zeros_like(c["kv_cache"]))
    top = float(c["q"].reshape(-1, d).norm(dim=1).max()) * float(finite[:, 0].norm(dim=-1).max()) * scale      # (sum |q k| <= |q| |k|)
    scores = 2 * (d * 2.0 ** -23 * top + 2.0 ** -20 * max(2.0 ** 7, softcap))
    return o, 2.0 ** -8 * o.abs() + 2.0 ** -8 * (a + o.abs()) + scores * a + 1e-30
