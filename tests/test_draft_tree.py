"""Drafted trees without a GPU: the restatements against what they restate, refusals, and the sizes that the attention takes."""
import ctypes
import math
import random

import pytest
import torch

from draft_tree_cases import attention_case, page_table, starts_of, tree_parents
from vllm_cpp_b200.ops import _lib, draft_tree, reference
from vllm_cpp_b200.ops.validate import OpArgumentError
from vllm_cpp_b200.spec_decode import greedy_rejection_sample


def test_the_masks_restatement():
    parents = torch.tensor([-1, 0, 0, 1, 3, -1, 0], dtype=torch.int32)
    bits, positions = draft_tree.ref_mask(parents, q_start=starts_of([5, 2]), seq_lens=torch.tensor([25, 2], dtype=torch.int32), max_nodes=65)
    assert bits.tolist() == [[1, 0], [3, 0], [5, 0], [11, 0], [27, 0], [1, 0], [3, 0]] and positions.tolist() == [20, 21, 21, 22, 23, 0, 1]
    chain = torch.arange(-1, 129, dtype=torch.int32)
    bits, _ = draft_tree.ref_mask(chain, q_start=starts_of([130]), seq_lens=torch.tensor([130], dtype=torch.int32), max_nodes=130)
    assert bits[63].tolist() == [-1, 0, 0] and bits[129].tolist() == [-1, -1, 3]


def test_the_restatements_of_more_than_1024_nodes():
    """Nodes past the 1024th are left out, and lie behind the context all the same."""
    n, c = 1030, 9
    q_start, lens = starts_of([n]), torch.tensor([n + c], dtype=torch.int32)
    bits, positions = draft_tree.ref_mask(torch.arange(-1, n - 1, dtype=torch.int32), q_start=q_start, seq_lens=lens, max_nodes=1024)
    assert positions[:1024].tolist() == list(range(c, c + 1024)) and not bool(bits[1024:].any())
    seen = draft_tree.seen_by(bits, q_start=q_start, seq_lens=lens)[0]
    assert seen.sum(1).tolist() == list(range(c + 1, c + 1025)) and bool(seen[:, :c].all()) and not bool(seen[:, c + 1024:].any())
    table, pages = page_table([n + c], 64, torch.Generator().manual_seed(1))
    cache = torch.arange(pages * 2 * 64 * 4).view(pages, 2, 64, 1, 4).float()
    before = cache.clone()
    draft_tree.ref_compact(cache, block_table=table, seq_lens=lens, q_start=q_start, path=torch.tensor([[0, 3, 1023, 1024, 1029]]))
    cell = lambda x, at: x[table[0, at // 64], :, at % 64]  # noqa: E731
    assert torch.equal(cell(cache, c + 1), cell(before, c + 3)) and torch.equal(cell(cache, c + 2), cell(before, c + 1023))
    assert all(torch.equal(cell(cache, c + j), cell(before, c + j)) for j in (0, 3, 4, 1023, 1024))


@pytest.mark.parametrize("window,softcap", [(0, 0.0), (40, 0.0), (0, 20.0)])
def test_the_attentions_restatement_of_a_chain_is_causal_attention(window, softcap):
    case, scale = attention_case([6, 1, 30], [50, 0, 77], hq=4, hkv=2, d=64, page=16, wide=1)
    got = draft_tree.ref_attention(scale=scale, window=window, softcap=softcap, **case)
    want = reference.paged_attention(case["q"].float(), case["kv_cache"], case["block_table"], case["seq_lens"], case["q_start"], 4, 2, 64, 16, scale,
                                     softcap, window)
    assert float((got - want).abs().max()) < 1e-4


@pytest.mark.parametrize("window", [1, 2, 7, 30, 31])
def test_the_attentions_restatement_of_a_chain_longer_than_its_window(window):
    """A window ends among the nodes too: causal attention in that window."""
    case, scale = attention_case([40, 1, 100], [50, 0, 0], hq=4, hkv=2, d=64, page=16, wide=1)
    got = draft_tree.ref_attention(scale=scale, window=window, **case)
    want = reference.paged_attention(case["q"].float(), case["kv_cache"], case["block_table"], case["seq_lens"], case["q_start"], 4, 2, 64, 16, scale, 0.0, window)
    assert float((got - want).abs().max()) < 1e-4


@pytest.mark.parametrize("window", [1, 2, 3, 20])
def test_the_attentions_restatement_of_a_path_in_a_window(window):
    """The last `window` of what its path, context and ancestors, holds."""
    case, scale = attention_case([60], [10], hq=2, hkv=1, d=64, page=16, wide=2, seed=4)
    got = draft_tree.ref_attention(scale=scale, dtype=torch.float64, window=window, **case)
    for node in (59, 31, 0):
        line = ([*range(10)] + [10 + j for j in range(60) if int(case["mask"][node, 0]) >> j & 1])[-window:]
        kv = case["kv_cache"][case["block_table"][0].long()].transpose(1, 2).reshape(-1, 2, 1, 64)[line].double()
        s = torch.einsum("hd,kd->hk", case["q"][node].view(2, 64).double(), kv[:, 0, 0]) * scale
        assert torch.allclose(got[node].view(2, 64), s.softmax(-1) @ kv[:, 1, 0], atol=1e-12)


def test_the_attentions_restatement_of_a_path_is_causal_attention_of_that_path():
    """A node of a tree sees what it would see if its ancestors stood alone behind the context."""
    case, scale = attention_case([17], [33], hq=2, hkv=1, d=64, page=16, wide=4, seed=4)
    got = draft_tree.ref_attention(scale=scale, dtype=torch.float64, **case)
    for node in (16, 9):
        line = [j for j in range(17) if int(case["mask"][node, 0]) >> j & 1]
        kv = case["kv_cache"][case["block_table"][0].long()].transpose(1, 2).reshape(-1, 2, 1, 64)
        cells = torch.cat([kv[:33], kv[[33 + j for j in line]]]).double()
        s = torch.einsum("hd,kd->hk", case["q"][node].view(2, 64).double(), cells[:, 0, 0]) * scale
        assert torch.allclose(got[node].view(2, 64), s.softmax(-1) @ cells[:, 1, 0], atol=1e-12)


def test_the_greedy_rule_is_the_greedy_rejection():
    gen = torch.Generator().manual_seed(1)
    sizes, V = [4, 1, 6, 3], 4
    logits = torch.randn((sum(sizes), V), generator=gen)
    tokens = torch.where(torch.rand(sum(sizes), generator=gen) < 0.7, logits.argmax(1).roll(1), torch.randint(0, V, (sum(sizes),), generator=gen))
    q_start = starts_of(sizes)
    drafts = torch.cat([tokens[int(a) + 1: int(b)] for a, b in zip(q_start, q_start[1:])])
    want = greedy_rejection_sample(logits.argmax(1), drafts, starts_of([n - 1 for n in sizes]), 5)
    got, path, count = draft_tree.ref_verify(logits, tokens, q_start=q_start, uniforms=torch.zeros(14), seeds=torch.zeros(4), steps=torch.zeros(4),
                                             max_tokens=6, temperature=torch.zeros(4))
    assert torch.equal(got, want) and count.tolist() == (want >= 0).sum(1).tolist()
    assert [p[:k] for p, k in zip(path.tolist(), count.tolist())] == [list(range(k)) for k in count.tolist()]


@pytest.mark.parametrize("drawn", [True, False])
def test_the_rule_keeps_the_targets_distribution(drawn):
    """Summed over what is drafted and integrated over the random numbers (each accepted or not, with its probability) the first
    token has the target's distribution: two children, all pairs of tokens."""
    gen = torch.Generator().manual_seed(5)
    p, q = (torch.softmax(torch.randn(4, generator=gen, dtype=torch.float64), 0) for _ in range(2))
    total = torch.zeros(4, dtype=torch.float64)
    for x in range(4):
        for y in range(4):
            if not drawn and (x, y) != (2, 0):
                continue
            weight, left = (q[x] * q[y], p.clone()) if drawn else (torch.ones(()).double(), p.clone())
            for t in (x, y):
                point = q if drawn else torch.eye(4, dtype=torch.float64)[t]
                a = min(1.0, float(left[t] / point[t]))
                total[t] += weight * a
                weight = weight * (1 - a)
                if weight <= 0:
                    break
                left = (left - point).clamp(min=0)
                left /= left.sum()
            total += weight * left
    assert torch.allclose(total, p, atol=1e-12)


@pytest.mark.parametrize("drawn", [True, False])
def test_the_rules_restatement_keeps_the_targets_distribution(drawn):
    """Two children of a root, all pairs of tokens: what each is accepted with is looked for among the random numbers (numbers below a border accept), and
    what is drawn after both are refused is the residual's draw. Summed over what is drafted, the first token has the target's distribution."""
    gen = torch.Generator().manual_seed(5)
    logits = torch.randn(4, generator=gen)
    p, q = torch.softmax(logits.double(), 0), torch.softmax(torch.randn(4, generator=gen).double(), 0)
    ids = torch.arange(40)

    def said(x, y, u, v):
        """The first tokens of 40 requests with these children and numbers: (accepted node or -1, token)."""
        n = len(ids)
        out, path, count = draft_tree.ref_verify(
            logits.expand(3 * n, 4), torch.tensor([0, x, y] * n), q_start=starts_of([3] * n), uniforms=torch.tensor([0.0, u, v] * n), seeds=ids, steps=ids * 7,
            max_tokens=2, parents=torch.tensor([-1, 0, 0] * n, dtype=torch.int32), draft_probs=q.float().expand(3 * n, 4) if drawn else None)
        return [(int(a[1]) if int(c) == 2 else -1, int(t[0])) for a, c, t in zip(path, count, out)]

    def border(accepts):
        low, high = 0.0, 1.0                                     # (numbers stay below one)
        for _ in range(22):
            mid = (low + high) / 2
            low, high = (mid, high) if accepts(mid) else (low, mid)
        return low
    ids, many = ids[:1], ids
    total, most = torch.zeros(4, dtype=torch.float64), 1 - 2.0 ** -23
    for x in range(4):
        for y in range(4):
            if not drawn and (x, y) != (2, 0):
                continue
            ids = many[:1]
            weight = q[x] * q[y] if drawn else 1.0
            first = border(lambda u: said(x, y, u, most)[0][0] == 1)
            total[x] += weight * first
            if first >= 1 - 2.0 ** -21:
                continue
            second = border(lambda v: said(x, y, most, v)[0][0] == 2)
            total[y] += weight * (1 - first) * second
            left = p.clone()
            for t in (x, y):
                left = (left - (q if drawn else torch.eye(4, dtype=torch.float64)[t])).clamp(min=0)
                left /= left.sum()
            total += weight * (1 - first) * (1 - second) * left
            if second < 1 - 2.0 ** -21:
                ids = many
                want = [int((left / draft_tree.race_numbers(i, 7 * i, 4)).argmax()) for i in range(len(many))]
                assert said(x, y, most, most) == [(-1, t) for t in want]
    assert torch.allclose(total, p, atol=2.0 ** -19)             # (borders to 2^-22, q in 32 bits)


def test_the_draw_of_the_rule_is_the_samplers():
    p = torch.softmax(torch.randn(300, generator=torch.Generator().manual_seed(2)) * 2, 0)
    for seed, step in ((3, 0), (2 ** 63 + 5, 77)):
        assert int((p.double() / draft_tree.race_numbers(seed, step, 300)).argmax()) == reference.race_sample(p, seed, step)


def test_the_compactions_restatement_reads_before_it_writes():
    table, pages = page_table([12], 4, torch.Generator().manual_seed(1))
    cache = torch.arange(pages * 2 * 4 * 8).view(pages, 2, 4, 1, 8).to(torch.float32)
    before = cache.clone()
    draft_tree.ref_compact(cache, block_table=table, seq_lens=torch.tensor([12]), q_start=starts_of([7]), path=torch.tensor([[0, 2, 3, 6, -1]]))
    cell = lambda c, at: c[table[0, at // 4], :, at % 4]  # noqa: E731
    for i, node in ((1, 2), (2, 3), (3, 6)):
        assert torch.equal(cell(cache, 5 + i), cell(before, 5 + node))
    assert torch.equal(cell(cache, 5), cell(before, 5)) and torch.equal(cell(cache, 9), cell(before, 9))


# ------------------------------------------------------------------------------------------------ refusals
def attention_args():
    case, scale = attention_case([5, 3], [10, 4], hq=4, hkv=2, d=64, page=16)
    return dict(case, scale=scale)


@pytest.mark.parametrize("what,change", [
    ("head_dim", lambda a: a.update(kv_cache=a["kv_cache"][..., :32].contiguous(), q=a["q"][:, :128].contiguous())),
    ("kv_cache is bf16", lambda a: a.update(kv_cache=a["kv_cache"].float())),
    ("kv_cache is bf16", lambda a: a.update(kv_cache=a["kv_cache"].transpose(2, 3))),
    ("q is", lambda a: a.update(q=a["q"].half())),
    ("q is", lambda a: a.update(q=a["q"][:, :192])),
    ("q is", lambda a: a.update(q=torch.zeros((8, 260), dtype=torch.bfloat16)[:, 4:])),
    ("q_start", lambda a: a.update(q_start=a["q_start"].long())),
    ("seq_lens", lambda a: a.update(seq_lens=a["seq_lens"][:1])),
    ("block_table", lambda a: a.update(block_table=a["block_table"][:1])),
    ("block_table", lambda a: a.update(block_table=a["block_table"].long())),
    ("mask is", lambda a: a.update(mask=a["mask"][:5])),
    ("mask is", lambda a: a.update(mask=a["mask"].int())),
    ("at most 16 words", lambda a: a.update(mask=torch.zeros((8, 17), dtype=torch.int64))),
    ("at most 128 query heads", lambda a: a.update(q=torch.zeros((8, 2 * 129 * 64), dtype=torch.bfloat16))),
    ("at most 8192 requests", lambda a: a.update(q_start=torch.zeros(8194, dtype=torch.int32), seq_lens=torch.zeros(8193, dtype=torch.int32),
                                                 block_table=torch.zeros((8193, 1), dtype=torch.int32))),
    ("block_size divides", lambda a: a.update(kv_cache=torch.zeros((3, 2, 48, 2, 64), dtype=torch.bfloat16))),
    ("block_size divides", lambda a: a.update(kv_cache=torch.zeros((3, 2, 4, 2, 64), dtype=torch.bfloat16))),
    ("kv_cache is bf16", lambda a: a.update(kv_cache=torch.zeros((3, 2, 0, 2, 64), dtype=torch.bfloat16))),
    ("kv_cache is bf16", lambda a: a.update(kv_cache=torch.zeros((3, 2, 16, 0, 64), dtype=torch.bfloat16))),
    ("kv_cache is bf16", lambda a: a.update(kv_cache=torch.zeros((3, 2, 16, 2, 0), dtype=torch.bfloat16))),
    ("one GPU", lambda a: a.update(tmp=torch.zeros(10))),
    ("scale", lambda a: a.update(scale=0.0)),
    ("scale", lambda a: a.update(scale=math.inf)),
    ("softcap", lambda a: a.update(softcap=-1.0)),
    ("window", lambda a: a.update(window=-128)),
    ("window", lambda a: a.update(window=16, positions=None)),
    ("out is", lambda a: a.update(out=a["q"])),
    ("out is", lambda a: a.update(out=torch.zeros((8, 128), dtype=torch.bfloat16))),
    ("out is", lambda a: a.update(out=torch.zeros((1, 256), dtype=torch.bfloat16).expand(8, 256))),
    ("tmp", lambda a: a.update(tmp=torch.zeros(7, dtype=torch.int32))),
    ("one GPU", lambda a: None),
])
def test_attention_refuses(what, change):
    args = attention_args()
    change(args)
    with pytest.raises(OpArgumentError, match=what):
        draft_tree.attention(**args)


@pytest.mark.parametrize("name", ["scale", "softcap"])
@pytest.mark.parametrize("value", [1e-50, 2.0 ** -150, 2.36e38, 1e39, 1e300, math.nan])
def test_attention_refuses_numbers_that_32_bits_do_not_hold(name, value):
    """Below half the least number of 32 bits a cap would be none and a scale 0; above 2.35e38 they overflow in log2 units."""
    with pytest.raises(OpArgumentError, match=f"{name} is|softcap not"):
        draft_tree.attention(**{**attention_args(), name: value})


def mask_args():
    return dict(parents=torch.tensor([-1, 0, 1], dtype=torch.int32), q_start=starts_of([3]), seq_lens=torch.tensor([7], dtype=torch.int32))


@pytest.mark.parametrize("what,change", [
    ("parents", lambda a: a.update(parents=a["parents"].long())),
    ("q_start", lambda a: a.update(q_start=a["q_start"].view(1, 2))),
    ("seq_lens", lambda a: a.update(seq_lens=a["seq_lens"][:0])),
    ("max_nodes", lambda a: a.update(max_nodes=0)),
    ("max_nodes", lambda a: a.update(max_nodes=1025)),
    ("max_nodes", lambda a: a.update(max_nodes=None)),
    ("bits", lambda a: a.update(bits=torch.zeros((3, 2), dtype=torch.int64))),
    ("positions", lambda a: a.update(positions=torch.zeros(3, dtype=torch.int32))),
    ("apart", lambda a: a.update(bits=(b := torch.zeros((3, 1), dtype=torch.int64)), positions=b[:, 0])),
    ("one GPU", lambda a: None),
])
def test_mask_refuses(what, change):
    args = mask_args()
    change(args)
    with pytest.raises(OpArgumentError, match=what):
        draft_tree.mask(**args)


def verify_args():
    return dict(logits=torch.zeros((3, 9)), tokens=torch.zeros(3, dtype=torch.int64), q_start=starts_of([3]), uniforms=torch.zeros(3),
                seeds=torch.zeros(1, dtype=torch.int64), steps=torch.zeros(1, dtype=torch.int64), max_tokens=3)


@pytest.mark.parametrize("what,change", [
    ("logits", lambda a: a.update(logits=a["logits"].bfloat16())),
    ("logits", lambda a: a.update(logits=torch.zeros((9, 3)).t())),
    ("778000 columns", lambda a: a.update(logits=torch.zeros((3, 778001)))),
    ("tokens", lambda a: a.update(tokens=a["tokens"].int())),
    ("uniforms", lambda a: a.update(uniforms=a["uniforms"][:2])),
    ("q_start", lambda a: a.update(q_start=a["q_start"].long())),
    ("seeds", lambda a: a.update(seeds=a["seeds"].int())),
    ("temperature", lambda a: a.update(temperature=torch.zeros(0))),
    ("parents", lambda a: a.update(parents=torch.zeros(2, dtype=torch.int32))),
    ("draft_probs", lambda a: a.update(draft_probs=torch.zeros((2, 9)))),
    ("draft_probs", lambda a: a.update(draft_probs=torch.zeros((3, 9), dtype=torch.float64))),
    ("max_tokens", lambda a: a.update(max_tokens=0)),
    ("one GPU", lambda a: None),
])
def test_verify_refuses(what, change):
    args = verify_args()
    change(args)
    with pytest.raises(OpArgumentError, match=what):
        draft_tree.verify(**args)


def compact_args():
    return dict(kv_caches=[torch.zeros((4, 2, 16, 1, 64), dtype=torch.bfloat16) for _ in range(2)], block_table=torch.zeros((1, 3), dtype=torch.int32),
                seq_lens=torch.tensor([20], dtype=torch.int32), q_start=starts_of([5]), path=torch.zeros((1, 3), dtype=torch.int32))


@pytest.mark.parametrize("what,change", [
    ("there is a cache", lambda a: a.update(kv_caches=[])),
    ("alike", lambda a: a["kv_caches"].append(torch.zeros((4, 2, 16, 1, 64)))),
    ("alike", lambda a: a["kv_caches"].append(torch.zeros((4, 2, 16, 2, 64), dtype=torch.bfloat16))),
    ("16-byte", lambda a: a.update(kv_caches=[torch.zeros((4, 2, 16, 1, 4), dtype=torch.bfloat16)])),
    ("alike", lambda a: a.update(kv_caches=[torch.zeros((4, 2, 3, 16, 64), dtype=torch.bfloat16).transpose(2, 3)])),
    ("twice", lambda a: a["kv_caches"].append(a["kv_caches"][0])),
    ("share no memory", lambda a: a.update(kv_caches=[(b := torch.zeros((7, 2, 16, 1, 64), dtype=torch.bfloat16))[3:], b[:4]])),
    ("seq_lens", lambda a: a.update(seq_lens=a["seq_lens"].long())),
    ("block_table", lambda a: a.update(block_table=a["block_table"].t())),
    ("path", lambda a: a.update(path=torch.zeros((2, 3), dtype=torch.int32))),
    ("path", lambda a: a.update(path=a["path"].long())),
    ("one GPU", lambda a: None),
])
def test_compact_refuses(what, change):
    args = compact_args()
    change(args)
    with pytest.raises(OpArgumentError, match=what):
        draft_tree.compact(**args)


def test_sizes_that_the_attention_takes():
    if not _lib.available():
        pytest.skip("kernel library not built")
    draft_tree._declare()

    def takes(**more):
        a = draft_tree.AttnArgs()
        for k, v in dict(dict(D=128, Hq=32, Hkv=8, block_size=32, max_blocks=4000, num_blocks=100000, num_reqs=64, total_q=2048, words=1), **more).items():
            setattr(a, k, v)
        return _lib.lib().b200_tree_attn_takes(ctypes.byref(a))
    assert takes() == 0 and takes(block_size=192) == 0 and takes(words=16, total_q=65536, num_reqs=8192) == 0 and takes(D=256, block_size=64) == 0
    for wrong in (dict(D=96), dict(Hq=30), dict(Hq=129, Hkv=1), dict(block_size=12), dict(block_size=48), dict(block_size=4), dict(words=0),
                  dict(D=256, block_size=96), dict(block_size=72)):
        assert takes(**wrong) == -1, wrong
    for large in (dict(words=17), dict(num_reqs=8193), dict(num_blocks=2 ** 25), dict(max_blocks=2 ** 26), dict(max_blocks=2 ** 25, words=16, total_q=2048)):
        assert takes(**large) == -4, large
