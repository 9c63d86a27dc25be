"""Drafted trees on a GPU: masks, attention against its definition in 64 bits, verification against the rule in 64 bits, compaction, and a
run of them together."""
import math
import random

import pytest
import torch

from draft_tree_cases import attention_bound, attention_case, page_table, starts_of, tree_parents
from vllm_cpp_b200 import ops
from vllm_cpp_b200.ops import draft_tree
from vllm_cpp_b200.ops.validate import OpArgumentError

pytestmark = pytest.mark.gpu
DEV = "cuda"


# ------------------------------------------------------------------------------------------------ mask
@pytest.mark.parametrize("sizes,most", [([1], 64), ([60], 64), ([64, 1, 0, 7], 64), ([65, 3], 128), ([200, 130, 1], 256), ([1024, 5], 1024), ([70], 64)])
@pytest.mark.parametrize("wide", [1, 4])
def test_masks_are_the_ancestors(sizes, most, wide):
    rng = random.Random(len(sizes) + wide)
    parents = torch.tensor([p for n in sizes for p in tree_parents(n, rng, wide)], dtype=torch.int32)
    q_start, lens = starts_of(sizes), torch.tensor([n + 13 * i for i, n in enumerate(sizes)], dtype=torch.int32)
    want = draft_tree.ref_mask(parents, q_start=q_start, seq_lens=lens, max_nodes=most)
    got = draft_tree.mask(parents.to(DEV), q_start=q_start.to(DEV), seq_lens=lens.to(DEV), max_nodes=most)
    assert all(torch.equal(g.cpu(), w) for g, w in zip(got, want))


def test_masks_of_odd_parents_and_rows_behind():
    """Parents that do not lie below their node are roots; rows of no request stay as they are."""
    parents = torch.tensor([5, 0, 2, 1, -7, 4, 99, 3, 0, 0], dtype=torch.int32, device=DEV)
    q_start, lens = torch.tensor([0, 8], dtype=torch.int32, device=DEV), torch.tensor([20], dtype=torch.int32, device=DEV)
    bits = torch.full((10, 1), 77, dtype=torch.int64, device=DEV)
    positions = torch.full((10,), 78, dtype=torch.int64, device=DEV)
    draft_tree.mask(parents, q_start=q_start, seq_lens=lens, bits=bits, positions=positions)
    assert bits[:, 0].tolist() == [1, 3, 4, 8 | 3, 16, 32 | 16, 64, 128 | 8 | 3, 77, 77]
    assert positions.tolist() == [12, 13, 12, 14, 12, 13, 12, 15, 78, 78]


# ------------------------------------------------------------------------------------------------ attention
def run_attention(case, scale, **more):
    T, cols = case["q"].shape
    out = torch.full((T, cols), 7.0, dtype=torch.bfloat16, device=DEV)
    got = draft_tree.attention(scale=scale, out=out, **case, **more)
    torch.cuda.synchronize()
    assert ops.read_status() == 0
    return got


def check_attention(case, scale, **more):
    got = run_attention(case, scale, **more)
    want, bound = attention_bound(case, scale, **more)
    rows = int(case["q_start"][-1])
    off = (got.double() - want).abs()[:rows]
    assert torch.isfinite(got[:rows].float()).all()
    assert bool((off <= bound[:rows]).all()), f"{float((off / bound[:rows]).max()):.2f} times the bound"
    assert bool((got[rows:] == 7).all())
    return got


SHAPES = [(4, 4, 64), (8, 2, 64), (6, 2, 128), (32, 8, 128), (16, 1, 128), (5, 1, 128), (8, 8, 128), (12, 1, 128), (8, 4, 256), (16, 2, 256), (3, 1, 256)]


@pytest.mark.parametrize("hq,hkv,d", SHAPES)
@pytest.mark.parametrize("sizes,contexts", [([1], [0]), ([1], [1]), ([7], [120]), ([5, 1, 0, 33], [0, 300, 50, 128]), ([16, 64, 3], [1000, 127, 2049])])
def test_attention_of_small_steps(hq, hkv, d, sizes, contexts):
    case, scale = attention_case(sizes, contexts, hq=hq, hkv=hkv, d=d, page=16, seed=hq + d, device=DEV)
    check_attention(case, scale)


@pytest.mark.parametrize("page", [8, 16, 32, 64, 128, 256])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_attention_over_pages_of_every_size(page, d):
    case, scale = attention_case([9, 30, 2], [77, 513, 1500], hq=8, hkv=2, d=d, page=page, seed=page, device=DEV)
    check_attention(case, scale)


@pytest.mark.parametrize("n", [31, 32, 33, 64, 65, 100, 129, 257])
@pytest.mark.parametrize("d", [128, 256])
def test_attention_of_large_trees(n, d):
    case, scale = attention_case([n, 4], [700, 60], hq=8, hkv=2, d=d, page=32, seed=n, wide=3, device=DEV)
    check_attention(case, scale)


def test_attention_of_the_largest_tree():
    case, scale = attention_case([1024], [300], hq=2, hkv=1, d=64, page=64, seed=1, device=DEV)
    check_attention(case, scale)


@pytest.mark.parametrize("context", [20000, 70001])
@pytest.mark.parametrize("n", [3, 61])
def test_attention_over_long_contexts(context, n):
    case, scale = attention_case([n], [context], hq=8, hkv=2, d=128, page=64, seed=n, device=DEV)
    check_attention(case, scale)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("window", [1, 5, 128, 300, 5000])
def test_attention_in_a_window(d, window):
    case, scale = attention_case([9, 40, 1, 17], [77, 900, 3000, 0], hq=6, hkv=2, d=d, page=16, seed=window, wide=1, device=DEV)
    check_attention(case, scale, window=window)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("window", [1, 2, 3, 8, 63, 130])
def test_attention_in_a_window_that_ends_among_the_nodes(d, window):
    """Trees and chains deeper than the window, capped and not; also where rows of no tree lie between them."""
    for wide, sizes in ((1, [9, 200, 1, 70]), (2, [64, 0, 300, 33])):
        case, scale = attention_case(sizes, [77, 20, 0, 500], hq=6, hkv=2, d=d, page=16, seed=window, wide=wide, device=DEV)
        check_attention(case, scale, window=window)
        check_attention(case, scale, window=window, softcap=20.0)


@pytest.mark.parametrize("window", [1, 3, 40])
def test_attention_in_a_window_of_lengths_below_the_nodes(window):
    """The first nodes have no cells; positions run from before the cache's first one."""
    for wide in (1, 2):
        case, scale = attention_case([70, 9, 100], [0, 5, 30], hq=6, hkv=2, d=128, page=16, seed=3, wide=wide, device=DEV)
        case["seq_lens"] -= 12
        case["positions"] -= 12
        check_attention(case, scale, window=window)


@pytest.mark.parametrize("window", [5, 64, 200, 1000])
def test_attention_of_chains_in_a_window_is_the_prefill_kernels(window):
    """Chains longer than a window, a prompt's among them: what attn_prefill computes, within both kernels' roundings."""
    sizes, contexts = [1000, 3, 130, 70], [0, 77, 1200, 3]
    case, scale = attention_case(sizes, contexts, hq=8, hkv=2, d=128, page=16, wide=1, device=DEV)
    got = run_attention(case, scale, window=window)
    req, q0 = ops_tiles(sizes)
    other = ops.attn_prefill(case["q"].contiguous(), case["kv_cache"], block_table=case["block_table"], seq_lens=case["seq_lens"], q_start=case["q_start"],
                             tile_req=req, tile_q0=q0, num_q_heads=8, num_kv_heads=2, head_dim=128, block_size=16, scale=scale, window=window)
    _, bound = attention_bound(case, scale, window=window)
    assert bool(((got.double() - other.double()).abs() <= 2 * bound).all())


@pytest.mark.parametrize("d", [64, 128, 256])
def test_attention_keeps_out_nodes_before_a_window(d):
    """NaN in an ancestor reaches the nodes below it that lie less than a window behind it, and no other."""
    case, scale = attention_case([100], [40], hq=8, hkv=2, d=d, page=16, seed=d, wide=2, device=DEV)
    clean = run_attention(case, scale, window=6).clone()
    node = max((case["positions"] == 45).nonzero().flatten().tolist(), key=lambda j: int((case["mask"][:, j // 64] >> (j % 64) & 1).sum()))
    bad = dict(case, kv_cache=case["kv_cache"].clone())
    bad["kv_cache"][int(case["block_table"][0, (40 + node) // 16]), :, (40 + node) % 16] = math.nan
    got = run_attention(bad, scale, window=6)
    below = (case["mask"][:, node // 64] >> (node % 64) & 1).bool()
    reached = below & (case["positions"] < 45 + 6)
    assert bool((below & ~reached).any()) and torch.equal(got[~reached], clean[~reached]) and bool(got[reached].isnan().all())


@pytest.mark.parametrize("window", [400, 2 ** 31 - 1])
def test_attention_in_a_window_that_holds_everything(window):
    """Lengths that are shorter than the request's nodes too."""
    case, scale = attention_case([70, 9, 100], [0, 250, 30], hq=6, hkv=2, d=128, page=16, seed=3, wide=2, device=DEV)
    for cut in (0, 5):
        case["seq_lens"] -= cut
        assert torch.equal(run_attention(case, scale, window=window), run_attention({**case}, scale))


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("softcap", [1e-38, 0.5, 30.0, 170.0, 200.0, 20000.0, 1e30])
@pytest.mark.parametrize("n", [40, 70])
def test_attention_with_capped_scores(d, softcap, n):
    case, scale = attention_case([9, n], [77, 900], hq=6, hkv=2, d=d, page=16, seed=3, device=DEV)
    check_attention(case, scale, softcap=softcap)
    check_attention(case, scale, softcap=softcap, window=200)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("softcap", [200.0, 1000.0, 20000.0, 1e30])
def test_attention_with_caps_far_above_the_scores(d, softcap):
    """A capped score is off by 2^-21 of its cap from a sixteenth of it on, and by some roundings of itself below: 2^-16 of the largest score either way. It counts twice
    in a weight (the sum too); the rest is what uncapped scores are off by."""
    case, scale = attention_case([9, 70], [77, 900], hq=6, hkv=2, d=d, page=16, seed=3, device=DEV)
    got = run_attention(case, scale, softcap=softcap).double()
    wide = {k: v.double() if v.dtype == torch.bfloat16 else v for k, v in case.items()}
    want = draft_tree.ref_attention(scale=scale, softcap=softcap, dtype=torch.float64, **wide)
    values = draft_tree.ref_attention(scale=scale, softcap=softcap, dtype=torch.float64, **dict(wide, kv_cache=torch.stack(
        [wide["kv_cache"][:, 0], wide["kv_cache"][:, 1].abs()], 1)))
    _, bound = attention_bound(case, scale)
    top = float(wide["q"].reshape(-1, d).norm(dim=1).max()) * float(wide["kv_cache"][:, 0].norm(dim=-1).max()) * scale
    assert bool(((got - want).abs() <= bound + 2 * 2.0 ** -16 * top * values).all())


@pytest.mark.parametrize("group", [17, 20, 33, 64, 65, 100, 127, 128])
def test_attention_of_many_query_heads_a_kv_head(group):
    for d, hkv in ((64, 2), (128, 1), (256, 1)):
        case, scale = attention_case([9, 0, 3, 1], [77, 5, 900, 0], hq=group * hkv, hkv=hkv, d=d, page=32, seed=group, device=DEV)
        check_attention(case, scale)
        check_attention(case, scale, window=50, softcap=25.0)


def test_attention_of_as_many_requests_as_a_call_takes():
    """8192 requests: 128 of them again and again."""
    rng = random.Random(6)
    sizes = [rng.randrange(0, 5) for _ in range(128)]
    case, scale = attention_case(sizes, [rng.randrange(0, 200) for _ in sizes], hq=4, hkv=2, d=64, page=16, seed=6, device=DEV)
    want, bound = attention_bound(case, scale)
    many = dict(case, **{k: case[k].repeat(64, *[1] * (case[k].dim() - 1)) for k in ("q", "block_table", "seq_lens", "mask", "positions")},
                q_start=starts_of(sizes * 64, DEV))
    got = run_attention(many, scale).double().view(64, *want.shape)
    assert bool(((got - want).abs() <= bound).all())


def test_attention_of_many_requests():
    rng = random.Random(5)
    sizes = [rng.randrange(0, 12) for _ in range(700)]
    case, scale = attention_case(sizes, [rng.randrange(0, 60) for _ in sizes], hq=4, hkv=2, d=64, page=16, seed=5, device=DEV)
    check_attention(case, scale)


def test_attention_of_rows_with_a_stride_and_rows_behind():
    case, scale = attention_case([9, 40], [77, 900], hq=8, hkv=2, d=128, page=16, seed=3, stride=512, pad=5, device=DEV)
    check_attention(case, scale)


def test_attention_of_nodes_that_see_nothing():
    """Nodes without a bit: the context alone, and zeros where there is none; bits past the request's nodes say nothing."""
    case, scale = attention_case([20, 9, 12], [300, 0, 0], hq=8, hkv=2, d=128, page=16, seed=3, device=DEV)
    case["mask"][::2] = 0
    case["mask"][21] = -1
    case["mask"][30] = -1
    got = check_attention(case, scale)
    nothing = [i for i in range(20, 41) if i % 2 == 0 and i != 30]
    assert bool((got[nothing] == 0).all()) and bool((got[:20] != 0).any(1).all())


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("contexts", [[100, 0], [700, 5], [40000, 300]])
def test_attention_keeps_what_is_hidden_out(d, contexts):
    """Infinities and NaN among keys and values that a node does not see (siblings, cells behind the request, keys before the window)
    leave its outputs as they are, bit for bit; nodes that see a value of infinity get it, in that dimension alone."""
    sizes = [24, 40]
    case, scale = attention_case(sizes, contexts, hq=8, hkv=2, d=d, page=16, seed=d, wide=5, device=DEV)
    clean = run_attention(case, scale).clone()
    from vllm_cpp_b200.ops.draft_tree import seen_by
    seen = seen_by(case["mask"], q_start=case["q_start"], seq_lens=case["seq_lens"])
    for r, (n, c) in enumerate(zip(sizes, contexts)):
        bad = dict(case, kv_cache=case["kv_cache"].clone())

        def cell(position):
            return bad["kv_cache"][int(case["block_table"][r, position // 16]), :, position % 16]
        node = n - 2
        cell(c + node)[0] = math.nan
        cell(c + node)[1, :, :] = math.nan
        for tail in range(n + c, -(-(n + c) // 16) * 16):
            cell(tail)[:] = math.nan
        bad["kv_cache"][0] = math.inf
        got = run_attention(bad, scale)
        first = int(case["q_start"][r])
        reached = torch.zeros(sum(sizes), dtype=torch.bool, device=DEV)
        reached[first: first + n] = seen[r][:, c + node]
        assert torch.equal(got[~reached], clean[~reached]) and bool(got[reached].isnan().all())
        bad = dict(case, kv_cache=case["kv_cache"].clone())
        cell(c + node)[1, 1, 3] = math.inf
        cell(c + node)[1, 0, d - 1] = -math.inf
        got = run_attention(bad, scale).view(-1, 8, d)
        want = clean.clone().view(-1, 8, d)
        want[reached, 4:, 3] = math.inf
        want[reached, :4, d - 1] = -math.inf
        assert torch.equal(got, want)


@pytest.mark.parametrize("d", [64, 128, 256])
def test_attention_keeps_out_what_lies_before_a_window(d):
    case, scale = attention_case([30], [900], hq=8, hkv=2, d=d, page=16, seed=d, wide=1, device=DEV)
    clean = run_attention(case, scale, window=400).clone()
    low = case["positions"] - 400                        # the last position that a node does not see
    bad = dict(case, kv_cache=case["kv_cache"].clone())
    key = int(low[10])
    bad["kv_cache"][int(case["block_table"][0, key // 16]), :, key % 16] = math.nan
    got = run_attention(bad, scale, window=400)
    reached = low < key
    assert int(reached.sum()) == 10 and torch.equal(got[~reached], clean[~reached]) and bool(got[reached].isnan().all())


def test_attention_of_keys_that_are_not_finite():
    """A NaN among a seen key's dims reaches the rows that see it; one that is hidden does not, capped or not."""
    case, scale = attention_case([12], [100], hq=8, hkv=2, d=128, page=16, seed=1, wide=3, device=DEV)
    from vllm_cpp_b200.ops.draft_tree import seen_by
    seen = seen_by(case["mask"], q_start=case["q_start"], seq_lens=case["seq_lens"])[0]
    for softcap in (0.0, 30.0):
        clean = run_attention(case, scale, softcap=softcap).clone()
        for value in (math.nan, math.inf):
            bad = dict(case, kv_cache=case["kv_cache"].clone())
            bad["kv_cache"][int(case["block_table"][0, 110 // 16]), 0, 110 % 16] = value
            got = run_attention(bad, scale, softcap=softcap)
            assert torch.equal(got[~seen[:, 110]], clean[~seen[:, 110]])
            if math.isnan(value):
                assert bool(got[seen[:, 110]].isnan().all())


def test_attention_of_nothing_and_of_short_lengths():
    """Steps without rows or requests; lengths below a request's nodes, whose first cells lie before the cache's first: nobody sees them."""
    case, scale = attention_case([12, 3], [100, 7], hq=8, hkv=2, d=128, page=16, seed=1, device=DEV)
    assert run_attention(dict(case, q=case["q"][:0]), scale).shape == (0, 1024)
    none = dict(case, q_start=case["q_start"][:1])
    assert bool((run_attention(none, scale) == 7).all())
    case["seq_lens"] = torch.tensor([5, 0], dtype=torch.int32, device=DEV)
    got = run_attention(case, scale)
    kv = case["kv_cache"][int(case["block_table"][0, 0])].double()
    for node in range(12):
        cells = [j - 7 for j in range(7, 12) if int(case["mask"][node, 0]) >> j & 1]
        want = torch.zeros((8, 128), dtype=torch.float64, device=DEV)
        if cells:
            k, v = (kv[i, cells].repeat_interleave(4, 1) for i in (0, 1))
            p = (torch.einsum("hd,khd->hk", case["q"][node].view(8, 128).double(), k) * scale).softmax(-1)
            want = torch.einsum("hk,khd->hd", p, v)
        # (weights and output rounded to bf16, 2^-8 of the largest value each, and as much again for scores in 32 bits)
        assert float((got[node].view(8, 128).double() - want).abs().max()) <= 3 * 2.0 ** -8 * float(kv[1].abs().max())
    assert bool((got[12:] == 0).all())


def test_attention_over_pages_outside_the_cache():
    """They count as keys and values of zeros, and nothing else is read."""
    case, scale = attention_case([9], [300], hq=8, hkv=2, d=128, page=16, seed=3, device=DEV)
    for entry in (-1, case["kv_cache"].shape[0], 2 ** 31 - 1, -2 ** 31):
        bad = dict(case, block_table=case["block_table"].clone())
        bad["block_table"][0, 3] = entry
        zeros = dict(case, kv_cache=case["kv_cache"].clone())
        zeros["kv_cache"][int(case["block_table"][0, 3])] = 0
        assert torch.equal(run_attention(bad, scale), run_attention(zeros, scale))


def test_attention_of_chains_is_the_prefill_kernels():
    """A chain is causal attention: what attn_prefill computes, within both kernels' roundings."""
    sizes, contexts = [6, 3, 40], [500, 77, 1200]
    case, scale = attention_case(sizes, contexts, hq=32, hkv=8, d=128, page=16, wide=1, device=DEV)
    got = run_attention(case, scale)
    req, q0 = ops_tiles(sizes)
    other = ops.attn_prefill(case["q"].contiguous(), case["kv_cache"], block_table=case["block_table"], seq_lens=case["seq_lens"], q_start=case["q_start"],
                             tile_req=req, tile_q0=q0, num_q_heads=32, num_kv_heads=8, head_dim=128, block_size=16, scale=scale)
    _, bound = attention_bound(case, scale)
    assert bool(((got.double() - other.double()).abs() <= 2 * bound).all())


def test_cells_past_32_bits():
    """Pages at the end of a cache of 2.6 G values: the same bits as at the beginning of a small one, values that are not finite included; moves too."""
    case, scale = attention_case([9, 40], [300, 900], hq=16, hkv=8, d=128, page=256, seed=5, device=DEV)
    small = case["kv_cache"]
    end = int(case["seq_lens"][0]) - 1                           # (the last node, which the others do not see)
    small[case["block_table"][0, end // 256].long(), 1, end % 256, :, 3] = math.inf
    large = torch.empty((5000, *small.shape[1:]), dtype=torch.bfloat16, device=DEV)
    large[-len(small):] = small
    there = dict(case, kv_cache=large, block_table=case["block_table"] + (5000 - len(small)))
    want = run_attention(case, scale)
    assert torch.equal(run_attention(there, scale).view(torch.int16), want.view(torch.int16)) and bool(torch.isinf(want).any())
    path = torch.tensor([[0, 2, 5, 8, -1], [0, 7, 8, 30, 39]], dtype=torch.int32, device=DEV)
    for c in (case, there):
        draft_tree.compact(c["kv_cache"], block_table=c["block_table"], seq_lens=c["seq_lens"], q_start=c["q_start"], path=path)
    assert torch.equal(large[-len(small):].view(torch.int16), small.view(torch.int16))


def test_cells_past_32_bits_of_values_and_31_of_pieces():
    """Pages at the end of a cache of 19 G values, which are 2.4 G pieces of 16 bytes: attention (a value that is not finite is read again by its address) and moves."""
    case, scale = attention_case([9, 40], [300, 900], hq=16, hkv=8, d=128, page=256, seed=5, device=DEV)
    small = case["kv_cache"]
    if torch.cuda.mem_get_info()[1] < 80 << 30:
        pytest.skip("a cache of 38 GB")
    end = int(case["seq_lens"][0]) - 1
    small[case["block_table"][0, end // 256].long(), 1, end % 256, :, 3] = math.inf
    large = torch.empty((36500, *small.shape[1:]), dtype=torch.bfloat16, device=DEV)
    large[-len(small):] = small
    there = dict(case, kv_cache=large, block_table=case["block_table"] + (36500 - len(small)))
    want = run_attention(case, scale)
    assert torch.equal(run_attention(there, scale).view(torch.int16), want.view(torch.int16)) and bool(torch.isinf(want).any())
    path = torch.tensor([[0, 2, 5, 8, -1], [0, 7, 8, 30, 39]], dtype=torch.int32, device=DEV)
    for c in (case, there):
        draft_tree.compact(c["kv_cache"], block_table=c["block_table"], seq_lens=c["seq_lens"], q_start=c["q_start"], path=path)
    assert torch.equal(large[-len(small):].view(torch.int16), small.view(torch.int16))


def ops_tiles(sizes):
    from vllm_cpp_b200.ops.reference import build_prefill_tiles
    req, q0 = build_prefill_tiles(sizes)
    return torch.tensor(req, dtype=torch.int32, device=DEV), torch.tensor(q0, dtype=torch.int32, device=DEV)


def test_attention_gives_the_same_bits_in_streams_and_graphs():
    case, scale = attention_case([9, 40, 3], [77, 9000, 200], hq=8, hkv=2, d=128, page=16, seed=3, device=DEV)
    want = run_attention(case, scale).clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = draft_tree.attention(scale=scale, **case)
    side.synchronize()
    assert torch.equal(got, want)
    # two graphs, each with its own scratch, replayed side by side; lengths change between replays
    # (the scratch lives as long as its graph: a capture's beginning gives memory that nobody holds back to the device)
    tmps = [draft_tree.scratch(torch.device(DEV, 0), 128) for _ in range(2)]
    graphs, outs = [], [torch.empty_like(want) for _ in range(2)]
    for tmp, out in zip(tmps, outs):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            draft_tree.attention(scale=scale, out=out, tmp=tmp, **case)
        graphs.append(g)
    case["seq_lens"][1] -= 3000
    want = run_attention(case, scale).clone()
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(5):
        for g, s in zip(graphs, streams):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, want) for o in outs)


def test_attention_refuses_on_the_gpu_too():
    """Refusals by the short checks of a call whose tensors are all on the GPU: nothing is launched."""
    case, scale = attention_case([5, 3], [10, 4], hq=4, hkv=2, d=64, page=16, device=DEV)
    zero = lambda *s, dtype=torch.bfloat16: torch.zeros(s, dtype=dtype, device=DEV)  # noqa: E731
    for what, change in (("bf16", dict(kv_cache=zero(3, 2, 0, 2, 64))), ("bf16", dict(kv_cache=zero(3, 2, 16, 0, 64))), ("bf16", dict(kv_cache=zero(3, 2, 16, 2, 0))),
                         ("block_size", dict(kv_cache=zero(3, 2, 48, 2, 64))), ("16 words", dict(mask=zero(8, 17, dtype=torch.int64))),
                         ("128 query heads", dict(q=zero(8, 2 * 129 * 64))), ("tmp", dict(tmp=zero(10, dtype=torch.float32))), ("scale", dict(scale=1e-50)),
                         ("softcap", dict(softcap=1e39)), ("window", dict(window=4, positions=None))):
        with pytest.raises(OpArgumentError, match=what):
            draft_tree.attention(**{**case, "scale": scale, **change})
    caches = zero(7, 2, 16, 1, 64)
    path = zero(2, 3, dtype=torch.int32)
    with pytest.raises(OpArgumentError, match="share no memory"):
        draft_tree.compact([caches[3:], caches[:4]], path=path, **{k: case[k] for k in ("block_table", "seq_lens", "q_start")})
    assert ops.read_status() == 0


def test_attention_on_another_device_than_the_current_one():
    if torch.cuda.device_count() < 2:
        pytest.skip("one GPU")
    case, scale = attention_case([9, 40, 3], [77, 900, 200], hq=8, hkv=2, d=128, page=16, seed=3, device="cuda:1")
    got = draft_tree.attention(scale=scale, **case)
    want = run_attention({k: v.to("cuda:0") for k, v in case.items()}, scale)
    assert torch.equal(got.cpu(), want.cpu())


# ------------------------------------------------------------------------------------------------ verify
def verify_case(sizes, vocab, *, wide=1, drawn=True, seed=0, spread=2.0, noise=0.7, stride=0, keep=0, cold=0.2):
    rng, gen = random.Random(seed), torch.Generator().manual_seed(seed)
    rows = sum(sizes)
    parents = torch.tensor([p for n in sizes for p in tree_parents(n, rng, wide)], dtype=torch.int32)
    q_start = starts_of(sizes)
    logits = torch.randn((rows, vocab + stride), generator=gen).mul_(spread)[:, :vocab]
    guess = logits + noise * torch.randn((rows, vocab), generator=gen)
    if keep:
        logits.masked_fill_(logits < logits.topk(keep, 1).values[:, -1:], -math.inf)
    first = torch.repeat_interleave(q_start[:-1].long(), q_start.diff().long())
    row = first + parents.long().clamp(min=0)
    probs = torch.softmax(guess, 1)
    tokens = torch.multinomial(probs[row], 1, generator=gen)[:, 0] if drawn else guess[row].topk(min(3, vocab), 1).indices[
        torch.arange(rows), torch.randint(0, min(3, vocab), (rows,), generator=gen)]
    case = dict(logits=logits, tokens=tokens, q_start=q_start, uniforms=torch.rand(rows, generator=gen),
                seeds=torch.randint(-2 ** 62, 2 ** 62, (len(sizes),), generator=gen), steps=torch.randint(0, 1000, (len(sizes),), generator=gen),
                max_tokens=max(max(sizes, default=1), 1), parents=None if wide == 1 else parents, draft_probs=probs if drawn else None,
                temperature=torch.where(torch.rand(len(sizes), generator=gen) < cold, 0.0, 1.0))
    return case


def on_gpu(case):
    moved = {}
    for k, v in case.items():
        moved[k] = v
        if isinstance(v, torch.Tensor):
            moved[k] = v.to(DEV)
            if k == "logits" and v.stride(0) != v.shape[1]:
                whole = torch.zeros((v.shape[0], v.stride(0)), device=DEV)
                whole[:, : v.shape[1]] = moved[k]
                moved[k] = whole[:, : v.shape[1]]
    return moved


def check_verify(case):
    got = [t.cpu() for t in draft_tree.verify(**on_gpu(case))]
    want = draft_tree.ref_verify(**case)
    for g, w, name in zip(got, want, ("tokens", "path", "count")):
        assert torch.equal(g, w), (name, (g != w).nonzero()[:4].tolist())
    return got


@pytest.mark.parametrize("drawn", [True, False])
@pytest.mark.parametrize("wide", [1, 3])
@pytest.mark.parametrize("vocab", [1, 2, 33, 1000, 2048, 2049, 4001])
def test_verify_against_the_rule_in_64_bits(vocab, wide, drawn):
    check_verify(verify_case([6, 1, 3, 12, 2], vocab, wide=wide, drawn=drawn, seed=vocab + wide, stride=3 if vocab == 33 else 0))


@pytest.mark.parametrize("drawn", [True, False])
def test_verify_of_long_rows_and_many_requests(drawn):
    check_verify(verify_case([4, 3], 33001, wide=2, drawn=drawn, seed=1))
    check_verify(verify_case([4], 220001, wide=2, drawn=drawn, seed=4, cold=0.0))
    check_verify(verify_case([3] * 150, 40, wide=2, drawn=drawn, seed=2))


@pytest.mark.parametrize("drawn", [True, False])
@pytest.mark.parametrize("wide", [1, 3])
@pytest.mark.parametrize("requests,vocab", [(5, 60001), (13, 90000), (16, 128256)])
def test_verify_of_long_rows_of_more_requests(requests, vocab, wide, drawn):
    """Eight CTAs a request, one or two rows at a time; greedy requests among them."""
    rng = random.Random(requests)
    check_verify(verify_case([rng.randrange(1, 6) for _ in range(requests)], vocab, wide=wide, drawn=drawn, seed=wide, noise=0.3, spread=2.0 if drawn else 5.0))


@pytest.mark.parametrize("drawn", [True, False])
def test_verify_of_as_many_columns_as_a_call_takes(drawn):
    check_verify(verify_case([3], 778000, wide=2, drawn=drawn, seed=1, cold=0.0))
    check_verify(verify_case([2] * 6, 400001, drawn=drawn, seed=2))


@pytest.mark.parametrize("drawn", [True, False])
def test_verify_of_filtered_logits(drawn):
    check_verify(verify_case([6, 1, 3, 12, 2], 1000, wide=3, drawn=drawn, seed=9, keep=5))


def test_verify_of_large_trees_and_short_results():
    case = verify_case([300, 64, 0, 65], 50, wide=4, drawn=True, seed=3, noise=0.1)
    check_verify(case)
    for most in (1, 2, 3):
        check_verify(dict(case, max_tokens=most))


def test_verify_without_drafts_is_the_samplers_draw():
    gen = torch.Generator().manual_seed(2)
    logits = torch.randn((40, 5000), generator=gen).mul_(3).to(DEV)
    seeds, steps = torch.arange(40, device=DEV), torch.arange(40, device=DEV) * 3
    tokens, path, count = draft_tree.verify(logits, torch.zeros(40, dtype=torch.int64, device=DEV), q_start=torch.arange(41, dtype=torch.int32, device=DEV),
                                            uniforms=torch.zeros(40, device=DEV), seeds=seeds, steps=steps, max_tokens=3)
    assert torch.equal(tokens[:, 0], ops.random_sample(ops.softmax(logits), seeds, steps)) and bool((count == 1).all())
    assert bool((path[:, 0] == 0).all()) and bool((path[:, 1:] == -1).all()) and bool((tokens[:, 1:] == -1).all())


def test_verify_of_odd_logits():
    """NaN and infinities among the logits, rows without a token, tokens outside the vocabulary, probabilities of NaN."""
    case = verify_case([3, 3, 3, 3, 3], 2500, drawn=True, seed=5, cold=0.0)
    l = case["logits"]
    l[0, 100:] = -math.inf
    l[3, ::2] = math.nan
    l[6, 77] = math.inf
    case["tokens"][7] = 77
    l[9] = -math.inf
    l[12] = torch.finfo(torch.float32).min
    case["tokens"][1] = 2500
    case["tokens"][4] = -1
    case["draft_probs"][3, 10] = math.nan
    got = check_verify(case)
    assert got[0][2, 0] == 77 and got[0][3, 0] == 0
    check_verify(dict(case, temperature=torch.zeros(5)))


@pytest.mark.parametrize("drawn", [True, False])
@pytest.mark.parametrize("offset", [0.0, 100.0, 3e3, -3e3, 2e5, 1e6, 1e30])
def test_verify_does_not_depend_on_what_all_logits_have_in_common(offset, drawn):
    """Logits far from 0, rounded to 32 bits before the rule in 64 bits sees them; where they are rounded to whole numbers, many share the largest."""
    for vocab, wide, whole in ((700, 1, False), (2500, 3, False), (2500, 3, True)):
        case = verify_case([4, 2, 7] * 8, vocab, wide=wide, drawn=drawn, seed=int(math.log2(abs(offset) + 1)), cold=0.1)
        case["logits"] = (case["logits"].round() if whole else case["logits"]) + offset
        check_verify(case)


@pytest.mark.parametrize("drawn", [True, False])
@pytest.mark.parametrize("vocab", [700, 2500])
@pytest.mark.parametrize("offset", [0.0, 100.0, 3e3, 2e5, 1e6])
def test_verify_accepts_up_to_the_border(offset, vocab, drawn):
    """One draft of each request, asked with numbers a little below and above what it is accepted with. Weights are off by 2^-20 at the most down to a 2^-16 of the
    largest (their argument's rounding, an exponential of 2^-22), their sum by as much and by 24 roundings of 2^-24, q and the number by one each: 2^-17.5 in all."""
    R = 200
    gen = torch.Generator().manual_seed(vocab)
    logits = torch.randn((R, vocab), generator=gen) * 1.5 + offset
    p = torch.softmax(logits.double(), 1)
    token = torch.where(torch.arange(R) % 2 == 0, logits.argmax(1), logits.topk(40, 1).indices[:, 39])
    of_token = p.gather(1, token[:, None])[:, 0]
    share = torch.rand(R, generator=gen) * 0.8 + 0.1                      # of the draws that are accepted
    probs = torch.full((R, vocab), 0.5 / vocab)
    border = of_token
    if drawn:
        probs.scatter_(1, token[:, None], (of_token / share).float()[:, None])
        border = of_token / probs.gather(1, token[:, None])[:, 0].double()
    for factor, accepted in ((1 - 2.0 ** -16, True), (1 + 2.0 ** -16, False)):
        _, _, count = draft_tree.verify(
            logits.repeat_interleave(2, 0).to(DEV), token.repeat_interleave(2).to(DEV), q_start=(torch.arange(R + 1) * 2).int().to(DEV),
            uniforms=(border * factor).float().repeat_interleave(2).to(DEV), seeds=torch.arange(R, device=DEV), steps=torch.arange(R, device=DEV), max_tokens=2,
            draft_probs=probs.repeat_interleave(2, 0).to(DEV) if drawn else None)
        assert bool((count == (2 if accepted else 1)).all()), (factor, int((count != (2 if accepted else 1)).sum()))


def test_verify_of_rows_with_one_likely_token():
    """All of a row's weight on one token, which its draft is: whatever the logit, it is accepted with every number below one."""
    R, V = 64, 2500
    top = torch.linspace(130.0, 30000.0, R)
    logits = torch.zeros((R, V))
    logits[:, 7] = top
    logits = logits.repeat_interleave(2, 0).to(DEV)
    common = dict(q_start=(torch.arange(R + 1) * 2).int().to(DEV), uniforms=torch.full((2 * R,), 1 - 2.0 ** -24, device=DEV),
                  seeds=torch.arange(R, device=DEV), steps=torch.arange(R, device=DEV), max_tokens=2)
    tokens = torch.full((2 * R,), 7, device=DEV)
    for probs in (None, torch.nn.functional.one_hot(tokens, V).float()):
        out, _, count = draft_tree.verify(logits, tokens, draft_probs=probs, **common)
        assert bool((count == 2).all()) and bool((out == 7).all())


def test_verify_of_the_same_draft_twice():
    """The second of two chosen drafts alike has no weight left; drawn ones count each for itself."""
    case = verify_case([5] * 60, 6, wide=9, drawn=False, seed=7, cold=0.0, spread=1.0)
    case["parents"] = torch.tensor([-1, 0, 0, 0, 0] * 60, dtype=torch.int32)
    case["tokens"] = torch.tensor([0, 2, 2, 4, 2] * 60)
    check_verify(case)
    probs = torch.softmax(torch.randn((300, 6), generator=torch.Generator().manual_seed(1)), 1)
    check_verify(dict(case, draft_probs=probs))


@pytest.mark.parametrize("drawn", [True, False])
@pytest.mark.parametrize("wide", [1, 3])
def test_verify_keeps_the_targets_distribution(drawn, wide):
    """First tokens of many requests with the same distributions: each token's count lies within 6 standard deviations."""
    R, V, n = 20000, 7, 4
    gen = torch.Generator().manual_seed(11)
    target, guess = torch.randn(V, generator=gen) * 1.5, torch.randn(V, generator=gen)
    p, q = torch.softmax(target, 0), torch.softmax(guess, 0)
    parents = [-1, 0, 1, 2] if wide == 1 else [-1, 0, 0, 0]
    tokens = torch.multinomial(q.expand(R, V), n, replacement=True, generator=gen) if drawn else torch.tensor([0, 3, 5, 1]).expand(R, n)
    out, _, count = draft_tree.verify(
        target.expand(R * n, V).contiguous().to(DEV), tokens.reshape(-1).contiguous().to(DEV), q_start=(torch.arange(R + 1) * n).int().to(DEV),
        parents=torch.tensor(parents * R, dtype=torch.int32, device=DEV), draft_probs=q.expand(R * n, V).contiguous().to(DEV) if drawn else None,
        uniforms=torch.rand(R * n, generator=gen).to(DEV), seeds=torch.arange(R).to(DEV), steps=torch.full((R,), 3).to(DEV), max_tokens=n)
    got = torch.bincount(out[:, 0].cpu(), minlength=V).double()
    assert bool(((got - R * p).abs() <= 6 * (R * p * (1 - p)).sqrt()).all()), (got / R, p)
    assert int(count.max()) > 1


def test_verify_of_steps_without_requests_or_rows():
    case = on_gpu(verify_case([2, 3], 50, seed=1))
    none = dict(case, q_start=case["q_start"][:1], seeds=case["seeds"][:0], steps=case["steps"][:0], temperature=None)
    assert [tuple(t.shape) for t in draft_tree.verify(**none)] == [(0, 3), (0, 3), (0,)]
    zero = torch.zeros(3, dtype=torch.int32, device=DEV)
    empty = {k: case[k][:0] for k in ("logits", "tokens", "uniforms", "draft_probs")}
    out, path, count = draft_tree.verify(**dict(case, q_start=zero, **empty))
    assert count.tolist() == [0, 0] and bool((out == -1).all()) and bool((path == -1).all())


@pytest.mark.parametrize("drawn", [True, False])
def test_verify_of_rows_at_every_alignment(drawn):
    """Rows that begin one, two or three columns off 16 bytes, and rows without a distance (the same logits for all nodes)."""
    for shift in (1, 2, 3):
        case = on_gpu(verify_case([4, 1, 6], 5003, wide=2, drawn=drawn, seed=shift))
        want = [t.clone() for t in draft_tree.verify(**case)]
        for name in ("logits", "draft_probs"):
            if case[name] is not None:
                flat = torch.full((case[name].numel() + 16,), 1e9, device=DEV)
                at = flat[shift: shift + case[name].numel()].view(case[name].shape)
                at.copy_(case[name])
                case[name] = at
        assert all(torch.equal(a, b) for a, b in zip(draft_tree.verify(**case), want))
    case = on_gpu(verify_case([4, 1, 6], 5003, wide=2, drawn=drawn, seed=9))
    case["logits"] = case["logits"][:1].expand(11, 5003)
    got = draft_tree.verify(**case)
    assert all(torch.equal(a, b) for a, b in zip(got, draft_tree.verify(**dict(case, logits=case["logits"].contiguous()))))


def test_verify_in_a_graph():
    case = on_gpu(verify_case([4, 6, 1], 3000, wide=2, seed=4))
    want = [t.clone() for t in draft_tree.verify(**case)]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = draft_tree.verify(**case)
    for _ in range(2):
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    case["uniforms"].fill_(0.0)
    want = draft_tree.verify(**case)
    g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


# ------------------------------------------------------------------------------------------------ compact
@pytest.mark.parametrize("page,hkv,d,dtype,layers", [(16, 2, 64, torch.bfloat16, 3), (32, 8, 128, torch.bfloat16, 70), (8, 1, 8, torch.bfloat16, 1),
                                                     (64, 3, 40, torch.float32, 2), (16, 1, 256, torch.bfloat16, 5)])
def test_compact_moves_the_path(page, hkv, d, dtype, layers):
    rng, gen = random.Random(page), torch.Generator().manual_seed(page)
    sizes, contexts = [30, 1, 0, 64, 9, 200], [5, 40, 3, 0, 130, 16]
    lengths = [a + b for a, b in zip(sizes, contexts)]
    table, pages = page_table(lengths, page, gen)
    caches = [torch.randn((pages, 2, page, hkv, d), generator=gen).to(dtype) for _ in range(layers)]
    path = torch.full((len(sizes), 70), -1, dtype=torch.int32)
    for r, n in enumerate(sizes):
        k = min(69, rng.randrange(0, n)) if n else 0
        if n:
            path[r, : k + 1] = torch.tensor([0] + sorted(rng.sample(range(1, n), k)), dtype=torch.int32)
    path[0, :7] = torch.tensor([0, 2, 3, 4, 5, 28, 29])          # (sources that are destinations, the nearest cells)
    args = dict(block_table=table, seq_lens=torch.tensor(lengths, dtype=torch.int32), q_start=starts_of(sizes), path=path)
    got = [c.to(DEV) for c in caches]
    draft_tree.compact(got, **{k: v.to(DEV) for k, v in args.items()})
    draft_tree.ref_compact(caches, **args)
    assert all(torch.equal(g.cpu(), c) for g, c in zip(got, caches))


def test_compact_passes_over_what_is_not_a_path():
    """Entries before their place, outside the request or behind a padding entry, and pages outside the cache, move nothing."""
    gen = torch.Generator().manual_seed(1)
    table, pages = page_table([60], 16, gen)
    cache = torch.randn((pages, 2, 16, 1, 64), generator=gen).to(torch.bfloat16)
    path = torch.tensor([[0, 0, 1, 20, -1, 5, 99, 6, 8, 30]], dtype=torch.int32)
    table[0, 2] = 1000                                           # (cells of the nodes 12 to 27, behind a context of 20)
    args = dict(block_table=table, seq_lens=torch.tensor([60], dtype=torch.int32), q_start=starts_of([40]), path=path)
    got = cache.to(DEV)
    draft_tree.compact(got, **{k: v.to(DEV) for k, v in args.items()})
    want = cache.clone()
    draft_tree.ref_compact(want, **args)
    assert torch.equal(got.cpu(), want) and not torch.equal(want, cache)


# ------------------------------------------------------------------------------------------------ more nodes than a request has
def test_nodes_past_the_1024th_are_left_out():
    """Their rows stay as they are; the others are as the restatements have them, the request's context included."""
    sizes, contexts = [1050, 3], [70, 9]
    case, scale = attention_case(sizes, contexts, hq=4, hkv=2, d=64, page=16, seed=2, wide=3, words=16, device=DEV)
    parents = torch.tensor([p for n in sizes for p in tree_parents(n, random.Random(1), 3)], dtype=torch.int32, device=DEV)
    bits = torch.full((sum(sizes), 16), 77, dtype=torch.int64, device=DEV)
    positions = torch.full((sum(sizes),), 78, dtype=torch.int64, device=DEV)
    at = dict(q_start=case["q_start"], seq_lens=case["seq_lens"])
    draft_tree.mask(parents, max_nodes=1024, bits=bits, positions=positions, **at)
    want = draft_tree.ref_mask(parents, max_nodes=1024, **at)
    node = torch.ones(sum(sizes), dtype=torch.bool, device=DEV)
    node[1024: 1050] = False
    assert torch.equal(bits[node], want[0][node]) and torch.equal(positions[node], want[1][node])
    assert bool((bits[~node] == 77).all()) and bool((positions[~node] == 78).all())
    case["mask"], case["positions"] = want
    for window in (0, 40):
        got = run_attention(case, scale, window=window)
        o, bound = attention_bound(case, scale, window=window)
        assert bool(((got.double() - o).abs() <= bound)[node].all()) and bool((got[~node] == 7).all())
    gen = torch.Generator().manual_seed(1)
    logits, ids = torch.randn((sum(sizes), 40), generator=gen), torch.tensor([5, 6])
    tokens = torch.randint(0, 40, (sum(sizes),), generator=gen)
    logits[torch.arange(1049), tokens[1: 1050]] = 60.0           # (a chain of drafts that are all accepted)
    steps = dict(logits=logits, tokens=tokens, q_start=starts_of(sizes), uniforms=torch.full((sum(sizes),), 0.5), seeds=ids, steps=ids, max_tokens=1060)
    out, path, count = draft_tree.verify(**on_gpu(steps))
    assert all(torch.equal(a.cpu(), b) for a, b in zip((out, path, count), draft_tree.ref_verify(**steps))) and int(count[0]) == 1024
    path = torch.tensor([[0, 3, 1023, 1024, 1049, -1], [0, 2, -1, -1, -1, -1]], dtype=torch.int32, device=DEV)
    moved, kept = case["kv_cache"].clone(), case["kv_cache"].clone()
    draft_tree.compact(moved, block_table=case["block_table"], path=path, **at)
    draft_tree.ref_compact(kept, block_table=case["block_table"], path=path, **at)
    assert torch.equal(moved, kept) and not torch.equal(moved, case["kv_cache"])


# ------------------------------------------------------------------------------------------------ together
def test_a_run_of_steps_with_trees():
    """A model of two layers decodes greedily with trees of drafts, some of them right, through the operators of a step: every token is the
    argmax of the model computed at once over all tokens so far in 32 bits, but for logits nearer than bf16 tells apart."""
    gen = torch.Generator().manual_seed(3)
    H, hq, hkv, D, V, L, page = 256, 4, 2, 64, 504, 2, 16
    w = lambda *s: (torch.randn(s, generator=gen) / math.sqrt(s[1])).to(torch.bfloat16).to(DEV)  # noqa: E731
    emb, head = w(V, H) * 16, w(V, H)
    qkv_w, o_w = [w((hq + 2 * hkv) * D, H) for _ in range(L)], [w(H, hq * D) for _ in range(L)]
    from vllm_cpp_b200.ops import reference
    cos_sin = ops.rope_table(reference.rope_inv_freq(D, 10000.0).to(DEV), 400)

    def oracle(tokens):
        """Logits after each of the tokens."""
        x = emb[torch.tensor(tokens, device=DEV)].float()
        n = len(tokens)
        for l in range(L):
            y = x @ qkv_w[l].float().t()
            q, k, v = reference.rope_kv(y, torch.arange(n, device=DEV), cos_sin, hq, hkv, D)
            s = torch.einsum("qhd,khd->hqk", q, k.repeat_interleave(hq // hkv, 1)) * D ** -0.5
            s = s.masked_fill(torch.triu(torch.ones(n, n, dtype=torch.bool, device=DEV), 1), -math.inf).softmax(-1)
            x = x + torch.einsum("hqk,khd->qhd", s, v.repeat_interleave(hq // hkv, 1)).flatten(1) @ o_w[l].float().t()
        return x @ head.float().t()

    rng = random.Random(1)
    R = 3
    said = [[rng.randrange(V) for _ in range(n)] for n in (5, 40, 17)]
    start = [len(x) for x in said]
    table, pages = page_table([200] * R, page, gen)
    table = table.to(DEV)
    caches = [torch.zeros((pages, 2, page, hkv, D), dtype=torch.bfloat16, device=DEV) for _ in range(L)]
    context, accepted, odd = [0] * R, 0, 0
    for step in range(14):
        nodes, parents, sizes = [], [], []
        for r in range(R):
            if step == 0:                                        # the prompt: a chain
                n = len(said[r])
                nodes += said[r]
                parents += [-1] + list(range(n - 1))
            else:
                right = []                                       # what greedy decoding would say next
                for _ in range(3):
                    right.append(int(oracle(said[r] + right)[-1].argmax()))
                wrong = [rng.randrange(V) for _ in range(4)]
                nodes += [said[r][-1], wrong[0], right[0], wrong[1], right[1], wrong[2], wrong[3] if rng.random() < 0.5 else right[2]]
                parents += [-1, 0, 0, 1, 2, 2, 4]
                n = 7
            sizes.append(n)
        rows = sum(sizes)
        q_start = starts_of(sizes, DEV)
        seq_lens = torch.tensor([c + n for c, n in zip(context, sizes)], dtype=torch.int32, device=DEV)
        up = torch.tensor(parents, dtype=torch.int32, device=DEV)
        ids = torch.tensor(nodes, device=DEV)
        bits, positions = draft_tree.mask(up, q_start=q_start, seq_lens=seq_lens)
        cell = torch.cat([torch.arange(c, c + n) for c, n in zip(context, sizes)]).to(DEV)
        of = torch.repeat_interleave(torch.arange(R, device=DEV), torch.tensor(sizes, device=DEV))
        slots = table[of, cell // page].long() * page + cell % page
        x = emb[ids].float()
        for l in range(L):
            qkv = ops.gemm(x.to(torch.bfloat16), qkv_w[l])
            ops.rope_kv(qkv, positions, cos_sin, num_q_heads=hq, num_kv_heads=hkv, head_dim=D, slot_mapping=slots, kv_cache=caches[l], block_size=page)
            a = draft_tree.attention(qkv[:, : hq * D], caches[l], block_table=table, seq_lens=seq_lens, q_start=q_start, mask=bits, scale=D ** -0.5)
            x = x + ops.gemm(a, o_w[l], out_dtype=torch.float32)
        logits = ops.gemm(x.to(torch.bfloat16), head, out_dtype=torch.float32)
        if step == 0:
            tokens = [[int(logits[int(q_start[r + 1]) - 1].argmax())] for r in range(R)]
            context = [len(s) for s in said]
        else:
            out, path, count = draft_tree.verify(logits, ids, q_start=q_start, parents=up, uniforms=torch.zeros(rows, device=DEV),
                                                 seeds=torch.zeros(R, dtype=torch.int64, device=DEV), steps=torch.zeros(R, dtype=torch.int64, device=DEV),
                                                 temperature=torch.zeros(R, device=DEV), max_tokens=5)
            draft_tree.compact(caches, block_table=table, seq_lens=seq_lens, q_start=q_start, path=path)
            tokens = [out[r, : int(count[r])].tolist() for r in range(R)]
            accepted += int(count.sum()) - R
            context = [c + int(k) for c, k in zip(context, count)]
        for r in range(R):
            for t in tokens[r]:
                l = oracle(said[r])[-1]
                # activations and products are rounded to bf16 a few times a layer: a hundredth of the logits' spread
                assert float(l.max() - l[t]) <= 0.03 * float(l.std()) * 5, (step, r)
                odd += int(l.argmax()) != t
                said[r].append(t)
    assert accepted > 50 and odd <= 5


def test_a_run_of_steps_that_samples():
    """A layer decodes with trees that a draft distribution drew: in every step masks, tokens, paths and cells are what the restatements make of the same
    inputs, tokens by the rule in 64 bits, and outputs of the attention lie within its bound."""
    gen, rng = torch.Generator().manual_seed(4), random.Random(2)
    H, hq, hkv, D, V, page, R = 256, 8, 2, 64, 2104, 16, 4
    w = lambda *s: (torch.randn(s, generator=gen) / math.sqrt(s[1])).to(torch.bfloat16).to(DEV)  # noqa: E731
    emb, head, qkv_w, o_w = w(V, H) * 16, w(V, H) * 3, w((hq + 2 * hkv) * D, H), w(H, hq * D)
    from vllm_cpp_b200.ops import reference
    cos_sin = ops.rope_table(reference.rope_inv_freq(D, 10000.0).to(DEV), 400)
    table, pages = page_table([200] * R, page, gen)
    table = table.to(DEV)
    cache = torch.zeros((pages, 2, page, hkv, D), dtype=torch.bfloat16, device=DEV)
    temperature = torch.tensor([0.8, 1.0, 0.0, 0.5], device=DEV)
    seeds = torch.tensor([3, 2 ** 40, 5, -9], device=DEV)
    context, roots, accepted = [0] * R, [rng.randrange(V) for _ in range(R)], 0
    for step in range(12):
        sizes = [rng.randrange(2, 9) for _ in range(R)]
        parents = torch.tensor([p for n in sizes for p in tree_parents(n, rng, 2)], dtype=torch.int32)
        q_start, rows = starts_of(sizes), sum(sizes)
        first = torch.repeat_interleave(q_start[:-1], q_start.diff()).long()
        ids = torch.zeros(rows, dtype=torch.int64)
        ids[q_start[:-1].long()] = torch.tensor(roots)
        guess = torch.empty((rows, V))
        for i in range(rows):                                    # (a draft of the next token by the last one alone)
            if parents[i] >= 0:
                ids[i] = torch.multinomial(guess[first[i] + parents[i]], 1, generator=gen)
            guess[i] = torch.softmax(emb[ids[i]].float() @ head.float().t(), 0).cpu()
        lens = torch.tensor([c + n for c, n in zip(context, sizes)], dtype=torch.int32)
        where = dict(q_start=q_start.to(DEV), seq_lens=lens.to(DEV))
        bits, positions = draft_tree.mask(parents.to(DEV), **where)
        assert all(torch.equal(a, b) for a, b in zip((bits, positions), draft_tree.ref_mask(parents.to(DEV), **where)))
        cell = torch.cat([torch.arange(c, c + n) for c, n in zip(context, sizes)]).to(DEV)
        of = torch.repeat_interleave(torch.arange(R), torch.tensor(sizes)).to(DEV)
        slots = table[of, cell // page].long() * page + cell % page
        x = emb[ids.to(DEV)]
        qkv = ops.gemm(x, qkv_w)
        ops.rope_kv(qkv, positions, cos_sin, num_q_heads=hq, num_kv_heads=hkv, head_dim=D, slot_mapping=slots, kv_cache=cache, block_size=page)
        case = dict(q=qkv[:, : hq * D], kv_cache=cache, block_table=table, mask=bits, positions=positions, **where)
        a = check_attention(case, D ** -0.5)
        logits = ops.gemm((x.float() + 0.3 * ops.gemm(a, o_w).float()).to(torch.bfloat16), head, out_dtype=torch.float32)
        logits /= torch.where(temperature > 0, temperature, 1.0)[of, None]
        given = dict(logits=logits, tokens=ids.to(DEV), parents=parents.to(DEV), draft_probs=guess.to(DEV), uniforms=torch.rand(rows, generator=gen).to(DEV),
                     seeds=seeds, steps=torch.full((R,), step, device=DEV), temperature=temperature, q_start=where["q_start"], max_tokens=6)
        got = draft_tree.verify(**given)
        want = draft_tree.ref_verify(**{k: v.cpu() if isinstance(v, torch.Tensor) else v for k, v in given.items()})
        assert all(torch.equal(g.cpu(), w) for g, w in zip(got, want))
        moved = cache.clone()
        draft_tree.compact(cache, block_table=table, path=got[1], **where)
        draft_tree.ref_compact(moved, block_table=table, path=got[1], **where)
        assert torch.equal(cache, moved)
        counts = got[2].tolist()
        roots = [int(got[0][r, k - 1]) for r, k in enumerate(counts)]
        context = [c + k for c, k in zip(context, counts)]
        accepted += sum(counts) - R
    assert accepted >= 10
