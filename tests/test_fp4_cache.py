"""The 4-bit KV cache on the CPU: its layout and rounding as restated in PyTorch, refusals of the operators, and engines that hold their cache
in it."""
import math

import pytest
import torch

import fp4_reference as F
from vllm_cpp_b200.ops import fp4_cache as C
from vllm_cpp_b200.ops import reference as ref
from vllm_cpp_b200.ops.validate import OpArgumentError


def _gen(seed=0):
    return torch.Generator().manual_seed(seed)


def _hard_rows(D, n, gen):
    """Rows with groups of every kind: normal values, zeros, values exactly between two codes, scales exactly between two of theirs,
    subnormal and vanishing scales, saturated ones, signed zeros."""
    x = torch.randn((n, D), generator=gen)
    g = x.view(n, D // 16, 16)
    kind = torch.arange(n * (D // 16)).view(n, D // 16) % 9
    ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, -0.25, -0.75, -1.25, -1.75, -2.5, -3.5, -5.0, 0.5])
    g[kind == 1] = 0
    g[kind == 2] = ties * 0.375
    g[kind == 3] = ties * 1.125
    g[kind == 4] = torch.cat([torch.tensor([6 * 1.0625]), torch.linspace(-3, 3, 15)])      # amax / 6 between 1 and 1.125
    g[kind == 5] = ties * 2.0 ** -16
    g[kind == 6] = ties * 2.0 ** -21
    g[kind == 7] = ties * 20000
    g[kind == 8] = -torch.zeros(16)
    return x.to(torch.bfloat16)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_restated_rounding_is_the_definitions(D):
    x = _hard_rows(D, 40, _gen(D))
    codes, s = C.ref_quantize(x)
    want = F.scales(x)
    s = C.scale_values(s)
    assert torch.equal(s.double(), want)
    levels = torch.tensor(C.LEVELS + tuple(-v for v in C.LEVELS), dtype=torch.float64)
    got = (levels[codes.long()].unflatten(-1, (-1, 16)) * s.double()[..., None]).flatten(-2)
    assert torch.equal(got, F.held(x, want))
    assert torch.equal(got.to(torch.bfloat16).double(), got)               # exact in bf16


def test_nan_and_infinity_in_a_group():
    x = torch.ones((1, 64))
    x[0, 3], x[0, 17], x[0, 40] = math.nan, math.inf, -math.inf
    codes, s = C.ref_quantize(x)
    s = C.scale_values(s)
    assert s[0].isnan().tolist() == [True, False, False, False]
    assert s[0, 1] == C.MOST_SCALE and codes[0, 17] == 7 and codes[0, 40] == 15 and codes[0, 16] == 0


@pytest.mark.parametrize("D,bs", [(64, 16), (128, 48), (256, 32)])
def test_write_then_read(D, bs):
    nb, H, n = 5, 3, 37
    x = _hard_rows(D, 2 * n * H, _gen(1)).view(2, n, H, D)
    cache = C.alloc(nb, H, bs, D, "cpu")
    assert cache[0].numel() == C.bytes_per_block(H, bs, D)
    slots = torch.randperm(nb * bs, generator=_gen(2))[:n]
    slots[5], slots[9] = -1, nb * bs
    C.ref_write(x[0], x[1], cache, slots)
    k, v = C.ref_read(cache, slots)
    ok = (slots >= 0) & (slots < nb * bs)
    for got, y in ((k, x[0]), (v, x[1])):
        assert torch.equal(got.double()[ok], F.held(y, F.scales(y))[ok])
        assert bool((got[~ok] == 0).all())
    # untouched slots stay zero
    rest = torch.ones(nb * bs, dtype=torch.bool)
    rest[slots[ok]] = False
    k, v = C.ref_read(cache, torch.arange(nb * bs)[rest])
    assert not k.any() and not v.any()


def test_written_again_the_values_stay():
    """Exchange with other programs in bf16 loses nothing: the largest code of a group with a normal scale is 6, so its scale comes back."""
    D, n = 128, 400
    x = (torch.randn((2, n, 1, D), generator=_gen(3)) * torch.exp(torch.randn((2, n, 1, 1), generator=_gen(4)) * 2)).to(torch.bfloat16)
    a, b = C.alloc(30, 1, 16, D, "cpu"), C.alloc(30, 1, 16, D, "cpu")
    slots = torch.arange(n)
    C.ref_write(x[0], x[1], a, slots)
    k, v = C.ref_read(a, slots)
    C.ref_write(k, v, b, slots)
    for u, w in zip((k, v), C.ref_read(b, slots)):
        assert torch.equal(u, w)


def test_restated_append_rounds_once():
    T, Hq, Hkv, D, rot = 9, 4, 2, 64, 32
    gen = _gen(5)
    qkv = torch.randn((T, (Hq + 2 * Hkv) * D), generator=gen).to(torch.bfloat16)
    table = ref.rope_table(ref.rope_inv_freq(rot, 1e4), 100)
    pos = torch.randint(0, 100, (T,), generator=gen)
    w = (1 + 0.1 * torch.randn((2, D), generator=gen)).to(torch.bfloat16)
    cache = C.alloc(2, Hkv, 16, D, "cpu")
    slots = torch.randperm(32, generator=gen)[:T]
    before = qkv.clone()
    C.ref_append(qkv, pos, table, cache, slots, num_q_heads=Hq, rot_dim=rot, q_norm=w[0], k_norm=w[1])
    x = before.view(T, Hq + 2 * Hkv, D)
    cos, sin = table[pos].chunk(2, -1)
    q, _ = F.rotated(x[:, :Hq], w[0], 1e-6, False, cos, sin, rot, True)
    k, big = F.rotated(x[:, Hq: Hq + Hkv], w[1], 1e-6, False, cos, sin, rot, True)
    assert bool(((qkv.view(T, -1, D)[:, :Hq].double() - q).abs() <= 2.0 ** -8 * q.abs() + 1e-6).all())
    assert torch.equal(qkv.view(T, -1, D)[:, Hq:], x[:, Hq:])             # k and v columns stay
    got_k, got_v = C.ref_read(cache, slots)
    F.check_held(got_k, k, big)
    F.check_held(got_v, x[:, Hq + Hkv:].double(), x[:, Hq + Hkv:].abs().double())


def test_restated_attention():
    gen = _gen(6)
    Hq, Hkv, D, bs = 6, 2, 64, 16
    cache = F.random_cache(9, Hkv, bs, D, gen)
    lens, new = [0, 1, 33, 50], [1, 1, 4, 50]
    table = torch.randint(0, 9, (4, 4), dtype=torch.int32, generator=gen)
    start = torch.tensor([0, 1, 2, 6, 56], dtype=torch.int32)
    q = torch.randn((56, Hq * D), generator=gen).to(torch.bfloat16)
    for window, cap in ((0, 0.0), (7, 0.0), (-16, 20.0)):
        out = C.ref_attention(q, cache, block_table=table, seq_lens=torch.tensor(lens, dtype=torch.int32), q_start=start, scale=0.125,
                              softcap=cap, window=window)
        for r, (n, m) in enumerate(zip(lens, new)):
            slots = (table[r].long()[:, None] * bs + torch.arange(bs)).flatten()[:n]
            k, v = C.ref_read(cache, slots)
            rows = slice(int(start[r]), int(start[r]) + m)
            want, size = F.attention(q[rows].view(m, Hq, D), k, v, n - m, 0.125, cap, window)
            F.check_attention(out[rows].view(m, Hq, D), want, size)


# ------------------------------------------------------------------------------------------------ refusals
def test_refusals_without_a_gpu():
    """Arguments are checked before anything is launched."""
    cache = C.alloc(2, 2, 16, 64, "cpu")
    q = torch.zeros((3, 256), dtype=torch.bfloat16)
    table, lens = torch.zeros((3, 2), dtype=torch.int32), torch.ones(3, dtype=torch.int32)
    slots = torch.zeros(3, dtype=torch.int64)
    good = dict(block_table=table, seq_lens=lens, scale=1.0, out=torch.zeros_like(q))

    def refused(rule, call, *a, **kw):
        with pytest.raises(OpArgumentError, match=rule):
            call(*a, **kw)
    refused("one GPU", C.decode, q, cache, **good)
    refused("one GPU", C.append, q, None, None, cache, slots, num_q_heads=0, offsets=(0, 0, 128))
    refused("one GPU", C.read, cache, slots)
    refused("one GPU", C.write, q[:, :128], q[:, 128:], cache, slots)
    refused("cache is uint8", C.decode, q, cache.view(torch.int8), **good)
    refused("cache is uint8", C.read, cache[..., :64 * 9], slots)
    refused("cache is uint8", C.read, cache.transpose(0, 1), slots)
    refused("q is", C.decode, q.float(), cache, **good)
    refused("q is", C.decode, q[:, :192], cache, **good)
    refused("q is", C.decode, q[:, :64], cache, **good)
    refused("q is", C.decode, torch.zeros((3, 257), dtype=torch.bfloat16)[:, 1:], cache, **good)
    refused("out is like q", C.decode, q, cache, **{**good, "out": q})
    refused("out is like q", C.decode, q, cache, **{**good, "out": torch.zeros((2, 256), dtype=torch.bfloat16)})
    refused("block_table", C.decode, q, cache, **{**good, "block_table": table.long()})
    refused("block_table", C.decode, q, cache, **{**good, "block_table": table[:, :0]})
    refused("softcap", C.decode, q, cache, softcap=-1.0, **good)
    refused("scale is positive", C.decode, q, cache, **{**good, "scale": 0.0})
    tiles = dict(q_start=torch.zeros(4, dtype=torch.int32), tile_req=slots.int(), tile_q0=slots.int())
    refused("one GPU", C.prefill, q, cache, **tiles, **good)
    qkv = torch.zeros((3, 640), dtype=torch.bfloat16)
    pos, cs = slots.clone(), torch.zeros((5, 64))
    for bad, rule in ((dict(num_q_heads=7), "inside the rows"), (dict(num_q_heads=6, offsets=(0, 4, 512)), "inside the rows"),
                      (dict(num_q_heads=6, q_head_stride=68), "inside the rows"), (dict(num_q_heads=6, rot_dim=32), "cos_sin"),
                      (dict(num_q_heads=6, q_norm=torch.ones(32, dtype=torch.bfloat16)), "norm weights"),
                      (dict(num_q_heads=6, q_out=torch.zeros((3, 64), dtype=torch.bfloat16)), "q_out")):
        refused(rule, C.append, qkv, pos, cs, cache, slots, **bad)
    refused("slots is int64", C.append, qkv, pos, cs, cache, slots.int(), num_q_heads=6)
    refused("cos_sin", C.append, qkv, pos[:2], cs, cache, slots, num_q_heads=6)
    refused("cos_sin", C.append, qkv, pos, cs.double(), cache, slots, num_q_heads=6)
    refused("qkv is", C.append, qkv.float(), pos, cs, cache, slots, num_q_heads=6)
    refused("head_dim", C.alloc, 2, 2, 24, 64, "cpu")
    refused("head_dim", C.alloc, 2, 2, 16, 96, "cpu")


def test_refusals_of_rows_that_share_memory_and_of_numbers_past_the_limits():
    cache = C.alloc(2, 2, 16, 64, "cpu")
    q = torch.zeros((3, 256), dtype=torch.bfloat16)
    table, lens = torch.zeros((3, 2), dtype=torch.int32), torch.ones(3, dtype=torch.int32)
    good = dict(block_table=table, seq_lens=lens, scale=1.0, out=torch.zeros_like(q))

    def refused(rule, call, *a, **kw):
        with pytest.raises(OpArgumentError, match=rule):
            call(*a, **kw)
    refused("out is like q", C.decode, q, cache, **{**good, "out": torch.zeros((1, 256), dtype=torch.bfloat16).expand(3, 256)})
    refused("window in 32 bits", C.decode, q, cache, window=2 ** 31, **good)
    refused("window in 32 bits", C.decode, q, cache, window=-2 ** 31, **good)
    refused("softcap finite", C.decode, q, cache, softcap=float("inf"), **good)
    refused("scale is positive", C.decode, q, cache, **{**good, "scale": float("nan")})
    many = torch.zeros((8193, 256), dtype=torch.bfloat16)
    refused("8192 sequences", C.decode, many, cache, block_table=table.new_zeros((8193, 1)), seq_lens=lens.new_zeros(8193), scale=1.0,
            out=torch.zeros_like(many))
    ints = torch.zeros(8194, dtype=torch.int32)
    refused("8000 tiles", C.prefill, q, cache, q_start=ints[:4], tile_req=ints[:8001], tile_q0=ints[:8001], **good)
    refused("8192 sequences", C.prefill, q, cache, q_start=ints, tile_req=ints[:1], tile_q0=ints[:1], scale=1.0, out=good["out"],
            block_table=table.new_zeros((8193, 1)), seq_lens=lens.new_zeros(8193))
    refused("q_start", C.prefill, q, cache, q_start=None, tile_req=ints[:1], tile_q0=ints[:1], **good)
    qkv, slots = torch.zeros((3, 640), dtype=torch.bfloat16), torch.zeros(3, dtype=torch.int64)
    refused("apart from one another", C.append, qkv, None, None, cache, slots, num_q_heads=4, q_head_stride=32)
    refused("apart from one another", C.append, qkv, None, None, cache, slots, num_q_heads=6, offsets=(0, 320, 512))
    refused("apart from one another", C.append, qkv[:1].expand(3, 640), None, None, cache, slots, num_q_heads=6)
    refused("q_out", C.append, qkv, None, None, cache, slots, num_q_heads=1, q_out=torch.zeros((1, 64), dtype=torch.bfloat16).expand(3, 64))
