"""Kernels of the 4-bit KV cache against the operators in 64 bits (fp4_reference.py, where the bounds are derived)."""
import math

import pytest
import torch

import fp4_reference as F
from test_fp4_cache import _hard_rows
from vllm_cpp_b200.ops import fp4_cache as C
from vllm_cpp_b200.ops import reference as ref
from vllm_cpp_b200.ops.validate import OpArgumentError

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _gen(seed=0):
    return torch.Generator().manual_seed(seed)


def _status():
    from vllm_cpp_b200 import ops
    return ops.read_status()


# -------------------------------------------------------------------------------------------- append, write, read
@pytest.mark.parametrize("D,bs,H", [(64, 16, 1), (128, 48, 3), (256, 32, 2)])
def test_write_is_the_restated_one_bit_for_bit(D, bs, H):
    nb, n = 7, 61
    x = _hard_rows(D, 2 * n * H, _gen(D)).view(2, n, H, D)
    x[0, 3, 0, 5], x[1, 4, 0, 20], x[1, 6, H - 1, 40] = math.nan, math.inf, -math.inf
    slots = torch.randperm(nb * bs, generator=_gen(1))[:n]
    slots[0], slots[7], slots[9] = -1, nb * bs, 1 << 40
    want = C.alloc(nb, H, bs, D, "cpu")
    C.ref_write(x[0], x[1], want, slots)
    cache = C.alloc(nb, H, bs, D, DEV)
    C.write(x[0].to(DEV), x[1].to(DEV), cache, slots.to(DEV))
    a, b = C.ref_expand(want), C.ref_expand(cache.cpu())
    assert torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(), b.nan_to_num())
    assert torch.equal(C.scale_values(want[..., 16 * D:]).nan_to_num(-1), C.scale_values(cache.cpu()[..., 16 * D:]).nan_to_num(-1))
    k, v = C.read(cache, slots.to(DEV))
    rk, rv = C.ref_read(want, slots)
    for got, r in ((k.cpu(), rk), (v.cpu(), rv)):
        assert torch.equal(got.isnan(), r.isnan()) and torch.equal(got.nan_to_num(), r.nan_to_num())


APPEND = [
    # T, Hq, Hkv, D, rot, neox, normed, gemma, block
    (1, 32, 8, 128, 128, True, False, False, 32),
    (3, 4, 1, 64, 64, True, True, False, 16),
    (257, 16, 8, 128, 128, True, True, True, 16),
    (70, 7, 1, 128, 64, True, False, False, 48),
    (33, 5, 5, 64, 20, True, True, False, 32),       # half of the rotated dims is no multiple of 8
    (33, 6, 3, 128, 96, False, False, False, 32),    # neighbouring pairs
    (12, 12, 2, 256, 256, True, True, False, 64),
    (12, 3, 3, 256, 10, False, True, True, 16),
    (900, 32, 4, 128, 128, True, False, False, 32),
    (40, 8, 2, 128, 0, True, True, False, 32),       # no rotation
]


@pytest.mark.parametrize("T,Hq,Hkv,D,rot,neox,normed,gemma,bs", APPEND)
@pytest.mark.parametrize("in_place", [False, True])
def test_append(T, Hq, Hkv, D, rot, neox, normed, gemma, bs, in_place):
    gen = _gen(T + D)
    gate = 2 if in_place and D == 128 else 1                    # q heads with a gate between them
    cols = Hq * D * gate + 2 * Hkv * D
    wide = torch.randn((T, cols + 24), generator=gen).to(torch.bfloat16).to(DEV)
    qkv = wide[:, 8: 8 + cols]
    before = qkv.clone()
    table = ref.rope_table(ref.rope_inv_freq(rot, 1e4), 5000).to(DEV) if rot else None
    pos = torch.randint(0, 5000, (T,), generator=gen).to(DEV)
    w = (1 + 0.2 * torch.randn((2, D), generator=gen)).to(torch.bfloat16).to(DEV)
    nb = -(-T // bs) + 2
    cache = C.alloc(nb, Hkv, bs, D, DEV)
    slots = torch.randperm(nb * bs, generator=gen)[:T].to(DEV)
    if T > 2:
        slots[1] = -1
    q_out = None if in_place else torch.empty((T, Hq * D), dtype=torch.bfloat16, device=DEV)
    offsets = (0, Hq * D * gate, (Hq * gate + Hkv) * D)
    C.append(qkv, pos, table, cache, slots, num_q_heads=Hq, rot_dim=rot or None, neox=neox, q_norm=w[0] if normed else None,
             k_norm=w[1] if normed else None, eps=1e-6, gemma=gemma, q_out=q_out, q_head_stride=D * gate, offsets=offsets)
    x_q = before[:, : Hq * D * gate].view(T, Hq, gate * D)[..., :D]
    x_k, x_v = (before[:, o: o + Hkv * D].view(T, Hkv, D) for o in offsets[1:])
    cos, sin = (table[pos][:, : rot // 2], table[pos][:, rot // 2:]) if rot else (None, None)
    q, q_big = F.rotated(x_q, w[0] if normed else None, 1e-6, gemma, cos, sin, rot, neox)
    k, k_big = F.rotated(x_k, w[1] if normed else None, 1e-6, gemma, cos, sin, rot, neox)
    if in_place:
        got = qkv[:, : Hq * D * gate].view(T, Hq, gate * D)
        assert torch.equal(got[..., D:], before[:, : Hq * D * gate].view(T, Hq, gate * D)[..., D:])
        got = got[..., :D]
        assert torch.equal(qkv[:, offsets[1]:], before[:, offsets[1]:])
    else:
        got = q_out.view(T, Hq, D)
        assert torch.equal(qkv, before)
    assert bool(((got.double() - q).abs() <= 2.0 ** -8 * q.abs() + 2.0 ** -18 * q_big).all())
    ok = slots >= 0
    gk, gv = C.read(cache, slots)
    F.check_held(gk[ok], k[ok], k_big[ok])
    v = x_v.double()
    assert torch.equal(gv.double()[ok], F.held(v, F.scales(v))[ok])
    assert not gk[~ok].any() and not gv[~ok].any()
    rest = torch.ones(nb * bs, dtype=torch.bool, device=DEV)
    rest[slots[ok]] = False
    assert not any(x.any() for x in C.read(cache, rest.nonzero()[:, 0]))        # nothing else was written


def test_positions_outside_the_table_give_nan():
    T, D = 4, 64
    qkv = torch.randn((T, 3 * D), generator=_gen()).to(torch.bfloat16).to(DEV)
    table = ref.rope_table(ref.rope_inv_freq(D, 1e4), 10).to(DEV)
    cache, slots = C.alloc(1, 1, 16, D, DEV), torch.arange(T, device=DEV)
    q = torch.empty((T, D), dtype=torch.bfloat16, device=DEV)
    C.append(qkv, torch.tensor([9, 10, -1, 1 << 40], device=DEV), table, cache, slots, num_q_heads=1, q_out=q)
    assert q.isnan().all(1).tolist() == [False, True, True, True]
    assert C.read(cache, slots)[0].isnan().flatten(1).all(1).tolist() == [False, True, True, True]


# -------------------------------------------------------------------------------------------------------- attention
def _pages(lens, bs, gen, spare=3):
    """A table of distinct pages in no order; entries behind a sequence's pages name a page that holds nothing of use."""
    need = [max(1, -(-n // bs)) for n in lens]
    perm = torch.randperm(sum(need), generator=gen) + spare
    table = torch.ones((len(lens), max(need) + 1), dtype=torch.int32)
    at = 0
    for r, n in enumerate(need):
        table[r, :n] = perm[at: at + n].int()
        at += n
    return table, sum(need) + spare


def _spoil(cache, table, lens, lows, bs):
    """NaN scales wherever no query may look: unused pages, slots behind a sequence and before every window."""
    nb, H, _, D = C.shape_of(cache)
    keep = torch.zeros((nb, bs), dtype=torch.bool)
    for r, (n, low) in enumerate(zip(lens, lows)):
        for i in range(max(0, low), n):
            keep[table[r, i // bs], i % bs] = True
    gone = ~keep.view(nb, 1, bs // 16, 16)
    ks = cache[..., 16 * D: 17 * D].unflatten(-1, (16, D // 16))
    vs = cache[..., 17 * D:].unflatten(-1, (D // 16, 16))
    ks.masked_fill_(gone[..., None], 0xff)
    vs.masked_fill_(gone[..., None, :], 0xff)


def _case(lens, new, Hq, Hkv, D, bs, window, seed):
    gen = _gen(seed)
    table, nb = _pages(lens, bs, gen)
    cache = F.random_cache(nb, Hkv, bs, D, gen)
    lows = [0 if window == 0 else n - m - window + 1 if window > 0 else max(0, n - m) // -window * -window for n, m in zip(lens, new)]
    _spoil(cache, table, lens, lows, bs)
    q = (torch.randn((sum(new), Hq * D), generator=gen) * torch.exp(torch.randn((sum(new), 1), generator=gen))).to(torch.bfloat16)
    return q, cache, table, torch.tensor(lens, dtype=torch.int32)


def _check(out, q, cache, table, lens, new, Hq, D, bs, scale, cap, window, causal=True):
    at = 0
    for r, (n, m) in enumerate(zip(lens, new)):
        slots = (table[r].long()[:, None] * bs + torch.arange(bs)).flatten()[:n]
        low = 0 if window == 0 else n - m - window + 1 if window > 0 else max(0, n - m) // -window * -window
        low = max(0, low) if m else 0
        k, v = C.ref_read(cache, slots)
        k, v = k.nan_to_num(), v.nan_to_num()
        qq = q[at: at + m].view(m, Hq, D)
        want, size = F.attention(qq.to(DEV), k.to(DEV), v.to(DEV), n - m, scale, cap, window, causal)
        F.check_attention(out[at: at + m].view(m, Hq, D), want, size)
        at += m


DECODE = [
    # lengths, Hq, Hkv, D, block, window, softcap
    ([1], 8, 8, 128, 16, 0, 0.0),
    ([0, 1, 15, 16, 17, 0], 32, 8, 128, 32, 0, 0.0),
    ([1000], 32, 8, 128, 32, 0, 0.0),
    ([31, 700, 2, 129, 5000, 0, 64], 16, 2, 128, 16, 0, 0.0),            # eight heads a group
    ([513, 40], 24, 2, 128, 64, 0, 0.0),                                 # twelve
    ([513, 40], 32, 2, 128, 64, 0, 0.0),                                 # sixteen
    ([333, 1, 90], 20, 1, 128, 32, 0, 0.0),                              # more than sixteen: several tiles
    ([333, 1, 90], 7, 1, 64, 48, 0, 0.0),
    ([2000, 17, 300, 48], 9, 3, 64, 16, 100, 0.0),
    ([2000, 17, 300, 48], 40, 4, 64, 128, -128, 30.0),
    ([2000, 17, 300, 48], 5, 5, 128, 32, 33, 20.0),
    ([257, 4096, 3], 8, 1, 256, 32, 0, 0.0),
    ([257, 4096, 3], 24, 2, 256, 16, 64, 50.0),
    ([9, 33, 128] * 90, 16, 8, 128, 32, 0, 0.0),                         # many short sequences
    ([70000], 8, 2, 128, 32, 0, 0.0),
    ([1] * 300, 4, 4, 64, 16, 0, 0.0),
]


@pytest.mark.parametrize("lens,Hq,Hkv,D,bs,window,cap", DECODE)
def test_decode(lens, Hq, Hkv, D, bs, window, cap):
    q, cache, table, n = _case(lens, [1] * len(lens), Hq, Hkv, D, bs, window, seed=len(lens) + D)
    scale = D ** -0.5
    out = torch.full_like(q, 7.0).to(DEV)
    args = dict(block_table=table.to(DEV), seq_lens=n.to(DEV), scale=scale, softcap=cap, window=window)
    got = C.decode(q.to(DEV), cache.to(DEV), out=out, **args)
    assert got is out
    _check(out, q, cache, table, lens, [1] * len(lens), Hq, D, bs, scale, cap, window)
    assert torch.equal(C.decode(q.to(DEV), cache.to(DEV), **args), out)                     # and the same bits again
    assert _status() == 0


PREFILL = [
    # lengths, new tokens, Hq, Hkv, D, block, window, softcap, causal
    ([1], [1], 4, 1, 128, 16, 0, 0.0, True),
    ([5, 40, 300], [5, 3, 300], 32, 8, 128, 32, 0, 0.0, True),
    ([129, 128, 127], [129, 128, 1], 16, 8, 128, 16, 0, 0.0, True),
    ([700, 0, 90], [200, 0, 90], 14, 2, 64, 32, 0, 0.0, True),
    ([1500], [1111], 8, 8, 128, 64, 0, 0.0, True),
    ([2500, 33], [37, 2], 12, 1, 128, 32, 0, 0.0, True),
    ([900, 300], [640, 300], 9, 3, 64, 16, 100, 0.0, True),
    ([900, 300], [640, 300], 8, 2, 128, 48, -256, 25.0, True),
    ([600, 50], [300, 50], 40, 2, 128, 32, 0, 0.0, True),                # twenty heads a group
    ([400, 31], [77, 31], 4, 2, 128, 32, 0, 0.0, False),
    ([400, 31], [77, 31], 6, 2, 256, 32, 50, 0.0, True),
    ([3000] * 9, [4, 5, 6, 1, 2, 3, 4, 5, 6], 32, 8, 128, 32, 0, 0.0, True),
    ([5000], [70], 32, 8, 128, 32, 0, 0.0, True),                        # few rows after a long context: every item is cut
    ([5000], [70], 4, 1, 64, 16, 0, 0.0, True),
    ([260, 3, 2000, 17], [130, 3, 5, 17], 24, 4, 128, 32, 0, 0.0, True), # sequences of both kernels
    ([130 + i for i in range(40)], [65 + i for i in range(40)], 8, 4, 128, 16, 0, 0.0, True),
    ([4000], [4000], 16, 2, 128, 32, 0, 0.0, True),
    ([4000, 500], [2048, 129], 8, 8, 64, 128, 700, 0.0, True),
    ([1300, 200], [900, 200], 16, 1, 128, 32, 0, 15.0, False),
    ([3000], [1500], 5, 1, 128, 16, -512, 0.0, True),
]


def _tiles(new):
    req, q0 = ref.build_prefill_tiles(new)
    return torch.tensor(req, dtype=torch.int32, device=DEV), torch.tensor(q0, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("lens,new,Hq,Hkv,D,bs,window,cap,causal", PREFILL)
def test_prefill(lens, new, Hq, Hkv, D, bs, window, cap, causal):
    q, cache, table, n = _case(lens, new, Hq, Hkv, D, bs, window, seed=sum(new))
    scale = D ** -0.5
    start = torch.tensor([0] + new).cumsum(0).int()
    req, q0 = _tiles(new)
    padded = torch.cat([q, torch.full((3, q.shape[1]), math.nan, dtype=q.dtype)]).to(DEV)    # rows behind the last sequence
    out = torch.full_like(padded, 7.0)
    args = dict(block_table=table.to(DEV), seq_lens=n.to(DEV), q_start=start.to(DEV), tile_req=req, tile_q0=q0, scale=scale, softcap=cap,
                window=window, causal=causal)
    C.prefill(padded, cache.to(DEV), out=out, **args)
    assert bool((out[sum(new):] == 7).all())
    _check(out, q, cache, table, lens, new, Hq, D, bs, scale, cap, window, causal)
    again = torch.full_like(out, 7.0)
    C.prefill(padded, cache.to(DEV), out=again, **args)
    assert torch.equal(again, out)
    assert _status() == 0


def test_queries_before_the_first_key_and_pages_outside_the_cache():
    """More new tokens than positions: the first rows see nothing and are zero. Table entries outside the cache are masked keys."""
    Hq, Hkv, D, bs = 4, 2, 64, 16
    gen = _gen(3)
    cache = F.random_cache(6, Hkv, bs, D, gen)
    q = torch.randn((10, Hq * D), generator=gen).to(torch.bfloat16)
    req, q0 = _tiles([10])
    table = torch.tensor([[1, 2, 3, 4]], dtype=torch.int32)
    out = C.prefill(q.to(DEV), cache.to(DEV), block_table=table.to(DEV), seq_lens=torch.tensor([6], dtype=torch.int32, device=DEV),
                    q_start=torch.tensor([0, 10], dtype=torch.int32, device=DEV), tile_req=req, tile_q0=q0, scale=0.1)
    assert not out[:4].any()
    k, v = C.ref_read(cache, torch.arange(16, 22))
    F.check_attention(out[4:].view(6, Hq, D).cpu(), *F.attention(q[4:].view(6, Hq, D), k, v, 0, 0.1, 0.0, 0))
    q = q[:3]
    table = torch.tensor([[1, -1, 3], [-5, 6, 1 << 30], [2, 6, 3]], dtype=torch.int32)
    n = torch.tensor([45, 48, 999], dtype=torch.int32)                  # (the last: longer than its row of the table)
    out = C.decode(q.to(DEV), cache.to(DEV), block_table=table.to(DEV), seq_lens=n.to(DEV), scale=0.1).cpu()
    assert not out[1].any()
    for r, slots in ((0, list(range(16, 32)) + list(range(48, 61))), (2, list(range(32, 48)) + list(range(48, 64)))):
        k, v = C.ref_read(cache, torch.tensor(slots))
        F.check_attention(out[r].view(1, Hq, D), *F.attention(q[r].view(1, Hq, D), k, v, len(slots), 0.1, 0.0, 0))


def test_pages_outside_the_cache_under_many_rows():
    Hq, Hkv, D, bs, n = 4, 2, 128, 16, 700
    gen = _gen(4)
    cache = F.random_cache(60, Hkv, bs, D, gen)
    table = torch.randperm(60, generator=gen)[: n // bs + 1].int()[None]
    gone = [3, 4, 17, 30]
    table[0, gone] = torch.tensor([-1, 60, 1 << 30, -(1 << 31)], dtype=torch.int32)
    q = torch.randn((n, Hq * D), generator=gen).to(torch.bfloat16)
    req, q0 = _tiles([n])
    out = C.prefill(q.to(DEV), cache.to(DEV), block_table=table.to(DEV), seq_lens=torch.tensor([n], dtype=torch.int32, device=DEV),
                    q_start=torch.tensor([0, n], dtype=torch.int32, device=DEV), tile_req=req, tile_q0=q0, scale=0.1).cpu()
    pos = torch.arange(n)
    there = ~torch.isin(pos // bs, torch.tensor(gone))
    k, v = C.ref_read(cache, table[0].long().clamp(0, 59)[pos // bs] * bs + pos % bs)
    for first in (0, 47, 48, 79, 80, 300, 699):                          # a row at a time, over the keys that it has
        seen = there & (pos <= first)
        want = F.attention(q[first].view(1, Hq, D), k[seen], v[seen], int(seen.sum()), 0.1, 0.0, 0)
        F.check_attention(out[first].view(1, Hq, D), *want)
    assert _status() == 0


def test_values_of_every_size():
    """Queries, keys and values far from 1, scores that rise along the sequence, and infinities and NaN that are somebody's keys."""
    D, bs, n = 128, 32, 600
    gen = _gen(8)
    x = torch.randn((2, n, 1, D), generator=gen)
    x[0] *= torch.linspace(0.01, 30, n)[:, None, None]                  # the running maximum is raised again and again
    x[1] *= torch.exp(4 * torch.randn((n, 1, 1), generator=gen))
    x = x.to(torch.bfloat16).to(DEV)
    table = torch.arange(n // bs + 1, dtype=torch.int32, device=DEV)[None]
    lens = torch.tensor([n], dtype=torch.int32, device=DEV)
    for size in (1e-30, 1e-3, 1.0, 1e4, 1e30):
        cache = C.alloc(n // bs + 1, 1, bs, D, DEV)
        C.write(x[0], x[1], cache, torch.arange(n, device=DEV))
        q = (torch.randn((1, 8 * D), generator=gen) * size).to(torch.bfloat16).to(DEV)
        scale = 0.02 / size
        out = C.decode(q, cache, block_table=table, seq_lens=lens, scale=scale)
        k, v = C.read(cache, torch.arange(n, device=DEV))
        F.check_attention(out.view(1, 8, D), *F.attention(q.view(1, 8, D), k, v, n - 1, scale, 0.0, 0))
    bad = x.clone()
    bad[1, 10, 0, 3] = math.nan                                         # a group of a value
    C.write(bad[0], bad[1], cache, torch.arange(n, device=DEV))
    out = C.decode(q, cache, block_table=table, seq_lens=lens, scale=scale).view(8, D)
    assert out[:, :16].isnan().all() and not out[:, 16:].isnan().any()
    bad[0, 10, 0, 3] = math.nan                                         # and of a key
    C.write(bad[0], bad[1], cache, torch.arange(n, device=DEV))
    assert C.decode(q, cache, block_table=table, seq_lens=lens, scale=scale).isnan().all()


def test_views_and_strides():
    """q and out inside wider rows, a table that is a part of a wider one, as an engine step hands them over."""
    lens, new, Hq, Hkv, D, bs = [100, 37, 260], [1, 1, 90], 8, 2, 128, 32
    q, cache, table, n = _case(lens, new, Hq, Hkv, D, bs, 0, seed=5)
    rows = torch.zeros((92, Hq * D + 512), dtype=torch.bfloat16, device=DEV)
    rows[:, 256: 256 + Hq * D] = q.to(DEV)
    qv = rows[:, 256: 256 + Hq * D]
    wide = torch.full((92, Hq * D + 64), 3.0, dtype=torch.bfloat16, device=DEV)
    ov = wide[:, 64:]
    big = torch.full((5, table.shape[1] + 7), 1 << 20, dtype=torch.int32, device=DEV)
    big[:3, : table.shape[1]] = table.to(DEV)
    bt = big[:3, : table.shape[1]]
    c, nd = cache.to(DEV), n.to(DEV)
    C.decode(qv[:2], c, block_table=bt[:2], seq_lens=nd[:2], scale=0.1, out=ov[:2])
    req, q0 = _tiles([90])
    C.prefill(qv[2:], c, block_table=bt[2:], seq_lens=nd[2:], q_start=torch.tensor([0, 90], dtype=torch.int32, device=DEV), tile_req=req,
              tile_q0=q0, scale=0.1, out=ov[2:])
    _check(ov, q, cache, table, lens, new, Hq, D, bs, 0.1, 0.0, 0)
    assert bool((wide[:, :64] == 3).all())


def test_nothing_to_do():
    cache = C.alloc(2, 2, 16, 64, DEV)
    q = torch.empty((0, 256), dtype=torch.bfloat16, device=DEV)
    table, none = torch.zeros((0, 1), dtype=torch.int32, device=DEV), torch.zeros(0, dtype=torch.int32, device=DEV)
    assert C.decode(q, cache, block_table=table, seq_lens=none, scale=1.0).shape == (0, 256)
    start = torch.zeros(1, dtype=torch.int32, device=DEV)
    assert C.prefill(q, cache, block_table=table, seq_lens=none, q_start=start, tile_req=none, tile_q0=none, scale=1.0).shape == (0, 256)
    slots = torch.zeros(0, dtype=torch.int64, device=DEV)
    C.append(torch.empty((0, 8 * 64), dtype=torch.bfloat16, device=DEV), None, None, cache, slots, num_q_heads=4)
    assert C.read(cache, slots)[0].shape == (0, 2, 64)


def test_refusals_on_a_gpu():
    cache = C.alloc(2, 2, 16, 64, DEV)
    q = torch.zeros((3, 256), dtype=torch.bfloat16, device=DEV)
    table, lens = torch.zeros((3, 2), dtype=torch.int32, device=DEV), torch.ones(3, dtype=torch.int32, device=DEV)
    for bad in (dict(block_table=table[:2]), dict(seq_lens=lens[:2]), dict(seq_lens=lens.long()), dict(seq_lens=lens.cpu()),
                dict(tmp=torch.empty(10, device=DEV))):
        with pytest.raises(OpArgumentError):
            C.decode(q, cache, **{**dict(block_table=table, seq_lens=lens, scale=1.0), **bad})
    with pytest.raises(OpArgumentError):
        C.read(cache, torch.zeros(3, dtype=torch.int64, device=DEV), torch.empty((3, 2, 64), device=DEV))


# --------------------------------------------------------------------------------------------------- run together
def test_a_sequence_grows_token_by_token():
    """Append and attend in turn, as an engine does: a prompt, then single tokens, over pages in no order. Each step against attention
    over what the cache should hold."""
    Hq, Hkv, D, bs, P, steps = 8, 2, 64, 16, 37, 20
    gen = _gen(11)
    total = P + steps
    rows = torch.randn((total, (Hq + 2 * Hkv) * D), generator=gen).to(torch.bfloat16).to(DEV)
    table = ref.rope_table(ref.rope_inv_freq(D, 1e4), 100).to(DEV)
    pages = torch.tensor([[4, 1, 3, 2]], dtype=torch.int32, device=DEV)
    pos = torch.arange(total, device=DEV)
    slots = pages[0].long()[pos // bs] * bs + pos % bs
    cache = C.alloc(5, Hkv, bs, D, DEV)
    cos, sin = table[pos].chunk(2, -1)
    x = rows.view(total, Hq + 2 * Hkv, D)
    q_all, _ = F.rotated(x[:, :Hq], None, 0, False, cos, sin, D, True)
    k_all, big = F.rotated(x[:, Hq: Hq + Hkv], None, 0, False, cos, sin, D, True)

    def step(a, b):
        qkv = rows[a:b].clone()
        C.append(qkv, pos[a:b], table, cache, slots[a:b], num_q_heads=Hq)
        n = torch.tensor([b], dtype=torch.int32, device=DEV)
        if b - a == 1:
            out = C.decode(qkv[:, : Hq * D], cache, block_table=pages, seq_lens=n, scale=0.125)
        else:
            req, q0 = _tiles([b - a])
            out = C.prefill(qkv[:, : Hq * D], cache, block_table=pages, seq_lens=n, tile_req=req, tile_q0=q0, scale=0.125,
                            q_start=torch.tensor([0, b - a], dtype=torch.int32, device=DEV))
        k, v = C.read(cache, slots[:b])
        F.check_held(k, k_all[:b], big[:b])
        q = qkv[:, : Hq * D].view(b - a, Hq, D)
        assert bool(((q.double() - q_all[a:b]).abs() <= 2.0 ** -8 * q_all[a:b].abs() + 1e-4).all())
        F.check_attention(out.view(b - a, Hq, D), *F.attention(q, k, v, a, 0.125, 0.0, 0))
    step(0, P)
    for t in range(P, total):
        step(t, t + 1)


def test_captured_and_replayed_with_other_lengths():
    lens, Hq, Hkv, D, bs = [900, 20, 333, 1], 16, 4, 128, 32
    q, cache, table, _ = _case(lens, [1] * 4, Hq, Hkv, D, bs, 0, seed=2)
    cache = F.random_cache(cache.shape[0], Hkv, bs, D, _gen(1))
    qd, c, bt = q.to(DEV), cache.to(DEV), table.to(DEV)
    n = torch.tensor(lens, dtype=torch.int32, device=DEV)
    out = torch.empty_like(qd)

    def run():
        C.decode(qd, c, block_table=bt, seq_lens=n, scale=0.09, out=out)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        run()
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        run()
    for now in ([5, 20, 0, 1], [900, 1, 333, 17], [0, 0, 0, 0], lens):
        n.copy_(torch.tensor(now, dtype=torch.int32))
        out.fill_(9)
        g.replay()
        torch.cuda.synchronize()
        _check(out, q, cache, table, now, [1] * 4, Hq, D, bs, 0.09, 0.0, 0)


def test_two_streams_at_once():
    """Calls side by side, each with scratch of its own (the default)."""
    Hq, Hkv, D, bs = 8, 2, 128, 32
    work = []
    for i, lens in enumerate(([3000, 50], [40, 2500, 900])):
        q, cache, table, n = _case(lens, [1] * len(lens), Hq, Hkv, D, bs, 0, seed=20 + i)
        args = (q.to(DEV), cache.to(DEV)), dict(block_table=table.to(DEV), seq_lens=n.to(DEV), scale=0.1)
        work.append((args, C.decode(*args[0], **args[1]), torch.cuda.Stream()))
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, ((a, kw), _, s) in enumerate(work):
            with torch.cuda.stream(s):
                got[i].append(C.decode(*a, **kw))
    torch.cuda.synchronize()
    for i, (_, want, _) in enumerate(work):
        assert all(torch.equal(x, want) for x in got[i])


BORDER = [
    # sequences on both sides of the line between the kernels (48 rows), and of the rule for row tiles of 8 and 16
    ([400] * 6, [11, 12, 13, 12, 1, 130], 16, 4, 128, 32),
    ([90, 49, 48, 47], [90, 49, 48, 47], 4, 4, 64, 16),
    ([700] * 5, [1, 2, 1, 1, 1], 8, 2, 128, 32),
    ([700] * 5, [3, 2, 1, 4, 2], 8, 2, 128, 32),
    ([300, 49, 70], [48, 49, 3], 3, 3, 256, 16),
]


@pytest.mark.parametrize("lens,new,Hq,Hkv,D,bs", BORDER)
def test_both_sides_of_the_choices(lens, new, Hq, Hkv, D, bs):
    q, cache, table, n = _case(lens, new, Hq, Hkv, D, bs, 0, seed=sum(lens))
    req, q0 = _tiles(new)
    out = C.prefill(q.to(DEV), cache.to(DEV), block_table=table.to(DEV), seq_lens=n.to(DEV), q_start=torch.tensor([0] + new).cumsum(0).int().to(DEV),
                    tile_req=req, tile_q0=q0, scale=0.1)
    _check(out, q, cache, table, lens, new, Hq, D, bs, 0.1, 0.0, 0)
    assert _status() == 0


@pytest.mark.parametrize("D,Hq,Hkv", [(64, 1, 1), (128, 2, 1), (128, 16, 1), (256, 1, 1)])
def test_as_many_sequences_as_a_call_takes(D, Hq, Hkv):
    """8192 sequences of 0 to 3 keys, in pages that neighbours share."""
    R, bs, gen = 8192, 16, _gen(D + Hq)
    cache = F.random_cache(9, Hkv, bs, D, gen)
    page = torch.randint(0, 9, (R, 1), generator=gen, dtype=torch.int32)
    n = torch.randint(0, 4, (R,), generator=gen, dtype=torch.int32)
    q = torch.randn((R, Hq * D), generator=gen).to(torch.bfloat16)
    got = C.decode(q.to(DEV), cache.to(DEV), block_table=page.to(DEV), seq_lens=n.to(DEV), scale=0.1).cpu()
    for at in range(9):
        for length in range(4):
            rows = ((page[:, 0] == at) & (n == length)).nonzero()[:, 0]
            if length == 0:
                assert not got[rows].any()
                continue
            k, v = C.ref_read(cache, torch.arange(at * bs, at * bs + length))
            want = F.attention(q[rows].view(len(rows), Hq, D), k, v, 0, 0.1, 0.0, 0, causal=False)
            F.check_attention(got[rows].view(len(rows), Hq, D), *want)
    assert _status() == 0


@pytest.mark.parametrize("window", [1, 2 ** 31 - 1, -(2 ** 31 - 1)])
def test_windows_of_one_key_and_past_every_sequence(window):
    lens, new, Hq, Hkv, D, bs = [300, 1, 65], [300, 1, 2], 4, 2, 128, 16
    q, cache, table, n = _case(lens, new, Hq, Hkv, D, bs, 1 if window == 1 else 0, seed=9)
    req, q0 = _tiles(new)
    args = dict(block_table=table.to(DEV), seq_lens=n.to(DEV), scale=0.1, window=window)
    out = C.prefill(q.to(DEV), cache.to(DEV), q_start=torch.tensor([0] + new).cumsum(0).int().to(DEV), tile_req=req, tile_q0=q0, **args)
    _check(out, q, cache, table, lens, new, Hq, D, bs, 0.1, 0.0, 1 if window == 1 else 0)
    last = torch.tensor(new).cumsum(0) - 1
    out = C.decode(q[last].to(DEV), cache.to(DEV), **args)
    _check(out, q[last], cache, table, lens, [1] * 3, Hq, D, bs, 0.1, 0.0, 1 if window == 1 else 0)


def test_a_tile_listed_twice_and_pages_that_sequences_share():
    lens, new, Hq, Hkv, D, bs = [700, 690], [300, 290], 8, 2, 128, 32
    q, cache, table, n = _case(lens, new, Hq, Hkv, D, bs, 0, seed=31)
    table[1] = table[0]
    req, q0 = _tiles(new)
    req, q0 = torch.cat([req, req[:2]]), torch.cat([q0, q0[:2]])
    out = C.prefill(q.to(DEV), cache.to(DEV), block_table=table.to(DEV), seq_lens=n.to(DEV), q_start=torch.tensor([0, 300, 590], dtype=torch.int32, device=DEV),
                    tile_req=req, tile_q0=q0, scale=0.1)
    _check(out, q, cache, table, lens, new, Hq, D, bs, 0.1, 0.0, 0)


def test_two_graphs_that_share_scratch():
    """Two steps captured over one scratch, replayed one after the other in both orders, with lengths that change."""
    Hq, Hkv, D, bs, new = 8, 2, 128, 32, [40, 3]
    one, two = ([900, 700], 2), ([1300, 64], 5)
    tmp = C.scratch(torch.device(DEV, torch.cuda.current_device()), D)
    req, q0 = _tiles(new)
    start = torch.tensor([0, 40, 43], dtype=torch.int32, device=DEV)
    graphs = []
    for lens, seed in (one, two):
        q, cache, table, n = _case(lens, new, Hq, Hkv, D, bs, 0, seed=seed)
        t = [x.to(DEV) for x in (q, cache, table, n)]
        out = torch.empty_like(t[0])

        def run(t=t, out=out):
            C.prefill(t[0], t[1], block_table=t[2], seq_lens=t[3], q_start=start, tile_req=req, tile_q0=q0, scale=0.1, out=out, tmp=tmp)
        run()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            run()
        graphs.append((g, out, (q, cache, table, lens), t))      # (the graph reads what t holds)
    for order in ((0, 1), (1, 0), (0, 0, 1)):
        for _, out, _, _ in graphs:
            out.fill_(5)
        for i in order:
            graphs[i][0].replay()
        torch.cuda.synchronize()
        for _, out, (q, cache, table, lens), _ in graphs:
            _check(out, q, cache, table, lens, new, Hq, D, bs, 0.1, 0.0, 0)


def test_two_threads_at_once():
    import threading
    Hq, Hkv, D, bs = 8, 2, 64, 32
    work = []
    for i, (lens, new) in enumerate((([500, 50], [200, 50]), ([40, 2500, 900], [3, 700, 9]))):
        q, cache, table, n = _case(lens, new, Hq, Hkv, D, bs, 0, seed=40 + i)
        req, q0 = _tiles(new)
        work.append(((q.to(DEV), cache.to(DEV)), dict(block_table=table.to(DEV), seq_lens=n.to(DEV), tile_req=req, tile_q0=q0, scale=0.1,
                                                      q_start=torch.tensor([0] + new).cumsum(0).int().to(DEV)), (q, cache, table, lens, new)))
    torch.cuda.synchronize()
    got, errors = [[], []], []

    def thread(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(10):
                    got[i].append(C.prefill(*work[i][0], **work[i][1]))
        except Exception as e:                                   # (a thread's exception does not end the test by itself)
            errors.append(e)
    threads = [threading.Thread(target=thread, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors
    for i, (_, _, (q, cache, table, lens, new)) in enumerate(work):
        for out in got[i]:
            _check(out, q, cache, table, lens, new, Hq, D, bs, 0.1, 0.0, 0)


APPEND_MANY = [
    # several passes a warp; heads that do not fill the last one, and passes with query and key heads
    (2050, 7, 3, 64, 20, True, True, False, 16),
    (5000, 7, 3, 64, 64, True, False, False, 32),
    (1400, 5, 3, 128, 96, False, True, True, 48),
    (700, 12, 2, 256, 256, True, True, False, 64),
    (9000, 0, 1, 128, 128, True, False, False, 16),
]


@pytest.mark.parametrize("T,Hq,Hkv,D,rot,neox,normed,gemma,bs", APPEND_MANY)
def test_append_of_many_tokens(T, Hq, Hkv, D, rot, neox, normed, gemma, bs):
    for in_place in (False, True):
        test_append(T, Hq, Hkv, D, rot, neox, normed, gemma, bs, in_place)


@pytest.mark.parametrize("n,H,D", [(20001, 1, 64), (9000, 3, 128), (6001, 5, 256)])
def test_read_of_many_tokens(n, H, D):
    """Slots in any order, some twice, some outside."""
    bs, nb, gen = 16, 40, _gen(n)
    cache = F.random_cache(nb, H, bs, D, gen)
    slots = torch.randint(-3, nb * bs + 3, (n,), generator=gen)
    k, v = C.read(cache.to(DEV), slots.to(DEV))
    rk, rv = C.ref_read(cache, slots)
    assert torch.equal(k.cpu(), rk) and torch.equal(v.cpu(), rv)


@pytest.mark.parametrize("D", [64, 128])
def test_as_many_tiles_as_a_call_takes(D):
    """8000 tiles: those of two prompts, over and over."""
    lens, new, Hq, Hkv, bs = [200, 150], [200, 150], 2, 1, 16
    q, cache, table, n = _case(lens, new, Hq, Hkv, D, bs, 0, seed=D)
    req, q0 = _tiles(new)
    out = C.prefill(q.to(DEV), cache.to(DEV), block_table=table.to(DEV), seq_lens=n.to(DEV), q_start=torch.tensor([0, 200, 350], dtype=torch.int32, device=DEV),
                    tile_req=req.repeat(2000), tile_q0=q0.repeat(2000), scale=0.1)
    _check(out, q, cache, table, lens, new, Hq, D, bs, 0.1, 0.0, 0)
    assert _status() == 0


@pytest.mark.parametrize("said", [3, 12, 13, 200, 10 ** 6])
def test_the_longest_sequence_only_chooses_between_kernels(said):
    """Whatever is said of it, also what is not so."""
    lens, new, Hq, Hkv, D, bs = [900, 300, 12, 77], [12, 13, 2, 40], 16, 4, 128, 32
    q, cache, table, n = _case(lens, new, Hq, Hkv, D, bs, 0, seed=77)
    req, q0 = _tiles(new)
    out = C.prefill(q.to(DEV), cache.to(DEV), block_table=table.to(DEV), seq_lens=n.to(DEV), q_start=torch.tensor([0] + new).cumsum(0).int().to(DEV),
                    tile_req=req, tile_q0=q0, scale=0.1, max_query_len=said)
    _check(out, q, cache, table, lens, new, Hq, D, bs, 0.1, 0.0, 0)
    assert _status() == 0


def test_refusals_of_lines_past_31_bits():
    """What the lengths allow at most, whatever they are: the kernels count cells in 31 bits."""
    from vllm_cpp_b200.ops._lib import KernelError
    cache = C.alloc(1, 1, 2048, 64, DEV)
    q = torch.zeros((128, 4 * 64), dtype=torch.bfloat16, device=DEV)
    lens, start = torch.full((1,), 128, dtype=torch.int32, device=DEV), torch.tensor([0, 128], dtype=torch.int32, device=DEV)
    ids = torch.zeros(8000, dtype=torch.int32, device=DEV)
    for pages, tiles, ok in ((1 << 14, 8000, False), (1 << 14, 1, True), (1 << 20, 1, False)):
        args = dict(block_table=torch.zeros((1, pages), dtype=torch.int32, device=DEV), seq_lens=lens, q_start=start, tile_req=ids[:tiles],
                    tile_q0=ids[:tiles], scale=0.1)
        if ok:
            assert not C.prefill(q, cache, **args).any()
        else:
            with pytest.raises(KernelError, match="-4"):
                C.prefill(q, cache, **args)


def test_sequences_that_share_query_rows():
    """Bounds that go back: the second sequence has no rows, the third those of the first, over keys of its own or the same."""
    lens, Hq, Hkv, D, bs = [100, 5, 100], 8, 2, 128, 16
    q, cache, table, n = _case(lens, [70, 0, 0], Hq, Hkv, D, bs, 0, seed=6)
    table[2] = table[0]
    req, q0 = _tiles([70, 0, 70])
    out = C.prefill(q.to(DEV), cache.to(DEV), block_table=table.to(DEV), seq_lens=n.to(DEV), q_start=torch.tensor([0, 70, 0, 70], dtype=torch.int32, device=DEV),
                    tile_req=req, tile_q0=q0, scale=0.1)
    _check(out, q, cache, table, [100], [70], Hq, D, bs, 0.1, 0.0, 0)


def test_bounds_that_overlap_until_the_line_is_too_long():
    """4096 sequences that each claim all query rows: more cells than 31 bits count. The call does nothing."""
    R, H, D, bs, keys = 8192, 16, 256, 2048, 32768
    cache = C.alloc(1, H, bs, D, DEV)
    q = torch.ones((16, 16 * H * D), dtype=torch.bfloat16, device=DEV)
    start = (torch.arange(R + 1, dtype=torch.int32, device=DEV) % 2) * 16
    ids = torch.zeros(1, dtype=torch.int32, device=DEV)
    out = torch.full_like(q, 7.0)
    C.prefill(q, cache, block_table=torch.zeros((R, keys // bs), dtype=torch.int32, device=DEV), q_start=start, tile_req=ids, tile_q0=ids,
              seq_lens=torch.full((R,), keys, dtype=torch.int32, device=DEV), scale=0.1, out=out)
    assert bool((out == 7.0).all())
    assert _status() == 0
