"""Results that a call writes lie apart from the rows that it reads: views of one buffer that share bytes are refused, columns of the same rows that
do not are taken."""
import pytest
import torch

import fp4_reference as F
from vllm_cpp_b200.ops import fp4_cache as C
from vllm_cpp_b200.ops import reference as ref
from vllm_cpp_b200.ops.validate import OpArgumentError, _apart_rows


def _refused(rule, call, *a, **kw):
    with pytest.raises(OpArgumentError, match=rule):
        call(*a, **kw)


def test_rows_that_share_bytes_are_found():
    """Against the sets of elements, for rows of any width and distance."""
    gen = torch.Generator().manual_seed(0)
    buf = torch.arange(400, dtype=torch.int16)
    seen = set()
    for _ in range(3000):
        views = []
        for _ in range(2):
            at, n, ld, w = (int(torch.randint(0, hi, (1,), generator=gen)) for hi in (120, 6, 40, 12))
            views.append(buf.as_strided((n, w), (ld, 1), at))
        a, b = views
        shared = bool(set(a.flatten().tolist()) & set(b.flatten().tolist()))
        assert _apart_rows(a, b) is not shared
        seen.add(shared)
    assert seen == {True, False}


def test_results_over_the_queries():
    cache = C.alloc(2, 2, 16, 64, "cpu")
    table, lens = torch.zeros((3, 2), dtype=torch.int32), torch.ones(3, dtype=torch.int32)
    good = dict(block_table=table, seq_lens=lens, scale=1.0)
    ids = torch.zeros(4, dtype=torch.int32)
    buf = torch.zeros((8, 640), dtype=torch.bfloat16)
    q = buf[1:4, :256]
    for out in (buf[1:4, :256], buf[2:5, :256], buf[3:6, :256], buf[:3, :256], buf[1:4, 8:264], buf[1:4, 248:504], buf.flatten()[640 + 128:][:768].view(3, 256)):
        _refused("out is like q", C.decode, q, cache, out=out, **good)
        _refused("out is like q", C.prefill, q, cache, out=out, q_start=ids, tile_req=ids, tile_q0=ids, **good)
    for out in (buf[4:7, :256], buf[1:4, 256:512], buf[1:4, 384:], buf[2:5, 256:512], buf.flatten()[640 * 4:][:768].view(3, 256)):
        _refused("one GPU", C.decode, q, cache, out=out, **good)           # (taken but for the device)
        _refused("one GPU", C.prefill, q, cache, out=out, q_start=ids, tile_req=ids, tile_q0=ids, **good)


def test_queries_over_keys_and_values():
    cache = C.alloc(2, 2, 16, 64, "cpu")
    slots = torch.zeros(3, dtype=torch.int64)
    buf = torch.zeros((8, 1280), dtype=torch.bfloat16)
    qkv = buf[1:4, :640]                                       # six heads, two of keys, two of values
    for q_out in (buf[1:4, :384], buf[1:4, 8:392], buf[1:4, 512:896], buf[2:5, 256:640], buf[0:3, 632:1016]):
        _refused("q_out lies apart", C.append, qkv, None, None, cache, slots, num_q_heads=6, q_out=q_out)
    for q_out in (buf[4:7, :384], buf[1:4, 640:1024], buf[2:5, 896:]):
        _refused("one GPU", C.append, qkv, None, None, cache, slots, num_q_heads=6, q_out=q_out)
    wide = buf[1:4]                                            # columns that are not read
    kw = dict(num_q_heads=2, q_head_stride=320, offsets=(0, 640, 768))
    _refused("one GPU", C.append, wide, None, None, cache, slots, q_out=wide[:, 64:192], **kw)
    _refused("one GPU", C.append, wide, None, None, cache, slots, q_out=wide[:, 896:1024], **kw)
    _refused("q_out lies apart", C.append, wide, None, None, cache, slots, q_out=wide[:, 56:184], **kw)
    _refused("q_out lies apart", C.append, wide, None, None, cache, slots, q_out=wide[:, 888:1016], **kw)


def test_keys_over_values_read_back():
    cache, slots = C.alloc(2, 2, 16, 64, "cpu"), torch.zeros(3, dtype=torch.int64)
    buf = torch.zeros((8, 2, 64), dtype=torch.bfloat16)
    _refused("k and v lie apart", C.read, cache, slots, buf[:3], buf[:3])
    _refused("k and v lie apart", C.read, cache, slots, buf[:3], buf[2:5])
    _refused("one GPU", C.read, cache, slots, buf[:3], buf[3:6])


@pytest.mark.gpu
def test_columns_of_the_same_rows():
    """Queries, their rotated form and results in one buffer, side by side."""
    Hq, Hkv, D, bs, n = 4, 2, 64, 16, 50
    gen = torch.Generator().manual_seed(1)
    cols = (Hq + 2 * Hkv) * D
    buf = torch.randn((n, cols + 2 * Hq * D), generator=gen).to(torch.bfloat16).cuda()
    before = buf.clone()
    qkv, q, out = buf[:, :cols], buf[:, cols: cols + Hq * D], buf[:, cols + Hq * D:]
    cache = C.alloc(4, Hkv, bs, D, "cuda")
    C.append(qkv, None, None, cache, torch.arange(n, device="cuda"), num_q_heads=Hq, q_out=q)
    assert torch.equal(buf[:, :cols], before[:, :cols]) and torch.equal(q, before[:, : Hq * D])
    table, lens = torch.arange(4, dtype=torch.int32, device="cuda")[None], torch.tensor([n], dtype=torch.int32, device="cuda")
    req, q0 = (torch.tensor(t, dtype=torch.int32, device="cuda") for t in ref.build_prefill_tiles([n]))
    start = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    C.prefill(q, cache, block_table=table, seq_lens=lens, q_start=start, tile_req=req, tile_q0=q0, scale=0.125, out=out)
    k, v = C.read(cache, torch.arange(n, device="cuda"))
    F.check_attention(out.view(n, Hq, D), *F.attention(q.view(n, Hq, D), k, v, 0, 0.125, 0.0, 0))
    C.decode(q[-1:], cache, block_table=table, seq_lens=lens, scale=0.125, out=out[:1])
    F.check_attention(out[:1].view(1, Hq, D), *F.attention(q[-1:].view(1, Hq, D), k, v, n - 1, 0.125, 0.0, 0))
    with pytest.raises(OpArgumentError, match="out is like q"):
        C.decode(q[:1], cache, block_table=table, seq_lens=lens, scale=0.125, out=buf[:1, cols + 8: cols + 8 + Hq * D])
    with pytest.raises(OpArgumentError, match="q_out lies apart"):
        C.append(qkv, None, None, cache, torch.arange(n, device="cuda"), num_q_heads=Hq, q_out=buf[:, 256: 512])
