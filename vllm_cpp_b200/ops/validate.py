"""One validation layer in front of the kernel launchers: every op lists its argument contract as
named rules over the tensors it is given; ``validate(op, **args)`` raises :class:`OpArgumentError`
naming the op, the rule that failed and the offending shapes before anything is launched. The C
launchers keep their own checks (they return -1); this layer is what turns a bad call into a
message a caller can act on, the same for every op.

Reference: the ``Validate*`` helpers of ``include/vt/ops.h`` / ``src/vt/ops.cpp`` (uniform
shape / dtype / layout errors in front of every backend).
"""
from __future__ import annotations

import itertools
import math

import torch


class OpArgumentError(ValueError):
    def __init__(self, op: str, rule: str, detail: str):
        super().__init__(f"{op}: {rule} ({detail})")
        self.op, self.rule = op, rule


def _desc(**t) -> str:
    parts = []
    for k, v in t.items():
        if isinstance(v, torch.Tensor):
            parts.append(f"{k}={tuple(v.shape)} {str(v.dtype).replace('torch.', '')} stride={tuple(v.stride())}")
        elif isinstance(v, list):
            parts.append(f"{k}=[{'; '.join(_desc(**{str(i): t}) for i, t in enumerate(v[:4]))}{'; ...' if len(v) > 4 else ''}]")
        elif v is not None:
            parts.append(f"{k}={v}")
    return ", ".join(parts)


def _rows16(t: torch.Tensor) -> bool:
    """Row-contiguous with 16-byte aligned rows: what a TMA tensor map needs."""
    return t.stride(-1) == 1 and (t.dim() < 2 or (t.stride(-2) * t.element_size()) % 16 == 0) \
        and t.data_ptr() % 16 == 0


BF16 = torch.bfloat16
# Numbers that are 0 in 32 bits; the largest whose log2(e)-fold is finite there.
LEAST_F32, MOST_LOG2_F32 = 2.0 ** -150, 2.35e38

RULES: dict[str, list] = {
    "gemm": [
        ("a and w are bf16", lambda a, w, **_: a.dtype == BF16 and w.dtype == BF16),
        ("a is [M, K] and w is [N, K] with the same K", lambda a, w, **_: a.dim() == 2 and w.dim() == 2
         and a.shape[1] == w.shape[1]),
        ("rows are contiguous and 16-byte aligned", lambda a, w, **_: _rows16(a) and _rows16(w)),
        ("out is [M, N], bf16 or fp32, row-contiguous", lambda a, w, out=None, **_: out is None or (
            out.shape == (a.shape[0], w.shape[0]) and out.dtype in (BF16, torch.float32) and out.stride(1) == 1)),
        ("bias is bf16 [N]", lambda w, bias=None, **_: bias is None or (bias.dtype == BF16 and bias.numel() == w.shape[0])),
        ("residual is bf16 [M, N]", lambda a, w, residual=None, **_: residual is None or (
            residual.dtype == BF16 and residual.shape == (a.shape[0], w.shape[0]))),
    ],
    "gemm_nvfp4": [
        ("packed operands are uint8 [rows, K/2] with the same K", lambda aq, wq, **_: aq.dtype == torch.uint8
         and wq.dtype == torch.uint8 and aq.dim() == 2 and wq.dim() == 2 and aq.shape[1] == wq.shape[1]),
        ("K is a multiple of 256", lambda aq, **_: (aq.shape[1] * 2) % 256 == 0),
        ("N is a multiple of 8", lambda wq, **_: wq.shape[0] % 8 == 0),
        ("scale chunks cover the padded rows", lambda aq, wq, sfa, sfw, **_: sfa.numel() >= -(-aq.shape[0] // 128) * 128
         * (aq.shape[1] // 8) and sfw.numel() >= -(-wq.shape[0] // 128) * 128 * (wq.shape[1] // 8)),
        ("global scales are fp32 scalars on the device", lambda g_a, g_w, aq, **_: g_a.dtype == torch.float32
         and g_w.dtype == torch.float32 and g_a.device == aq.device and g_w.device == aq.device),
    ],
    "rmsnorm": [
        ("x is [T, H] bf16, row-contiguous", lambda x, **_: x.dim() == 2 and x.dtype == BF16 and x.stride(1) == 1),
        ("weight has H elements", lambda x, weight, **_: weight.numel() == x.shape[1]),
        ("residual is contiguous [T, H]", lambda x, residual=None, **_: residual is None or (
            residual.is_contiguous() and residual.shape == x.shape)),
    ],
    "attn_decode": [
        ("q is [B, Hq * D] bf16, row-contiguous", lambda q, num_q_heads, head_dim, **_: q.dim() == 2
         and q.dtype == BF16 and q.shape[1] == num_q_heads * head_dim and q.stride(1) == 1),
        ("kv_cache is [blocks, 2, block_size, Hkv, D]", lambda kv_cache, num_kv_heads, head_dim, block_size, **_:
         kv_cache.dim() == 5 and tuple(kv_cache.shape[1:]) == (2, block_size, num_kv_heads, head_dim)),
        ("Hq is a multiple of Hkv", lambda num_q_heads, num_kv_heads, **_: num_q_heads % num_kv_heads == 0),
        ("head_dim is 64, 128 or 256", lambda head_dim, **_: head_dim in (64, 128, 256)),
        ("block_table and seq_lens are int32 with B rows", lambda q, block_table, seq_lens, **_:
         block_table.dtype == torch.int32 and seq_lens.dtype == torch.int32 and block_table.shape[0] >= q.shape[0]
         and seq_lens.numel() >= q.shape[0]),
    ],
    "attn_prefill": [
        ("q is [T, Hq * D] bf16, row-contiguous", lambda q, num_q_heads, head_dim, **_: q.dim() == 2
         and q.dtype == BF16 and q.shape[1] == num_q_heads * head_dim and q.stride(1) == 1),
        ("kv_cache is [blocks, 2, block_size, Hkv, D]", lambda kv_cache, num_kv_heads, head_dim, block_size, **_:
         kv_cache.dim() == 5 and tuple(kv_cache.shape[1:]) == (2, block_size, num_kv_heads, head_dim)),
        ("head_dim is 64, 128 or 256", lambda head_dim, **_: head_dim in (64, 128, 256)),
        ("page size divides or is a multiple of 64", lambda block_size, **_: block_size >= 8 and block_size % 8 == 0
         and (64 % block_size == 0 or block_size % 64 == 0)),
        ("tile table entries are int32", lambda tile_req, tile_q0, **_: tile_req.dtype == torch.int32
         and tile_q0.dtype == torch.int32 and tile_req.numel() == tile_q0.numel()),
    ],
    "moe_grouped_gemm": [
        ("w is [E, N, K] bf16", lambda w, **_: w.dim() == 3 and w.dtype == BF16),
        ("xs is [rows, K] bf16 with the weights' K", lambda xs, w, **_: xs.dim() == 2 and xs.dtype == BF16
         and xs.shape[1] == w.shape[2]),
        ("N and K are multiples of 8", lambda w, **_: w.shape[1] % 8 == 0 and w.shape[2] % 8 == 0),
    ],
}


def _fp4_cache(cache, **_) -> bool:
    return cache.dim() == 4 and cache.dtype == torch.uint8 and cache.is_contiguous() and cache.shape[3] in (64 * 18, 128 * 18, 256 * 18) \
        and cache.shape[2] > 0 and cache.data_ptr() % 16 == 0


def _on_gpu(*tensors) -> bool:
    """All of them (None apart) on one GPU."""
    dev = {t.device for t in tensors if t is not None}
    return len(dev) == 1 and next(iter(dev)).type == "cuda"


def _ids(t, dtype, n) -> bool:
    return t.dtype == dtype and t.dim() == 1 and t.numel() >= n and t.is_contiguous()


def _bf16_rows(t) -> bool:
    return t.dim() == 2 and t.dtype == BF16 and (t.shape[0] <= 1 or _rows16(t)) and (t.shape[1] <= 1 or t.stride(1) == 1) and t.data_ptr() % 16 == 0


def _apart(t) -> bool:
    """Rows that a kernel may write: none begins inside another."""
    return t.shape[0] <= 1 or t.stride(0) >= t.shape[1]


def _apart_from_keys(H, D, num_q_heads, stride, offsets) -> bool:
    """Query heads that a kernel may write in place lie apart from one another and from the keys and values."""
    heads = [(offsets[0] + i * stride, offsets[0] + i * stride + D) for i in range(num_q_heads)]
    return (num_q_heads <= 1 or stride >= D) and not any(a < o + H * D and o < b for a, b in heads for o in offsets[1:])


def _apart_rows(a, b) -> bool:
    """No byte of the rows of ``a`` is one of the rows of ``b`` (2-d, columns side by side, any distance between rows)."""
    if a.numel() == 0 or b.numel() == 0:
        return True
    (pa, na, la, wa), (pb, nb, lb, wb) = ((t.data_ptr(), t.shape[0], t.stride(0) * t.element_size() if t.shape[0] > 1 else 0,
                                           t.shape[1] * t.element_size()) for t in (a, b))
    if pa + (na - 1) * la + wa <= pb or pb + (nb - 1) * lb + wb <= pa:
        return True
    first = pa + la * torch.arange(na)
    other = pb + lb * torch.arange(nb)
    # of a's rows as many end at or before a row of b as begin before its end
    return torch.equal(torch.searchsorted(first, other + wb), torch.searchsorted(first + wa, other, right=True))


def _apart_from_heads(q_out, qkv, cache, num_q_heads, stride, offsets) -> bool:
    """Query rows that go elsewhere lie apart from the heads that are read."""
    D, T = cache.shape[3] // 18, qkv.shape[0]
    read = [(offsets[0] + i * stride, D) for i in range(num_q_heads)] + [(o, cache.shape[1] * D) for o in offsets[1:]]
    return _apart_rows(q_out[:T], qkv) or all(_apart_rows(q_out[:T], qkv[:, at: at + n]) for at, n in read)


_FP4_CACHE = ("cache is uint8 [blocks, kv heads, block_size / 16, 18 head_dim], contiguous, head_dim 64, 128 or 256", _fp4_cache)
_FP4_ATTN = [
    _FP4_CACHE,
    ("q is [rows, Hq * head_dim] bf16 with rows on 16-byte boundaries, Hq a multiple of the kv heads", lambda q, cache, **_: _bf16_rows(q)
     and q.shape[1] > 0 and q.shape[1] % (cache.shape[3] // 18 * cache.shape[1]) == 0),
    ("out is like q and apart from it, its rows apart from one another", lambda q, out, **_: _bf16_rows(out) and out.shape == q.shape and _apart(out)
     and _apart_rows(q, out)),
    ("block_table is int32 [sequences, pages], rows contiguous", lambda block_table, **_: block_table.dtype == torch.int32
     and block_table.dim() == 2 and block_table.shape[1] > 0 and (block_table.shape[1] == 1 or block_table.stride(1) == 1)),
    ("scale is positive, softcap finite and not negative, window in 32 bits", lambda scale, softcap, window=0, **_: scale > 0
     and 0 <= softcap < math.inf and -2 ** 31 < window < 2 ** 31),
    ("there are at most 8192 sequences and 8000 tiles", lambda q, block_table, seq_lens, tile_req=None, q_start=None, **_: (
        q.shape[0] if q_start is None else min(block_table.shape[0], seq_lens.numel(), q_start.numel() - 1)) <= 8192 and (
            tile_req is None or tile_req.numel() <= 8000)),
    ("tmp is fp32 and large enough", lambda cache, q_start=None, tmp=None, **_: tmp is None or (
        tmp.dtype == torch.float32 and tmp.is_contiguous() and tmp.data_ptr() % 16 == 0
        and tmp.numel() >= _fp4_scratch(cache, q_start is not None))),
    ("all tensors are on one GPU", lambda q, cache, block_table, seq_lens, out, q_start=None, tile_req=None, tile_q0=None, tmp=None, **_:
     _on_gpu(q, cache, block_table, seq_lens, out, q_start, tile_req, tile_q0, tmp)),
]


def _fp4_scratch(cache, prefill) -> int:
    from .fp4_cache import scratch_floats
    return scratch_floats(cache.device, cache.shape[3] // 18, prefill)


RULES.update({
    "fp4_append": [
        _FP4_CACHE,
        ("qkv is [T, columns] bf16 with rows on 16-byte boundaries", lambda qkv, **_: _bf16_rows(qkv)),
        ("q, k and v lie inside the rows, their columns multiples of 8", lambda qkv, cache, num_q_heads, q_head_stride, offsets, **_:
         num_q_heads >= 0 and all(o >= 0 and o % 8 == 0 for o in (*offsets, q_head_stride)) and max(
             offsets[0] + (num_q_heads - 1) * q_head_stride + cache.shape[3] // 18 if num_q_heads else 0,
             max(offsets[1:]) + cache.shape[1] * (cache.shape[3] // 18)) <= qkv.shape[1]),
        ("query heads turned in place lie apart from one another, from the keys and from the values", lambda qkv, cache, num_q_heads, q_head_stride,
         offsets, q_out, **_: q_out is not None or (
             _apart(qkv) and _apart_from_keys(cache.shape[1], cache.shape[3] // 18, num_q_heads, q_head_stride, offsets))),
        ("slots is int64 [T]", lambda qkv, slots, **_: _ids(slots, torch.int64, qkv.shape[0])),
        ("cos_sin is fp32 [positions, rot_dim] with positions int64 [T], rot_dim even and at most head_dim",
         lambda qkv, cache, cos_sin, positions, rot_dim, **_: cos_sin is None or (
             cos_sin.dtype == torch.float32 and cos_sin.dim() == 2 and cos_sin.is_contiguous() and cos_sin.shape[0] > 0
             and cos_sin.shape[1] == rot_dim and rot_dim % 2 == 0 and 0 < rot_dim <= cache.shape[3] // 18
             and positions is not None and _ids(positions, torch.int64, qkv.shape[0]))),
        ("norm weights are bf16 [head_dim] on 16-byte boundaries", lambda cache, q_norm, k_norm, **_: all(
            w is None or (w.dtype == BF16 and w.is_contiguous() and w.numel() == cache.shape[3] // 18 and w.data_ptr() % 16 == 0)
            for w in (q_norm, k_norm))),
        ("q_out is [T, Hq * head_dim] bf16 with rows on 16-byte boundaries", lambda qkv, cache, num_q_heads, q_out, **_: q_out is None or (
            q_out.dtype == BF16 and q_out.dim() == 2 and (q_out.numel() == 0 or _bf16_rows(q_out) and _apart(q_out)) and q_out.shape[0] >= qkv.shape[0] and q_out.shape[1] == num_q_heads * (cache.shape[3] // 18))),
        ("q_out lies apart from what is read of qkv", lambda qkv, cache, num_q_heads, q_head_stride, offsets, q_out, **_: q_out is None
         or num_q_heads == 0 or _apart_from_heads(q_out, qkv, cache, num_q_heads, q_head_stride, offsets)),
        ("all tensors are on one GPU", lambda qkv, cache, slots, positions, cos_sin, q_norm, k_norm, q_out, **_:
         _on_gpu(qkv, cache, slots, positions, cos_sin, q_norm, k_norm, q_out)),
    ],
    "fp4_write": [
        _FP4_CACHE,
        ("k and v are [n, kv heads * head_dim] bf16 with rows on 16-byte boundaries", lambda k, v, cache, **_: all(
            _bf16_rows(x) and x.shape[1] == cache.shape[1] * (cache.shape[3] // 18) for x in (k, v)) and k.shape == v.shape),
        ("slots is int64 [n]", lambda k, slots, **_: _ids(slots, torch.int64, k.shape[0])),
        ("all tensors are on one GPU", lambda k, v, cache, slots, **_: _on_gpu(k, v, cache, slots)),
    ],
    "fp4_read": [
        _FP4_CACHE,
        ("slots is int64 [n]", lambda slots, **_: _ids(slots, torch.int64, 0)),
        ("k and v are bf16 [n, kv heads, head_dim], contiguous", lambda cache, slots, k=None, v=None, **_: all(
            x is None or (x.dtype == BF16 and x.is_contiguous() and x.data_ptr() % 16 == 0
                          and tuple(x.shape) == (slots.numel(), cache.shape[1], cache.shape[3] // 18)) for x in (k, v))),
        ("k and v lie apart from one another", lambda k=None, v=None, **_: k is None or v is None or _apart_rows(k.flatten(1), v.flatten(1))),
        ("all tensors are on one GPU", lambda cache, slots, k=None, v=None, **_: _on_gpu(cache, slots, k, v)),
    ],
    "fp4_decode": _FP4_ATTN + [
        ("block_table and seq_lens (int32) have a row for each of q", lambda q, block_table, seq_lens, **_:
         block_table.shape[0] >= q.shape[0] and _ids(seq_lens, torch.int32, q.shape[0])),
    ],
    "fp4_prefill": [
        ("q_start, seq_lens, tile_req and tile_q0 are int32", lambda seq_lens, q_start, tile_req, tile_q0, **_: q_start is not None and _ids(q_start, torch.int32, 1)
         and _ids(seq_lens, torch.int32, 0) and _ids(tile_req, torch.int32, 0) and _ids(tile_q0, torch.int32, tile_req.numel())),
    ] + _FP4_ATTN,
})


def _paged_cache(c) -> bool:
    return c.dim() == 5 and c.shape[1] == 2 and min(c.shape[2:]) > 0 and c.is_contiguous() and c.data_ptr() % 16 == 0


def _table(t, reqs) -> bool:
    return t.dtype == torch.int32 and t.dim() == 2 and t.shape[0] >= reqs and t.shape[1] > 0 and (t.shape[1] == 1 or t.stride(1) == 1)


_TREE_REQS = ("q_start is int32 [requests + 1], seq_lens int32 [requests]", lambda q_start, seq_lens, **_: _ids(q_start, torch.int32, 1)
              and _ids(seq_lens, torch.int32, q_start.numel() - 1))
RULES.update({
    "tree_mask": [
        ("parents is int32 [T]", lambda parents, **_: _ids(parents, torch.int32, 0)),
        _TREE_REQS,
        ("max_nodes is 1 to 1024", lambda max_nodes, **_: 0 < max_nodes <= 1024),
        ("bits is int64 [T, ceil(max_nodes / 64)] and positions int64 [T], contiguous", lambda parents, max_nodes, bits, positions, **_: (
            bits is None or (bits.dtype == torch.int64 and tuple(bits.shape) == (parents.numel(), (max_nodes + 63) // 64) and bits.is_contiguous()))
         and (positions is None or (_ids(positions, torch.int64, 0) and positions.numel() == parents.numel()))),
        ("bits, positions and what is read lie apart", lambda parents, q_start, seq_lens, bits, positions, **_: _all_apart(
            [t for t in (bits, positions) if t is not None], [parents, q_start, seq_lens])),
        ("all tensors are on one GPU", lambda parents, q_start, seq_lens, bits, positions, **_: _on_gpu(parents, q_start, seq_lens, bits, positions)),
    ],
    "tree_attention": [
        ("kv_cache is bf16 [blocks, 2, block_size, kv heads, head_dim], contiguous, head_dim 64, 128 or 256", lambda kv_cache, **_:
         _paged_cache(kv_cache) and kv_cache.dtype == BF16 and kv_cache.shape[4] in (64, 128, 256)),
        ("block_size divides 64, from 8 on, or is a multiple of it", lambda kv_cache, **_: kv_cache.shape[2] in (8, 16, 32) or kv_cache.shape[2] % 64 == 0),
        ("q is [T, Hq * head_dim] bf16 with rows on 16-byte boundaries, Hq a multiple of the kv heads", lambda q, kv_cache, **_: _bf16_rows(q)
         and q.shape[1] > 0 and q.shape[1] % (kv_cache.shape[3] * kv_cache.shape[4]) == 0),
        ("there are at most 128 query heads a kv head", lambda q, kv_cache, **_: q.shape[1] <= 128 * kv_cache.shape[3] * kv_cache.shape[4]),
        ("out is like q and apart from it, its rows apart from one another", lambda q, out, **_: _bf16_rows(out) and out.shape == q.shape
         and _apart(out) and _apart_rows(q, out)),
        _TREE_REQS,
        ("there are at most 8192 requests", lambda q_start, **_: q_start.numel() <= 8193),
        ("block_table is int32 [requests, pages], rows contiguous", lambda block_table, q_start, **_: _table(block_table, q_start.numel() - 1)),
        ("mask is int64 [T, words], contiguous, at most 16 words", lambda q, mask, **_: mask.dtype == torch.int64 and mask.dim() == 2 and mask.shape[0] >= q.shape[0]
         and 0 < mask.shape[1] <= 16 and mask.is_contiguous()),
        ("scale is positive, softcap not negative, both within 32 bits", lambda scale, softcap, **_: LEAST_F32 < scale <= MOST_LOG2_F32
         and (softcap == 0 or LEAST_F32 < softcap <= MOST_LOG2_F32)),
        ("window is not negative and below 2^31, and has positions int64 [T]", lambda q, window, positions, **_: 0 <= window < 2 ** 31
         and (window == 0 or (positions is not None and _ids(positions, torch.int64, q.shape[0])))),
        ("tmp is fp32 and large enough", lambda kv_cache, tmp, **_: tmp is None or (tmp.dtype == torch.float32 and tmp.is_contiguous()
         and tmp.data_ptr() % 16 == 0 and tmp.numel() >= _tree_scratch(kv_cache))),
        ("all tensors are on one GPU", lambda q, kv_cache, block_table, seq_lens, q_start, mask, out, tmp, positions, window, **_: _on_gpu(
            q, kv_cache, block_table, seq_lens, q_start, mask, out, tmp, positions if window else None)),
    ],
    "tree_verify": [
        ("logits is fp32 [T, V], rows contiguous", lambda logits, **_: logits.dim() == 2 and logits.dtype == torch.float32 and logits.shape[1] > 0
         and (logits.shape[1] == 1 or logits.stride(1) == 1)),
        ("logits has at most 778000 columns", lambda logits, **_: logits.shape[1] <= 778000),
        ("tokens is int64 [T], uniforms fp32 [T]", lambda logits, tokens, uniforms, **_: _ids(tokens, torch.int64, logits.shape[0])
         and _ids(uniforms, torch.float32, logits.shape[0])),
        ("q_start is int32 [requests + 1]", lambda q_start, **_: _ids(q_start, torch.int32, 1)),
        ("seeds and steps are int64 [requests], temperature fp32 [requests]", lambda q_start, seeds, steps, temperature, **_: all(
            _ids(t, torch.int64, q_start.numel() - 1) for t in (seeds, steps)) and (
                temperature is None or _ids(temperature, torch.float32, q_start.numel() - 1))),
        ("parents is int32 [T]", lambda logits, parents, **_: parents is None or _ids(parents, torch.int32, logits.shape[0])),
        ("draft_probs is fp32 [T, V], rows contiguous", lambda logits, draft_probs, **_: draft_probs is None or (
            draft_probs.shape == logits.shape and draft_probs.dtype == torch.float32 and (logits.shape[1] == 1 or draft_probs.stride(1) == 1))),
        ("max_tokens is at least 1", lambda max_tokens, **_: max_tokens >= 1),
        ("all tensors are on one GPU", lambda logits, tokens, q_start, uniforms, seeds, steps, parents, draft_probs, temperature, **_: _on_gpu(
            logits, tokens, q_start, uniforms, seeds, steps, parents, draft_probs, temperature)),
    ],
    "tree_compact": [
        ("there is a cache", lambda caches, **_: len(caches) > 0),
        ("caches are [blocks, 2, block_size, kv heads, head_dim], contiguous and alike, cells of 16-byte pieces", lambda caches, **_: all(
            _paged_cache(c) and c.shape == caches[0].shape and c.dtype == caches[0].dtype
            and c.shape[3] * c.shape[4] * c.element_size() % 16 == 0 for c in caches)),
        ("no cache is there twice", lambda caches, **_: len({c.data_ptr() for c in caches}) == len(caches)),
        ("the caches share no memory", lambda caches, **_: all(b - a >= caches[0].numel() * caches[0].element_size() for a, b in itertools.pairwise(
            sorted(c.data_ptr() for c in caches)))),
        _TREE_REQS,
        ("block_table is int32 [requests, pages], rows contiguous", lambda block_table, q_start, **_: _table(block_table, q_start.numel() - 1)),
        ("path is int32 [requests, steps], contiguous", lambda path, q_start, **_: path.dtype == torch.int32 and path.dim() == 2
         and path.shape[0] == q_start.numel() - 1 and path.is_contiguous()),
        ("all tensors are on one GPU", lambda caches, block_table, seq_lens, q_start, path, **_: _on_gpu(*caches, block_table, seq_lens, q_start, path)),
    ],
})


def _all_apart(written, read) -> bool:
    """No two of the contiguous tensors share a byte, but for those that are only read."""
    spans = [(t.data_ptr(), t.data_ptr() + t.numel() * t.element_size()) for t in written + read]
    return not any(a < d and c < b for i, (a, b) in enumerate(spans[: len(written)]) for c, d in spans[i + 1:])


def _tree_scratch(kv_cache) -> int:
    from .draft_tree import scratch_floats
    return scratch_floats(kv_cache.device, kv_cache.shape[4]) if kv_cache.is_cuda else 0


def validate(op: str, **args) -> None:
    """Raises :class:`OpArgumentError` for the first rule of ``op`` the arguments break."""
    for rule, ok in RULES[op]:
        try:
            good = bool(ok(**args))
        except (KeyError, TypeError, IndexError, AttributeError) as e:
            raise OpArgumentError(op, rule, f"could not be evaluated: {e}; {_desc(**args)}") from None
        if not good:
            raise OpArgumentError(op, rule, _desc(**args))
