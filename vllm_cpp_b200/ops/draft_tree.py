"""Speculative decoding with trees of drafted tokens: ancestors' masks, attention over a paged cache, verification of what a request
that samples was offered, and the accepted path's cache cells.

A step holds ``n`` nodes of each request, rows ``q_start[r]..q_start[r + 1]`` (int32 ``[requests + 1]``, ascending): node 0 is the last
accepted token, every other a draft whose parent is an earlier node. Their keys and values lie in the cache behind the request's
context, node ``j`` at position ``c + j``, ``c = seq_lens[r] - n``; their rotary positions are ``c`` plus their depth (:func:`mask`). A step:

* ``bits, positions = mask(parents, ...)``;
* in every layer ``ops.rope_kv(..., positions, slot_mapping=...)`` with the slots of ``c + j``, then ``attention(..., mask=bits)``;
* ``tokens, path, count = verify(logits, ...)``;
* ``compact(kv_caches, path=path, ...)``: the context is ``c + count`` cells now, and the last of ``tokens`` the next root.

A chain of drafts is the tree whose parents count up; :func:`verify` takes ``parents=None`` for it. At most 1024 nodes a request: rows past them
are left out (nothing sees, accepts or moves them, their outputs stay as they are), and count among the cells behind the context.
bf16 queries and caches ``[num_blocks, 2, block_size, kv heads, head_dim]`` for the attention. Rows behind the last request are not
touched. The ``ref_*`` functions restate the operators in plain PyTorch (any device).
"""
from __future__ import annotations

import array
import ctypes
import functools
import math
import operator
from typing import Optional, Sequence, Union

import torch

from . import _lib, reference
from ._lib import check, lib, stream_ptr
from .validate import LEAST_F32, MOST_LOG2_F32, OpArgumentError, validate

MOST_NODES, MOST_COLUMNS = 1024, 778000
BF16, _I32, _I64, _F32 = torch.bfloat16, torch.int32, torch.int64, torch.float32
_P, _L, _I, _F = ctypes.c_void_p, ctypes.c_longlong, ctypes.c_int, ctypes.c_float


class AttnArgs(ctypes.Structure):
    _fields_ = [("q", _P), ("out", _P), ("ldq", _L), ("ldo", _L), ("ldt", _L), ("cache", _P), ("num_blocks", _L), ("block_table", _P),
                ("seq_lens", _P), ("q_start", _P), ("mask", _P), ("positions", _P), ("parts", _P), ("max_blocks", _I), ("num_reqs", _I),
                ("total_q", _I), ("words", _I), ("Hq", _I), ("Hkv", _I), ("D", _I), ("block_size", _I), ("window", _I), ("scale", _F),
                ("softcap", _F)]


class VerifyArgs(ctypes.Structure):
    _fields_ = [("logits", _P), ("probs", _P), ("ldl", _L), ("ldp", _L), ("tokens", _P), ("parents", _P), ("q_start", _P), ("uniforms", _P),
                ("seeds", _P), ("steps", _P), ("temperature", _P), ("out", _P), ("path", _P), ("count", _P), ("num_reqs", _I), ("total", _I),
                ("V", _I), ("most", _I)]


class CompactArgs(ctypes.Structure):
    _fields_ = [("caches", _P), ("block_table", _P), ("seq_lens", _P), ("q_start", _P), ("path", _P), ("num_blocks", _L), ("ldt", _L),
                ("cell_bytes", _L), ("num_caches", _I), ("max_blocks", _I), ("num_reqs", _I), ("total", _I), ("most", _I), ("block_size", _I)]


_address, _contiguous, _device, _shape, _dtype = (torch.Tensor.data_ptr, torch.Tensor.is_contiguous, torch.Tensor.get_device,
                                                  operator.attrgetter("shape"), operator.attrgetter("dtype"))
_declared = False
_attn = _mask = _verify = _compact = None


def _declare():
    global _declared, _attn, _mask, _verify, _compact
    if _declared:
        return
    for name, args in (("b200_tree_attn", AttnArgs), ("b200_tree_verify", VerifyArgs), ("b200_tree_compact", CompactArgs)):
        _lib.declare(name, [ctypes.POINTER(args), _P], _I)
    _lib.declare("b200_tree_attn_takes", [ctypes.POINTER(AttnArgs)], _I)
    _lib.declare("b200_tree_attn_scratch", [_I], _L)
    _lib.declare("b200_tree_mask", [_P, _P, _P, _I, _I, _I, _P, _P, _P], _I)
    l = lib()
    _attn, _mask, _verify, _compact = l.b200_tree_attn, l.b200_tree_mask, l.b200_tree_verify, l.b200_tree_compact
    _declared = True


def _launch(t: torch.Tensor, call, what: str, *args) -> None:
    """On the current stream of the device of ``t``, whichever device is current."""
    if t.get_device() == torch._C._cuda_getDevice():
        check(call(*args, stream_ptr()), what)
    else:
        with torch.cuda.device(t.device):
            check(call(*args, stream_ptr()), what)


def _ids(t, dtype, dev, least) -> bool:
    return t.dtype is dtype and t.get_device() == dev and t.dim() == 1 and t.numel() >= least and t.is_contiguous()


def mask(parents: torch.Tensor, *, q_start: torch.Tensor, seq_lens: torch.Tensor, max_nodes: int = 64, bits: Optional[torch.Tensor] = None,
         positions: Optional[torch.Tensor] = None) -> tuple[torch.Tensor, torch.Tensor]:
    """``parents`` int32 ``[T]``, a node's within its request (-1 and what is not below the node's own number: a root) ->
    ``bits`` int64 ``[T, ceil(max_nodes / 64)]``, bit ``j`` of a row (64 a word) set for the node itself and those above it, and ``positions`` int64 ``[T]``.
    ``max_nodes``: of the largest tree. The trees' sizes are known on the device alone: in a larger one the nodes past it have no bit, and nothing sees them, they themselves
    included."""
    try:
        (T,), (reqs,) = parents.shape, q_start.shape
        dev = parents.get_device()
        ok = (dev >= 0 and _ids(parents, _I32, dev, 0) and _ids(q_start, _I32, dev, 1) and _ids(seq_lens, _I32, dev, reqs - 1)
              and 0 < max_nodes <= MOST_NODES and bits is None and positions is None)
    except (TypeError, ValueError, AttributeError):
        ok = False
    if not ok:
        validate("tree_mask", parents=parents, q_start=q_start, seq_lens=seq_lens, max_nodes=max_nodes, bits=bits, positions=positions)
        T, reqs = parents.shape[0], q_start.shape[0]
    words = (max_nodes + 63) // 64
    _declare()
    if bits is None:
        bits = parents.new_empty((T, words), dtype=_I64)
    if positions is None:
        positions = parents.new_empty((T,), dtype=_I64)
    _launch(parents, _mask, "tree_mask", parents.data_ptr(), q_start.data_ptr(), seq_lens.data_ptr(), reqs - 1, T, words, bits.data_ptr(),
            positions.data_ptr())
    return bits, positions


_scratch_floats: dict = {}


def scratch_floats(device: torch.device, head_dim: int) -> int:
    key = (device.index, head_dim)
    n = _scratch_floats.get(key)
    if n is None:
        _declare()
        with torch.cuda.device(device):
            n = _scratch_floats[key] = lib().b200_tree_attn_scratch(head_dim)
    return n


def scratch(device: torch.device, head_dim: int) -> torch.Tensor:
    """What :func:`attention` takes as ``tmp``: parts of requests that several CTAs share. Calls that may run at the same time (streams,
    graphs replayed side by side) need one each, which lives as long as a graph that was captured with it."""
    return torch.empty(scratch_floats(device, head_dim), dtype=_F32, device=device)


def attention(q: torch.Tensor, kv_cache: torch.Tensor, *, block_table: torch.Tensor, seq_lens: torch.Tensor, q_start: torch.Tensor,
              mask: torch.Tensor, scale: float, positions: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
              softcap: float = 0.0, window: int = 0, tmp: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of the nodes ``q`` ``[T, Hq * D]`` (any row stride in steps of 8): each sees its request's context and the nodes whose bits
    are set in its row of ``mask`` (int64 ``[T, words]``, as :func:`mask` makes it, or any other); a node that sees nothing gives zeros. ``window``:
    of the context and of those nodes it sees only what lies less than ``window`` before it; that takes the nodes' ``positions``, as :func:`mask` makes
    them (from ``c`` to ``c + n - 1``). What a node does not see does not reach it, infinities and NaN among the values
    included. Entries of ``block_table`` outside the cache count as keys and values of zeros. ``out`` shares no memory with the rows of ``q``. ``tmp``:
    :func:`scratch`, allocated if not given. head_dim 64, 128 or 256, at most 128 query heads a kv head, pages that divide a tile of 64
    tokens or are whole tiles; at most 8192 requests. ``scale`` and ``softcap`` are held in
    32 bits: below 2.35e38, and not so small that they would be 0."""
    given = out is not None
    try:
        (T, cols), (nb, two, bs, H, D), (treqs, pages), (reqs,), (rows, words) = q.shape, kv_cache.shape, block_table.shape, q_start.shape, mask.shape
        (ldq, q1), (ldt, t1), dev, qp, cp = q.stride(), block_table.stride(), q.get_device(), q.data_ptr(), kv_cache.data_ptr()
        ok = (dev >= 0 and dev == kv_cache.get_device() == block_table.get_device() == mask.get_device() and q.dtype is BF16
              and kv_cache.dtype is BF16 and block_table.dtype is _I32 and mask.dtype is _I64 and two == 2 and H > 0 and cols > 0
              and (D == 128 or D == 64 or D == 256) and cols % (D * H) == 0 and kv_cache.is_contiguous() and q1 == t1 == 1 and pages > 0
              and treqs >= reqs - 1 and (qp | cp | 2 * ldq) % 16 == 0 and rows >= T and 0 < words <= 16 and mask.is_contiguous()
              and cols <= 128 * D * H and bs >= 8 and (64 % bs == 0 or bs % 64 == 0) and reqs <= 8193
              and _ids(seq_lens, _I32, dev, reqs - 1) and _ids(q_start, _I32, dev, 1)
              and LEAST_F32 < scale <= MOST_LOG2_F32 and (softcap == 0 or LEAST_F32 < softcap <= MOST_LOG2_F32)
              and 0 <= window < 2 ** 31 and (window == 0 or _ids(positions, _I64, dev, T)))
        if ok and given:
            (orows, ocols), (ldo, o1), op_ = out.shape, out.stride(), out.data_ptr()
            ok = (orows == T and ocols == cols and out.dtype is BF16 and out.get_device() == dev and o1 == 1 and (op_ | 2 * ldo) % 16 == 0
                  and (T <= 1 or ldo >= cols) and (op_ >= qp + 2 * ((T - 1) * ldq + cols) or qp >= op_ + 2 * ((T - 1) * ldo + cols)))
        if ok and tmp is not None:
            ok = (tmp.dtype is _F32 and tmp.get_device() == dev and tmp.is_contiguous() and tmp.data_ptr() % 16 == 0
                  and tmp.numel() >= scratch_floats(q.device, D))
    except (TypeError, ValueError, AttributeError):
        ok = False
    if not given:
        out = q.new_empty(q.shape)
        op_, ldo = out.data_ptr(), out.stride(0) if out.dim() == 2 else 0
    if not ok:
        validate("tree_attention", q=q, kv_cache=kv_cache, block_table=block_table, seq_lens=seq_lens, q_start=q_start, mask=mask, scale=scale,
                 positions=positions, out=out, softcap=softcap, window=window, tmp=tmp)
        (T, cols), (nb, two, bs, H, D), pages, reqs, words = q.shape, kv_cache.shape, block_table.shape[1], q_start.shape[0], mask.shape[1]
        ldq, ldt, ldo, qp, cp, op_ = q.stride(0), block_table.stride(0), out.stride(0), q.data_ptr(), kv_cache.data_ptr(), out.data_ptr()
    _declare()
    if tmp is None:
        tmp = q.new_empty(scratch_floats(q.device, D), dtype=_F32)
    a = AttnArgs()
    a.q, a.out, a.cache, a.num_blocks, a.block_size, a.Hq, a.Hkv, a.D = qp, op_, cp, nb, bs, cols // D, H, D
    a.ldq, a.ldo = (ldq, ldo) if T > 1 else (cols, cols)         # (the stride of a single row says nothing)
    a.block_table, a.ldt, a.max_blocks, a.seq_lens, a.q_start = block_table.data_ptr(), ldt, pages, seq_lens.data_ptr(), q_start.data_ptr()
    a.mask, a.words, a.num_reqs, a.total_q, a.parts = mask.data_ptr(), words, reqs - 1, T, tmp.data_ptr()
    if window:
        a.positions, a.window = positions.data_ptr(), window
    a.scale, a.softcap = scale, softcap
    _launch(q, _attn, "tree_attention", a)
    return out


def verify(logits: torch.Tensor, tokens: torch.Tensor, *, q_start: torch.Tensor, uniforms: torch.Tensor, seeds: torch.Tensor,
           steps: torch.Tensor, max_tokens: int, parents: Optional[torch.Tensor] = None, draft_probs: Optional[torch.Tensor] = None,
           temperature: Optional[torch.Tensor] = None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Accepts drafts so that the tokens that come out have the distribution of the target, softmax of ``logits`` (fp32 ``[T, V]``, a node's
    row says what follows it; temperature, filters and penalties are applied to them before). ``tokens`` int64 ``[T]`` (the roots' do not matter; one
    outside the vocabulary is refused), ``parents`` as in :func:`mask` (None: chains). ``draft_probs`` fp32 ``[T, V]``: a node's row is the distribution that its children
    were drawn from, each for itself; None: children that were chosen (n-grams, likeliest tokens). ``uniforms`` fp32 ``[T]`` in [0, 1) decide
    on each node; the last token is drawn as :func:`vllm_cpp_b200.ops.random_sample` draws, from ``seeds`` and ``steps`` int64
    ``[requests]``. ``temperature`` fp32 ``[requests]`` (not applied) names the greedy requests, those below 1e-5: they accept the argmax.

    -> ``tokens`` int64 ``[requests, max_tokens]``, the accepted ones and one more, then -1; ``path`` int32 of the same shape, the root and the accepted
    nodes, then -1; ``count`` int32 ``[requests]``, tokens of each. The walk ends after ``max_tokens - 1`` accepted drafts. NaN logits count
    as -inf; where nothing is left to draw from, the likeliest token comes out. At most 778000 columns."""
    try:
        (T, V), (ld, one), dev, (reqs,) = logits.shape, logits.stride(), logits.get_device(), q_start.shape
        ok = (dev >= 0 and logits.dtype is _F32 and (one == 1 or V == 1) and V > 0 and _ids(tokens, _I64, dev, T) and _ids(q_start, _I32, dev, 1)
              and _ids(uniforms, _F32, dev, T) and _ids(seeds, _I64, dev, reqs - 1) and _ids(steps, _I64, dev, reqs - 1) and max_tokens > 0
              and V <= MOST_COLUMNS and (parents is None or _ids(parents, _I32, dev, T)) and (temperature is None or _ids(temperature, _F32, dev, reqs - 1)))
        if ok and draft_probs is not None:
            ok = (draft_probs.shape == logits.shape and draft_probs.dtype is _F32 and draft_probs.get_device() == dev
                  and (draft_probs.stride(1) == 1 or V == 1))
    except (TypeError, ValueError, AttributeError):
        ok = False
    if not ok:
        validate("tree_verify", logits=logits, tokens=tokens, q_start=q_start, uniforms=uniforms, seeds=seeds, steps=steps, max_tokens=max_tokens,
                 parents=parents, draft_probs=draft_probs, temperature=temperature)
        (T, V), ld, reqs = logits.shape, logits.stride(0), q_start.shape[0]
    _declare()
    R = reqs - 1
    out, path, count = tokens.new_empty((R, max_tokens)), q_start.new_empty((R, max_tokens)), q_start.new_empty((R,))
    a = VerifyArgs()
    a.logits, a.ldl, a.tokens, a.q_start, a.uniforms = logits.data_ptr(), ld, tokens.data_ptr(), q_start.data_ptr(), uniforms.data_ptr()
    a.seeds, a.steps, a.out, a.path, a.count = seeds.data_ptr(), steps.data_ptr(), out.data_ptr(), path.data_ptr(), count.data_ptr()
    if draft_probs is not None:
        a.probs, a.ldp = draft_probs.data_ptr(), draft_probs.stride(0)
    if parents is not None:
        a.parents = parents.data_ptr()
    if temperature is not None:
        a.temperature = temperature.data_ptr()
    a.num_reqs, a.total, a.V, a.most = R, T, V, max_tokens
    _launch(logits, _verify, "tree_verify", a)
    return out, path, count


def compact(kv_caches: Union[torch.Tensor, Sequence[torch.Tensor]], *, block_table: torch.Tensor, seq_lens: torch.Tensor,
            q_start: torch.Tensor, path: torch.Tensor) -> None:
    """Keys and values of accepted nodes move behind their context, in place and in every one of the caches (``[num_blocks, 2, block_size, kv
    heads, head_dim]``, alike, of any type, apart from one another): cell ``c + path[r, i]`` to cell ``c + i``. ``path`` int32 ``[requests, steps]`` as :func:`verify`
    gives it; entries that are not behind their own place (padding too) move nothing. ``seq_lens`` still counts all nodes."""
    caches = [kv_caches] if isinstance(kv_caches, torch.Tensor) else list(kv_caches)
    try:
        first = caches[0]
        shape, dev = first.shape, first.get_device()
        (nb, two, bs, H, D), (treqs, pages), (ldt, t1), (reqs,), (prows, most) = shape, block_table.shape, block_table.stride(), q_start.shape, path.shape
        cell = H * D * first.element_size()
        at = list(map(_address, caches))
        line = sorted(at)
        ok = (dev >= 0 and two == 2 and bs > 0 and cell > 0 and cell % 16 == 0 and pages > 0 and t1 == 1 and block_table.dtype is _I32 and block_table.get_device() == dev
              and treqs >= reqs - 1 and _ids(seq_lens, _I32, dev, reqs - 1) and _ids(q_start, _I32, dev, 1) and path.dtype is _I32
              and path.get_device() == dev and path.is_contiguous() and prows == reqs - 1
              and min(map(operator.sub, line[1:], line), default=nb * 2 * bs * cell) >= nb * 2 * bs * cell
              and not functools.reduce(operator.or_, at) % 16 and all(map(_contiguous, caches))
              and [*map(_device, caches)].count(dev) == [*map(_dtype, caches)].count(first.dtype) == [*map(_shape, caches)].count(shape) == len(at))
    except (TypeError, ValueError, AttributeError, IndexError):
        ok = False
    if not ok:
        validate("tree_compact", caches=caches, block_table=block_table, seq_lens=seq_lens, q_start=q_start, path=path)
        (nb, two, bs, H, D), pages, ldt, reqs, most = caches[0].shape, block_table.shape[1], block_table.stride(0), q_start.shape[0], path.shape[1]
        cell, at = H * D * caches[0].element_size(), [c.data_ptr() for c in caches]
    _declare()
    a = CompactArgs()
    held = array.array("Q", at)
    a.caches, a.num_caches = held.buffer_info()[0], len(at)
    a.block_table, a.ldt, a.max_blocks, a.seq_lens, a.q_start = block_table.data_ptr(), ldt, pages, seq_lens.data_ptr(), q_start.data_ptr()
    a.path, a.most, a.num_blocks, a.block_size, a.cell_bytes, a.num_reqs, a.total = path.data_ptr(), most, nb, bs, cell, reqs - 1, 2 ** 31 - 1
    _launch(caches[0], _compact, "tree_compact", a)


# ------------------------------------------------------------------------------ restatements
def _rows(q_start, T):
    """(first row, nodes, cells) of each request: those past the 1024th are no nodes, but their cells lie behind its context too."""
    at = [min(max(int(x), 0), T) for x in q_start.tolist()]
    return [(a, min(max(0, b - a), MOST_NODES), max(0, b - a)) for a, b in zip(at, at[1:])]


def _signed(x: int) -> int:
    return x - (1 << 64) if x >> 63 else x


def ref_mask(parents, *, q_start, seq_lens, max_nodes=64):
    words = (max_nodes + 63) // 64
    bits = torch.zeros((parents.numel(), words), dtype=_I64, device=parents.device)
    positions = torch.zeros((parents.numel(),), dtype=_I64, device=parents.device)
    up = parents.tolist()
    for r, (first, n, cells) in enumerate(_rows(q_start, parents.numel())):
        held, depth = [], []
        for j in range(n):
            p = up[first + j] if 0 <= up[first + j] < j else -1
            held.append((held[p] if p >= 0 else 0) | 1 << j)
            depth.append(depth[p] + 1 if p >= 0 else 0)
            for w in range(words):
                bits[first + j, w] = _signed(held[j] >> 64 * w & (1 << 64) - 1)
            positions[first + j] = int(seq_lens[r]) - cells + depth[j]
    return bits, positions


def seen_by(mask, *, q_start, seq_lens, positions=None, window=0) -> list:
    """For each request the truth values ``[n, seq_lens[r]]``: which positions its nodes see."""
    out = []
    for r, (first, n, cells) in enumerate(_rows(q_start, mask.shape[0])):
        length = max(0, int(seq_lens[r]))
        c, key = length - cells, torch.arange(length, device=mask.device)
        node = (key - c).clamp(min=0)
        word = mask[first: first + n][:, (node // 64).clamp(max=mask.shape[1] - 1)]
        bit = (word >> (node % 64) & 1).bool() & (node < 64 * mask.shape[1])
        seen = torch.where(key < c, torch.ones_like(bit), bit)
        if window > 0:
            at = positions[first: first + n].clamp(min=c, max=c + n - 1)
            lies = torch.where(key < c, key, at[node.clamp(max=n - 1)]) if n else key
            seen &= lies > at[:, None] - window
        out.append(seen)
    return out


def ref_attention(q, kv_cache, *, block_table, seq_lens, q_start, mask, scale, positions=None, softcap=0.0, window=0,
                  dtype=torch.float32) -> torch.Tensor:
    """:func:`attention` with sums in ``dtype``, in that type; rows of no request are zeros."""
    nb, _, bs, H, D = kv_cache.shape
    T, Hq = q.shape[0], q.shape[1] // D
    out = torch.zeros((T, Hq, D), dtype=dtype, device=q.device)
    seen_all = seen_by(mask, q_start=q_start, seq_lens=seq_lens, positions=positions, window=window)
    for r, (first, n, _) in enumerate(_rows(q_start, T)):
        seen = seen_all[r]
        length = seen.shape[1]
        if not n or not length:
            continue
        kv = kv_cache[block_table[r, : -(-length // bs)].long()]
        k, v = (kv[:, i].reshape(-1, H, D)[:length].to(dtype).repeat_interleave(Hq // H, 1) for i in (0, 1))
        s = torch.einsum("nhd,khd->hnk", q[first: first + n].reshape(n, Hq, D).to(dtype), k) * scale
        if softcap > 0:
            s = softcap * torch.tanh(s / softcap)
        s = s.masked_fill(~seen[None], -math.inf)
        top = s.amax(-1, keepdim=True)
        p = torch.exp(s - torch.where(top == -math.inf, torch.zeros_like(top), top))
        # (0 times an infinity or NaN that is not seen is nothing)
        o = torch.einsum("hnk,khd->nhd", p, torch.nan_to_num(v, nan=0.0, posinf=0.0, neginf=0.0))
        odd = ~torch.isfinite(v)
        for key in odd.flatten(1).any(1).nonzero().flatten().tolist():
            w = torch.where(odd[key], v[key], torch.zeros_like(v[key]))
            o = o + torch.where(seen[:, key, None, None], w, torch.zeros_like(w))
        total = p.sum(-1).t()[..., None]
        out[first: first + n] = o / torch.where(total == 0, torch.ones_like(total), total)
    return out.flatten(1)


def race_numbers(seed: int, step: int, vocab: int) -> torch.Tensor:
    """The exponentially distributed numbers, fp64 ``[vocab]``, that a draw with ``seed`` and ``step`` divides by."""
    m = (1 << 64) - 1
    u = [((reference.splitmix64(seed & m ^ reference.splitmix64((step * 0x100000001B3 + i) & m)) >> 11) + 0.5) / 9007199254740992.0
         for i in range(vocab)]
    return -torch.log(torch.tensor(u, dtype=torch.float64))


def ref_verify(logits, tokens, *, q_start, uniforms, seeds, steps, max_tokens, parents=None, draft_probs=None, temperature=None):
    """:func:`verify` in 64 bits, one refusal after another (on the host)."""
    T, V = logits.shape
    rows = _rows(q_start, T)
    out = torch.full((len(rows), max_tokens), -1, dtype=_I64)
    path, count = torch.full((len(rows), max_tokens), -1, dtype=_I32), torch.zeros(len(rows), dtype=_I32)
    for r, (first, n, _) in enumerate(rows):
        if not n:
            continue
        node, depth, greedy = 0, 0, temperature is not None and float(temperature[r]) < 1e-5
        path[r, 0] = 0
        while True:
            l = logits[first + node].double().cpu()
            l = torch.where(l.isnan(), torch.full_like(l, -math.inf), l)
            top = l.max()
            p = torch.where(l == top, torch.ones_like(l), torch.exp(l - top)) * (l > -math.inf)
            p = p / p.sum().clamp(min=1e-300)
            best = int(l.argmax()) if top > -math.inf else 0
            below = [j for j in range(node + 1, n) if (j - 1 if parents is None else int(parents[first + j])) == node]
            taken = -1
            for j in below if depth + 1 < max_tokens else ():
                x, u = int(tokens[first + j]), float(uniforms[first + j])
                inside = 0 <= x < V
                if greedy:
                    if inside and top > -math.inf and x == best:
                        taken = j
                        break
                    continue
                q = torch.zeros(V, dtype=torch.float64)
                if draft_probs is not None:
                    q = draft_probs[first + node].double().cpu().nan_to_num(nan=0.0).clamp(min=0)
                elif inside:
                    q[x] = 1
                if inside and u * float(q[x]) < float(p[x]):
                    taken = j
                    break
                p = (p - q).clamp(min=0)
                p = p / p.sum().clamp(min=1e-300)
            if taken < 0:
                last = best
                if not greedy and float(p.sum()) > 0:
                    last = int((p / race_numbers(int(seeds[r]), int(steps[r]), V)).argmax())
                out[r, depth], count[r] = last, depth + 1
                break
            out[r, depth], path[r, depth + 1] = tokens[first + taken], taken
            node, depth = taken, depth + 1
    return out, path, count


def ref_compact(kv_caches, *, block_table, seq_lens, q_start, path) -> None:
    caches = [kv_caches] if isinstance(kv_caches, torch.Tensor) else list(kv_caches)
    nb, _, bs = caches[0].shape[:3]
    for r, (first, n, cells) in enumerate(_rows(q_start, 2 ** 31 - 1)):
        c, held = int(seq_lens[r]) - cells, []

        def cell(position):
            return int(block_table[r, position // bs]), position % bs
        for i in range(1, min(path.shape[1], n)):
            node = int(path[r, i])
            if i < node < n and c + i >= 0:
                (b, o), to = cell(c + node), cell(c + i)
                if 0 <= b < nb and 0 <= to[0] < nb:
                    held += [(x, to, x[b, :, o].clone()) for x in caches]
        for x, (b, o), kv in held:
            x[b, :, o] = kv
