"""A paged KV cache held in 4 bits: what writes it, what reads it back, and the attention over it.

A layer's cache is uint8 ``[num_blocks, kv heads, block_size / 16, 18 * head_dim]`` (:func:`alloc`), 9 bits for 2 bytes of a bf16
cache; slots and block tables are those of the bf16 cache. Groups of 16 neighbouring head dimensions share a scale,
``s = max |x| / 6`` in 5 exponent and 3 mantissa bits (the upper half of an f16 behind its sign), and hold codes ``e2m1(x / s)``, both
rounded to nearest, ties to even. Code times scale is exact in bf16. Magnitudes past 6 * 10240 saturate, a NaN makes its group NaN. Within the last dimension, 16 tokens:
key codes ``[16, D / 2]`` (the even dimension in the low nibble), value codes ``[16, D / 2]`` whose 16-byte piece ``n`` lies at
``n ^ 2 (token // 4)``, key scales ``[16, D / 16]``, value scales ``[D / 16, 16]``.

head_dim 64, 128 or 256; block_size a multiple of 16; bf16 queries, keys and values in rows on 16-byte boundaries. The ``ref_*``
functions restate the operators in plain PyTorch (any device; a NaN in a cache aside).
"""
from __future__ import annotations

import ctypes
import math
from typing import Optional

import torch

from . import _lib, reference
from ._lib import check, lib, stream_ptr
from .validate import OpArgumentError, validate

CELL = 16                      # tokens of a cell
LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
MOST_SCALE = 10240.0           # (6 times it is still an f16)
BF16 = torch.bfloat16

_P, _L, _I, _F = ctypes.c_void_p, ctypes.c_longlong, ctypes.c_int, ctypes.c_float


class AppendArgs(ctypes.Structure):
    _fields_ = [("q", _P), ("k", _P), ("v", _P), ("q_out", _P), ("ldq", _L), ("ldk", _L), ("ldv", _L), ("ldo", _L),
                ("positions", _P), ("cos_sin", _P), ("q_norm", _P), ("k_norm", _P), ("slots", _P), ("cache", _P),
                ("num_blocks", _L), ("table_rows", _L), ("T", _I), ("Hq", _I), ("Hkv", _I), ("D", _I), ("rot", _I),
                ("q_head_stride", _I), ("block_size", _I), ("neox", _I), ("gemma", _I), ("eps", _F)]


class AttnArgs(ctypes.Structure):
    _fields_ = [("q", _P), ("out", _P), ("ldq", _L), ("ldo", _L), ("ldt", _L), ("cache", _P), ("num_blocks", _L),
                ("block_table", _P), ("seq_lens", _P), ("q_start", _P), ("tile_req", _P), ("tile_q0", _P), ("parts", _P),
                ("max_blocks", _I), ("num_reqs", _I), ("total_q", _I), ("num_tiles", _I), ("Hq", _I), ("Hkv", _I), ("D", _I),
                ("block_size", _I), ("window", _I), ("causal", _I), ("most_q", _I), ("scale", _F), ("softcap", _F)]


class ReadArgs(ctypes.Structure):
    _fields_ = [("cache", _P), ("slots", _P), ("k", _P), ("v", _P), ("num_blocks", _L), ("n", _L), ("block_size", _I), ("Hkv", _I),
                ("D", _I)]


_declared = False
_append = _read = _attn = None      # the library's entry points


def _declare():
    global _declared, _append, _read, _attn
    if _declared:
        return
    for name, args in (("b200_fp4_append", AppendArgs), ("b200_fp4_read", ReadArgs), ("b200_fp4_attn", AttnArgs)):
        _lib.declare(name, [ctypes.POINTER(args), _P], _I)
    _lib.declare("b200_fp4_attn_scratch", [_I, _I], _L)
    _lib.declare("b200_fp4_attn_takes", [ctypes.POINTER(AttnArgs)], _I)
    l = lib()
    _append, _read, _attn = l.b200_fp4_append, l.b200_fp4_read, l.b200_fp4_attn
    _declared = True


def bytes_per_block(num_kv_heads: int, block_size: int, head_dim: int) -> int:
    return num_kv_heads * (block_size // CELL) * 18 * head_dim


def alloc(num_blocks: int, num_kv_heads: int, block_size: int, head_dim: int, device) -> torch.Tensor:
    """The zeroed cache of a layer."""
    if head_dim not in (64, 128, 256) or block_size <= 0 or block_size % CELL:
        raise OpArgumentError("fp4_cache.alloc", "head_dim is 64, 128 or 256 and block_size a multiple of 16",
                              f"head_dim={head_dim}, block_size={block_size}")
    return torch.zeros((num_blocks, num_kv_heads, block_size // CELL, 18 * head_dim), dtype=torch.uint8, device=device)


def shape_of(cache: torch.Tensor) -> tuple[int, int, int, int]:
    """(num_blocks, kv heads, block_size, head_dim) of a cache."""
    n, h, c, b = cache.shape
    return n, h, c * CELL, b // 18


def _launch(t: torch.Tensor, call, args, what: str) -> None:
    """On the current stream of the device of ``t``, whichever device is current."""
    if t.get_device() == torch._C._cuda_getDevice():
        check(call(args, stream_ptr()), what)
    else:
        with torch.cuda.device(t.device):
            check(call(args, stream_ptr()), what)


def append(qkv: torch.Tensor, positions: Optional[torch.Tensor], cos_sin: Optional[torch.Tensor], cache: torch.Tensor,
           slots: torch.Tensor, *, num_q_heads: int, rot_dim: Optional[int] = None, neox: bool = True,
           q_norm: Optional[torch.Tensor] = None, k_norm: Optional[torch.Tensor] = None, eps: float = 1e-6, gemma: bool = False,
           q_out: Optional[torch.Tensor] = None, q_head_stride: Optional[int] = None,
           offsets: Optional[tuple[int, int, int]] = None) -> None:
    """Per-head RMSNorm of q and k (weights bf16 ``[D]``, optional) and rotation of merged ``[T, q | k | v]`` rows; q in place or to
    ``q_out`` ``[T, Hq * D]`` (apart from the heads of ``qkv``), k and v into the cache. ``cos_sin``: fp32 ``[positions, cos | sin]`` (None: no rotation), ``rot_dim``
    its width, pairs half of it apart (``neox``) or neighbours. ``offsets``: columns where q, k and v begin; ``q_head_stride``:
    columns between q heads. The slots of a call differ; slots outside the cache (-1) write nothing, and a position
    outside the table makes its row NaN. The k and v columns of ``qkv`` stay as they are."""
    nb, H, bs, D = shape_of(cache) if cache.dim() == 4 else (0, 0, 0, 0)
    hs = D if q_head_stride is None else q_head_stride
    if offsets is None:
        offsets = (0, num_q_heads * D, (num_q_heads + H) * D)
    rot = (D if cos_sin is None else cos_sin.shape[1]) if rot_dim is None else rot_dim
    # (the rules of ops.validate for the plain call of a model's layer, in a fraction of their time)
    try:
        (T, cols), (ld, one), dev, (n,), at = qkv.shape, qkv.stride(), qkv.get_device(), slots.shape, qkv.data_ptr()
        ok = (dev >= 0 and dev == cache.get_device() == slots.get_device() and D in (64, 128, 256) and cache.shape[3] == 18 * D
              and bs > 0 and cache.dtype is torch.uint8 and cache.is_contiguous() and qkv.dtype is BF16 and one == 1
              and slots.dtype is torch.int64 and slots.is_contiguous() and n >= T and hs == D and num_q_heads >= 0
              and offsets == (0, num_q_heads * D, (num_q_heads + H) * D) and cols >= (num_q_heads + 2 * H) * D
              and (at | cache.data_ptr() | 2 * ld) % 16 == 0 and (T <= 1 or ld >= cols))
        if ok and cos_sin is not None:
            rows, width = cos_sin.shape
            ok = (cos_sin.dtype is torch.float32 and cos_sin.is_contiguous() and width == rot and rows > 0 and 0 < rot <= D and rot % 2 == 0
                  and positions.dtype is torch.int64 and positions.is_contiguous() and positions.dim() == 1 and positions.numel() >= T
                  and dev == cos_sin.get_device() == positions.get_device())
        if ok and q_out is not None:
            ok = (q_out.dtype is BF16 and q_out.get_device() == dev and q_out.dim() == 2 and q_out.stride(1) == 1 and q_out.shape[0] >= T
                  and q_out.shape[1] == num_q_heads * D and (q_out.data_ptr() | 2 * q_out.stride(0)) % 16 == 0
                  and (T <= 1 or q_out.stride(0) >= q_out.shape[1]) and num_q_heads > 0)
            if ok:
                out, ldo = q_out.data_ptr(), q_out.stride(0)
                ok = out >= at + 2 * ((T - 1) * ld + cols) or at >= out + 2 * ((T - 1) * ldo + q_out.shape[1])
        for w in (q_norm, k_norm):
            if ok and w is not None:
                ok = w.dtype is BF16 and w.get_device() == dev and w.numel() == D and w.is_contiguous() and w.data_ptr() % 16 == 0
    except (TypeError, ValueError, AttributeError):
        ok = False
    if not ok:
        validate("fp4_append", qkv=qkv, cache=cache, slots=slots, positions=positions, cos_sin=cos_sin, q_norm=q_norm, k_norm=k_norm,
                 q_out=q_out, num_q_heads=num_q_heads, rot_dim=rot, q_head_stride=hs, offsets=offsets)
        T, ld, at = qkv.shape[0], qkv.stride(0), qkv.data_ptr()
    _declare()
    a = AppendArgs()
    a.q, a.k, a.v = at + 2 * offsets[0], at + 2 * offsets[1], at + 2 * offsets[2]
    if T > 1:                      # (the stride of a single row says nothing)
        a.ldq = a.ldk = a.ldv = ld
    if q_out is not None and num_q_heads:
        a.q_out, a.ldo = q_out.data_ptr(), q_out.stride(0) if T > 1 else 0
    if cos_sin is not None:
        a.positions, a.cos_sin, a.table_rows, a.rot = positions.data_ptr(), cos_sin.data_ptr(), cos_sin.shape[0], rot
    if q_norm is not None:
        a.q_norm = q_norm.data_ptr()
    if k_norm is not None:
        a.k_norm = k_norm.data_ptr()
    a.num_blocks, a.Hkv, a.block_size, a.slots, a.cache = nb, H, bs, slots.data_ptr(), cache.data_ptr()
    a.T, a.Hq, a.D, a.q_head_stride, a.neox, a.gemma, a.eps = T, num_q_heads, D, hs, neox, gemma, eps
    _launch(qkv, _append, a, "fp4_append")


def write(k: torch.Tensor, v: torch.Tensor, cache: torch.Tensor, slots: torch.Tensor) -> None:
    """Keys and values ``[n, Hkv * D]`` (or ``[n, Hkv, D]``) that are normed and rotated already, into the cache. What :func:`read`
    gave comes back to the same values, but for groups whose scale was below 2^-14."""
    k, v = k.flatten(1), v.flatten(1)
    validate("fp4_write", k=k, v=v, cache=cache, slots=slots)
    _declare()
    a = AppendArgs()
    a.num_blocks, a.Hkv, a.block_size, a.D = shape_of(cache)
    a.k, a.v, a.ldk, a.ldv = k.data_ptr(), v.data_ptr(), *((k.stride(0), v.stride(0)) if k.shape[0] > 1 else (0, 0))
    a.slots, a.cache, a.T, a.eps = slots.data_ptr(), cache.data_ptr(), k.shape[0], 1.0
    _launch(k, _append, a, "fp4_write")


def read(cache: torch.Tensor, slots: torch.Tensor, k: Optional[torch.Tensor] = None,
         v: Optional[torch.Tensor] = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Keys and values bf16 ``[n, Hkv, D]`` that the cache holds for ``slots`` (int64 ``[n]``); zeros for slots outside the cache."""
    nb, H, bs, D = shape_of(cache) if cache.dim() == 4 else (0, 0, 0, 0)
    if not (k is None and v is None and cache.get_device() >= 0 and slots.get_device() == cache.get_device() and D in (64, 128, 256)
            and cache.shape[3] == 18 * D and bs > 0 and cache.dtype is torch.uint8 and cache.is_contiguous() and cache.data_ptr() % 16 == 0
            and slots.dtype is torch.int64 and slots.dim() == 1 and slots.is_contiguous()):
        validate("fp4_read", cache=cache, slots=slots, k=k, v=v)
    _declare()
    a = ReadArgs()
    a.num_blocks, a.Hkv, a.block_size, a.D = nb, H, bs, D
    n = a.n = slots.numel()
    if k is None:
        k = cache.new_empty((n, H, D), dtype=BF16)
    if v is None:
        v = torch.empty_like(k)
    a.cache, a.slots, a.k, a.v = cache.data_ptr(), slots.data_ptr(), k.data_ptr(), v.data_ptr()
    _launch(cache, _read, a, "fp4_read")
    return k, v


_scratch_floats: dict = {}


def scratch_floats(device: torch.device, head_dim: int, prefill: bool) -> int:
    key = (device.index, head_dim, bool(prefill))
    n = _scratch_floats.get(key)
    if n is None:
        _declare()
        with torch.cuda.device(device):
            n = _scratch_floats[key] = lib().b200_fp4_attn_scratch(head_dim, prefill)
    return n


def scratch(device: torch.device, head_dim: int, prefill: bool = True) -> torch.Tensor:
    """What ``decode`` and (with ``prefill``) ``prefill`` take as ``tmp``: parts of sequences that several CTAs share. Calls that may
    run at the same time (streams, graphs replayed side by side) need one each."""
    return torch.empty(scratch_floats(device, head_dim, prefill), dtype=torch.float32, device=device)


def steps_fit(*, head_dim: int, num_q_heads: int, num_kv_heads: int, block_size: int, max_blocks: int, max_reqs: int, max_tokens: int,
              max_tiles: int) -> bool:
    """Whether ``decode`` and ``prefill`` take every step of up to so many sequences, query tokens and tiles with tables of ``max_blocks``
    entries a sequence (no GPU is needed to say)."""
    _declare()

    def taken(tokens, reqs, tiles=0, most_q=0):
        a = AttnArgs()
        a.D, a.Hq, a.Hkv, a.block_size, a.max_blocks = head_dim, num_q_heads, num_kv_heads, block_size, max_blocks
        a.total_q, a.num_reqs, a.num_tiles, a.most_q, a.q_start = tokens, reqs, tiles, most_q, 1 if tiles else None
        return lib().b200_fp4_attn_takes(a) == 0
    # both kernels; one sequence; the row kernel alone, as for sequences of at most 48 rows, with row tiles of 16 and, where they are most, of 8
    group = max(1, num_q_heads // num_kv_heads)
    few = min(max_tokens, max_reqs * max(1, 48 // group))
    return (taken(max_reqs, max_reqs) and taken(max_tokens, max_reqs, max_tiles) and taken(max_tokens, 1, max_tiles)
            and taken(few, max_reqs, max_tiles, 1) and taken(max(1, min(few, 8 * max_reqs // group)), max_reqs, max_tiles, 1))


_I32 = torch.int32
_MOST = 2 ** 31


def _attend(op, q, cache, block_table, seq_lens, q_start, tile_req, tile_q0, scale, out, softcap, window, causal, tmp, most_q=0):
    # What the rules of ops.validate say, in a fraction of their time (a decode step calls this in every layer); they name what is
    # wrong, and decide what is rare.
    given = out is not None
    try:
        (rows, cols), (nb, H, cells, width), (reqs, pages), (n,) = q.shape, cache.shape, block_table.shape, seq_lens.shape
        (ldq, q1), (ldt, t1) = q.stride(), block_table.stride()
        dev, D, qp, cp = q.get_device(), width // 18, q.data_ptr(), cache.data_ptr()
        ok = (dev >= 0 and dev == cache.get_device() == block_table.get_device() == seq_lens.get_device()
              and q.dtype is BF16 and cache.dtype is torch.uint8 and block_table.dtype is _I32
              and seq_lens.dtype is _I32 and (D == 128 or D == 64 or D == 256) and width == 18 * D and cells > 0 and pages > 0 and cols > 0
              and cols % (D * H) == 0 and cache.is_contiguous() and seq_lens.is_contiguous() and q1 == t1 == 1 and scale > 0
              and 0 <= softcap < math.inf and -_MOST < window < _MOST and (qp | cp | 2 * ldq) % 16 == 0)
        if ok and given:
            (orows, ocols), (ldo, o1), op_ = out.shape, out.stride(), out.data_ptr()
            ok = (orows == rows and ocols == cols and out.dtype is BF16 and out.get_device() == dev and o1 == 1
                  and (op_ | 2 * ldo) % 16 == 0 and (rows <= 1 or ldo >= cols)
                  and (op_ >= qp + 2 * ((rows - 1) * ldq + cols) or qp >= op_ + 2 * ((rows - 1) * ldo + cols)))
        if ok and tmp is not None:
            ok = (tmp.dtype is torch.float32 and tmp.get_device() == dev and tmp.is_contiguous()
                  and tmp.data_ptr() % 16 == 0 and tmp.numel() >= scratch_floats(q.device, D, op == "fp4_prefill"))
        if op == "fp4_decode":
            ok = ok and reqs >= rows and n >= rows and rows <= 8192
        else:
            ok = ok and (q_start.dtype is tile_req.dtype is tile_q0.dtype is _I32 and q_start.dim() == tile_req.dim() == tile_q0.dim() == 1
                         and dev == q_start.get_device() == tile_req.get_device() == tile_q0.get_device() and 8193 >= q_start.numel() > 0
                         and q_start.is_contiguous() and tile_req.is_contiguous() and tile_q0.is_contiguous()
                         and tile_q0.numel() >= tile_req.numel() <= 8000)
    except (TypeError, ValueError, AttributeError):
        ok = False
    if not given:
        out = q.new_empty(q.shape)
        op_, ldo = out.data_ptr(), out.stride(0) if out.dim() == 2 else 0
    if not ok:
        validate(op, q=q, cache=cache, block_table=block_table, seq_lens=seq_lens, q_start=q_start, tile_req=tile_req,
                 tile_q0=tile_q0, out=out, scale=scale, softcap=softcap, window=window, tmp=tmp)
        (rows, cols), (nb, H, cells, width), (reqs, pages), (n,) = q.shape, cache.shape, block_table.shape, seq_lens.shape
        D, qp, cp, op_, ldq, ldo, ldt = width // 18, q.data_ptr(), cache.data_ptr(), out.data_ptr(), q.stride(0), out.stride(0), block_table.stride(0)
    _declare()
    if tmp is None:
        tmp = q.new_empty(scratch_floats(q.device, D, op == "fp4_prefill"), dtype=torch.float32)
    a = AttnArgs()
    a.num_blocks, a.Hkv, a.block_size, a.Hq, a.D = nb, H, cells * CELL, cols // D, D
    a.q, a.out, a.cache, a.parts = qp, op_, cp, tmp.data_ptr()
    if rows > 1:                   # (the stride of a single row says nothing)
        a.ldq, a.ldo = ldq, ldo
    a.block_table, a.ldt, a.max_blocks = block_table.data_ptr(), ldt, pages
    a.seq_lens, a.total_q, a.num_reqs = seq_lens.data_ptr(), rows, rows
    if op == "fp4_prefill":
        a.q_start, a.num_reqs = q_start.data_ptr(), min(q_start.numel() - 1, reqs, n)
        a.tile_req, a.tile_q0, a.num_tiles = tile_req.data_ptr(), tile_q0.data_ptr(), tile_req.numel()
        a.most_q = max(0, min(most_q, rows))
    a.window, a.causal, a.scale, a.softcap = window, causal, scale, softcap
    _launch(q, _attn, a, op)
    return out


def decode(q: torch.Tensor, cache: torch.Tensor, *, block_table: torch.Tensor, seq_lens: torch.Tensor, scale: float,
           out: Optional[torch.Tensor] = None, softcap: float = 0.0, window: int = 0,
           tmp: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of one query row a sequence, ``q`` ``[B, Hq * D]``, at its last position. ``seq_lens`` int32 ``[B]`` counts the row's own
    key; 0: zeros come out. ``window`` as in :func:`vllm_cpp_b200.ops.attn_decode`; entries of ``block_table`` outside the cache count as
    masked keys. ``out`` shares no memory with the rows of ``q``. ``tmp``: :func:`scratch`, allocated if not given. At most 8192 sequences."""
    return _attend("fp4_decode", q, cache, block_table, seq_lens, None, None, None, scale, out, softcap, window, True, tmp)


def prefill(q: torch.Tensor, cache: torch.Tensor, *, block_table: torch.Tensor, seq_lens: torch.Tensor, q_start: torch.Tensor,
            tile_req: torch.Tensor, tile_q0: torch.Tensor, scale: float, out: Optional[torch.Tensor] = None, softcap: float = 0.0,
            window: int = 0, causal: bool = True, tmp: Optional[torch.Tensor] = None, max_query_len: int = 0) -> torch.Tensor:
    """Attention of the query rows ``q_start[r]..q_start[r + 1]`` of each sequence, the last of its ``seq_lens[r]`` positions.
    ``tile_req`` / ``tile_q0`` list their 128-row tiles, as in :func:`vllm_cpp_b200.ops.attn_prefill`. Sequences are as many as ``q_start``,
    ``block_table`` and ``seq_lens`` all have; rows outside every sequence stay as they are. A NaN that the cache holds reaches the
    queries that see its key, and no others. ``max_query_len``, the rows of the longest sequence, only chooses between kernels (0: not
    known, which costs a step of few rows a sequence one launch more). At head_dim 256 many rows take several times what they take over
    a bf16 cache.

    At most 8192 sequences and 8000 tiles; what a table of this width allows is counted in 31 bits (:func:`steps_fit`: 32 heads over 8 of
    128 dims with tables for four million tokens, of 256 dims for one million, in steps of 8192 tokens and 256 sequences are within; a
    ``KernelError`` says what is not). The bounds of ``q_start`` ascend: where they go back so often that the sequences come to more than
    that, the call writes nothing."""
    return _attend("fp4_prefill", q, cache, block_table, seq_lens, q_start, tile_req, tile_q0, scale, out, softcap, window, causal, tmp, max_query_len)


# ------------------------------------------------------------------------------ restatements
def scale_values(b: torch.Tensor) -> torch.Tensor:
    """Scale bytes as fp32."""
    return (b.to(torch.int16) << 7).view(torch.float16).float()


def ref_quantize(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """``x`` ``[..., D]`` -> codes ``[..., D]``, scale bytes ``[..., D / 16]``, both uint8."""
    g = x.float().unflatten(-1, (-1, 16))
    top = g.abs().amax(-1)                                       # (a NaN stays one)
    s = (top / torch.full_like(top, 6.0)).clamp(max=MOST_SCALE)
    step = torch.ldexp(torch.ones_like(s), (torch.frexp(s)[1] - 1).clamp(min=-14) - 3)
    scale = ((torch.round(s / step) * step).half().view(torch.int16) >> 7).to(torch.uint8)
    scale = torch.where(s.isnan(), torch.full_like(scale, 0xff), scale)
    s = scale_values(scale)[..., None]
    r = torch.where(s == 0, torch.zeros_like(g), g.abs() / s)
    code = sum((r > b if i % 2 == 0 else r >= b).to(torch.uint8) for i, b in enumerate((0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)))
    return (code | torch.signbit(g).to(torch.uint8) << 3).flatten(-2), scale


def _value_order(D: int, device) -> torch.Tensor:
    """Where 16-byte piece n of a cell's value codes lies."""
    n = torch.arange(D // 2, device=device)
    return n ^ (2 * (n // (D // 32) // 4))


def ref_write(k: torch.Tensor, v: torch.Tensor, cache: torch.Tensor, slots: torch.Tensor) -> None:
    nb, H, bs, D = shape_of(cache)
    ok = (slots >= 0) & (slots < nb * bs)
    slot = slots[ok]
    b, c, t = slot // bs, slot % bs // CELL, slot % CELL
    kc, ks = ref_quantize(k[ok].reshape(-1, H, D))
    vc, vs = ref_quantize(v[ok].reshape(-1, H, D))
    order = _value_order(D, cache.device).view(CELL, D // 32)
    row, groups = torch.arange(D // 2, device=cache.device), torch.arange(D // 16, device=cache.device)
    cells = cache.permute(0, 2, 1, 3)                            # [blocks, cells, heads, bytes]
    for i in range(slot.numel()):
        cell, tok = cells[b[i], c[i]], int(t[i])
        cell[:, tok * (D // 2) + row] = kc[i, :, 0::2] | kc[i, :, 1::2] << 4
        cell[:, 8 * D + order[tok][row // 16] * 16 + row % 16] = vc[i, :, 0::2] | vc[i, :, 1::2] << 4
        cell[:, 16 * D + tok * (D // 16) + groups] = ks[i]
        cell[:, 17 * D + groups * CELL + tok] = vs[i]


def ref_append(qkv, positions, cos_sin, cache, slots, *, num_q_heads, rot_dim=None, neox=True, q_norm=None, k_norm=None, eps=1e-6,
               gemma=False, q_out=None, q_head_stride=None, offsets=None) -> None:
    nb, H, bs, D = shape_of(cache)
    T, hs = qkv.shape[0], D if q_head_stride is None else q_head_stride
    o = (0, num_q_heads * D, (num_q_heads + H) * D) if offsets is None else offsets
    rot = 0 if cos_sin is None else cos_sin.shape[1] if rot_dim is None else rot_dim
    q = torch.stack([qkv[:, o[0] + i * hs: o[0] + i * hs + D] for i in range(num_q_heads)], 1).float() if num_q_heads else None
    k, v = (qkv[:, o[i]: o[i] + H * D].reshape(T, H, D).float() for i in (1, 2))

    def turned(x, w):
        if w is not None:
            x = x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + eps) * (w.float() + float(gemma))
        if not rot:
            return x
        inside = (positions >= 0) & (positions < cos_sin.shape[0])
        cs = cos_sin[torch.where(inside, positions, 0)]
        cs = torch.where(inside[:, None], cs, torch.full_like(cs, math.nan))
        return reference.apply_rope(x, cs[:, : rot // 2], cs[:, rot // 2:], rot, neox)
    k = turned(k, k_norm)
    if num_q_heads:
        q = turned(q, q_norm).to(qkv.dtype)
        if q_out is not None:
            q_out[:T, : num_q_heads * D] = q.flatten(1)
        else:
            for i in range(num_q_heads):
                qkv[:, o[0] + i * hs: o[0] + i * hs + D] = q[:, i]
    ref_write(k, v, cache, slots)


def ref_expand(cache: torch.Tensor) -> torch.Tensor:
    """The cache as bf16 ``[num_blocks, 2, block_size, Hkv, D]`` (exact)."""
    nb, H, bs, D = shape_of(cache)
    levels = torch.tensor(LEVELS + tuple(-x for x in LEVELS), device=cache.device)

    def values(codes, scales):                                   # [..., 16, D / 2], [..., 16, D / 16] bytes
        both = levels[torch.stack([codes & 15, codes >> 4], -1).flatten(-2).int()]
        return (both.unflatten(-1, (-1, 16)) * scale_values(scales)[..., None]).flatten(-2)
    k = values(cache[..., : 8 * D].unflatten(-1, (CELL, D // 2)), cache[..., 16 * D: 17 * D].unflatten(-1, (CELL, D // 16)))
    vc = cache[..., 8 * D: 16 * D].unflatten(-1, (D // 2, 16))[..., _value_order(D, cache.device), :]
    v = values(vc.flatten(-2).unflatten(-1, (CELL, D // 2)), cache[..., 17 * D:].unflatten(-1, (D // 16, CELL)).transpose(-1, -2))
    both = torch.stack([k, v], 1)                                # [nb, 2, H, cells, 16, D]
    return both.flatten(3, 4).transpose(2, 3).contiguous().to(BF16)


def ref_read(cache: torch.Tensor, slots: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    nb, H, bs, D = shape_of(cache)
    ok = (slots >= 0) & (slots < nb * bs)
    at = torch.where(ok, slots, 0)
    blocks, where = torch.unique(at // bs, return_inverse=True)
    held = ref_expand(cache[blocks])
    k, v = held[where, 0, at % bs], held[where, 1, at % bs]
    zero = torch.zeros((), dtype=BF16, device=cache.device)
    return torch.where(ok[:, None, None], k, zero), torch.where(ok[:, None, None], v, zero)


def ref_attention(q, cache, *, block_table, seq_lens, q_start, scale, softcap=0.0, window=0, causal=True) -> torch.Tensor:
    """:func:`prefill` (and, with ``q_start`` 0, 1, 2.., :func:`decode`) over the pages that the sequences use; their table entries lie
    inside the cache."""
    nb, H, bs, D = shape_of(cache)
    used = [int(-(-int(n) // bs)) for n in seq_lens]
    ids = torch.cat([block_table[r, :n] for r, n in enumerate(used)] or [block_table.new_zeros(0)]).long()
    blocks, where = torch.unique(ids, return_inverse=True)
    table = torch.zeros((len(used), max(used, default=0) or 1), dtype=torch.int32, device=cache.device)
    at = 0
    for r, n in enumerate(used):
        table[r, :n] = where[at: at + n].int()
        at += n
    kv = ref_expand(cache[blocks]) if blocks.numel() else ref_expand(cache[:1])
    return reference.paged_attention(q, kv, table, seq_lens, q_start, q.shape[1] // D, H, D, bs, scale, softcap, window, causal)
