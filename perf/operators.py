"""Operators over a paged KV cache held in 4 bits, as a serving step uses them: what is measured, in plain torch and through
``vllm_cpp_b200.ops.fp4_cache``.

``append``: merged ``[q | k | v]`` rows of a step are normed per head (optionally) and rotated; q goes on, k and v go into the
cache in groups of 16 dimensions, each with a scale (largest magnitude / 6) of 5 exponent and 3 mantissa bits, which are an f16's
behind its sign, and e2m1 codes of value / scale. What comes back: q, and the keys and values that the cache now holds for these
tokens.
``decode``: attention of one new token a sequence over its cached keys and values.
``prefill``: attention of several new tokens a sequence (prompts, portions of prompts, drafts to verify), causal from the end.

Cache of a layer: uint8 ``[pages, kv heads, page tokens / 16, 18 D]``. 16 tokens of a head are one cell: key codes ``[16, D / 2]``
(low nibble first), value codes the same but with 16-byte piece ``n`` at ``n ^ 2 (token / 4)``, key scales ``[16, D / 16]``, value
scales ``[D / 16, 16]``.
"""
import math
import random

import torch

own = False

LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
MOST = 10240.0                 # largest scale: 6 times it is still an f16
NONE = -1                      # slot of a padding row


def _spread(n, low, high):
    """``n`` lengths between ``low`` and ``high`` in an order that jumps about."""
    return [low + (high - low) * ((i * 7919 + n * 31) % 97) // 96 for i in range(n)]


def listed():
    a = dict(op="append", page=32, d=128, rot=128, norm=False)
    d = dict(op="decode", page=32, d=128, window=0, softcap=0.0)
    p = dict(op="prefill", page=32, d=128, window=0, softcap=0.0)
    cases = {
        # one user's next token: the latency of a layer's cache write
        "append, one token": dict(a, tokens=1, pad=0, hq=32, hkv=8),
        # a full decode batch of a model with normed heads, padded to a graph's size
        "append, a decode batch": dict(a, tokens=250, pad=6, hq=16, hkv=8, norm=True),
        # a prefill step of 8192 tokens
        "append, a full step": dict(a, tokens=8192, pad=0, hq=32, hkv=8),
        # one user in a chat
        "decode, one chat": dict(d, batch=1, low=1000, high=1000, hq=32, hkv=8),
        # one user with a long document
        "decode, one long context": dict(d, batch=1, low=120001, high=120001, hq=32, hkv=8),
        # a loaded server, ragged contexts, eight query heads a key head
        "decode, 60 requests": dict(d, batch=60, low=17, high=3000, hq=32, hkv=4),
        # a full server
        "decode, 256 requests": dict(d, batch=256, low=200, high=3800, hq=32, hkv=8),
        # 64-dim heads in a sliding window with capped scores
        "decode, window": dict(d, batch=33, low=1, high=9000, hq=24, hkv=8, d=64, window=1024, softcap=30.0),
        # ragged short prompts in one step
        "prefill, short prompts": dict(p, reqs=13, q_low=3, q_high=211, c_low=0, c_high=0, hq=32, hkv=8),
        # drafts of a batch verified: a few new tokens each after a long context
        "prefill, drafts": dict(p, reqs=48, q_low=2, q_high=6, c_low=100, c_high=4000, hq=32, hkv=8),
        # a portion of a long prompt after the portions before it
        "prefill, a later portion": dict(p, reqs=1, q_low=1999, q_high=1999, c_low=30000, c_high=30000, hq=32, hkv=8),
        # a long prompt in one step
        "prefill, 8192 tokens": dict(p, reqs=1, q_low=8192, q_high=8192, c_low=0, c_high=0, hq=32, hkv=8),
    }
    return [dict(name=k, **v) for k, v in cases.items()]


def draw(rng):
    def log(low, high):
        return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))

    op = rng.choice(["append", "decode", "prefill"])
    hkv = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 2, 3, 4, 5, 6, 7, 8, 12, 16])
    while hkv * group > 32:
        group = rng.choice([1, 2, 3, 4, 5, 6, 7, 8, 12, 16])
    c = dict(op=op, page=rng.choice([16, 32, 64, 128]), d=rng.choice([64, 128, 128]), hq=hkv * group, hkv=hkv)
    if op == "append":
        c.update(tokens=log(1, 8000), pad=rng.choice([0, 0, 3]), rot=rng.choice([c["d"], c["d"], c["d"] // 2]), norm=rng.random() < 0.4)
        return c
    c.update(window=rng.choice([0, 0, 0, log(16, 4000)]), softcap=rng.choice([0.0, 0.0, 0.0, 25.0]))
    if op == "decode":
        batch = log(1, 256)
        high = min(100000, log(1, max(2, 500000 // batch)))
        c.update(batch=batch, low=log(1, high), high=high)
        return c
    reqs = log(1, 40)
    q_high = log(2, max(3, 5000 // reqs))
    c_high = rng.choice([0, log(1, max(2, 30000 // reqs))])
    c.update(reqs=reqs, q_low=log(1, q_high), q_high=q_high, c_low=rng.randint(0, c_high), c_high=c_high)
    return c


def _lengths(c):
    """(new tokens, all tokens) of each sequence."""
    if c["op"] == "decode":
        return [1] * c["batch"], _spread(c["batch"], c["low"], c["high"])
    q = _spread(c["reqs"], c["q_low"], c["q_high"])
    return q, [a + b for a, b in zip(q, _spread(c["reqs"], c["c_low"], c["c_high"])[::-1])]


def _page_table(lengths, page, gen):
    """Pages of the sequences, in no order; page 0 belongs to none. Behind a sequence's pages: page 0."""
    counts = [max(1, -(-n // page)) for n in lengths]
    total = sum(counts) + 1
    perm = (torch.randperm(total - 1, generator=gen, device="cuda") + 1).to(torch.int32)
    table = torch.zeros((len(lengths), max(counts)), dtype=torch.int32, device="cuda")
    have = torch.arange(max(counts), device="cuda")[None] < torch.tensor(counts, device="cuda")[:, None]
    table[have] = perm
    return table, total


def _random_cache(pages, hkv, page, d, gen):
    """Codes and scales of normal values; scales differ from group to group, some dimensions are large."""
    cells = page // 16
    n = pages * hkv * cells
    cache = torch.empty((n, 18 * d), dtype=torch.uint8, device="cuda")
    step = max(1, (1 << 28) // (16 * d))
    for at in range(0, n, step):
        part = cache[at: at + step]
        x = torch.randn((part.shape[0], 16 * d, 2), generator=gen, device="cuda", dtype=torch.float16)
        mag = (x.abs() * 4).round_().clamp_(max=7).to(torch.uint8)
        code = mag | ((x < 0).to(torch.uint8) << 3)
        part[:, : 16 * d] = code[..., 0] | (code[..., 1] << 4)
        s = torch.randn((part.shape[0], 2 * d), generator=gen, device="cuda").mul_(0.5).exp_().mul_(0.2)
        part[:, 16 * d:] = _scale_bytes(s)
    return cache.view(pages, hkv, cells, 18 * d)


def prepare(case, seed):
    c = case
    gen = torch.Generator(device="cuda").manual_seed(seed)
    d, page, hq, hkv = c["d"], c["page"], c["hq"], c["hkv"]
    s = {"case": c}
    if c["op"] == "append":
        n, rot = c["tokens"], c["rot"]
        t = n + c["pad"]
        far = 40000
        x = torch.randn((t, (hq + 2 * hkv) * d), generator=gen, device="cuda")
        x *= torch.randn((1, (hq + 2 * hkv) * d), generator=gen, device="cuda").mul_(0.7).exp_()
        inv = 10000.0 ** (-torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / rot)
        angle = torch.arange(far, device="cuda", dtype=torch.float64)[:, None] * inv
        s["table"] = torch.cat([angle.cos(), angle.sin()], 1).float()
        s["qkv"] = x.to(torch.bfloat16)
        s["positions"] = torch.randint(0, far, (t,), generator=gen, device="cuda")
        pages = -(-n // page) + 3
        s["cache"] = torch.zeros((pages, hkv, page // 16, 18 * d), dtype=torch.uint8, device="cuda")
        s["slots"] = torch.cat([torch.randperm(pages * page, generator=gen, device="cuda")[:n],
                                torch.full((c["pad"],), NONE, device="cuda", dtype=torch.int64)])
        w = (1 + 0.2 * torch.randn((2, d), generator=gen, device="cuda")).to(torch.bfloat16)
        s["q_norm"], s["k_norm"] = (w[0], w[1]) if c["norm"] else (None, None)
        s["q_out"] = torch.empty((t, hq * d), dtype=torch.bfloat16, device="cuda")
        return s
    new, lengths = _lengths(c)
    s["table"], pages = _page_table(lengths, page, gen)
    s["cache"] = _random_cache(pages, hkv, page, d, gen)
    t = sum(new)
    s["q"] = torch.randn((t, hq * d), generator=gen, device="cuda").mul_(3).to(torch.bfloat16)     # scores of a spread of about two
    s["out"] = torch.empty_like(s["q"])
    s["lengths"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    s["starts"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
    tiles = [(r, at) for r, n in enumerate(new) for at in range(0, n, 128)]
    s["tile_req"] = torch.tensor([r for r, _ in tiles], dtype=torch.int32, device="cuda")
    s["tile_q0"] = torch.tensor([at for _, at in tiles], dtype=torch.int32, device="cuda")
    s["most_new"], s["most"] = max(new), max(lengths)
    return s


# ------------------------------------------------------------------------------------------------ the plain forms
def _scale_bytes(s):
    """Scales of few bits -> the bits of an f16 behind its sign, its last seven left off."""
    return (s.half().view(torch.int16) >> 7).to(torch.uint8)


def _scale_values(b):
    return (b.to(torch.int16) << 7).view(torch.float16).float()


def _codes_and_scales(x):
    """fp32 [..., D] -> codes [..., D] (0..15), scales [..., D / 16]."""
    g = x.unflatten(-1, (-1, 16))
    six = torch.full((), 6.0, dtype=torch.float64, device=x.device)
    s = g.abs().amax(-1).double() / six
    step = torch.ldexp(torch.ones_like(s), (torch.frexp(s)[1] - 1).clamp(min=-14) - 3)
    scale = (torch.round(s / step) * step).clamp(max=MOST)
    r = g.abs().double() / scale[..., None]
    r = torch.where(scale[..., None] > 0, r, torch.zeros_like(r))
    # the nearest of the levels, of two that are equally near the one with an even code
    code = ((r > 0.25).int() + (r >= 0.75).int() + (r > 1.25).int() + (r >= 1.75).int() + (r > 2.5).int() + (r >= 3.5).int()
            + (r > 5.0).int())
    code = code + 8 * torch.signbit(g).int()
    return code.flatten(-2), scale.float()


def _values(codes, scales, levels):
    """codes [..., D], scales [..., D / 16] -> fp32 [..., D]."""
    return (levels[codes.int()].unflatten(-1, (-1, 16)) * scales[..., None]).flatten(-2)


def _levels(dtype=torch.float32):
    v = torch.tensor(LEVELS, device="cuda", dtype=dtype)
    return torch.cat([v, -v])


def _value_order(d):
    """Where 16-byte piece n of a cell's value codes is."""
    n = torch.arange(d // 2, device="cuda")
    return n ^ (2 * (n // (d // 32) // 4))


def _pack(codes):
    return (codes[..., 0::2] | (codes[..., 1::2] << 4)).to(torch.uint8)


def _unpack(b):
    return torch.stack([b & 15, b >> 4], -1).flatten(-2)


def _cells(cells, d):
    """Bytes [..., 18 D] of cells -> (keys, values) fp32 [..., 16, D]."""
    levels = _levels()
    k = _unpack(cells[..., : 8 * d].unflatten(-1, (16, d // 2)))
    v = cells[..., 8 * d: 16 * d].unflatten(-1, (d // 2, 16))[..., _value_order(d), :]
    v = _unpack(v.flatten(-2).unflatten(-1, (16, d // 2)))
    ks = _scale_values(cells[..., 16 * d: 17 * d].unflatten(-1, (16, d // 16)))
    vs = _scale_values(cells[..., 17 * d:].unflatten(-1, (d // 16, 16)).transpose(-1, -2))
    return _values(k, ks, levels), _values(v, vs, levels)


def _normed(x, w):
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w.float() if w is not None else x


def _rotated(x, cos, sin, rot):
    a, b, rest = x[..., : rot // 2], x[..., rot // 2: rot], x[..., rot:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, rest], -1)


def _append_plain(s):
    c = s["case"]
    d, page, hq, hkv, rot = c["d"], c["page"], c["hq"], c["hkv"], c["rot"]
    t = s["qkv"].shape[0]
    x = s["qkv"].float().view(t, hq + 2 * hkv, d)
    q, k, v = x[:, :hq], x[:, hq: hq + hkv], x[:, hq + hkv:]
    cs = s["table"][s["positions"]][:, None]
    q = _rotated(_normed(q, s["q_norm"]), cs[..., : rot // 2], cs[..., rot // 2:], rot)
    k = _rotated(_normed(k, s["k_norm"]), cs[..., : rot // 2], cs[..., rot // 2:], rot)
    kc, ks = _codes_and_scales(k)
    vc, vs = _codes_and_scales(v)
    # into the cache: each token's bytes at its cell
    slots = s["slots"]
    used = (slots >= 0).nonzero()[:, 0]
    slot = slots[used]
    blk, cell, tok = slot // page, slot % page // 16, slot % 16
    at = (blk[:, None], torch.arange(hkv, device="cuda")[None], cell[:, None])
    cache = s["cache"]
    n = tok[:, None] * (d // 2) + torch.arange(d // 2, device="cuda")[None]                          # byte of a row of codes
    cache[at[0][..., None], at[1][..., None], at[2][..., None], n[:, None]] = _pack(kc[used])
    swapped = ((n // 16) ^ (2 * (tok[:, None] // 4))) * 16 + n % 16
    cache[at[0][..., None], at[1][..., None], at[2][..., None], 8 * d + swapped[:, None]] = _pack(vc[used])
    group = torch.arange(d // 16, device="cuda")[None]
    cache[at[0][..., None], at[1][..., None], at[2][..., None], (16 * d + tok[:, None] * (d // 16) + group)[:, None]] = \
        _scale_bytes(ks[used])
    cache[at[0][..., None], at[1][..., None], at[2][..., None], (17 * d + group * 16 + tok[:, None])[:, None]] = \
        _scale_bytes(vs[used])
    levels = _levels()
    there = (slots >= 0)[:, None, None]
    k, v = _values(kc, ks, levels) * there, _values(vc, vs, levels) * there
    return q.flatten(1).to(torch.bfloat16), k.to(torch.bfloat16), v.to(torch.bfloat16)


def _attention_plain(s):
    """All sequences at once, padded to the longest."""
    c = s["case"]
    d, page, hq, hkv = c["d"], c["page"], c["hq"], c["hkv"]
    b, m, n = s["table"].shape[0], s["most_new"], s["table"].shape[1] * page
    k, v = _cells(s["cache"][s["table"].long()], d)                     # [B, pages, hkv, cells, 16, D]
    k, v = (x.transpose(1, 2).reshape(b, hkv, n, d) for x in (k, v))
    new = s["starts"][1:] - s["starts"][:-1]
    step = torch.arange(m, device="cuda")
    real = step[None] < new[:, None]
    rows = (s["starts"][:-1, None] + step[None]).clamp(max=s["q"].shape[0] - 1)
    q = s["q"].float().view(-1, hkv, hq // hkv, d)[rows].permute(0, 2, 3, 1, 4).reshape(b, hkv, -1, d)
    score = (q @ k.transpose(-1, -2)).view(b, hkv, hq // hkv, m, n).mul_(1 / math.sqrt(d))
    if c["softcap"] > 0:
        score = score.div_(c["softcap"]).tanh_().mul_(c["softcap"])
    at = (s["lengths"] - new)[:, None] + step[None]                     # position of each query
    key = torch.arange(n, device="cuda")
    seen = key[None, None] <= at[..., None]
    if c["window"] > 0:
        seen = seen & (key[None, None] > at[..., None] - c["window"])
    score.masked_fill_(~seen[:, None, None], -math.inf)
    score.sub_(score.amax(-1, keepdim=True)).exp_()
    score.div_(score.sum(-1, keepdim=True))
    v = torch.where(key[None, None, :, None] < s["lengths"][:, None, None, None], v, torch.zeros((), device="cuda"))
    out = (score.view(b, hkv, -1, n) @ v).view(b, hkv, hq // hkv, m, d).permute(0, 3, 1, 2, 4).reshape(b, m, hq * d)
    return out[real].to(torch.bfloat16)


# ----------------------------------------------------------------------------------------- the framework's operators
def _append_own(s):
    from vllm_cpp_b200.ops import fp4_cache
    c = s["case"]
    fp4_cache.append(s["qkv"], s["positions"], s["table"], s["cache"], s["slots"], num_q_heads=c["hq"], rot_dim=c["rot"],
                     q_norm=s["q_norm"], k_norm=s["k_norm"], eps=1e-6, q_out=s["q_out"])
    k, v = fp4_cache.read(s["cache"], s["slots"])
    return s["q_out"], k, v


def _attention_own(s):
    from vllm_cpp_b200.ops import fp4_cache
    c = s["case"]
    common = dict(block_table=s["table"], seq_lens=s["lengths"], scale=1 / math.sqrt(c["d"]), out=s["out"], softcap=c["softcap"],
                  window=c["window"])
    if c["op"] == "decode":
        return fp4_cache.decode(s["q"], s["cache"], **common)
    return fp4_cache.prefill(s["q"], s["cache"], q_start=s["starts"], tile_req=s["tile_req"], tile_q0=s["tile_q0"], **common)


def run(state):
    append = state["case"]["op"] == "append"
    if own:
        return _append_own(state) if append else _attention_own(state)
    return _append_plain(state) if append else _attention_plain(state)


def _seen(c):
    """(pairs of query token and visible key, keys that some query of their sequence sees), over all sequences."""
    new, lengths = _lengths(c)
    w = c["window"]
    pairs = keys = 0
    for n, total in zip(new, lengths):
        first = total - n                                                # position of the first query
        if w <= 0:
            pairs += n * first + n * (n + 1) // 2
            keys += total
        else:
            short = max(0, min(n, w - first))                            # queries whose window is not full
            pairs += short * first + short * (short + 1) // 2 + (n - short) * w
            keys += total - max(0, first - w + 1)
    return pairs, keys


def work(case):
    c = case
    d, hq, hkv = c["d"], c["hq"], c["hkv"]
    held = 2 * (d // 2 + d // 16)                                       # bytes of a token's key and value of a head
    if c["op"] == "append":
        t, n = c["tokens"] + c["pad"], c["tokens"]
        moved = t * (hq + 2 * hkv) * d * 2 + t * hq * d * 2 + t * hkv * 2 * d * 2 + n * hkv * held + t * (c["rot"] * 4 + 16)
        return {"bytes": moved, "flops": t * (hq + hkv) * d * 4 + t * hkv * 2 * d * 4}
    new, lengths = _lengths(c)
    pairs, keys = _seen(c)
    table = sum(-(-n // c["page"]) for n in lengths) * 4
    return {"bytes": keys * hkv * held + 2 * sum(new) * hq * d * 2 + table, "flops": 4 * pairs * hq * d}


# ------------------------------------------------------------------------------------------ the definition, in 64 bits
_SCALES = [(m / 8 * 2.0 ** -14) if e == 0 else (1 + m / 8) * 2.0 ** (e - 15) for e in range(31) for m in range(8)]
_USED = [v for v in _SCALES if v <= MOST]


def _nearest(x, values):
    """Index of the nearest of the ascending ``values``, ties to the even index."""
    v = torch.tensor(values, dtype=torch.float64, device=x.device)
    mid = (v[1:] + v[:-1]) / 2
    low = torch.searchsorted(mid, x.contiguous(), right=False)
    tie = (low < len(values) - 1) & (x == mid[low.clamp(max=len(values) - 2)])
    return torch.where(tie & (low % 2 == 1), low + 1, low)


def _quantised(x):
    g = x.reshape(*x.shape[:-1], -1, 16)
    top = g.abs().amax(-1) / torch.tensor(6.0, dtype=torch.float64, device=x.device)
    s = torch.tensor(_USED, dtype=torch.float64, device=x.device)[_nearest(top, _USED)]
    s = s[..., None]
    r = torch.where(s > 0, g.abs() / torch.where(s > 0, s, torch.ones_like(s)), torch.zeros_like(g))
    held = torch.tensor(LEVELS, dtype=torch.float64, device=x.device)[_nearest(r, list(LEVELS))] * s
    return torch.where(g < 0, -held, held).reshape(x.shape)


def _append_exact(s):
    c = s["case"]
    d, hq, hkv, half = c["d"], c["hq"], c["hkv"], c["rot"] // 2
    x = s["qkv"].double().reshape(-1, hq + 2 * hkv, d)
    cos, sin = (u.unsqueeze(1) for u in s["table"].double()[s["positions"]].split(half, 1))
    turned = []
    for head in range(hq + hkv):
        h = x[:, head: head + 1]
        w = s["q_norm"] if head < hq else s["k_norm"]
        if w is not None:
            h = h / torch.sqrt(h.pow(2).sum(-1, keepdim=True) / d + 1e-6) * w.double()
        z = torch.complex(h[..., :half], h[..., half: 2 * half]) * torch.complex(cos, sin)
        turned.append(torch.cat([z.real, z.imag, h[..., 2 * half:]], -1))
    y = torch.cat(turned, 1)
    there = (s["slots"] >= 0).double()[:, None, None]
    return y[:, :hq].flatten(1), _quantised(y[:, hq:]) * there, _quantised(x[:, hq + hkv:]) * there


def _held(cell, d):
    """Keys and values [tokens, D] of cells [n, 18 D], in 64 bits."""
    n = cell.shape[0]
    level = torch.tensor([-v if i >= 8 else v for i, v in enumerate(LEVELS * 2)], dtype=torch.float64, device=cell.device)

    def values(codes, scale):
        both = torch.empty((n, 16, d), dtype=torch.float64, device=cell.device)
        both[..., 0::2], both[..., 1::2] = level[(codes % 16).long()], level[(codes // 16).long()]
        return (both * scale.repeat_interleave(16, -1)).reshape(n * 16, d)

    scales = torch.tensor(_SCALES, dtype=torch.float64, device=cell.device)[cell[:, 16 * d:].long()]
    keys = values(cell[:, : 8 * d].reshape(n, 16, d // 2), scales[:, :d].reshape(n, 16, d // 16))
    rows = torch.empty((n, 16, d // 2), dtype=torch.uint8, device=cell.device)
    for token in range(16):
        for piece in range(d // 32):
            at = 8 * d + 16 * ((token * (d // 32) + piece) ^ (2 * (token // 4)))
            rows[:, token, 16 * piece: 16 * piece + 16] = cell[:, at: at + 16]
    return keys, values(rows, scales[:, d:].reshape(n, d // 16, 16).transpose(1, 2))


def _attention_exact(s):
    c = s["case"]
    d, page, hq, hkv = c["d"], c["page"], c["hq"], c["hkv"]
    new, lengths = _lengths(c)
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    first = 0
    for r, (m, total) in enumerate(zip(new, lengths)):
        pages = s["cache"][s["table"][r, : -(-total // page)].long()]
        at = torch.arange(total - m, total, device="cuda")[:, None]
        key = torch.arange(total, device="cuda")[None]
        hidden = key > at
        if c["window"] > 0:
            hidden = hidden | (at - key >= c["window"])
        for h in range(hkv):
            k, v = _held(pages[:, h].reshape(-1, 18 * d), d)
            for g in range(hq // hkv):
                cols = slice((h * (hq // hkv) + g) * d, (h * (hq // hkv) + g + 1) * d)
                z = s["q"][first: first + m, cols].double() @ k[:total].t() / math.sqrt(d)
                if c["softcap"] > 0:
                    z = c["softcap"] * torch.tanh(z / c["softcap"])
                out[first: first + m, cols] = torch.softmax(z.masked_fill(hidden, -math.inf), -1) @ v[:total]
        first += m
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return _append_exact(s) if case["op"] == "append" else _attention_exact(s)


if __name__ == "__main__":
    for case in listed() + [draw(random.Random(i)) for i in range(5)]:
        print(case.get("name", "drawn"), case, work(case))
