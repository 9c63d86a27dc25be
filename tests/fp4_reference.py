"""The operators of the 4-bit KV cache in 64 bits, written from their definition, and bounds on how far a kernel may be off.

Bounds. bf16 results round by at most 2^-8 of the value. Attention: probabilities are rounded to f16 (2^-11 of each) before they meet the
values, and scores are sums in 32 bits of exact products; a matrix instruction of 16 products adds at most about 2^-22 of the largest
partial sum, so over a head of at most 256 dims a score of the tests' size (|q| |k| scale below 100, at most 16 instructions) is off by less
than 16 * 100 * 2^-22 < 2^-11. Numerator and denominator together: the result is off by at most 2^-10 of the same average of |v|,
which leaves 2^-9 with the exponentials' own errors (2^-22) and soft caps (tanh, some 2^-22 of the cap). Probabilities that are f16
subnormals are off by up to 2^-25 where the largest is at least 2^7: 2^-32 of the largest for each key, at most n 2^-32 max |v| of the
result. Appended keys: sums of two fp32
products and a norm's sum over at most 256 dims keep a rotated value within 2^-18 of the magnitudes that went into it, so the code lies
between those of the values that far below and above."""
import math

import torch

LEVELS = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)
SCALES = torch.tensor([(m / 8 * 2.0 ** -14) if e == 0 else (1 + m / 8) * 2.0 ** (e - 15) for e in range(31) for m in range(8)],
                      dtype=torch.float64)
SCALES = SCALES[SCALES <= 10240]


def nearest(x, values):
    """The nearest of the ascending ``values`` to each of ``x`` >= 0, of two the one with the even index."""
    v = values.to(x.device)
    mid = (v[1:] + v[:-1]) / 2
    i = torch.searchsorted(mid, x.contiguous())
    tie = (i < mid.numel()) & (x == mid[i.clamp(max=mid.numel() - 1)])
    return v[torch.where(tie & (i % 2 == 1), i + 1, i)]


def scales(x):
    """[..., D] -> the scales [..., D / 16], in 64 bits."""
    return nearest(x.double().unflatten(-1, (-1, 16)).abs().amax(-1) / 6, SCALES)


def held(x, s):
    """What the cache keeps of ``x`` [..., D] with the scales ``s`` [..., D / 16]."""
    g, s = x.double().unflatten(-1, (-1, 16)), s.double()[..., None]
    r = torch.where(s > 0, g.abs() / torch.where(s > 0, s, torch.ones_like(s)), torch.zeros_like(g))
    return (torch.sign(g) * nearest(r, LEVELS) * s).flatten(-2)


def rotated(x, w, eps, gemma, cos, sin, rot, neox):
    """(heads [T, H, D] normed and rotated, the magnitudes that went into each value), 64 bits."""
    x = x.double()
    if w is not None:
        x = x / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + eps) * (w.double() + (1 if gemma else 0))
    if not rot:
        return x, x.abs()
    i = torch.arange(rot, device=x.device)
    j = i % (rot // 2) if neox else i // 2
    minus = i < rot // 2 if neox else i % 2 == 0
    other = x[..., torch.where(minus, i + (rot // 2 if neox else 1), i - (rot // 2 if neox else 1))]
    c, s = cos.double()[:, None, j], sin.double()[:, None, j] * torch.where(minus, -1.0, 1.0).double()
    y, big = x.clone(), x.abs()
    y[..., :rot] = x[..., :rot] * c + other * s
    big[..., :rot] = (x[..., :rot] * c).abs() + (other * s).abs()
    return y, big


def check_held(got, y, big):
    """``got`` [T, H, D], read back from the cache, is what ``y`` within 2^-18 ``big`` may have become."""
    got, off = got.double(), big * 2.0 ** -18
    top_low, top_high = ((y.abs() + k * off).clamp(min=0).unflatten(-1, (-1, 16)).amax(-1) / 6 for k in (-1, 1))
    s_low, s_high = nearest(top_low, SCALES), nearest(top_high, SCALES)
    ok = torch.zeros(got.unflatten(-1, (-1, 16)).shape[:-1], dtype=torch.bool, device=got.device)
    for s in (s_low, s_high):                                  # (at most two neighbouring scales are in reach)
        low, high = held(y - off, s), held(y + off, s)
        ok |= ((got >= low) & (got <= high)).unflatten(-1, (-1, 16)).all(-1)
    assert bool(ok.all()), f"{int((~ok).sum())} of {ok.numel()} groups are not what the cache should hold"


def attention(q, k, v, first, scale, softcap, window, causal=True):
    """One sequence: q [m, Hq, D] at positions first.., k and v [n, Hkv, D] -> (out, the same average of |v| and the share of
    subnormal probabilities, in units of 2^-9) [m, Hq, D], 64 bits; a row that sees nothing is zero."""
    m, n, G = q.shape[0], k.shape[0], q.shape[1] // k.shape[1]
    if n == 0:
        zero = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
        return zero, zero
    k, v = k.double().repeat_interleave(G, 1), v.double().repeat_interleave(G, 1)
    s = torch.einsum("mhd,nhd->hmn", q.double(), k) * scale
    if softcap:
        s = softcap * torch.tanh(s / softcap)
    at, key = torch.arange(first, first + m, device=q.device)[:, None], torch.arange(n, device=q.device)[None]
    seen = key <= at if causal else (key <= n).expand(m, n).clone()
    if window > 0:
        seen = seen & (key > at - window)
    elif window < 0:
        seen = seen & (key >= at.clamp(min=0) // -window * -window)
    s = s.masked_fill(~seen, -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True).clamp(min=-1e300))
    p = torch.where(seen, p, torch.zeros_like(p))
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-300)
    return torch.einsum("hmn,nhd->mhd", p, v), torch.einsum("hmn,nhd->mhd", p, v.abs()) + n * 2.0 ** -23 * v.abs().max()


def check_attention(got, want, size):
    err = (got.double() - want).abs()
    tol = 2.0 ** -8 * want.abs() + 2.0 ** -9 * size + 1e-30
    assert bool((err <= tol).all()), f"off by {float((err / tol).max()):.3g} times the bound at {int((err > tol).sum())} of {err.numel()}"


def random_cache(nb, H, bs, D, gen, device="cpu"):
    """Random codes and scales between 2^-5 and 2."""
    c = torch.randint(0, 256, (nb, H, bs // 16, 18 * D), dtype=torch.uint8, generator=gen)
    c[..., 16 * D:] = torch.randint(80, 129, c[..., 16 * D:].shape, dtype=torch.uint8, generator=gen)
    return c.to(device)
