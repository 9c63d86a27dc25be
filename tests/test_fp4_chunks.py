"""Chunks of a 4-bit cache that travel as bf16: the values come back, but in groups whose scale is below 2^-14."""
import time

import torch

import fp4_reference as F
from test_lmcache import MockServer
from vllm_cpp_b200.ops import fp4_cache
from vllm_cpp_b200.worker.lmcache import LMCacheStore


def test_values_come_back_but_for_the_smallest_groups():
    srv = MockServer()
    srv.start()
    H, D, bs, n = 2, 64, 16, 64
    gen = torch.Generator().manual_seed(0)
    # groups from 2^-24 to past the largest scale, and NaN
    x = torch.randn((2, n, H * D), generator=gen) * torch.exp2(torch.randint(-24, 18, (2, n, H * D // 16), generator=gen).float()).repeat_interleave(16, -1)
    x[0, 3, 5] = float("nan")
    x = x.to(torch.bfloat16)
    cache = fp4_cache.alloc(4, H, bs, D, "cpu")
    fp4_cache.ref_write(x[0], x[1], cache, torch.arange(n))
    store = LMCacheStore(f"lm://127.0.0.1:{srv.port}", "tiny", [cache], bs, chunk_size=32)
    tokens, blocks = list(range(n + 6)), [0, 1, 2, 3]
    assert store.store(tokens, blocks) == 2
    deadline = time.monotonic() + 5.0
    while len(srv.store) < 2 and time.monotonic() < deadline:
        time.sleep(0.01)
    back = torch.zeros_like(cache)
    other = LMCacheStore(f"lm://127.0.0.1:{srv.port}", "tiny", [back], bs, chunk_size=32, connect=False)
    other.client = store.client
    assert other.load(tokens, blocks, n) == n
    differ = 0
    for a, b, y in zip(fp4_cache.ref_read(cache, torch.arange(n)), fp4_cache.ref_read(back, torch.arange(n)), x):
        s = F.scales(y.view(n, H, D))
        small = (s < 2.0 ** -14).repeat_interleave(16, -1)
        same = (a == b) | (a.isnan() & b.isnan())
        assert bool(same[~small].all())
        differ += int((~same).sum())
    assert differ > 0                                          # (the smallest do change: what is said of them is not idle)
    store.client.close()
