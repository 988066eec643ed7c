"""GPU: calls whose blocks take several tokens of a request together - more than 128 MiB of keys, a hundred units and more, every four or two
consecutive places of one row - with sliding windows, soft caps, sinks, places without a token and two head sets, against fp64.  The bounds are
those of test_paged_attention_gpu.py, whose small calls of windows never come to share a block."""
from types import SimpleNamespace

import numpy as np
import pytest
import torch

from basalt_b200 import paged
from tests.test_paged_attention_gpu import check

pytestmark = pytest.mark.gpu
BF, F32, F8 = torch.bfloat16, torch.float32, torch.float8_e4m3fn


def served(seed, requests, shortest, longest, hk, D, kind, page=64):
    g, rng = torch.Generator(device="cuda").manual_seed(seed), np.random.default_rng(seed)
    lengths = rng.integers(shortest, longest, requests).tolist()
    per = -(-longest // page)
    scales = (0.3 + 0.4 * torch.rand((2, hk), generator=g, device="cuda")) if kind == F8 else (None, None)
    cache = paged.KVCache.empty(requests * per, hk, page, D, kind, None, *scales)
    for c in (cache.k, cache.v):
        c.copy_(torch.randn(c.shape, generator=g, device="cuda").to(kind))
    table = torch.randperm(requests * per, generator=torch.Generator().manual_seed(seed)).to(torch.int32).view(requests, per).cuda()
    host = SimpleNamespace(k=cache.k.cpu(), v=cache.v.cpu(), k_scale=cache.k_scale, v_scale=cache.v_scale, n_kv_heads=hk)
    return cache, table, lengths, host, g


def shares(new, row, pos, window, hk, hq, D, kind):
    """The rule by which a block takes `new` places together, on the host: their rows, the keys' bytes, the units."""
    keys = lambda t: min(pos[t] + 1, window or 2 ** 31) if row[t] >= 0 else 0  # noqa: E731
    groups = [range(t, min(t + new, len(row))) for t in range(0, len(row), new)]
    live = [[t for t in x if keys(t)] for x in groups]
    one_row = all(len({row[t] for t in x}) <= 1 for x in live)
    tokens, filled = sum(map(len, live)), sum(map(bool, live))
    full = tokens >= 3 * filled if new == 4 else tokens == 2 * filled
    size = sum(max(map(keys, x)) for x in live if x) * hk * D * 2 * (2 if kind == BF else 1)
    per = 16 if hq // hk > 8 and D <= 128 else 8
    sets = hk * -(-(hq // hk) // per)
    warps = 1 if sets == hk else 2 if sets == 2 * hk else 4
    return len(row) <= 512 and one_row and full and size >= 1.1 * 2 ** 27 and filled * (sets // warps) >= 100 and warps * new <= 4


CASES = [
    # new, kind, hq, hk, D, requests, shortest, longest, window
    (4, BF, 32, 8, 128, 50, 1500, 2500, 1200),
    (4, F8, 16, 8, 256, 50, 1500, 2500, 900),
    (4, BF, 18, 2, 64, 100, 3500, 4500, 3333),         # nine heads of a kv head: a second column tile
    (2, BF, 24, 8, 128, 50, 1500, 2500, 1201),
    (2, BF, 24, 1, 128, 120, 3000, 4000, 2900),        # two sets of heads and two tokens a block, 16 heads a warp
    (2, F8, 16, 1, 256, 120, 3000, 4000, 2901),        # the same of 8 heads a warp
]


@pytest.mark.parametrize("new,kind,hq,hk,D,requests,shortest,longest,window", CASES)
def test_windows_that_share_a_block(lib, cuda, new, kind, hq, hk, D, requests, shortest, longest, window):
    cache, table, lengths, host, g = served(new * D + hq, requests, shortest, longest, hk, D, kind)
    row = [r for r in range(requests) for _ in range(new)]
    pos = [x - new + i for x in lengths for i in range(new)]
    if new == 4:
        # a place without a token first, inside and last in its four, a four of none, and a last one cut short
        for t in (8, 4 * 5 + 1, 4 * 9 + 3, 4 * 20, 4 * 20 + 1, 4 * 20 + 2, 4 * 20 + 3):
            row[t] = -1
        row, pos = row[:-1], pos[:-1]
        which = [0, 3, 8, 9, 11, 20, 21, 22, 38, 39, 80, 83, 100, len(row) - 3, len(row) - 1]
    else:
        row[40] = row[41] = -1
        which = [0, 1, 38, 39, 40, 41, 42, 99, len(row) - 2, len(row) - 1]
    q = (torch.randn((len(row), hq, D), generator=g, device="cuda") * 2).to(BF)
    dev = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
    sinks = torch.randn(hq, generator=g, device="cuda") * 2
    sinks[0] += 6
    work = paged.attention_workspace(cache, len(row), hq)
    for kw in (dict(), dict(window=window), dict(sinks=sinks, softcap=20.0), dict(window=window, sinks=sinks, softcap=15.0)):
        assert shares(new, row, pos, kw.get("window", 0), hk, hq, D, kind)
        call = lambda: paged.paged_attention(q, cache, table, dev(pos), dev(row), out_dtype=F32, with_lse=True, workspace=work, **kw)  # noqa: E731
        (out, lse), (again, lse2) = call(), call()
        assert torch.equal(out, again) and torch.equal(lse, lse2)
        check(q, host, table, pos, row, out, lse, tokens=which, **kw)
        assert torch.isfinite(out).all() and all((out[t] == 0).all() for t in range(len(row)) if row[t] < 0)
        # every token alone, without the window's others
        for t in range(0, len(row), 37):
            one, one_lse = paged.paged_attention(q[t:t + 1], cache, table, dev(pos[t:t + 1]), dev(row[t:t + 1]), out_dtype=F32, with_lse=True, **kw)
            assert (one[0] - out[t]).abs().max() < 1e-4
            assert torch.equal(one_lse[0], lse[t]) or (one_lse[0] - lse[t]).abs().max() < 1e-4
    # a token among the fours that belongs to another row: no sharing, the same rows
    row[1] = 2
    out, lse = paged.paged_attention(q, cache, table, dev(pos), dev(row), out_dtype=F32, with_lse=True, workspace=work)
    check(q, host, table, pos, row, out, lse, tokens=which[:4])
