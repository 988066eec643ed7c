"""GPU: sinks at the ends of their type.  e^sink is the denominator's own term: infinite, it takes all the weight (rows of zeros, an infinite
logarithm); 0, it takes none (minus infinity, the lowest value)."""
import pytest
import torch

from basalt_b200 import paged

pytestmark = pytest.mark.gpu
INF, LOW = float("inf"), torch.finfo(torch.float32).min


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float8_e4m3fn])
@pytest.mark.parametrize("lengths", [[50, 0, 1], [6000, 0, 700]])      # units of one block, and units that several blocks join
def test_infinite_and_lowest_sinks(lib, cuda, kind, lengths):
    g = torch.Generator(device="cuda").manual_seed(31)
    pages = -(-max(lengths) // 16)
    cache = paged.KVCache.empty(3 * pages, 2, 16, 128, kind, None, *((torch.ones(2, device="cuda"),) * 2 if kind != torch.bfloat16 else ()))
    for c in (cache.k, cache.v):
        c.copy_(torch.randn(c.shape, generator=g, device="cuda").to(kind))
    table = torch.arange(3 * pages, dtype=torch.int32, device="cuda").view(3, -1)
    pos = torch.tensor([x - 1 for x in lengths], dtype=torch.int32, device="cuda")
    q = torch.randn((3, 8, 128), generator=g, device="cuda").bfloat16()
    call = lambda sinks: paged.paged_attention(q, cache, table, pos, sinks=sinks, out_dtype=torch.float32, with_lse=True)  # noqa: E731
    none, none_lse = call(None)
    some = torch.tensor([1.0, INF, -INF, 0.5, LOW, INF, -2.0, -INF], device="cuda")
    finite = torch.where(some == INF, torch.zeros(8, device="cuda"), some)
    out, lse = call(some)
    want, want_lse = call(finite)
    for h in range(8):
        if some[h] == INF:
            assert (out[:, h] == 0).all() and (lse[:, h] == INF).all()
        else:
            assert torch.equal(out[:, h], want[:, h]) and torch.equal(lse[:, h], want_lse[:, h])
        if some[h] <= LOW:      # the tokens that see keys
            assert torch.equal(out[::2, h], none[::2, h]) and torch.equal(lse[::2, h], none_lse[::2, h])
