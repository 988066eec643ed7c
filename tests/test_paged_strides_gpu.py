"""GPU: axes of one element have no step: whatever stride torch reports for them, the tensor is as dense as another."""
import pytest
import torch

from basalt_b200 import moe, paged

pytestmark = pytest.mark.gpu
BF, I32 = torch.bfloat16, torch.int32


def odd(t, axis):
    """t with another stride reported for its axis of one element."""
    assert t.shape[axis] == 1
    stride = list(t.stride())
    stride[axis] = 7
    return t.as_strided(t.shape, stride, t.storage_offset())


def test_one_head_one_page_one_token(lib, cuda):
    g = torch.Generator(device="cuda").manual_seed(1)
    k, v = (torch.randn((6, 1, 16, 128), generator=g, device="cuda").to(BF) for _ in range(2))
    table = torch.arange(6, dtype=I32, device="cuda").view(6, 1)
    pos = torch.tensor([15, 3, 0, 8, -1, 9], dtype=I32, device="cuda")
    q = torch.randn((6, 1, 128), generator=g, device="cuda").to(BF)
    cache, same = paged.KVCache(k, v), paged.KVCache(odd(k, 1), odd(v, 1))
    want, _ = paged.paged_attention(q, cache, table, pos)
    for args in ((odd(q, 1), cache, table), (q, same, table), (q, cache, odd(table, 1)), (q.transpose(0, 1).contiguous().transpose(0, 1), cache, table)):
        assert torch.equal(paged.paged_attention(*args, pos)[0], want)
    one, _ = paged.paged_attention(odd(q[:1], 0), cache, odd(table[:1], 0), pos)
    assert torch.equal(one, want[:1])
    rope = paged.Rope(torch.ones(64, device="cuda"))
    slot = torch.arange(6, device="cuda")
    first = paged.rope_append(q, q, q, cache, slot, pos, rope)
    stored = cache.k.clone()
    assert torch.equal(paged.rope_append(odd(q, 1), odd(q, 1), odd(q, 1), same, slot, pos, rope), first) and torch.equal(same.k, stored)


def test_a_plan_over_rows_of_one_page(lib, cuda):
    ints = lambda *a: torch.tensor(a, dtype=I32, device="cuda")  # noqa: E731
    tables = []
    for wrap in (lambda t: t, lambda t: odd(t, 1)):
        table = torch.full((3, 1), -1, dtype=I32, device="cuda")
        out = paged.PagePlan(3, 21)
        paged.page_plan(ints(0, 0, 0), ints(4, 1, 16), wrap(table), ints(8, 7, 6, 5), ints(4), 16, out)
        tables.append((table, out.slot, out.pos))
    assert all(torch.equal(a, b) for a, b in zip(*tables)) and tables[0][0].flatten().tolist() == [5, 6, 7]


def test_norms_of_one_value_and_one_row(lib, cuda):
    g = torch.Generator(device="cuda").manual_seed(2)
    for shape, axis in (((5, 1), 1), ((1, 64), 0)):
        y, x = (torch.randn(shape, generator=g, device="cuda") for _ in range(2))
        w = torch.ones(shape[1], device="cuda")
        want = moe.block_norm(y, x, w, pre_w=w)
        got = moe.block_norm(odd(y, axis), odd(x, axis), w, gate=None, pre_w=w, out=odd(torch.empty(shape, device="cuda"), axis))
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
