"""GPU: attention of calls of more than 512 places as a page plan gives them - a prompt's hundreds of tokens beside decoding rows, several
tokens of a row, places without a token at the end - against fp64.  The bounds are those of test_paged_attention_gpu.py."""
from types import SimpleNamespace

import numpy as np
import pytest
import torch

from basalt_b200 import paged
from tests.test_paged_attention_gpu import check, make

pytestmark = pytest.mark.gpu
BF, F32, F8 = torch.bfloat16, torch.float32, torch.float8_e4m3fn


def step(seed, places, hk, D, page, kind, prompt=600, decoding=40):
    """A step's plan over a cache that holds its keys already: row 0 brings a prompt, row 1 seven tokens behind 333, row 2 has nothing to do, the
    others decode a token behind 0 to 900 keys."""
    rng = np.random.default_rng(seed)
    before = [0, 333, 50] + rng.integers(0, 900, decoding).tolist()
    new = [prompt, 7, 0] + [1] * decoding
    after = [a + b for a, b in zip(before, new)]
    cache, table, g = make(seed, after, hk, D, page, kind)
    held = [-(-x // page) for x in before]
    fresh = [i for r, x in enumerate(after) for i in table[r, held[r]:-(-x // page)].tolist()]
    wanted = table.clone()
    dev = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
    for r, x in enumerate(held):
        table[r, x:] = -1
    plan = paged.PagePlan(len(after), places)
    # the stack gives the rows the pages that make() has filled
    paged.page_plan(dev(before), dev(new), table, dev(fresh[::-1]), dev([len(fresh)]), page, plan)
    plan.check_status()
    assert torch.equal(table, wanted) and plan.seq_len.tolist() == after
    on_host = SimpleNamespace(k=cache.k.cpu(), v=cache.v.cpu(), k_scale=cache.k_scale, v_scale=cache.v_scale, n_kv_heads=hk)
    return cache, table, plan, g, sum(new), on_host


def sample(rng, tokens, prompt, places):
    """Edges of the prompt, of its tiles and of the step, and some between."""
    edges = [0, 1, 7, 8, 15, 16, 17, 63, 64, 65, prompt - 1, prompt, prompt + 6, prompt + 7, tokens - 1]
    return sorted({*edges, *rng.integers(0, tokens, 12).tolist(), *(x for x in (511, 512, 513, 1023, 1024, 1025) if x < tokens), *range(tokens, places, 41)})


@pytest.mark.parametrize("places,prompt", [(648, 600), (700, 600), (1400, 600), (1500, 1300)])
@pytest.mark.parametrize("kind,hq,hk,D,page", [(BF, 8, 2, 128, 16), (F8, 8, 2, 64, 8), (BF, 20, 1, 128, 64), (F8, 16, 8, 128, 32), (BF, 9, 3, 64, 16), (BF, 12, 4, 256, 16)])
def test_a_prompt_beside_decoding_rows(lib, cuda, places, prompt, kind, hq, hk, D, page):
    cache, table, plan, g, tokens, host = step(places + hq, places, hk, D, page, kind, prompt)
    q = (torch.randn((places, hq, D), generator=g, device="cuda") * 2).to(BF)
    pos, row = plan.pos.tolist(), plan.row.tolist()
    assert row[tokens:] == [-1] * (places - tokens) and tokens > 512
    which = sample(np.random.default_rng(D), tokens, prompt, places)
    work = paged.attention_workspace(cache, places, hq)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    for kw in (dict(), dict(window=100), dict(softcap=20.0, sinks=torch.randn(hq, generator=g, device="cuda") * 2), dict(window=37, softcap=30.0, sinks=torch.zeros(hq, device="cuda"))):
        call = lambda: paged.paged_attention(q, cache, table, plan.pos, plan.row, out_dtype=F32, with_lse=True, workspace=work, status=status, **kw)  # noqa: E731
        (out, lse), (again, lse2) = call(), call()
        assert torch.equal(out, again) and torch.equal(lse, lse2) and status.item() == 0
        check(q, host, table, pos, row, out, lse, tokens=which, **kw)
        assert torch.isfinite(out).all() and (out[tokens:] == 0).all()
        if "sinks" in kw:
            assert torch.equal(lse[tokens:], kw["sinks"].expand(places - tokens, -1))
        else:
            assert torch.isneginf(lse[tokens:]).all() and torch.isfinite(lse[:tokens]).all()
    # without the padding: the same rows but for their last bits
    short, _ = paged.paged_attention(q[:tokens], cache, table, plan.pos, plan.row, out_dtype=F32, workspace=work)
    full, _ = paged.paged_attention(q, cache, table, plan.pos, plan.row, out_dtype=F32, workspace=work)
    assert (short - full[:tokens]).abs().max() < 1e-4


def test_rows_and_positions_beyond_the_table(lib, cuda):
    """Left out, or cut to the row's end, and said so; the other tokens as they are."""
    cache, table, plan, g, tokens, host = step(3, 700, 2, 128, 16, BF)
    q = torch.randn((700, 8, 128), generator=g, device="cuda").to(BF)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    row, pos = plan.row.clone(), plan.pos.clone()
    row[5], row[610] = table.shape[0], 10 ** 9
    out, lse = paged.paged_attention(q, cache, table, pos, row, out_dtype=F32, with_lse=True, status=status)
    assert status.item() == 64
    left = [r if r < table.shape[0] else -1 for r in row.tolist()]
    check(q, host, table, pos.tolist(), left, out, lse, tokens=[0, 4, 5, 6, 599, 609, 610, 611, tokens - 1, tokens])
    # a table of one row whose places are all filled: the last of them
    full = paged.KVCache.empty(4, 2, 16, 128)
    for c in (full.k, full.v):
        c.copy_(torch.randn(c.shape, generator=g, device="cuda"))
    one = torch.arange(4, dtype=torch.int32, device="cuda").view(1, 4)
    status.zero_()
    pos = torch.arange(700, dtype=torch.int32, device="cuda") % 64
    pos[600] = 2 ** 31 - 1
    out, lse = paged.paged_attention(q, full, one, pos, torch.zeros_like(pos), out_dtype=F32, with_lse=True, status=status)
    assert status.item() == 64
    pos[600] = 63
    check(q, full, one, pos.tolist(), [0] * 700, out, lse, tokens=[0, 63, 64, 127, 599, 600, 601, 699])
