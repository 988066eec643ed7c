"""GPU: objects that keep addresses (a Rope, a PagePlan) are refused where they lie on another device than the call.  Nothing is launched with
such an address: a stand-in for the library takes the calls, and a call that reaches it fails the test."""
import pytest
import torch

from basalt_b200 import capi, paged

pytestmark = pytest.mark.gpu
dev = "cuda"


@pytest.fixture
def nothing_launched(monkeypatch):
    class Library:
        def __getattr__(self, name):
            def call(*args):
                pytest.fail(f"{name} was called")
            return call
    return lambda: monkeypatch.setattr(capi, "lib", Library)


def test_a_rope_of_another_device(lib, cuda, nothing_launched):
    cache = paged.KVCache.empty(10, 2, 16, 128)
    rows = torch.zeros((3, 2, 128), dtype=torch.bfloat16, device=dev)
    slot, pos = torch.arange(3, device=dev), torch.zeros(3, dtype=torch.int32, device=dev)
    rope = paged.Rope(torch.ones(64, device=dev))
    paged.rope_append(rows, rows, rows, cache, slot, pos, rope)
    rope.index = torch.cuda.current_device() + 1      # as one that was made while another device was current
    nothing_launched()
    with pytest.raises(ValueError, match="rope"):
        paged.rope_append(rows, rows, rows, cache, slot, pos, rope)


@pytest.mark.parametrize("where", ["cpu", "another"])
def test_a_plan_of_another_device(lib, cuda, nothing_launched, where):
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    good = dict(seq_len=ints(0, 0, 0), n_new=ints(1, 2, 3), block_table=torch.zeros((3, 8), dtype=torch.int32, device=dev),
                free_list=torch.arange(30, dtype=torch.int32, device=dev), free_count=ints(30), page_size=16)
    out = paged.PagePlan(3, 64)
    paged.page_plan(**good, out=out)
    if where == "cpu":
        out = paged.PagePlan(3, 64, device="cpu")
    else:
        out.index = torch.cuda.current_device() + 1      # as one that was made while another device was current
    nothing_launched()
    with pytest.raises(ValueError, match="plan"):
        paged.page_plan(**good, out=out)
