"""GPU: the listed cases of perf/operators.py through the library's calls, against their 64-bit definitions (the page plan against its plain
form, whole numbers), and the same bits on a second pass, with another state's pass between, and on the same inputs made again.

Bounds, of the norm of an output's error over its norm, from the roundings: bf16 keeps 8 bits, so each value is within 2^-8 of itself, and so is
the whole; e4m3 4 bits, 2^-4; fp32 rows of sums, 2^-17.  What lies under the roundings adds 2^-14 where values are turned, summed or normed."""
import pytest
import torch

from perf import operators

pytestmark = pytest.mark.gpu
ROUNDING = {torch.bfloat16: 2.0 ** -8, torch.float8_e4m3fn: 2.0 ** -4, torch.float32: 2.0 ** -17}
# a tenth of the largest one's requests: its definition goes token by token
CASES = [{**c, "requests": c["requests"] // 10} if c["name"] == "attention-256-e4m3" else c for c in operators.listed()]


def bits(out):
    return {k: v.clone().view(torch.uint8) for k, v in out.items()}


def run(case, seed):
    return operators.run(operators.prepare(case, seed))


@pytest.mark.parametrize("case", CASES, ids=[c["name"] for c in CASES])
def test_listed_case(lib, cuda, monkeypatch, case):
    monkeypatch.setattr(operators, "own", True)
    state, other = operators.prepare(case, 3), operators.prepare(case, 4)
    got = {k: v.clone() for k, v in operators.run(state).items()}
    first = bits(got)
    operators.run(other)
    for again in (bits(operators.run(state)), bits(run(case, 3))):
        assert first.keys() == again.keys() and all(torch.equal(first[k], again[k]) for k in first)
    want = operators.exact(case, 3)
    if want is None:
        monkeypatch.setattr(operators, "own", False)
        plain = run(case, 3)
        assert got.keys() == plain.keys() and all(torch.equal(got[k], plain[k]) for k in got)
        return
    for k, x in got.items():
        off, size = (x.double() - want[k]).norm().item(), want[k].norm().item()
        print(f"{case['name']:24s} {k:8s} {str(x.dtype)[6:]:14s} {off / size:.3g}")
        assert off <= (ROUNDING[x.dtype] + 2.0 ** -14 * (x.dtype != torch.float32)) * size
