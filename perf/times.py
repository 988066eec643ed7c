"""Times the cases of perf/operators.py through the library's calls on this GPU, and says how far their outputs are from 64 bits.

    python perf/times.py [--seed N] [--exact] [NAME ...]

A case has three states of different seeds that its passes take in turn.  Call: passes issued one after the other from Python, wall time a
pass (median of seven runs).  Device: twenty passes in a CUDA graph, by events around its replay (median of seven).  States under 126 MB in
all stay in L2.  Bytes: what the three states cannot do without, at their own lengths, as a mean.
"""
import argparse
import sys
import time
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

from perf import operators  # noqa: E402

PASSES, RUNS = 20, 7


def middle(values):
    return sorted(values)[len(values) // 2]


def call_us(states, n=60):
    got = []
    for _ in range(RUNS):
        torch.cuda.synchronize()
        began = time.perf_counter()
        for i in range(n):
            operators.run(states[i % len(states)])
        torch.cuda.synchronize()
        got.append((time.perf_counter() - began) / n * 1e6)
    return middle(got)


def device_us(states):
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for i in range(PASSES):
            operators.run(states[i % len(states)])
    got = []
    for _ in range(RUNS + 3):
        start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        start.record()
        graph.replay()
        end.record()
        end.synchronize()
        got.append(start.elapsed_time(end) / PASSES * 1e3)
    return middle(got[3:])


def needed(case, states):
    """Bytes of a pass: operators.work()'s, with the lengths that the states of an attention case have in place of their mean."""
    size = operators.work(case)["bytes"]
    if case["op"] != "attention":
        return size
    n, new = case["requests"], case["window_tokens"]
    most = case["window"] + new - 1 if case["window"] else 2 ** 31 - 1
    keys = sum(s["pos"].view(n, new)[:, -1].add(1).clamp(max=most).sum().item() for s in states) / len(states)
    a_key = case["kv_heads"] * 2 * case["dim"] * (2 if case["cache"] == "bf16" else 1)
    rows = n * new * case["q_heads"] * (case["dim"] * (2 + (2 if case["out"] == "bf16" else 4)) + 4)
    return keys * a_key + rows + 4 * keys / case["page"]


def main():
    args = argparse.ArgumentParser()
    args.add_argument("names", nargs="*")
    args.add_argument("--seed", type=int, default=5)
    args.add_argument("--exact", action="store_true", help="errors against 64 bits too: seconds for the largest cases")
    args = args.parse_args()
    operators.own = True
    for case in operators.listed():
        if args.names and case["name"] not in args.names:
            continue
        states = [operators.prepare(case, args.seed + i) for i in range(3)]
        for s in states * 2:
            operators.run(s)
        call, device, size = call_us(states), device_us(states), needed(case, states)
        print(f"{case['name']:24s} call {call:8.2f} us  device {device:8.2f} us  {size / 1e6:8.2f} MB  {size / device / 1e6:5.2f} TB/s", flush=True)
        if args.exact:
            got, want = operators.run(states[0]), operators.exact(case, args.seed)
            for k in want or ():
                print(f"    {k:8s} {str(got[k].dtype)[6:]:14s} off by {((got[k].double() - want[k]).norm() / want[k].norm()).item():.3g} of its norm")
        del states
        torch.cuda.empty_cache()


if __name__ == "__main__":
    main()
