"""perf/operators.py's calls of the operators on rows: small cases on the current stream, on another one, and captured."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

ON_STREAMS = """
import torch
from perf import operators as cases

small = [dict(op="lookup", type="bf16", ids="i64", tokens=300, rows=500, d=256, scale=2.0, absent=0.1),
         dict(op="lookup_grad", type="f32", out="f32", ids="u32", tokens=900, rows=70, d=40, scale=1.0, absent=0.0),
         dict(op="to", type="f16", tokens=200, choices=2, groups=9, d=72, skew=0.5, dropped=0.1),
         dict(op="product", x="i8", out="f32", m=40, n=50, k=96, groups=0, bias=True, skew=0.0, dropped=0.0)]

def values(out):
    return [t.double().cpu() for t in (out.values() if isinstance(out, dict) else [out])]

side = torch.cuda.Stream()
for case in small:
    cases.own = False
    first = cases.prepare(case, 3)
    want = values(cases.run(first))
    # how far two fp32 results may be apart: each is off by its roundings times 2^-24 times the sum of the terms' magnitudes
    bar = 0.0
    if case["op"] == "lookup_grad":
        at = first["at"].long()
        terms = torch.zeros((70, 40), device="cuda", dtype=torch.float64).index_add_(0, at, first["given"].double().abs())
        count = torch.bincount(at, minlength=70)[:, None]
        bar = (2 * (count + 2) * 2.0 ** -24 * terms).cpu()
    elif case["op"] == "product":  # the sum is exact on both sides: below 2^24; two scales and the bias
        bar = 2 * 4 * 2.0 ** -24 * (want[0].abs() + 2 * first["bias"].double().abs().cpu())
    cases.own = True

    def check(out):
        for got, w in zip(values(out), want):
            assert ((got - w).abs() <= bar).all(), case

    check(cases.run(cases.prepare(case, 3)))
    with torch.cuda.stream(side):
        # nothing orders the side stream with the first one: the state is made on it, and everything of the call has to be too
        waste = torch.ones((1 << 28,), device="cuda")
        for _ in range(20):
            waste.mul_(1.0)
        state = cases.prepare(case, 3)
        check(cases.run(state))
        if case["op"] == "lookup":
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                out = cases.run(state)
            for _ in range(3):
                state["result"].zero_()
                graph.replay()
                check(out)
        del waste
torch.cuda.synchronize()
print("cases: ok", len(cases._operators))
"""


def test_own_calls_are_queued_on_the_current_stream():
    """In a process of its own: torch brings a HIP runtime, which has to be the first one that a process loads."""
    r = subprocess.run([sys.executable, "-c", ON_STREAMS], cwd=ROOT, capture_output=True, text=True, timeout=110)
    assert r.returncode == 0 and "cases: ok 2" in r.stdout, r.stdout[-2000:] + r.stderr[-4000:]
