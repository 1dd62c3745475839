"""The first call of a host thread that has not touched the device yet runs the kernels that later ones run: autograd's thread in the
first backward pass of a process, or a thread of the program."""
import subprocess
import sys
import threading

import pytest
import torch as th

from helpers import ROOT, chunked
from custom_op_benchmark_b200 import graphop, graphs

pytestmark = pytest.mark.gpu
DEV = "cuda:0"

TWO_STEPS = """
import sys
sys.path.insert(0, %r); sys.path.insert(0, %r)
import torch as th
from test_terms_gpu import Layer
from custom_op_benchmark_b200 import graphs, wrapper
kind = %r
layer = Layer(graphs.banded_graph(2, 400, 60), kind.startswith("diff"), 7 if kind.endswith("bucket") else 0, 2,
              32 if kind.startswith("diff") else 64, th.bfloat16, seed=61)
plans = layer.plans()
assert plans[0].dense_band and plans[1].dense_band
leaves = [t.cuda().requires_grad_(True) for t in (layer.q, layer.k, layer.v)]
up = layer.d_o.cuda()
def step():
    if kind == "plain":
        return th.autograd.grad(wrapper.GraphAttentionPlanned.apply(*plans, *leaves, layer.scale), leaves, up)
    return layer.step(plans)
with th.profiler.profile(activities=[th.profiler.ProfilerActivity.CUDA]) as prof:
    first = step()
    th.cuda.synchronize()
ran = " ".join(e.name for e in prof.events())
assert "banded::" in ran and "group_walk_kernel" not in ran, ran
assert all(th.equal(a, b) for a, b in zip(first, step()))
print("fine")
"""


@pytest.mark.parametrize("kind", ["plain", "bucket", "diff", "diff_bucket"])
def test_the_first_backward_of_a_process(kind):
    res = subprocess.run([sys.executable, "-c", TWO_STEPS % (ROOT, ROOT + "/tests", kind)], capture_output=True, text=True, timeout=300)
    assert res.returncode == 0 and res.stdout.strip().endswith("fine"), res.stdout[-2000:] + res.stderr[-2000:]


def test_a_new_thread():
    g = graphs.banded_graph(2, 400, 60)
    rows, cols = [t.to(DEV) for t in chunked(g, 32)], [t.to(DEV) for t in chunked(g, 32, transposed=True)]
    plans = graphop.GraphPlan(rows[0], rows[1], None, rows[3], g.n_dst), graphop.GraphPlan(*cols, g.n_src)
    gen = th.Generator(device=DEV).manual_seed(62)
    q, k, v, d_o = (th.randn(800, 2, 64, generator=gen, device=DEV).bfloat16() for _ in range(4))
    bucket = th.randint(0, 9, (g.n_edges,), generator=gen, device=DEV).int()
    table = th.randn(9, 2, generator=gen, device=DEV).bfloat16()

    def calls():
        o, lse, sums = graphop.attention_bucket_forward_planned(plans[0], q, k, v, bucket, table, 0.1, True)
        return [o, *graphop.attention_bucket_backward_planned(*plans, q, k, v, bucket, table, sums, lse, d_o, 0.1)]
    want, got = calls(), []
    th.cuda.synchronize()
    thread = threading.Thread(target=lambda: got.extend(calls()))
    thread.start()
    thread.join()
    th.cuda.synchronize()
    assert len(got) == len(want) and all(th.equal(a, b) for a, b in zip(got, want))
