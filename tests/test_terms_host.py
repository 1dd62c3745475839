"""Attention layers with learned score terms, more of what needs no GPU."""
import math
import os
import subprocess

import pytest
import torch as th

from helpers import ROOT, random_graph
from custom_op_benchmark_b200 import build
from oracle import terms_f64 as ref


@pytest.mark.parametrize("diff", [False, True])
def test_reference_leaves_masked_edges_out_of_a_spoilt_row(diff):
    """A query of NaN with live and masked edges: every gradient is what it is on the graph without the masked ones."""
    g = random_graph(9, 30, [6] * 9, 3)
    gen = th.Generator().manual_seed(4)
    rn = lambda *s: th.randn(*s, generator=gen, dtype=th.float64)  # noqa: E731
    h, d = 2, 4
    x = dict(q=rn(9, 2 * h if diff else h, d), k=rn(30, 2 * h if diff else h, d), v=rn(30, h, 2 * d if diff else d), scale=0.5,
             table=rn(5, 2 * h if diff else h), lam=rn(h) if diff else None, d_o=rn(9, h, 2 * d if diff else d))
    dst, src = ref.dst_of_edges(g.indptr), g.indices.long()
    bucket = th.randint(0, 4, (g.n_edges,), generator=gen).int()
    masked = th.arange(g.n_edges) % 3 == 0
    bucket[masked] = th.tensor([-1, 4, 5]).repeat(g.n_edges)[: int(masked.sum())].int()
    x["table"][4] = -math.inf
    x["q"][5, 0] = math.nan
    r, few = ref.attention(dst, src, bucket=bucket, **x), ref.attention(dst[~masked], src[~masked], bucket=bucket[~masked], **x)
    for name in ["o", "lse", "dq", "dk", "dv", "d_table"] + ["d_lam"] * diff:
        assert th.equal(th.isnan(r[name]), th.isnan(few[name])), name
        assert th.equal(th.nan_to_num(r[name]), th.nan_to_num(few[name])), name
    assert bool(th.isnan(r["dq"][5]).any()) and not bool(th.isnan(r["d_table"][4]).any())


def test_every_shape_fits_the_workspace_it_asks_for(tmp_path):
    """A program that takes a call's buffers as the library does, over all head counts and widths of all types, without a device."""
    exe = tmp_path / "terms_workspace"
    res = subprocess.run([build._nvcc(), "-std=c++17", "-O1", "-gencode", "arch=compute_100a,code=sm_100a", "-I" + build.CSRC,
                          os.path.join(ROOT, "tests", "terms_workspace.cu"), "-o", str(exe)], capture_output=True, text=True)
    assert res.returncode == 0, res.stderr
    res = subprocess.run([str(exe)], capture_output=True, text=True)
    assert res.returncode == 0, res.stdout
