"""Attention layers with learned score terms, more of what needs no GPU."""
import ctypes
import math
import os
import subprocess

import pytest
import torch as th

from helpers import ROOT, random_graph
from custom_op_benchmark_b200 import _capi, build, graphop, wrapper
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


def _band_plan(n, degree, span):
    """What the size functions read of a plan: numbers, and pointers that are there."""
    return _capi.Plan(n_chunks=n, n_edges=n * degree, n_nodes=n, node_lo=4096, node_deg=4096, node_first=4096, tile_lo=4096,
                      flags=_capi.PLAN_DENSE_BAND, band_span=span)


@pytest.mark.parametrize("n", [300, 4096, 40000, 200000])
@pytest.mark.parametrize("h", [1, 8])
@pytest.mark.parametrize("op,buckets", [(_capi.TERMS_BUCKET_BWD, 32), (_capi.TERMS_DIFF_BWD, 32), (_capi.TERMS_BUCKET_FWD, 32),
                                        (_capi.TERMS_DIFF_FWD, 0)])
def test_a_plan_that_the_tiles_serve_asks_for_their_room(n, h, op, buckets):
    lib = _capi.lib()
    diff, backward = op in (_capi.TERMS_DIFF_FWD, _capi.TERMS_DIFF_BWD), op in (_capi.TERMS_BUCKET_BWD, _capi.TERMS_DIFF_BWD)
    d, columns = (32, 2 * h) if diff else (64, h)

    def sizes(degree, span, elem=2, d=d, buckets=buckets, rows=n, second=True):
        plan = _band_plan(n, degree, span)
        other = ctypes.byref(plan) if backward and second else None
        return (lib.graphop_terms_workspace_bytes_planned(op, ctypes.byref(plan), other, rows, rows, h, d, buckets, elem),
                lib.graphop_terms_workspace_bytes(op, n * degree, rows, h, d, buckets, elem, 4))
    # window 8: 17 neighbours, 192 columns
    planned, plain = sizes(17, 144)
    assert planned >= plain
    if buckets:
        per_element = 2 + 3 * columns if backward else 1         # ids of both sides, score gradients
        assert planned >= (n // 128) * 128 * 192 * per_element
    for other in (sizes(11, 144), sizes(17, 144, elem=4), sizes(17, 144, d=2 * d), sizes(17, 144, rows=n + 1), sizes(17, 385),
                  sizes(17, 144, buckets=256)):
        assert other[0] == other[1] > 0
    if backward:
        assert sizes(17, 144, second=False)[0] == 0
    assert lib.graphop_terms_workspace_bytes_planned(op, None, None, n, n, h, d, buckets, 2) == 0


def test_the_version_belongs_to_the_plan_struct(tmp_path):
    """A library that writes a longer struct than its caller has says so: when the struct grows, so does the version."""
    src, exe = tmp_path / "version.c", tmp_path / "version"
    src.write_text('#include <stdio.h>\n#include "graphop_b200.h"\n'
                   'int main(void) { printf("%d %d\\n", GRAPHOP_VERSION, (int)sizeof(graphop_plan_t)); return 0; }\n')
    res = subprocess.run(["gcc", "-std=c99", "-I" + os.path.join(ROOT, "include"), str(src), "-o", str(exe)], capture_output=True, text=True)
    assert res.returncode == 0, res.stderr
    version, size = map(int, subprocess.run([str(exe)], capture_output=True, text=True).stdout.split())
    assert _capi.lib().graphop_version() == version
    assert ctypes.sizeof(_capi.Plan) == size
    assert (version, size) == (101, 112)       # 100: 96


class _Context:
    """What torch.autograd.Function hands a forward."""

    def __init__(self, needs):
        self.needs_input_grad = needs

    def save_for_backward(self, *tensors):
        self.saved = tensors


@pytest.mark.parametrize("planned", [False, True])
@pytest.mark.parametrize("wanted", [False, True])
def test_the_unrounded_sums_are_kept_where_a_gradient_is_asked_for(monkeypatch, planned, wanted):
    """The Functions without the compiled nodes: the bias layer's sums are a tensor of float32 as large as q."""
    name, seen, t = "attention_bucket_forward" + ("_planned" if planned else ""), [], th.zeros(2, 1, 16)

    def forward(*args, keep_sums):
        seen.append(keep_sums)
        return (t, t, t) if keep_sums else (t, t)
    monkeypatch.setattr(graphop, name, forward)
    if planned:
        monkeypatch.setattr(graphop, "check_plan_rows", lambda *a: None)
    function, n_graph = (wrapper.GraphAttentionBucketPlanned, 2) if planned else (wrapper.GraphAttentionBucket, 7)
    needs = [False] * (n_graph + 6)
    needs[n_graph + 4] = wanted                 # the table
    ctx = _Context(tuple(needs))
    assert function.forward(ctx, *[None] * n_graph, t, t, t, None, t, 1.0) is t
    assert seen == [wanted] and (ctx.saved[-2] is t) == wanted


def test_a_bucket_holds_the_distances_that_exactly_so_many_limits_do_not_exceed():
    """As the docstring says: the buckets do not overlap, and the reference puts every distance into the same one."""
    assert "exactly b of them" in graphop.bucket_limits.__doc__
    at = graphop.bucket_limits(10, 300)
    x = th.arange(400)
    want = ref.relative_buckets(th.zeros(400, dtype=th.int64), x, 10, 300, False, th.zeros(1, dtype=th.int64), -x)
    for b in range(10):
        assert ((want == b) == (th.tensor([sum(a <= d for a in at) for d in x.tolist()]) == b)).all()


@pytest.mark.parametrize("count,reach,both,match", [(32, 2 ** 63, False, "64-bit"), (32, 10 ** 400, True, "64-bit"),
                                                    (1025, 10 ** 6, False, "1024"), (2050, 10 ** 6, True, "1024"), (10 ** 6, 10 ** 9, True, "1024")])
def test_buckets_beyond_what_the_library_takes_are_refused_as_such(count, reach, both, match):
    """Not as an overflow of the packing, and before a limit is computed; nothing of the graph is looked at."""
    with pytest.raises(ValueError, match=match):
        graphop.relative_buckets(None, None, None, count, reach, both)
    with pytest.raises(ValueError, match=match):
        graphop.relative_buckets_planned(None, count, reach, both)


def test_the_largest_limits_fit_their_packing():
    at = graphop.bucket_limits(1024, 2 ** 63 - 1)
    assert len(at) == 1023 and at == sorted(at) and at[-1] < 2 ** 63
    assert len(graphop._limits(2048, 2 ** 63 - 1, True)) == 1023 * 8
