"""Attention layers with learned score terms, what needs no GPU: bucket limits, the reference itself (against differences and
counting), the C header against the binding and the library, refusals of the entry points before any CUDA call."""
import ctypes
import math
import os
import re
import subprocess

import pytest
import torch as th

from helpers import ROOT, random_graph
from custom_op_benchmark_b200 import _capi, graphop, wrapper
from oracle import terms_f64 as ref


# ------------------------------------------------------------------------------------------
# buckets of relative positions
# ------------------------------------------------------------------------------------------
@pytest.mark.parametrize("count,reach", [(2, 5), (3, 2), (16, 128), (16, 9), (32, 128), (31, 1000), (160, 2 ** 20), (8, 2 ** 40)])
def test_limits_are_the_smallest_distance_of_every_bucket(count, reach):
    at = graphop.bucket_limits(count, reach)
    half, m = count // 2, count - count // 2
    assert len(at) == count - 1 and at == sorted(at) and at[:half] == list(range(1, half + 1))
    for t, x in enumerate(at[half:], 1):
        assert x ** m * half ** t >= reach ** t * half ** m
        assert x == half or (x - 1) ** m * half ** t < reach ** t * half ** m
    # the formula in floating point, away from the borders
    for x in range(half, min(reach, 2000)):
        v = m * math.log(x / half) / math.log(reach / half)
        if abs(v - round(v)) > 1e-9:
            assert sum(a <= x for a in at) == min(count - 1, half + math.floor(v)), x


def test_limits_at_exact_borders():
    # 8 exact distances, then powers of 2^(1/2): 16, 32, 64, 128 are borders to the last digit
    assert graphop.bucket_limits(16, 128) == [1, 2, 3, 4, 5, 6, 7, 8, 12, 16, 23, 32, 46, 64, 91]


@pytest.mark.parametrize("count,reach", [(1, 10), (0, 10), (8, 4), (8, 3), (16, 8)])
def test_limits_refuse(count, reach):
    with pytest.raises(ValueError):
        graphop.bucket_limits(count, reach)


def test_reference_counts_as_the_limits_do():
    dst, src = th.arange(60).repeat_interleave(60), th.arange(60).repeat(60)
    for both in (True, False):
        got = ref.relative_buckets(dst, src, 12, 40, both)
        at = graphop.bucket_limits(6 if both else 12, 40)
        for b, x in zip(got.tolist(), (src - dst).tolist()):
            d = abs(x) if both else max(-x, 0)
            assert b == sum(a <= d for a in at) + (6 if both and x > 0 else 0)


# ------------------------------------------------------------------------------------------
# the reference: its gradients against differences
# ------------------------------------------------------------------------------------------
@pytest.mark.parametrize("diff,buckets", [(False, 5), (True, 0), (True, 5)])
def test_reference_gradients_are_differences(diff, buckets):
    g = random_graph(7, 6, [0, 3, 1, 9, 2, 4, 5], 3)
    gen = th.Generator().manual_seed(4)
    rn = lambda *s: th.randn(*s, generator=gen, dtype=th.float64)  # noqa: E731
    h, d = 2, 4
    x = {"q": rn(7, 2 * h if diff else h, d), "k": rn(6, 2 * h if diff else h, d), "v": rn(6, h, 2 * d if diff else d)}
    more = {}
    if diff:
        x["lam"] = rn(h)
    if buckets:
        x["table"] = rn(buckets, 2 * h if diff else h)
        x["table"][1, 0] = -math.inf
        more["bucket"] = th.randint(-1, buckets + 1, (g.n_edges,), generator=gen).int()
    dst, src, d_o = ref.dst_of_edges(g.indptr), g.indices.long(), rn(7, h, 2 * d if diff else d)
    r = ref.attention(dst, src, scale=0.7, d_o=d_o, **x, **more)
    names = {"q": "dq", "k": "dk", "v": "dv", "lam": "d_lam", "table": "d_table"}
    eps = 1e-6
    for name, t in x.items():
        flat = t.view(-1)
        for i in th.randperm(flat.numel(), generator=gen)[:12].tolist():
            if not math.isfinite(float(flat[i])):
                assert float(r[names[name]].view(-1)[i]) == 0
                continue
            keep = float(flat[i])
            ends = []
            for step in (eps, -eps):
                flat[i] = keep + step
                ends.append(float((ref.attention(dst, src, scale=0.7, **x, **more)["o"] * d_o).sum()))
            flat[i] = keep
            # central differences: a third of the third derivative times eps^2, and cancellation 1e-16 / eps
            assert abs((ends[0] - ends[1]) / (2 * eps) - float(r[names[name]].view(-1)[i])) < 1e-7, (name, i)


# ------------------------------------------------------------------------------------------
# boundary
# ------------------------------------------------------------------------------------------
def _header_symbols():
    text = open(os.path.join(ROOT, "include", "graphop_terms.h")).read()
    typed = text[text.index("#define GRAPHOP_DECLARE_TERMS(SUF"):text.index("#define GRAPHOP_DECLARE_TERMS_PLANNED")]
    planned = text[text.index("#define GRAPHOP_DECLARE_TERMS_PLANNED"):text.index("GRAPHOP_DECLARE_TERMS(f32_i32")]
    names = ["%s_%s" % (op, s) for op in re.findall(r"int (graphop_\w+)_##SUF", typed)
             for s in re.findall(r"^GRAPHOP_DECLARE_TERMS\((\w+),", text, re.M)]
    names += ["%s_%s" % (op, s) for op in re.findall(r"int (graphop_\w+)_##SUF", planned)
              for s in re.findall(r"^GRAPHOP_DECLARE_TERMS_PLANNED\((\w+),", text, re.M)]
    return sorted(names + re.findall(r"^(?:int|size_t) (graphop_\w+)\(", text, re.M))


def test_header_binding_and_library_agree():
    assert _header_symbols() == sorted(_capi.terms_symbols())
    out = subprocess.run(["nm", "-D", "--defined-only", _capi.LIB_PATH], capture_output=True, text=True).stdout
    exported = set(re.findall(r" T (graphop_\w+)", out))
    assert not [s for s in _header_symbols() if s not in exported]


def test_a_c_program_compiles_against_the_header(tmp_path):
    src = tmp_path / "consumer.c"
    src.write_text('#include "graphop_terms.h"\n'
                   "int main(void) { return graphop_terms_workspace_bytes(GRAPHOP_TERMS_DIFF_BWD, 100, 10, 2, 16, 8, 4, 4) == 0; }\n")
    exe = tmp_path / "consumer"
    lib = _capi.LIB_PATH
    res = subprocess.run(["gcc", "-std=c99", "-Wall", "-Wextra", "-pedantic", "-Werror", "-I" + os.path.join(ROOT, "include"), str(src),
                          "-o", str(exe), "-L" + os.path.dirname(lib), "-l:" + os.path.basename(lib),
                          "-Wl,-rpath," + os.path.dirname(lib)], capture_output=True, text=True)
    assert res.returncode == 0, res.stderr
    assert subprocess.run([str(exe)]).returncode == 0


def test_workspace_grows_with_what_it_holds():
    size = _capi.lib().graphop_terms_workspace_bytes
    for op in range(4):
        assert 0 < size(op, 1000, 100, 4, 32, 8, 4, 4) < size(op, 100_000, 100, 4, 32, 8, 4, 4) < size(op, 100_000, 100, 4, 32, 8, 4, 8)
    assert size(4, 1000, 100, 4, 32, 8, 4, 4) == 0 and size(0, -1, 100, 4, 32, 8, 4, 4) == 0
    assert size(1, 1000, 100, 4, 32, 16385, 4, 4) == 0
    # the pairs of every edge and map
    assert size(_capi.TERMS_DIFF_BWD, 100_000, 100, 4, 32, 0, 4, 4) > 100_000 * 8 * 8


def _forward_code(**change):
    """Status of a forward call whose arguments are refused before anything is read: pointers are numbers."""
    a = dict(row=4096, indptr=4096, indices=4096, chunks=4, q=4096, k=4096, v=4096, lam=4096, bucket=4096, table=4096, nb=8, o=4096,
             parts=4096, lse=4096, e=10, n=5, m=5, h=2, d=16, ws=4096, wsb=0)
    a.update(change)
    lib = _capi.lib()
    got = [lib.graphop_attention_diff_forward_f32_i32(
        a["row"], a["indptr"], a["indices"], a["chunks"], a["q"], a["k"], a["v"], a["lam"], a["bucket"], a["table"], a["nb"], 1.0,
        a["o"], a["parts"], a["lse"], a["e"], a["n"], a["m"], a["h"], a["d"], a["ws"], a["wsb"], None)]
    got.append(lib.graphop_attention_bucket_forward_f32_i32(
        a["row"], a["indptr"], a["indices"], a["chunks"], a["q"], a["k"], a["v"], a["bucket"], a["table"], a["nb"], 1.0, a["o"],
        a["parts"], a["lse"], a["e"], a["n"], a["m"], a["h"], a["d"], a["ws"], a["wsb"], None))
    return got


@pytest.mark.parametrize("change,code", [
    (dict(), _capi.ERR_WORKSPACE), (dict(ws=4097), _capi.ERR_WORKSPACE), (dict(ws=None), _capi.ERR_WORKSPACE),
    (dict(d=12), _capi.ERR_UNSUPPORTED), (dict(d=2), _capi.ERR_UNSUPPORTED), (dict(h=200, d=64), _capi.ERR_UNSUPPORTED),
    (dict(q=4100), _capi.ERR_UNSUPPORTED), (dict(nb=16385), _capi.ERR_UNSUPPORTED),
    (dict(e=-1), _capi.ERR_INVALID_ARGUMENT), (dict(e=2 ** 31), _capi.ERR_INVALID_ARGUMENT), (dict(h=0), _capi.ERR_INVALID_ARGUMENT),
    (dict(q=None), _capi.ERR_INVALID_ARGUMENT), (dict(row=None), _capi.ERR_INVALID_ARGUMENT), (dict(indices=None), _capi.ERR_INVALID_ARGUMENT),
    (dict(bucket=None), _capi.ERR_INVALID_ARGUMENT), (dict(table=None), _capi.ERR_INVALID_ARGUMENT), (dict(nb=-1), _capi.ERR_INVALID_ARGUMENT),
    (dict(lse=None), _capi.ERR_INVALID_ARGUMENT), (dict(o=None), _capi.ERR_INVALID_ARGUMENT), (dict(n=0), _capi.ERR_INVALID_ARGUMENT),
])
def test_entry_points_refuse_before_any_cuda_call(change, code):
    assert _forward_code(**change) == [code, code]


def test_entry_points_refuse_each_their_own():
    assert _forward_code(lam=None)[0] == _capi.ERR_INVALID_ARGUMENT
    assert _forward_code(lse=4100) == [_capi.ERR_INVALID_ARGUMENT, _capi.ERR_WORKSPACE]   # a pair of maps is read as one
    assert _forward_code(nb=0) == [_capi.ERR_WORKSPACE, _capi.ERR_INVALID_ARGUMENT]       # the bias is the differential layer's option
    lib = _capi.lib()
    zeros = (ctypes.c_int64 * 3)(5, 4, 9)
    assert lib.graphop_relative_buckets_i32(4096, 4096, 4096, 1, None, None, zeros, 3, 1, 4096, 4, None) == _capi.ERR_INVALID_ARGUMENT
    assert lib.graphop_relative_buckets_i32(4096, 4096, 4096, 1, None, None, zeros, 1024, 1, 4096, 4, None) == _capi.ERR_UNSUPPORTED
    assert lib.graphop_relative_buckets_planned_i32(None, None, None, zeros, 1, 1, 4096, None) == _capi.ERR_INVALID_ARGUMENT


def test_python_refuses_host_tensors():
    t, x = th.zeros(2, dtype=th.int64), th.zeros(2, 2, 16)
    with pytest.raises(RuntimeError, match="row must be a CUDA tensor"):
        graphop.relative_buckets(t, t, t, 32, 128)
    with pytest.raises(RuntimeError, match="row must be a CUDA tensor"):
        graphop.attention_bucket_forward(t, t, t, x, x, x, t.int(), th.zeros(4, 2), 1.0)
    for function, last in ((wrapper.GraphAttentionBucket, (t.int(), th.zeros(4, 2), 1.0)), (wrapper.GraphAttentionDiff, (th.zeros(1), 1.0))):
        with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
            function.apply(t, t, t, t, t, t, t, x, x, x, *last)
