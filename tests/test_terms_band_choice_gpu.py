"""Which kernels a call on a dense-band plan runs (tensor cores where a node has enough neighbours for the columns that a tile computes,
else the walkers), that either answer is right, and bands whose two sides have different numbers of tiles."""
import ctypes
import threading

import pytest
import torch as th

from custom_op_benchmark_b200 import _capi, graphop, graphs
from oracle import terms_f64 as ref
from test_terms_gpu import KIND_IDS, KINDS, Layer

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
STAGED = th.finfo(th.bfloat16).eps / 2      # probabilities and score gradients enter the products as bfloat16


def _kernels(call):
    with th.profiler.profile(activities=[th.profiler.ProfilerActivity.CUDA]) as prof:
        out = call()
        th.cuda.synchronize()
    return out, " ".join(e.name for e in prof.events())


def _slanted(n_dst, n_src, per, degree):
    """Node i sees `degree` sources from per * i on (per may be a fraction)."""
    lo = (th.arange(n_dst, dtype=th.float64) * per).long().clamp(max=n_src - degree)
    dst = th.arange(n_dst).repeat_interleave(degree)
    return graphs.coo_to_graph(dst, (lo[:, None] + th.arange(degree)).flatten(), n_dst, n_src)


def _layer(g, diff, buckets, h, seed):
    layer = Layer(g, diff, buckets, h, 32 if diff else 64, th.bfloat16, seed=seed)
    if buckets:
        layer.bucket[::7] = -1
    return layer


# (graph, tensor cores): neighbours against a sixteenth of the columns, 192 of a window of 8, 256 of a window of 64, 128 of the blocks
CHOICES = [("window_8_short", graphs.banded_graph(1, 300, 8), True), ("window_8", graphs.banded_graph(2, 1500, 8), True),
           ("window_12", graphs.banded_graph(1, 4096, 12), True), ("window_4", graphs.banded_graph(1, 2000, 4), False),
           ("window_64", graphs.banded_graph(1, 700, 64), True), ("blocks_of_8", graphs.block_diagonal_graph(80, 8), True),
           ("blocks_of_7", graphs.block_diagonal_graph(80, 7), False), ("blocks_of_1", graphs.block_diagonal_graph(300, 1), False),
           ("one_node", graphs.banded_graph(1, 1, 4), False)]


@pytest.mark.parametrize("name,g,tiles", CHOICES, ids=[c[0] for c in CHOICES])
@pytest.mark.parametrize("diff,buckets", KINDS, ids=KIND_IDS)
@pytest.mark.parametrize("h", [1, 8])
def test_the_rule(name, g, tiles, diff, buckets, h):
    layer = _layer(g, diff, buckets, h, 51)
    plans = layer.plans()
    assert plans[0].dense_band and plans[1].dense_band
    got, ran = _kernels(lambda: layer.step(plans))
    for kernel in ("terms_forward_kernel", "terms_backward_kernel"):
        assert (kernel in ran) == tiles, ran
    assert ("group_walk_kernel" in ran) != tiles, ran
    layer.check(got, STAGED if tiles else 0.0)


RECTANGLES = [("more_sources", _slanted(400, 800, 2, 40)), ("more_destinations", _slanted(800, 400, 0.5, 24)),
              ("far_more_sources", _slanted(130, 1100, 2, 100))]


@pytest.mark.parametrize("name,g", RECTANGLES, ids=[r[0] for r in RECTANGLES])
@pytest.mark.parametrize("diff,buckets", KINDS, ids=KIND_IDS)
@pytest.mark.parametrize("h", [1, 3])
def test_rectangular_bands(name, g, diff, buckets, h):
    layer = _layer(g, diff, buckets, h, 52)
    plans = layer.plans()
    got, ran = _kernels(lambda: layer.step(plans))
    assert "terms_forward_kernel" in ran and "terms_backward_kernel" in ran, ran
    layer.check(got, STAGED)


@pytest.mark.parametrize("diff,buckets", KINDS[::2], ids=KIND_IDS[::2])
def test_without_the_plans_workspace_the_walkers_run(diff, buckets):
    """The C entry point with the size that a chunk-table call asks for."""
    h, n = 8, 300
    layer = _layer(graphs.banded_graph(1, n, 8), diff, buckets, h, 53)
    d, op = (32, _capi.TERMS_DIFF_BWD) if diff else (64, _capi.TERMS_BUCKET_BWD)
    plans = layer.plans()
    lib = _capi.lib()
    few = lib.graphop_terms_workspace_bytes(op, layer.g.n_edges, n, h, d, buckets, 2, 4)
    enough = lib.graphop_terms_workspace_bytes_planned(op, plans[0].ref(), plans[1].ref(), n, n, h, d, buckets, 2)
    assert enough > few
    q, k, v, d_o = (t.to(DEV) for t in (layer.q, layer.k, layer.v, layer.d_o))
    lam = layer.lam.to(DEV) if diff else None
    bucket, table = layer.terms()
    # the walkers' forward, with its sums: the chunk-table call
    rows = [layer.rows[0], layer.rows[1], layer.rows[3]]
    if diff:
        o, lse, sums = graphop.attention_diff_forward(*rows, q, k, v, lam, layer.scale, bucket, table)
    else:
        o, lse, sums = graphop.attention_bucket_forward(*rows, q, k, v, bucket, table, layer.scale, True)
    out = [th.empty_like(t) for t in (q, k, v)] + ([th.empty_like(lam)] if diff else []) + [th.empty_like(table)]
    p = lambda t: t.data_ptr()  # noqa: E731
    name = "graphop_attention_%s_backward_planned_bf16" % ("diff" if diff else "bucket")
    args = [p(q), p(k), p(v)] + ([p(lam)] if diff else []) + [p(bucket), p(table), buckets, p(sums), p(lse), p(d_o), ctypes.c_double(layer.scale)]
    for size, tiles in ((few, False), (enough, True)):
        ws = th.empty(size, dtype=th.uint8, device=DEV)
        rc, ran = _kernels(lambda: getattr(lib, name)(plans[0].ref(), plans[1].ref(), *args, *[p(t) for t in out], n, n, h, d, p(ws), size,
                                                      th.cuda.current_stream().cuda_stream))
        assert rc == _capi.OK and ("terms_backward_kernel" in ran) == tiles, ran
        layer.check([o] + out, STAGED if tiles else 0.0)
    assert getattr(lib, name)(plans[0].ref(), plans[1].ref(), *args, *[p(t) for t in out], n, n, h, d, p(ws), 4096,
                              th.cuda.current_stream().cuda_stream) == _capi.ERR_WORKSPACE


def test_bands_on_several_threads_and_streams():
    """Blocks of different kernels share the SMs' tensor memory and shared memory; everyone gets the bits of a call alone."""
    layers = [_layer(graphs.banded_graph(2, 700, w), diff, buckets, 4, 54) for w, (diff, buckets) in zip((64, 30, 128), KINDS)]
    plans = [layer.plans() for layer in layers]
    want = [layer.step(p) for layer, p in zip(layers, plans)]
    wrong = []

    def work(i):
        with th.cuda.stream(th.cuda.Stream()):
            for _ in range(10):
                got = layers[i].step(plans[i])
                th.cuda.current_stream().synchronize()
                if not all(th.equal(a, b) for a, b in zip(got, want[i])):
                    wrong.append(i)
    th.cuda.synchronize()
    threads = [threading.Thread(target=work, args=(i % 3,)) for i in range(6)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
