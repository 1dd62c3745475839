"""The layers with learned score terms on dense-band plans in bfloat16 (tensor-core kernels), against the float64 edge-list reference."""
import math

import pytest
import torch as th

from helpers import random_graph
from custom_op_benchmark_b200 import graphop, graphs
from oracle import terms_f64 as ref
from test_terms_gpu import KIND_IDS, KINDS, Layer

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
STAGED = th.finfo(th.bfloat16).eps / 2      # probabilities and score gradients enter the products as bfloat16


def _layer(g, diff, buckets, h, seed=1, relative=False):
    """Heads of 64 features of v."""
    layer = Layer(g, diff, buckets, h, 32 if diff else 64, th.bfloat16, seed=seed)
    if buckets and relative:
        layer.bucket = ref.relative_buckets(ref.dst_of_edges(g.indptr), g.indices.long(), buckets, 4 * buckets)
    return layer


def _uneven_band(n, seed):
    """Every node's neighbours are a run of its own length (nothing now and then), within 384 of a tile's."""
    gen = th.Generator().manual_seed(seed)
    lo = (th.arange(n) - th.randint(0, 100, (n,), generator=gen)).clamp(min=0)
    deg = th.randint(0, 120, (n,), generator=gen)
    deg[th.rand(n, generator=gen) < 0.1] = 0
    hi = (lo + deg).clamp(max=n)
    deg = (hi - lo).clamp(min=0)
    dst = th.repeat_interleave(th.arange(n), deg)
    begin = th.cumsum(deg, 0) - deg
    return graphs.coo_to_graph(dst, th.arange(dst.numel()) - begin[dst] + lo[dst], n)


def _growing_band(n, seed):
    """Runs of uneven length whose ends both grow, so that the transposed graph is a band as well; the first nodes have none."""
    gen = th.Generator().manual_seed(seed)
    lo = th.randint(0, n, (n,), generator=gen).sort().values
    hi = th.maximum(th.randint(0, n, (n,), generator=gen).sort().values, lo) + 1
    lo, hi = th.maximum(lo, th.arange(n) - 60).clamp(max=n - 1), th.minimum(hi, th.arange(n) + 60).clamp(max=n)
    deg = (hi - lo).clamp(min=0)
    deg[:20] = 0
    dst = th.repeat_interleave(th.arange(n), deg)
    begin = th.cumsum(deg, 0) - deg
    return graphs.coo_to_graph(dst, th.arange(dst.numel()) - begin[dst] + lo[dst], n)


def _fan(n_dst, n_src):
    """More sources than destinations: each sees a run of 2 of its own."""
    dst = th.arange(n_dst).repeat_interleave(2)
    return graphs.coo_to_graph(dst, th.arange(2 * n_dst), n_dst, n_src)


GRAPHS = [("one_tile", graphs.banded_graph(1, 100, 9)), ("one_node", graphs.banded_graph(1, 1, 4)), ("ragged", graphs.banded_graph(1, 301, 64)),
          ("two_wide", graphs.banded_graph(2, 400, 128)), ("blocks", graphs.block_diagonal_graph(9, 30)), ("uneven", _uneven_band(517, 3)), ("growing", _growing_band(517, 4)),
          ("blocks_of_one", graphs.block_diagonal_graph(300, 1)), ("fan", _fan(90, 200))]


@pytest.mark.parametrize("name,g", GRAPHS, ids=[x[0] for x in GRAPHS])
@pytest.mark.parametrize("diff,buckets", KINDS, ids=KIND_IDS)
@pytest.mark.parametrize("h", [1, 3])
def test_training_step(name, g, diff, buckets, h):
    layer = _layer(g, diff, buckets, h)
    plans = layer.plans()
    assert plans[0].dense_band and (plans[1].dense_band or name == "uneven")   # there the backward goes to the walkers
    layer.check(layer.step(plans), STAGED)
    if buckets:
        layer.bucket = th.randint(-2, buckets + 2, layer.bucket.shape, generator=layer.gen).int()
        layer.table[2, 0] = -math.inf
        layer.table[4, -1] = th.finfo(th.bfloat16).min
        layer.check(layer.step(plans), STAGED)


@pytest.mark.parametrize("diff,buckets", [(False, 32), (True, 32), (False, 255), (False, 256), (True, 2)])
def test_relative_positions_and_table_sizes(diff, buckets):
    layer = _layer(GRAPHS[3][1], diff, buckets, 2, seed=2, relative=buckets <= 32)
    layer.check(layer.step(layer.plans()), STAGED)


@pytest.mark.parametrize("diff,buckets", KINDS, ids=KIND_IDS)
def test_forward_alone(diff, buckets):
    layer = _layer(GRAPHS[2][1], diff, buckets, 4, seed=3)
    r = layer.reference(False)
    b = ref.bounds(r, layer.q, layer.k, layer.v, layer.scale, layer.dt, layer.bucket, layer.table, STAGED)
    plan = layer.plans()[0]
    o, lse, *parts = layer.forward(plan)
    ref.assert_within(o, r["o"], b["o"], "o")
    ref.assert_within(lse, r["lse"], b["lse"], "lse")
    if diff:
        ref.assert_within(parts[0], r["parts"], b["parts"], "parts")
        bare = layer.forward(plan, keep_parts=False)
        assert th.equal(bare[0], o) and th.equal(bare[1], lse)


@pytest.mark.parametrize("diff,buckets", KINDS, ids=KIND_IDS)
def test_the_same_bits_every_time(diff, buckets):
    layer = _layer(GRAPHS[3][1], diff, buckets, 3, seed=4)
    plans = layer.plans()
    first = layer.step(plans)
    for _ in range(3):
        assert all(th.equal(a, b) for a, b in zip(first, layer.step(plans)))


@pytest.mark.parametrize("diff,buckets", [KINDS[0], KINDS[2]], ids=["bucket", "diff_bucket"])
def test_what_takes_no_part_may_hold_anything(diff, buckets):
    """Nodes of NaN and infinities whose edges are all masked, by their bucket or by the table: 0 * NaN inside a tile's products."""
    g = GRAPHS[3][1]
    layer = _layer(g, diff, buckets, 2, seed=5)
    layer.table[6] = -math.inf
    dst, src = ref.dst_of_edges(g.indptr), g.indices.long()
    gone_dst, gone_src = th.zeros(g.n_dst, dtype=th.bool), th.zeros(g.n_src, dtype=th.bool)
    gone_dst[[3, 77, 500]] = True
    gone_src[[3, 200, 201, 799]] = True
    gone = gone_dst[dst] | gone_src[src] | (dst == 17)
    layer.bucket[gone & (th.arange(g.n_edges) % 3 == 0)] = -1
    layer.bucket[gone & (th.arange(g.n_edges) % 3 == 1)] = 6
    layer.bucket[gone & (th.arange(g.n_edges) % 3 == 2)] = buckets
    layer.bucket[~gone] = layer.bucket[~gone] % 6
    for t in (layer.q, layer.d_o):
        t[gone_dst] = math.nan
    for t in (layer.k, layer.v):
        t[gone_src] = math.nan
    layer.v[200] = math.inf
    layer.check(layer.step(layer.plans()), STAGED)


def test_a_row_next_to_the_band_may_hold_anything():
    """Two sequences share a tile: the one's NaN does not reach the other."""
    g = graphs.banded_graph(2, 40, 40)
    for diff, buckets in KINDS:
        layer = _layer(g, diff, buckets, 1, seed=6)
        want = layer.step(layer.plans())
        for t in (layer.q, layer.k, layer.v, layer.d_o):
            t[40:] = math.nan
        got = layer.step(layer.plans())
        bound = ref.bounds(layer_clean(layer, 40), layer.q[:40], layer.k[:40], layer.v[:40], layer.scale, layer.dt,
                           None if layer.bucket is None else layer.bucket[:1600], layer.table, STAGED)
        for name, a, b in list(zip(layer.names(), got, want))[:4]:
            ref.assert_within(a[:40], b[:40].cpu().double(), 2 * bound[name], name)
            assert bool(th.isnan(a[40:]).all())


def layer_clean(layer, n):
    """The reference of a layer's first n nodes, which see nothing else."""
    g = layer.g
    dst, src = ref.dst_of_edges(g.indptr), g.indices.long()
    keep = dst < n
    bucket = None if layer.bucket is None else layer.bucket[keep]
    return ref.attention(dst[keep], src[keep], layer.q[:n], layer.k[:n], layer.v[:n], layer.scale, bucket, layer.table, layer.lam, layer.d_o[:n])


def test_nothing_left_in_a_tile():
    layer = _layer(GRAPHS[3][1], False, 7, 2, seed=7)
    dst = ref.dst_of_edges(layer.g.indptr)
    layer.bucket[dst < 300] = -1
    got = layer.step(layer.plans())
    layer.check(got, STAGED)
    assert bool((got[0][:300] == 0).all()) and bool((got[1][:300] == 0).all())


def test_a_band_that_is_none_goes_to_the_walkers():
    g = random_graph(300, 300, [5] * 300, 8)
    layer = _layer(g, False, 7, 2, seed=8)
    plans = layer.plans()
    assert not plans[0].dense_band
    layer.check(layer.step(plans))


def test_large_sizes_against_the_walkers():
    """More tiles than the chip takes at a time; the walkers' answer to the same call on chunk tables is within both bounds."""
    g = graphs.banded_graph(2, 3001, 100)
    for diff, buckets in KINDS:
        layer = _layer(g, diff, buckets, 4, seed=9)
        for a, b, name in zip(layer.step(layer.plans()), layer.step(), layer.names()):
            a, b = a.detach().float(), b.detach().float()
            # every element is off by at most a few roundings of its terms: in the 2-norm, 2^-8 for the stored value and as much for
            # each of the two staged factors
            assert float((a - b).norm()) <= 4 * STAGED * float(b.norm()), name
