"""What takes no part stays out of every gradient also where the query itself is not finite: a live query of NaN or infinity, or
one that sees a key of NaN, next to masked edges, on the walkers and on the tensor cores."""
import math

import pytest
import torch as th

from helpers import random_graph
from custom_op_benchmark_b200 import graphs
from oracle import terms_f64 as ref
from test_terms_gpu import KIND_IDS, KINDS, Layer

pytestmark = pytest.mark.gpu
STAGED = th.finfo(th.bfloat16).eps / 2      # probabilities and score gradients enter the products as bfloat16


def _spoilt(layer, how, node, diff):
    """The edges of `node` become masked, by their id or by an entry of the table, but for the first two.  Returns the layer's clean reference and
    bounds (everything finite) and what the two live edges may reach: source rows and buckets."""
    dst, src = ref.dst_of_edges(layer.g.indptr), layer.g.indices.long()
    mine = (dst == node).nonzero().flatten()
    live, gone = mine[:2], mine[2:]
    assert len(gone) > 3
    layer.table[6] = -math.inf                  # no part for either map
    layer.table[5, 0] = -math.inf               # none for the first one
    layer.bucket[layer.bucket >= 5] = 4
    layer.bucket[gone] = th.tensor([-1, 6, 7])[th.arange(len(gone)) % 3].int()
    layer.bucket[live] = 1
    r = layer.reference()
    b = ref.bounds(r, layer.q, layer.k, layer.v, layer.scale, layer.dt, layer.bucket, layer.table, layer.staged)
    if how == "query":
        layer.q[node, :, 0] = math.nan
    elif how == "infinite":
        layer.q[node, :, 0] = math.inf
    else:
        layer.k[src[live[0]], :, 0] = math.nan
    return r, b, src[live].unique(), dst[(src[:, None] == src[live][None]).any(1)].unique()


def _check(layer, r, b, got, how, node, sources, seen_by):
    """Whatever the spoilt score does not reach is what it is without it."""
    dead_dst = seen_by if how == "key" else th.tensor([node])       # rows whose softmax is spoilt
    dst, src = ref.dst_of_edges(layer.g.indptr), layer.g.indices.long()
    spoilt = (dst[:, None] == dead_dst[None]).any(1)
    live = r["part"].any(1)
    dead_src = src[spoilt & live].unique()
    for name, t in zip(layer.names(), got):
        t, want, bound = t.detach().cpu().double(), r[name], b[name]
        if name == "d_lam":
            continue                                                # a sum over all queries
        if name == "d_table":
            keep = th.ones(len(want), dtype=th.bool)
            keep[layer.bucket[spoilt & live].unique().long()] = False
            assert bool(keep[5:].all())
            assert bool((t[5:] == 0).all()), name
        else:
            keep = th.ones(len(want), dtype=th.bool)
            keep[dead_dst if name in ("o", "dq") else dead_src] = False
        assert bool(keep.any())
        ref.assert_within(t[keep], want[keep], bound[keep], name)


@pytest.mark.parametrize("diff,buckets", KINDS[::2], ids=KIND_IDS[::2])
@pytest.mark.parametrize("dt", [th.float32, th.float64, th.bfloat16], ids=str)
@pytest.mark.parametrize("how", ["query", "infinite", "key"])
@pytest.mark.parametrize("planned", [False, True])
def test_walkers(diff, buckets, dt, how, planned):
    g = random_graph(90, 400, [12] * 90, 31, dedup=True)
    layer = Layer(g, diff, buckets, 3, 16, dt, seed=31)
    layer.staged = 0.0
    spoilt = _spoilt(layer, how, 40, diff)
    got = layer.step(layer.plans() if planned else None)
    _check(layer, *spoilt[:2], got, how, 40, *spoilt[2:])


@pytest.mark.parametrize("diff,buckets", KINDS[::2], ids=KIND_IDS[::2])
@pytest.mark.parametrize("how", ["query", "infinite", "key"])
def test_tensor_cores(diff, buckets, how):
    g = graphs.banded_graph(2, 400, 40)
    layer = Layer(g, diff, buckets, 2, 32 if diff else 64, th.bfloat16, seed=32)
    layer.staged = STAGED
    spoilt = _spoilt(layer, how, 300, diff)
    plans = layer.plans()
    assert plans[0].dense_band and plans[1].dense_band
    _check(layer, *spoilt[:2], layer.step(plans), how, 300, *spoilt[2:])

@pytest.mark.parametrize("dt", [th.float32, th.bfloat16], ids=str)
@pytest.mark.parametrize("planned", [False, True])
def test_one_map_masked_where_the_other_is_not(dt, planned):
    """Map 0 of node 77 is spoilt by two live edges; its other edges take part in map 1 alone, and nothing of them changes."""
    g = graphs.banded_graph(1, 200, 20)
    layer = Layer(g, True, 7, 2, 32, dt, seed=33)
    dst, src = ref.dst_of_edges(g.indptr), g.indices.long()
    layer.table[5, 0] = -math.inf
    layer.bucket[layer.bucket == 5] = 4
    layer.bucket[layer.bucket == 1] = 0
    mine = (dst == 77).nonzero().flatten()
    layer.bucket[mine] = 5                      # map 0 of head 0 sees nothing of these
    layer.bucket[mine[:2]] = 1
    r = layer.reference()
    staged = STAGED if planned and dt == th.bfloat16 else 0.0
    b = ref.bounds(r, layer.q, layer.k, layer.v, layer.scale, layer.dt, layer.bucket, layer.table, staged)
    layer.q[77, 0] = math.nan
    got = dict(zip(layer.names(), layer.step(layer.plans() if planned else None)))
    assert bool(th.isnan(got["o"][77, 0]).all()) and bool((got["d_table"][5, 0] == 0).all())
    keep = {name: th.ones(len(r[name]), dtype=th.bool) for name in ("o", "dq", "dk", "dv", "d_table")}
    keep["o"][77] = keep["dq"][77] = False
    keep["dk"][src[mine[:2]]] = keep["dv"][src[mine[:2]]] = False
    keep["d_table"][1] = False
    for name, rows in keep.items():
        ref.assert_within(got[name].detach().cpu()[rows], r[name][rows], b[name][rows], name)
