"""Attention layers with learned score terms on the GPU against the float64 edge-list reference (oracle/terms_f64.py), held to the
bounds that its error analysis derives from the types."""
import math

import pytest
import torch as th

from helpers import chunked, graph_zoo, random_graph
from custom_op_benchmark_b200 import graphop, graphs, wrapper
from custom_op_benchmark_b200.part_csr import partition_csr
from oracle import terms_f64 as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
ZOO = graph_zoo()


class Layer:
    """One layer's inputs on a graph, on the device and (as rounded) on the host."""

    def __init__(self, g, diff, buckets, h, d, dt, idt=th.int32, seed=1, chunk=32):
        gen = th.Generator().manual_seed(seed)
        make = lambda *s: th.randn(*s, generator=gen, dtype=th.float64).to(dt)  # noqa: E731
        self.g, self.diff, self.dt, self.scale = g, diff, dt, d ** -0.5
        maps, width = (2 * h, 2 * d) if diff else (h, d)
        self.q, self.k, self.v, self.d_o = make(g.n_dst, maps, d), make(g.n_src, maps, d), make(g.n_src, h, width), make(g.n_dst, h, width)
        self.lam = (th.rand(h, generator=gen, dtype=th.float64) + 0.2).to(dt) if diff else None
        self.bucket = self.table = None
        if buckets:
            self.table = make(buckets, maps)
            self.bucket = th.randint(0, buckets, (g.n_edges,), generator=gen).int()
        self.rows = [t.to(DEV) for t in chunked(g, chunk, dtype=idt)]
        self.cols = [t.to(DEV) for t in chunked(g, chunk, transposed=True, dtype=idt)]
        self.gen = gen

    def plans(self):
        return (graphop.GraphPlan(self.rows[0], self.rows[1], None, self.rows[3], self.g.n_dst),
                graphop.GraphPlan(*self.cols, self.g.n_src))

    def terms(self):
        return [] if self.table is None else [self.bucket.to(DEV), self.table.to(DEV)]

    def reference(self, d_o=True):
        dst, src = ref.dst_of_edges(self.g.indptr), self.g.indices.long()
        return ref.attention(dst, src, self.q, self.k, self.v, self.scale, self.bucket, self.table, self.lam, self.d_o if d_o else None)

    def forward(self, plan=None, **more):
        q, k, v = (t.to(DEV) for t in (self.q, self.k, self.v))
        graph, kind = ([plan], "_planned") if plan else ([self.rows[0], self.rows[1], self.rows[3]], "")
        if self.diff:
            return getattr(graphop, "attention_diff_forward" + kind)(*graph, q, k, v, self.lam.to(DEV), self.scale, *self.terms(), **more)
        return getattr(graphop, "attention_bucket_forward" + kind)(*graph, q, k, v, *self.terms(), self.scale)

    def step(self, plans=None, leaves=None):
        """o and the gradients of q, k, v (, lam)(, table) through the autograd Functions."""
        x = leaves or [t.to(DEV).requires_grad_(True) for t in (self.q, self.k, self.v, self.lam, self.table) if t is not None]
        graph, kind = (plans, "Planned") if plans else ([self.rows[0], self.rows[1], self.rows[3], *self.cols], "")
        bias = [] if self.table is None else [self.bucket.to(DEV), x[-1]]
        if self.diff:
            o = getattr(wrapper, "GraphAttentionDiff" + kind).apply(*graph, *x[:4], self.scale, *bias)
        else:
            o = getattr(wrapper, "GraphAttentionBucket" + kind).apply(*graph, *x[:3], *bias, self.scale)
        return [o, *th.autograd.grad(o, x, self.d_o.to(DEV))]

    def names(self):
        return ["o", "dq", "dk", "dv"] + (["d_lam"] if self.diff else []) + ([] if self.table is None else ["d_table"])

    def check(self, got, staged=0.0):
        r = self.reference()
        b = ref.bounds(r, self.q, self.k, self.v, self.scale, self.dt, self.bucket, self.table, staged)
        for name, t in zip(self.names(), got):
            ref.assert_within(t, r[name], b[name], name)


KINDS = [(False, 7), (True, 0), (True, 7)]
KIND_IDS = ["bucket", "diff", "diff_bucket"]
SHAPES = [(th.float32, th.int32, 4, 32), (th.float32, th.int64, 1, 64), (th.float64, th.int64, 2, 16), (th.bfloat16, th.int32, 8, 32),
          (th.bfloat16, th.int64, 3, 16), (th.float32, th.int32, 5, 8)]


@pytest.mark.parametrize("name,g", ZOO, ids=[z[0] for z in ZOO])
@pytest.mark.parametrize("diff,buckets", KINDS, ids=KIND_IDS)
@pytest.mark.parametrize("dt,idt,h,d", SHAPES, ids=lambda x: str(x).replace("torch.", ""))
def test_training_step(name, g, diff, buckets, dt, idt, h, d):
    layer = Layer(g, diff, buckets, h, d, dt, idt)
    if buckets:
        layer.bucket[::5] = th.randint(-2, buckets + 2, layer.bucket[::5].shape, generator=layer.gen).int()
        layer.table[2, 0] = -math.inf
        layer.table[4, -1] = th.finfo(dt).min
    layer.check(layer.step())
    plans = layer.plans()
    # a dense band in bfloat16 with 64 features per head of v: probabilities and score gradients enter the products as bfloat16
    dense = dt == th.bfloat16 and layer.v.shape[2] == 64 and plans[0].dense_band
    layer.check(layer.step(plans), th.finfo(dt).eps / 2 if dense else 0.0)


@pytest.mark.parametrize("diff,buckets", KINDS, ids=KIND_IDS)
@pytest.mark.parametrize("dt,h,d", [(th.float32, 1, 4), (th.float32, 2, 8), (th.float32, 16, 16), (th.float32, 3, 128), (th.float32, 1, 256),
                                    (th.float32, 1, 512), (th.float64, 1, 2), (th.float64, 4, 64), (th.float64, 1, 256), (th.bfloat16, 1, 8),
                                    (th.bfloat16, 12, 64), (th.bfloat16, 4, 128), (th.bfloat16, 1, 1024), (th.bfloat16, 32, 16)],
                         ids=lambda x: str(x).replace("torch.", ""))
def test_every_row_shape(diff, buckets, dt, h, d):
    g = ZOO[3][1]
    layer = Layer(g, diff, buckets, h, d, dt, seed=2)
    layer.check(layer.step())


@pytest.mark.parametrize("diff,buckets", KINDS, ids=KIND_IDS)
def test_forward_statistics_and_parts(diff, buckets):
    layer = Layer(ZOO[2][1], diff, buckets, 4, 32, th.float32, seed=3)
    r = layer.reference(False)
    b = ref.bounds(r, layer.q, layer.k, layer.v, layer.scale, layer.dt, layer.bucket, layer.table)
    for plan in (None, layer.plans()[0]):
        o, lse, *parts = layer.forward(plan)
        ref.assert_within(o, r["o"], b["o"], "o")
        ref.assert_within(lse, r["lse"], b["lse"], "lse")
        if diff:
            ref.assert_within(parts[0], r["parts"], b["parts"], "parts")
            bare = layer.forward(plan, keep_parts=False)
            assert bare[2] is None and th.equal(bare[0], o) and th.equal(bare[1], lse)


@pytest.mark.parametrize("diff,buckets", KINDS, ids=KIND_IDS)
def test_the_same_bits_every_time_and_on_plans(diff, buckets):
    layer = Layer(ZOO[3][1], diff, buckets, 4, 32, th.float32, seed=4)
    first = layer.step()
    for plans in (None, layer.plans()):
        for a, b in zip(first, layer.step(plans)):
            assert th.equal(a, b)


@pytest.mark.parametrize("diff,buckets", [KINDS[0], KINDS[2]], ids=["bucket", "diff_bucket"])
@pytest.mark.parametrize("dt", [th.float32, th.bfloat16, th.float64], ids=str)
def test_what_takes_no_part_may_hold_anything(diff, buckets, dt):
    """Padding: a fifth of the nodes on either side holds NaN and infinities, and every edge of theirs is masked, by its bucket or by
    the table; some nodes have nothing left."""
    g = ZOO[0][1]
    layer = Layer(g, diff, buckets, 4, 32, dt, seed=5)
    layer.table[6] = -math.inf
    dst, src = ref.dst_of_edges(g.indptr), g.indices.long()
    gone_dst, gone_src = th.arange(g.n_dst) % 5 == 1, th.arange(g.n_src) % 5 == 2
    gone = gone_dst[dst] | gone_src[src] | (dst == 17)
    layer.bucket[gone & (th.arange(g.n_edges) % 2 == 0)] = -1
    layer.bucket[gone & (th.arange(g.n_edges) % 4 == 1)] = 6
    layer.bucket[gone & (th.arange(g.n_edges) % 4 == 3)] = buckets
    layer.bucket[~gone] = layer.bucket[~gone] % 6
    for t in (layer.q, layer.d_o):
        t[gone_dst] = math.nan
    layer.q[6] = math.inf
    for t in (layer.k, layer.v):
        t[gone_src] = math.nan
    layer.v[7] = -math.inf
    got = layer.step()
    layer.check(got)
    assert bool((got[0][gone_dst.to(DEV)] == 0).all()) and bool((got[1][gone_dst.to(DEV)] == 0).all())
    o, lse = layer.forward()[:2]
    assert bool((lse[gone_dst.to(DEV)] == -math.inf).all()) and bool((o[17] == 0).all())


def test_nothing_left_anywhere():
    for diff, buckets in (KINDS[0], KINDS[2]):
        layer = Layer(ZOO[3][1], diff, buckets, 2, 16, th.float32, seed=6)
        layer.bucket.fill_(-1)
        for t in layer.step():
            assert bool((t == 0).all())


def test_large_biases_and_scores():
    """Scores of thousands, positive and negative, and rows that all carry the same large bias."""
    for diff, buckets in KINDS:
        layer = Layer(ZOO[3][1], diff, buckets, 2, 32, th.float32, seed=7)
        layer.q *= 20
        if buckets:
            layer.table[:] = layer.table * 100 - 1000
        layer.check(layer.step())


def test_a_scale_of_zero_leaves_the_bias():
    layer = Layer(ZOO[3][1], False, 7, 2, 32, th.float32, seed=8)
    layer.scale = 0.0
    got = layer.step()
    layer.check(got)
    assert bool((got[1] == 0).all()) and bool((got[2] == 0).all()) and bool((got[4] != 0).any())


@pytest.mark.parametrize("buckets,h", [(1, 1), (2, 33), (300, 8), (2000, 16), (16384, 1), (16384, 3)])
def test_table_sizes(buckets, h):
    g = ZOO[6][1]
    layer = Layer(g, False, buckets, h, 16, th.float32, seed=9)
    layer.check(layer.step())


def test_a_large_table_in_double_precision():
    layer = Layer(ZOO[6][1], False, 16384, 2, 16, th.float64, seed=10)
    layer.check(layer.step())


@pytest.mark.parametrize("chunk", [None, 1, 32])
@pytest.mark.parametrize("diff,buckets", KINDS, ids=KIND_IDS)
def test_single_tokens_over_long_rows(diff, buckets, chunk):
    """Decoding: a destination per sequence, of nothing, one and many cached rows in any order."""
    lengths = [0, 1, 4099, 0, 33, 700]
    gen = th.Generator().manual_seed(11)
    pool = 6000
    slots = th.randperm(pool, generator=gen)[: sum(lengths)]
    dst = th.repeat_interleave(th.arange(6), th.tensor(lengths))
    g = graphs.coo_to_graph(dst, slots, 6, pool, index_dtype=th.int32)
    for dt, h, d in ((th.bfloat16, 4, 64), (th.float32, 2, 32)):
        layer = Layer(g, diff, buckets, h, d, dt, seed=12, chunk=chunk)
        r = layer.reference(False)
        b = ref.bounds(r, layer.q, layer.k, layer.v, layer.scale, dt, layer.bucket, layer.table)
        o, lse = layer.forward()[:2]
        ref.assert_within(o, r["o"], b["o"], "o")
        ref.assert_within(lse, r["lse"], b["lse"], "lse")


@pytest.mark.parametrize("both", [True, False])
@pytest.mark.parametrize("idt", [th.int32, th.int64])
@pytest.mark.parametrize("count,reach", [(2, 5), (32, 128), (31, 60), (320, 5000)])
def test_relative_buckets(both, idt, count, reach):
    if both and (count % 2 or count // 2 < 2):
        with pytest.raises(ValueError):
            graphop.relative_buckets(*[th.zeros(n, dtype=idt, device=DEV) for n in (1, 2, 1)], count, reach, both)
        return
    for name, g in ZOO:
        rows = [t.to(DEV) for t in chunked(g, 32, dtype=idt)]
        graph = [rows[0], rows[1], rows[3]]
        plan = graphop.GraphPlan(rows[0], rows[1], None, rows[3], g.n_dst)
        dst, src = ref.dst_of_edges(g.indptr), g.indices.long()
        gen = th.Generator().manual_seed(13)
        far = th.randint(-2 ** 31, 2 ** 31 - 1, (g.n_dst + g.n_src,), generator=gen)
        for pos in ((None, None), (far[: g.n_dst] // 2 ** 20, far[g.n_dst:] // 2 ** 20), (far[: g.n_dst], far[g.n_dst:])):
            on = [None if p is None else p.to(DEV, idt) for p in pos]
            want = ref.relative_buckets(dst, src, count, reach, both, *pos)
            for got in (graphop.relative_buckets(*graph, count, reach, both, *on), graphop.relative_buckets_planned(plan, count, reach, both, *on)):
                assert got.dtype == th.int32 and th.equal(got.cpu(), want), name


def test_relative_buckets_of_far_positions_and_uncovered_ones():
    row, ptr = th.tensor([0, 1], device=DEV), th.tensor([1, 3, 4], device=DEV)       # position 0 and 4 belong to no chunk
    idx = th.tensor([0, 0, 1, 1, 0], device=DEV)
    at = th.tensor([-2 ** 62, 2 ** 62], device=DEV)
    got = graphop.relative_buckets(row, ptr, idx, 32, 128, True, at, at)
    assert got.tolist() == [-1, 0, 31, 0, -1]
    assert graphop.relative_buckets(row, ptr, idx, 32, 128, False, at.flip(0), at).tolist() == [-1, 31, 0, 0, -1]


@pytest.mark.parametrize("diff,buckets", KINDS, ids=KIND_IDS)
def test_graphs_without_edges_nodes_or_chunks(diff, buckets):
    h, d = 2, 16
    maps, width = (2 * h, 2 * d) if diff else (h, d)
    none = th.zeros(0, dtype=th.int32, device=DEV)
    for n, m, e, covered in ((5, 3, 0, True), (0, 3, 0, True), (5, 0, 0, True), (5, 3, 6, False)):
        ptr = th.zeros(1, dtype=th.int32, device=DEV)
        idx = th.zeros(e, dtype=th.int32, device=DEV)
        x = [th.randn(*s, device=DEV).requires_grad_(True) for s in ((n, maps, d), (m, maps, d), (m, h, width))]
        more = [th.randn(h, device=DEV).requires_grad_(True)] if diff else []
        bias = [th.zeros(e, dtype=th.int32, device=DEV), th.randn(buckets, maps, device=DEV).requires_grad_(True)] if buckets else []
        graph = [none, ptr, idx, none, ptr, idx, idx]
        o = wrapper.GraphAttentionDiff.apply(*graph, *x, *more, 0.5, *bias) if diff else wrapper.GraphAttentionBucket.apply(*graph, *x, *bias, 0.5)
        assert o.shape == (n, h, width) and bool((o == 0).all())
        for t in th.autograd.grad(o, x + more + bias[1:], th.ones_like(o)):
            assert bool((t == 0).all())


def test_refusals():
    layer = Layer(ZOO[0][1], True, 7, 4, 32, th.float32)
    q, k, v, lam, d_o = (t.to(DEV) for t in (layer.q, layer.k, layer.v, layer.lam, layer.d_o))
    bucket, table = layer.terms()
    graph = [layer.rows[0], layer.rows[1], layer.rows[3]]
    plan_r, plan_t = layer.plans()

    def diff(match, q=q, k=k, v=v, lam=lam, bucket=bucket, table=table):
        with pytest.raises(RuntimeError, match=match):
            graphop.attention_diff_forward(*graph, q, k, v, lam, 1.0, bucket, table)
        with pytest.raises(RuntimeError, match=match):
            graphop.attention_diff_forward_planned(plan_r, q, k, v, lam, 1.0, bucket, table)
    diff("must be \\(n, 2h, d\\)", v=v[:, :2].contiguous())
    diff("must be \\(n, 2h, d\\)", v=v[:, :, :32].contiguous())
    diff("must be \\(n, 2h, d\\)", q=q[:, :7].contiguous(), k=k[:, :7].contiguous())
    diff("disagree", k=k[:, :6].contiguous())
    diff("disagree", v=v[:-1].contiguous())
    diff("must be contiguous", k=k.transpose(0, 1).contiguous().transpose(0, 1))
    diff("lam must be", lam=lam[:3].contiguous())
    diff("share dtype", lam=lam.double())
    diff("share dtype", table=table.bfloat16())
    diff("come together", bucket=None)
    diff("come together", table=None)
    diff("bucket must be", bucket=bucket.long())
    diff("bucket must be", bucket=bucket[:-1].contiguous())
    diff("table must be", table=table[:, :4].contiguous())
    diff("must be a CUDA tensor", bucket=bucket.cpu())
    diff("not supported", q=q[:, :, :24].contiguous(), k=k[:, :, :24].contiguous(), v=v[:, :, :48].contiguous())
    diff("not implemented for 'Half'", q=q.half(), k=k.half(), v=v.half(), lam=lam.half(), table=table.half())
    diff("not supported", table=th.zeros(16385, 8, device=DEV))
    with pytest.raises(RuntimeError, match="a row for each of the plan"):
        graphop.attention_diff_forward_planned(plan_r, q[:-1].contiguous(), k, v, lam, 1.0)
    o, lse, parts = graphop.attention_diff_forward_planned(plan_r, q, k, v, lam, 1.0)
    no_ids = graphop.GraphPlan(layer.cols[0], layer.cols[1], None, layer.cols[3], layer.g.n_src)
    with pytest.raises(RuntimeError, match="must have edge ids"):
        graphop.attention_diff_backward_planned(plan_r, no_ids, q, k, v, lam, parts, lse, d_o, 1.0)
    with pytest.raises(RuntimeError, match="forward's shapes"):
        graphop.attention_diff_backward_planned(plan_r, plan_t, q, k, v, lam, parts, lse[:-1], d_o, 1.0)
    with pytest.raises(RuntimeError, match="forward's shapes"):
        graphop.attention_diff_backward_planned(plan_r, plan_t, q, k, v, lam, parts, lse, d_o[:-1], 1.0)
    with pytest.raises(RuntimeError, match="must be given"):
        graphop.attention_bucket_forward(*graph, q, k, k, None, None, 1.0)
    for pos, match in ((th.zeros(64, device=DEV), "dst_pos"), (th.zeros(64, dtype=th.int32), "must be a CUDA tensor"),
                       (th.zeros(63, dtype=th.int32, device=DEV), "a position for every node")):
        with pytest.raises(RuntimeError, match=match):
            graphop.relative_buckets_planned(plan_r, 32, 128, True, pos, None)
    with pytest.raises(RuntimeError, match="index type"):
        graphop.relative_buckets(*graph, 32, 128, True, th.zeros(64, dtype=th.int64, device=DEV), None)


def test_a_plan_that_names_more_sources_than_there_are_rows_is_refused():
    """Before the forward reads them, with and without the compiled nodes."""
    layer = Layer(ZOO[0][1], True, 7, 4, 32, th.float32)
    q, k, v, lam = (t.to(DEV) for t in (layer.q, layer.k, layer.v, layer.lam))
    bucket, table = layer.terms()
    plans = layer.plans()
    short = [k[:-1].contiguous(), v[:-1].contiguous()]
    bias = [bucket, table[:, :4].contiguous()]
    calls = [lambda f: f(*plans, q, *short, lam, 1.0, bucket, table),
             lambda f: f(*plans, v, short[1], short[1], *bias, 1.0)]
    for cls, call in zip((wrapper.GraphAttentionDiffPlanned, wrapper.GraphAttentionBucketPlanned), calls):
        for apply in (cls.apply, super(cls, cls).apply):
            with pytest.raises(RuntimeError, match="a row for each of the plan"):
                call(apply)


@pytest.mark.parametrize("both,reach,last", [(False, 3865, 1023), (False, 3870, 1024), (False, 3874, 1025), (True, 23103, 1023),
                                             (True, 23137, 1024), (True, 23171, 1025)])
def test_limits_around_the_table_by_distance(both, reach, last):
    """Limits that end at 1024 or before make a table of the distances, others are searched; distances on both sides of the last one."""
    assert graphop.bucket_limits(5 if both else 10, reach)[-1] == last
    n = 2300
    at = th.arange(n) * (1 - 2 * (th.arange(n) % 2)) if both else -th.arange(n)
    graph = [th.zeros(1, dtype=th.int64, device=DEV), th.tensor([0, n], device=DEV), th.arange(n, device=DEV)]
    zero = th.zeros(1, dtype=th.int64)
    want = ref.relative_buckets(th.zeros(n, dtype=th.int64), th.arange(n), 10, reach, both, zero, at)
    assert th.equal(graphop.relative_buckets(*graph, 10, reach, both, zero.to(DEV), at.to(DEV)).cpu(), want)
    plan = graphop.GraphPlan(graph[0], graph[1], None, graph[2], 1)
    assert th.equal(graphop.relative_buckets_planned(plan, 10, reach, both, zero.to(DEV), at.to(DEV)).cpu(), want)


@pytest.mark.parametrize("diff,buckets", KINDS, ids=KIND_IDS)
@pytest.mark.parametrize("name", ["zoo", "band"])
def test_more_rows_than_the_graph_names(diff, buckets, name):
    """A padded batch: node rows behind the last one of a plan or of a chunk table come out as zeros, whatever they hold."""
    g = ZOO[2][1] if name == "zoo" else graphs.banded_graph(1, 300, 60)
    d = 64 if not diff else 32
    layer = Layer(g, diff, buckets, 2, d, th.bfloat16, seed=21)
    plans = layer.plans()
    for on in (None, plans):
        want = layer.step(on)
        x = [t.to(DEV) for t in (layer.q, layer.k, layer.v, layer.lam, layer.table) if t is not None]
        pad = [th.full((5, *t.shape[1:]), math.nan, dtype=t.dtype, device=DEV) for t in x[:3]]
        leaves = [th.cat([t, p]).requires_grad_(True) for t, p in zip(x[:3], pad)] + [t.requires_grad_(True) for t in x[3:]]
        d_o, layer.d_o = layer.d_o, th.cat([layer.d_o, th.zeros(5, *layer.d_o.shape[1:], dtype=layer.dt)])
        got = layer.step(on, leaves)
        layer.d_o = d_o
        for n, w, t in zip(layer.names(), want, got):
            if t.shape != w.shape:
                assert bool((t[len(w):] == 0).all()), n
                t = t[: len(w)]
            assert not bool(th.isnan(t).any()), n
        layer.check([t[: len(w)] for t, w in zip(got, want)], th.finfo(th.bfloat16).eps / 2 if name == "band" else 0.0)


@pytest.mark.parametrize("diff,buckets", KINDS[::2], ids=KIND_IDS[::2])
def test_ids_and_biases_at_odd_addresses(diff, buckets):
    """Neither the ids nor the table nor lam have to be aligned to more than their elements; node tensors that are not are refused."""
    def odd(t):
        room = th.empty(t.numel() + 1, dtype=t.dtype, device=DEV)
        room[1:] = t.reshape(-1).to(DEV)
        return room[1:].view(t.shape)

    for g in (ZOO[2][1], graphs.banded_graph(1, 300, 60)):
        layer = Layer(g, diff, buckets, 2, 32 if diff else 64, th.bfloat16, seed=22)
        for plan in (None, layer.plans()[0]):
            graph, kind = ([plan], "_planned") if plan else ([layer.rows[0], layer.rows[1], layer.rows[3]], "")
            q, k, v = (t.to(DEV) for t in (layer.q, layer.k, layer.v))
            call = getattr(graphop, ("attention_diff_forward" if diff else "attention_bucket_forward") + kind)
            terms = [odd(layer.bucket), odd(layer.table)]
            more = lambda q: call(*graph, q, k, v, odd(layer.lam), layer.scale, *terms) if diff else call(*graph, q, k, v, *terms, layer.scale)  # noqa: E731
            assert all(th.equal(a, b) for a, b in zip(more(q)[:2], layer.forward(plan)[:2]))
            with pytest.raises(RuntimeError, match="not supported"):
                more(odd(q))


@pytest.mark.parametrize("reach", [2 ** 32 - 2 ** 20, 2 ** 40])
def test_limits_and_distances_around_32_bits(reach):
    """Limits within 32 bits and beyond, distances from -2^62 to 2^62 with those around every limit and around 2^32."""
    near = [x + i for x in graphop.bucket_limits(10, reach) + [2 ** 32, 2 ** 31, 2 ** 62] for i in (-1, 0, 1)]
    at = th.tensor(near + [-x for x in near] + [0])
    n = len(at)
    assert (graphop.bucket_limits(10, reach)[-1] >= 2 ** 32) == (reach > 2 ** 32)
    graph = [th.zeros(1, dtype=th.int64, device=DEV), th.tensor([0, n], device=DEV), th.arange(n, device=DEV)]
    plan = graphop.GraphPlan(graph[0], graph[1], None, graph[2], 1)
    zero = th.zeros(1, dtype=th.int64)
    for both, count in ((False, 10), (True, 20)):
        want = ref.relative_buckets(th.zeros(n, dtype=th.int64), th.arange(n), count, reach, both, zero, at)
        assert th.equal(graphop.relative_buckets(*graph, count, reach, both, zero.to(DEV), at.to(DEV)).cpu(), want)
        assert th.equal(graphop.relative_buckets_planned(plan, count, reach, both, zero.to(DEV), at.to(DEV)).cpu(), want)
