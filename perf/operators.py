"""Performance cases of the attention layers with learned score terms: a bias by buckets, the bucket ids themselves, and
differential attention.

A case is a dict of plain values:
    op       "bucket"   attention with a learned bias by buckets: scores scale * q.k + table[bucket[edge], head]
             "diff"     differential attention: (softmax of map 1 - lam * softmax of map 2) v, heads are pairs of maps;
                        with buckets > 0 both maps have the bias (2 * heads columns in the table)
             "relative" the bucket of every edge from the two ends' positions
    graph    "blocks" (batch x length, fully connected blocks), "band" (batch x length, +-window), "regular" (nodes,
             degree), "uniform" (nodes, edges), "rmat" (scale, edge_factor), "cache" (seqs sequences, each with one new
             token that attends to its own cached slots: up to length of them, scattered over a pool)
    heads, dim (features of a map), dtype ("float32", "float64", "bfloat16"), index ("int32", "int64"), train (forward and
    backward, or forward alone), entry ("chunks": chunk tables; "plans": graph plans the program keeps), buckets, reach
    (the distance of the last bucket), both (buckets for both directions), masked (share of edges that take no part)

A "cache" pass is what a decoding step does: bucket ids of the new edges, then the layer.
"""
import math

import torch as th

own = False

DEV = "cuda"
DTYPES = {"float32": th.float32, "float64": th.float64, "bfloat16": th.bfloat16}
INDEX = {"int32": th.int32, "int64": th.int64}
ITEM = {"float32": 4, "float64": 8, "bfloat16": 2, "int32": 4, "int64": 8}
MOST = 2.2e9      # edges * features of a row of the largest training case: drawn ones stay below


def _case(name, op, graph, heads=1, dim=1, dtype="float32", index="int32", train=True, entry="chunks", buckets=32, reach=128,
          both=True, masked=0.0, **sizes):
    c = dict(op=op, graph=graph, heads=heads, dim=dim, dtype=dtype, index=index, train=train, entry=entry, buckets=buckets,
             reach=reach, both=both, masked=masked)
    if name:
        c["name"] = name
    c.update(sizes)
    return c


def listed():
    return [
        # a few short sentences, fully connected, a training step on chunk tables: launches and host work
        _case("bucket_blocks_small", "bucket", "blocks", 8, 64, index="int64", buckets=32, batch=8, length=30),
        # the benchmark's small attention layer with a bias by edge type, a twentieth of the edges padding
        _case("bucket_er_small", "bucket", "regular", 8, 64, entry="plans", buckets=64, masked=0.05, nodes=4096, degree=16),
        # the benchmark's banded local attention with relative positions, two sequences, training step
        _case("bucket_band_train", "bucket", "band", 8, 64, "bfloat16", entry="plans", batch=2, length=8192, window=128),
        # a power-law graph with a bias by hop distance, chunk tables
        _case("bucket_rmat18_train", "bucket", "rmat", 4, 64, buckets=128, scale=18, edge_factor=16),
        # decoding: one token of each of 32 sequences over their cached rows, ids and layer in every step
        _case("bucket_cache_step", "bucket", "cache", 8, 128, "bfloat16", train=False, reach=4096, both=False, seqs=32,
              length=8192),
        # ids of a few sentences
        _case("relative_blocks_small", "relative", "blocks", index="int64", train=False, batch=16, length=30),
        # ids of the benchmark's four banded sequences
        _case("relative_band", "relative", "band", train=False, batch=4, length=8192, window=128),
        # a few short sentences through the differential layer
        _case("diff_blocks_small", "diff", "blocks", 8, 32, index="int64", buckets=0, batch=8, length=30),
        # the power-law graph, differential
        _case("diff_rmat18_train", "diff", "rmat", 4, 32, entry="plans", buckets=0, scale=18, edge_factor=16),
        # banded local attention, differential, two sequences, training step
        _case("diff_band_train", "diff", "band", 8, 32, "bfloat16", entry="plans", buckets=0, batch=2, length=8192, window=128),
        # a sampled neighbourhood with edge types, odd sizes and an odd number of heads
        _case("diff_bucket_sampled", "diff", "uniform", 3, 32, "bfloat16", "int64", buckets=33, masked=0.1, nodes=60_013,
              edges=600_007),
        # decoding with the differential layer and relative positions
        _case("diff_bucket_cache_step", "diff", "cache", 8, 64, "bfloat16", train=False, reach=4096, both=False, seqs=7,
              length=20_011),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["bucket", "bucket", "bucket", "relative", "diff", "diff", "diff"])
    index = rng.choice(["int32", "int64"])
    buckets, reach, both = rng.choice([8, 16, 31, 32, 64, 128, 320]), _log(rng, 64, 10_000), rng.random() < 0.6
    if both:
        buckets += buckets & 1
    reach = max(reach, buckets + 1)
    entry = rng.choice(["chunks", "plans"])
    if op == "relative":
        if rng.random() < 0.5:
            return _case(None, op, "band", 1, 1, index=index, train=False, buckets=buckets, reach=reach, both=both,
                         entry=entry, batch=rng.randint(1, 5), length=_log(rng, 300, 8000), window=_log(rng, 8, 128))
        return _case(None, op, "uniform", 1, 1, index=index, train=False, buckets=buckets, reach=reach, both=both, entry=entry,
                     nodes=_log(rng, 200, 200_000), edges=_log(rng, 2_000, 8_000_000))
    dtype = rng.choice(["float32", "float32", "bfloat16", "bfloat16", "float64"])
    dim = rng.choice([16, 32, 64, 128] if op == "bucket" else [16, 32, 64])
    heads = rng.choice([1, 2, 3, 4, 6, 8, 12, 16])
    width = heads * dim * (1 if op == "bucket" else 2)
    while width * ITEM[dtype] > 4096 or width > 1024:
        heads = max(1, heads // 2)
        width = heads * dim * (1 if op == "bucket" else 2)
    if op == "diff" and rng.random() < 0.5:
        buckets = 0
    cap = 0.8 * MOST / width * 4 / max(4, ITEM[dtype])      # edges
    kind = rng.choice(["band", "band", "rmat", "uniform", "regular", "blocks", "cache", "cache"])
    masked = rng.choice([0.0, 0.0, 0.1, 0.5])
    if kind == "cache":
        if op == "diff" and rng.random() < 0.5:
            buckets = 32
        seqs = _log(rng, 1, 64)
        return _case(None, op, kind, heads, dim, dtype, index, False, "chunks", buckets, reach, False, 0.0, seqs=seqs,
                     length=_log(rng, 50, min(40_000, 300_000 // seqs)))
    if kind == "band":
        window = _log(rng, 8, 200)
        total = int(min(_log(rng, 300, 40_000), cap / (2 * window + 1)))
        batch = min(rng.choice([1, 1, 2, 5]), max(1, total // 200))
        sizes = dict(batch=batch, length=max(50, total // batch), window=window)
    elif kind == "rmat":
        ef = rng.randint(6, 20)
        sizes = dict(scale=rng.randint(9, max(9, min(18, int(math.log2(cap / (ef + 1)))))), edge_factor=ef)
    elif kind == "blocks":
        length = rng.randint(5, 60)
        sizes = dict(batch=max(1, int(min(_log(rng, 2, 1000), cap / length ** 2))), length=length)
    else:
        nodes = _log(rng, 200, 250_000)
        degree = max(2, int(min(math.exp(rng.uniform(math.log(2), math.log(60))), cap / nodes)))
        sizes = dict(nodes=nodes, degree=degree) if kind == "regular" else dict(nodes=nodes, edges=int(nodes * degree * 1.013))
    return _case(None, op, kind, heads, dim, dtype, index, rng.random() < 0.8, entry, buckets, reach, both, masked, **sizes)


# ------------------------------------------------------------------------------------------
# graphs: (destination, source) of every edge, sorted by destination; nodes on either side
# ------------------------------------------------------------------------------------------
def _edges(case, gen):
    kind = case["graph"]

    def ids(count, n):
        return th.randint(0, n, (count,), generator=gen, device=DEV)
    if kind in ("blocks", "band"):
        n, length = case["batch"] * case["length"], case["length"]
        node = th.arange(n, device=DEV)
        first = node - node % length
        lo, hi = first, first + length - 1
        if kind == "band":
            lo, hi = th.maximum(lo, node - case["window"]), th.minimum(hi, node + case["window"])
        dst = node.repeat_interleave(hi - lo + 1)
        begin = th.cumsum(hi - lo + 1, 0) - (hi - lo + 1)
        return dst, th.arange(dst.numel(), device=DEV) - begin[dst] + lo[dst], n, n
    if kind == "cache":
        # lengths from nothing to the longest, spread over their logarithm; slots in the order the pool gave them out
        n, most = case["seqs"], case["length"]
        share = th.linspace(0, 1, n, device=DEV, dtype=th.float64) if n > 1 else th.ones(1, device=DEV, dtype=th.float64)
        lengths = ((most + 1) ** share[th.randperm(n, generator=gen, device=DEV)] - 1).round().long()
        dst = th.arange(n, device=DEV).repeat_interleave(lengths)
        pool = n * most
        return dst, th.randperm(pool, generator=gen, device=DEV)[: dst.numel()], n, pool
    if kind == "rmat":
        n, want = 1 << case["scale"], case["edge_factor"] << case["scale"]
        dst, src = (th.zeros(want + want // 4, dtype=th.int64, device=DEV) for _ in range(2))
        for _ in range(case["scale"]):
            u = th.rand(dst.numel(), generator=gen, device=DEV)
            dst = (dst << 1) | (u >= 0.76)
            src = (src << 1) | ((u >= 0.57) & (u < 0.76) | (u >= 0.95))
        keys = th.unique((dst * n + src)[dst != src])
        keys = keys[th.randperm(keys.numel(), generator=gen, device=DEV)]
        keys = keys[:want] if keys.numel() >= want else keys.repeat(-(-want // keys.numel()))[:want]
        keys = th.cat([keys, th.arange(n, device=DEV) * (n + 1)]).sort().values
        return keys // n, keys % n, n, n
    n = case["nodes"]
    if kind == "regular":
        dst = th.arange(n, device=DEV).repeat_interleave(case["degree"])
    else:
        dst = ids(case["edges"], n).sort().values
    return dst, ids(dst.numel(), n), n, n


def _chunk_table(owner_sorted, n, index):
    """The CSR of sorted owners cut into chunks of up to 32 positions: owner of each chunk, chunk boundaries."""
    deg = th.bincount(owner_sorted, minlength=n)
    ptr = th.cat([deg.new_zeros(1), th.cumsum(deg, 0)])
    pieces = (deg + 31) // 32
    row = th.arange(n, device=DEV).repeat_interleave(pieces)
    nth = th.arange(row.numel(), device=DEV) - (th.cumsum(pieces, 0) - pieces)[row]
    starts = ptr[row] + 32 * nth
    return row.to(index), th.cat([starts, ptr[-1:]]).to(index)


def prepare(case, seed):
    gen = th.Generator(device=DEV).manual_seed(seed)
    index, dt = INDEX[case["index"]], DTYPES[case["dtype"]]
    dst, src, n, m = _edges(case, gen)
    e, h, d, diff = dst.numel(), case["heads"], case["dim"], case["op"] == "diff"
    row, ptr = _chunk_table(dst, n, index)
    st = {"case": case, "dst": dst, "src": src, "n": n, "m": m, "rows": [row, ptr, src.to(index)], "pos": (None, None)}
    if case["train"]:
        order = src.sort(stable=True).indices
        col, ptr_t = _chunk_table(src[order], m, index)
        st["cols"] = [col, ptr_t, order.to(index), dst[order].to(index)]
    if case["graph"] == "cache":
        # the new token stands behind its cached ones, wherever their slots lie
        lengths = th.bincount(dst, minlength=n)
        slot_pos = th.zeros(m, dtype=th.int64, device=DEV)
        slot_pos[src] = th.arange(e, device=DEV) - (th.cumsum(lengths, 0) - lengths)[dst]
        st["pos"] = (lengths.to(index), slot_pos.to(index))
    if case["op"] == "relative":
        # packed sequences out of which tokens were dropped: a node stands one to four places behind the one before it
        place = th.cumsum(th.randint(1, 5, (max(n, m),), generator=gen, device=DEV), 0).to(index)
        st["pos"] = (place[:n].contiguous(), place[:m].contiguous())
    if own and case["entry"] == "plans":      # what the framework's program keeps of a graph (it has them without these operators)
        from custom_op_benchmark_b200 import graphop
        st["plans"] = [graphop.GraphPlan(row, ptr, None, st["rows"][2], n)]
        if case["train"]:
            st["plans"].append(graphop.GraphPlan(*st["cols"], m))
    if case["op"] == "relative":
        return st
    make = th.float64 if dt == th.float64 else th.float32

    def normal(*shape, mag=1.0):
        return (th.randn(*shape, generator=gen, device=DEV, dtype=make) * mag).to(dt)
    maps = 2 * h if diff else h
    width = 2 * d if diff else d
    st["in"] = [normal(n, maps, d), normal(m, maps, d), normal(m, h, width)]
    if diff:
        st["in"].append((th.rand(h, generator=gen, device=DEV, dtype=make) * 0.6 + 0.2).to(dt))
    st["bucket"] = None
    if case["buckets"]:
        st["in"].append(normal(case["buckets"], maps, mag=0.7))
        if case["graph"] in ("band", "blocks"):
            st["bucket"] = _relative_plain(st)
        elif case["graph"] != "cache":
            st["bucket"] = th.randint(0, case["buckets"], (e,), generator=gen, device=DEV).int()
        if case["masked"]:
            st["bucket"][th.rand(e, generator=gen, device=DEV) < case["masked"]] = -1
    st["grad"] = normal(n, h, width)
    if case["train"]:
        for t in st["in"]:
            t.requires_grad_(True)
    return st


# ------------------------------------------------------------------------------------------
# plain forms
# ------------------------------------------------------------------------------------------
def _relative_plain(st):
    """Distances below half of a direction's buckets have their own, longer ones share the rest evenly over the logarithm."""
    case, (dst_pos, src_pos) = st["case"], st["pos"]
    rel = (st["src"] if src_pos is None else src_pos[st["src"]]) - (st["dst"] if dst_pos is None else dst_pos[st["dst"]])
    count = case["buckets"] // 2 if case["both"] else case["buckets"]
    x = rel.long().abs() if case["both"] else (-rel.long()).clamp(min=0)
    half = count // 2
    steps = th.log(x.clamp(min=1).double() / half) * ((count - half) / math.log(case["reach"] / half))
    far = (half + (steps + 1e-9).floor().long()).clamp(max=count - 1)     # 1e-9: a distance on a border belongs behind it
    found = th.where(x < half, x, far)
    if case["both"]:
        found = found + count * (rel > 0)
    return found.int()


def _softmax_plain(st, q, k, table, bucket, scale):
    """Probabilities of every edge (edges, maps), the log of their denominators (n, maps), the edges that take part."""
    dst, n, maps = st["dst"], st["n"], q.size(1)
    s = (q[dst] * k[st["src"]]).sum(-1) * scale
    if table is not None:
        inside = (bucket >= 0) & (bucket < table.size(0))
        bias = table[bucket.clamp(0, table.size(0) - 1).long()]
        s = th.where(inside[:, None] & (bias > -1e38), s + bias, -math.inf)
    where = dst[:, None].expand(-1, maps)
    top = s.new_full((n, maps), -math.inf).scatter_reduce(0, where, s, "amax")
    w = th.exp(s - th.where(top == -math.inf, 0.0, top)[dst])
    total = s.new_zeros(n, maps).index_add(0, dst, w)
    return w / th.where(total == 0, 1.0, total)[dst], th.where(total == 0, -math.inf, top + total.log())


def _attention_plain(st, train):
    case, dst, src, n, m = st["case"], st["dst"], st["src"], st["n"], st["m"]
    wide = th.float64 if case["dtype"] == "float64" else th.float32
    given = [t.detach() for t in st["in"]]
    q, k, v = (t.to(wide) for t in given[:3])
    diff, scale, h = case["op"] == "diff", case["dim"] ** -0.5, case["heads"]
    lam = given[3].to(wide) if diff else None
    table = given[-1].to(wide) if case["buckets"] else None
    bucket = _relative_plain(st) if table is not None and case["graph"] == "cache" else st["bucket"]
    p, lse = _softmax_plain(st, q, k, table, bucket, scale)
    ve = v[src]
    if diff:
        weight = p[:, 0::2] - lam * p[:, 1::2]
    else:
        weight = p
    o = v.new_zeros(n, *v.shape[1:]).index_add(0, dst, weight[..., None] * ve)
    dt = st["in"][0].dtype
    if not train:
        return [o.to(dt), lse]
    g = st["grad"].to(wide)
    ge = g[dst]
    dp = (ge * ve).sum(-1)
    del ve
    dv = v.new_zeros(v.shape).index_add(0, src, weight[..., None] * ge)
    del ge
    if diff:
        dp = dp.repeat_interleave(2, 1)
    delta = p.new_zeros(n, p.size(1)).index_add(0, dst, p * dp)
    ds = p * (dp - delta[dst])
    if diff:
        d_lam = -delta[:, 1::2].sum(0)
        sign = th.ones_like(delta[0])
        sign[1::2] = -lam
        ds = ds * sign
    dq = th.zeros_like(q).index_add(0, dst, (ds * scale)[..., None] * k[src])
    dk = th.zeros_like(k).index_add(0, src, (ds * scale)[..., None] * q[dst])
    out = [o.to(dt), dq.to(dt), dk.to(dt), dv.to(dt)]
    if diff:
        out.append(d_lam.to(dt))
    if table is not None:
        inside = (bucket >= 0) & (bucket < table.size(0))
        out.append(th.zeros_like(table).index_add(0, bucket[inside].long(), ds[inside]).to(dt))
    return out


# ------------------------------------------------------------------------------------------
# one pass
# ------------------------------------------------------------------------------------------
def _own(st):
    from custom_op_benchmark_b200 import graphop, wrapper
    case, (dst_pos, src_pos), plans = st["case"], st["pos"], st.get("plans")
    given = (case["buckets"], case["reach"], case["both"], dst_pos, src_pos)
    if case["op"] == "relative":
        return graphop.relative_buckets_planned(plans[0], *given) if plans else graphop.relative_buckets(*st["rows"], *given)
    x, scale, diff = st["in"], case["dim"] ** -0.5, case["op"] == "diff"
    bucket = st["bucket"]
    if case["graph"] == "cache" and case["buckets"]:
        bucket = graphop.relative_buckets(*st["rows"], *given)
    terms = [bucket, x[-1]] if case["buckets"] else []
    if not case["train"]:
        graph, kind = ([plans[0]], "_planned") if plans else (st["rows"], "")
        if diff:
            o, lse, _ = getattr(graphop, "attention_diff_forward" + kind)(*graph, *x[:4], scale, *terms, keep_parts=False)
        else:
            o, lse = getattr(graphop, "attention_bucket_forward" + kind)(*graph, *x[:3], *terms, scale)
        return [o, lse]
    graph, kind = (plans, "Planned") if plans else (st["rows"] + st["cols"], "")
    if diff:
        o = getattr(wrapper, "GraphAttentionDiff" + kind).apply(*graph, *x[:4], scale, *terms)
    else:
        o = getattr(wrapper, "GraphAttentionBucket" + kind).apply(*graph, *x[:3], *terms, scale)
    return [o.detach()] + list(th.autograd.grad(o, x, st["grad"]))


def run(st):
    if own:
        return _own(st)
    with th.no_grad():
        return _relative_plain(st) if st["case"]["op"] == "relative" else _attention_plain(st, st["case"]["train"])


# ------------------------------------------------------------------------------------------
# what a pass cannot do without
# ------------------------------------------------------------------------------------------
def _counts(case):
    """Destinations, sources that edges name, edges."""
    k = case["graph"]
    if k in ("blocks", "band"):
        n = case["batch"] * case["length"]
        w = min(case.get("window", case["length"]), case["length"] - 1)
        e = n * case["length"] if k == "blocks" else case["batch"] * (case["length"] * (2 * w + 1) - w * (w + 1))
        return n, n, e
    if k == "cache":
        most = case["length"]
        n = case["seqs"]
        e = most if n == 1 else sum(round((most + 1) ** (j / (n - 1)) - 1) for j in range(n))
        return case["seqs"], e, e
    if k == "rmat":
        return 1 << case["scale"], 1 << case["scale"], (1 << case["scale"]) * (case["edge_factor"] + 1)
    return case["nodes"], case["nodes"], case["nodes"] * case["degree"] if k == "regular" else case["edges"]


def work(case):
    n, m, e = _counts(case)
    h, d, s, i = case["heads"], case["dim"], ITEM[case["dtype"]], ITEM[case["index"]]
    graph = (n + 1 + e) * i
    if case["op"] == "relative":
        return {"bytes": graph + 4 * e + max(n, m) * i, "flops": 2 * e}
    maps, acc = (2, max(4, s)) if case["op"] == "diff" else (1, max(4, s))
    row = h * maps * d * s                                     # a node's row of q, k, v or o alike
    table = case["buckets"] * h * maps * s
    ids = (2 * m * i if case["graph"] == "cache" else 4 * e) if case["buckets"] else 0
    b, f = graph + ids + table + 2 * (n + m) * row + n * h * maps * acc, (4 if maps == 1 else 8) * e * h * d
    if case["train"]:        # dO in, dq, dk, dv out, the transposed graph with its edge ids, the learned terms' gradients
        b += (2 * n + 2 * m) * row + (m + 1 + 2 * e) * i + table + (2 * h * s if maps == 2 else 0)
        f += (10 if maps == 1 else 20) * e * h * d
    return {"bytes": int(b), "flops": int(f)}


# ------------------------------------------------------------------------------------------
# in 64 bits, from the definitions: one map after the other, gradients by differentiation
# ------------------------------------------------------------------------------------------
def exact(case, seed):
    if case["op"] == "relative":
        return None
    st = prepare(case, seed)
    n, m, h, diff, scale = st["n"], st["m"], case["heads"], case["op"] == "diff", case["dim"] ** -0.5
    x = [t.detach().double() for t in st["in"]]
    bucket = _relative_plain(st) if case["buckets"] and case["graph"] == "cache" else st["bucket"]
    maps, per = (2, 2) if diff else (1, 1)
    g = st["grad"].double()
    grads, out, lse = [th.zeros_like(t) for t in x], th.zeros_like(g), th.full((n, h * maps), -math.inf, dtype=th.float64, device=DEV)
    for head in range(h):
        leaves = [x[0][:, per * head: per * (head + 1)].clone(), x[1][:, per * head: per * (head + 1)].clone(), x[2][:, head].clone()]
        if diff:
            leaves.append(x[3][head].clone())
        if case["buckets"]:
            leaves.append(x[-1][:, per * head: per * (head + 1)].clone())
        for t in leaves:
            t.requires_grad_(case["train"])
        q, k, v = leaves[:3]
        o = 0
        for j in range(maps):
            dst, src, score = st["dst"], st["src"], 0
            if case["buckets"]:
                b = bucket.long()
                part = (b >= 0) & (b < case["buckets"])
                part[part.clone()] = (leaves[-1][b[part], j] > -1e38).detach()
                dst, src = dst[part], src[part]
                score = leaves[-1][b[part], j]
            score = th.einsum("ed,ed->e", q[dst, j], k[src, j]) * scale + score
            top = th.full((n,), -math.inf, dtype=th.float64, device=DEV).index_reduce(0, dst, score.detach(), "amax")
            top = th.where(top == -math.inf, 0.0, top)
            w = th.exp(score - top[dst])
            sums = th.zeros(n, dtype=th.float64, device=DEV).index_add(0, dst, w)
            some = sums.detach() > 0
            lse[some, per * head + j] = (top + sums.detach().log())[some]
            summed = th.zeros(n, v.size(1), dtype=th.float64, device=DEV).index_add(0, dst, w[:, None] * v[src])
            one = summed / th.where(some, sums, 1.0)[:, None]
            o = one if j == 0 else o - leaves[3] * one
        out[:, head] = o.detach()
        if case["train"]:
            got = th.autograd.grad(o, leaves, g[:, head])
            grads[0][:, per * head: per * (head + 1)], grads[1][:, per * head: per * (head + 1)] = got[0], got[1]
            grads[2][:, head] = got[2]
            if diff:
                grads[3][head] = got[3]
            if case["buckets"]:
                grads[-1][:, per * head: per * (head + 1)] = got[-1]
            del got
        del o, one, w, score, summed, leaves, q, k, v
    return [out] + grads if case["train"] else [out, lse]
