"""Float64 edge-list reference of the attention layers with learned score terms (bias by buckets, differential attention).
TEST CHECKER ONLY: nothing in the product package imports it, and it calls none of the package's kernels.

Every edge is a row of (edges, maps) arrays; plain attention has one map per head, the differential layer two.  A position takes no
part where its bucket is no row of the table or the table's entry is at most -1e38: it is left out of every sum, whatever its rows
hold.  ``bounds`` follows the same sums with the rounding errors that a kernel of given types makes at each step.
"""
import torch as th

F64 = th.float64


def dst_of_edges(indptr):
    ip = indptr.to(th.int64)
    return th.repeat_interleave(th.arange(ip.numel() - 1, device=ip.device), ip[1:] - ip[:-1])


def _rows(t, idx, part):
    """t[idx] in float64 with zeros where no map of the edge takes part (part: (edges, maps))."""
    x = t.index_select(0, idx).to(F64)
    keep = part if part.size(1) == x.size(1) else part.view(part.size(0), x.size(1), -1).any(-1)
    return th.where(keep[:, :, None], x, th.zeros((), dtype=F64, device=x.device))


def relative_buckets(dst, src, num_buckets, max_distance, bidirectional=True, dst_pos=None, src_pos=None):
    """Buckets by counting in whole numbers: distance x of a direction with `count` buckets is in bucket x below half of
    them, else in half + t for the largest t < count - half with x^m * half^t >= max_distance^t * half^m, m = count - half."""
    out = []
    for n, c in zip(dst.tolist(), src.tolist()):
        x = (c if src_pos is None else int(src_pos[c])) - (n if dst_pos is None else int(dst_pos[n]))
        count = num_buckets // 2 if bidirectional else num_buckets
        half, m, d = count // 2, count - count // 2, abs(x) if bidirectional else max(-x, 0)
        b = d
        if d >= half:
            t = 0
            while t + 1 < m and d ** m * half ** (t + 1) >= max_distance ** (t + 1) * half ** m:
                t += 1
            b = half + t
        out.append(b + (count if bidirectional and x > 0 else 0))
    return th.tensor(out, dtype=th.int32)


def attention(dst, src, q, k, v, scale, bucket=None, table=None, lam=None, d_o=None):
    """Everything of one layer, as a dict: o, lse, parts (differential), and with d_o dq, dk, dv, d_table, d_lam; besides, what
    ``bounds`` needs (p, g, dp, ...)."""
    diff, n, maps = lam is not None, q.shape[0], q.shape[1]
    dev = q.device
    part = th.ones(dst.numel(), maps, dtype=th.bool, device=dev)
    bias = th.zeros(dst.numel(), maps, dtype=F64, device=dev)
    if table is not None:
        inside = (bucket >= 0) & (bucket < table.shape[0])
        row = table.to(F64)[bucket.clamp(0, table.shape[0] - 1).long()]
        part = inside[:, None] & ~(row <= -1e38)
        bias = th.where(part, row, th.zeros_like(row))
    qe, ke = _rows(q, dst, part), _rows(k, src, part)
    s = (qe * ke).sum(-1) * scale + bias
    s = th.where(part, s, th.full_like(s, -float("inf")))
    where = dst[:, None].expand(-1, maps)
    top = th.full((n, maps), -float("inf"), dtype=F64, device=dev).scatter_reduce(0, where, s, "amax")
    top0 = th.where(top == -float("inf"), th.zeros_like(top), top)
    w = th.where(part, th.exp(s - top0[dst]), th.zeros_like(s))
    total = th.zeros(n, maps, dtype=F64, device=dev).index_add(0, dst, w)
    p = th.where(part, w / th.where(total == 0, th.ones_like(total), total)[dst], th.zeros_like(w))   # the total may be NaN
    r = dict(dst=dst, src=src, part=part, bias=bias, p=p, qe=qe, ke=ke, lse=th.where(total == 0, top, top0 + total.log()))
    ve = _rows(v, src, part)
    per = ve if not diff else ve.repeat_interleave(2, 1)           # the row of v that a map's probability multiplies
    sums = th.zeros(n, maps, v.shape[2], dtype=F64, device=dev).index_add(0, dst, p[..., None] * per)
    sign = th.ones(maps, dtype=F64, device=dev)
    if diff:
        sign[1::2] = -lam.to(F64)
        r["parts"] = sums.view(n, maps // 2, 2, -1)
    signed = sums * sign[:, None]
    r.update(sums=sums, sign=sign, per=per, o=signed if not diff else signed[:, 0::2] + signed[:, 1::2])
    if d_o is None:
        return r
    ge = _rows(d_o, dst, part)
    gper = ge if not diff else ge.repeat_interleave(2, 1)
    dp = (gper * per).sum(-1)
    d_full = th.nan_to_num(d_o.to(F64)) if not diff else th.nan_to_num(d_o.to(F64)).repeat_interleave(2, 1)
    delta = (d_full * sums).sum(-1)
    g = th.where(part, sign * p * (dp - delta[dst]), th.zeros_like(p))
    wt = sign * p
    wt = wt if not diff else wt[:, 0::2] + wt[:, 1::2]
    r.update(ge=ge, gper=gper, dp=dp, delta=delta, g=g, d_full=d_full)
    r["dq"] = scale * th.zeros(q.shape, dtype=F64, device=dev).index_add(0, dst, g[..., None] * ke)
    r["dk"] = scale * th.zeros(k.shape, dtype=F64, device=dev).index_add(0, src, g[..., None] * qe)
    r["dv"] = th.zeros(v.shape, dtype=F64, device=dev).index_add(0, src, wt[..., None] * ge)
    if diff:
        r["d_lam"] = -delta[:, 1::2].sum(0)
    if table is not None:
        inside = (bucket >= 0) & (bucket < table.shape[0])
        r["d_table"] = th.zeros(table.shape, dtype=F64, device=dev).index_add(0, bucket[inside].long(), g[inside])
    return r


def bounds(r, q, k, v, scale, dtype, bucket=None, table=None, staged=0.0):
    """How far a kernel's outputs may be from ``attention``'s, by first-order error analysis.  Inputs are exact; sums are held
    in `acc` (float32, or float64 for float64 tensors) with unit roundoff a, in any order (a sum of t terms is off by at most a t
    times the sum of magnitudes); stored tensors of `dtype` are off by u of their value; 2^x by 2^-21 in float32 (the hardware's
    2^-22, and its argument), 2^-51 in float64, and below the smallest normal number of `acc` it is zero; `staged`: the unit roundoff
    of the type in which probabilities and score gradients enter the products, 0 where they do not leave the accumulator type; the
    table's gradient then sums score gradients cut to 16 bits of mantissa."""
    acc = th.float64 if dtype == th.float64 else th.float32
    u, a = th.finfo(dtype).eps / 2, th.finfo(acc).eps / 2
    x, tiny = 2.0 ** -51 if acc == th.float64 else 2.0 ** -21, 2 * th.finfo(acc).tiny   # of a weight and of the scaled sum it joins
    dst, src, p, n, d, D = r["dst"], r["src"], r["p"], q.shape[0], q.shape[2], v.shape[2]
    dev, maps, diff = q.device, q.shape[1], "parts" in r
    zeros = lambda *shape: th.zeros(*shape, dtype=F64, device=dev)  # noqa: E731
    deg = th.bincount(dst, minlength=n).to(F64)
    deg_t = th.bincount(src, minlength=k.shape[0]).to(F64)
    # scores: d products and their sum, the scale, the change of base and the bias
    es = a * (d + 8) * (scale * (r["qe"].abs() * r["ke"].abs()).sum(-1) + r["bias"].abs()) + a
    row_es = zeros(n, maps).scatter_reduce(0, dst[:, None].expand(-1, maps), es, "amax")
    # the running maximum, rescaled sums and their total; in the backward the stored lse
    lse = th.where(th.isfinite(r["lse"]), r["lse"].abs(), zeros(n, maps))
    e_lse = row_es + a * (deg[:, None] + 8) + x + 4 * a * lse
    ep = es + e_lse[dst] + 2 * x + 4 * a
    out = {"lse": e_lse}
    e_sum = zeros(n, maps, D).index_add(0, dst, (p * (ep + staged) + tiny)[..., None] * r["per"].abs())
    e_sum += a * (deg[:, None, None] + 4) * zeros(n, maps, D).index_add(0, dst, p[..., None] * r["per"].abs())
    signed = e_sum * r["sign"].abs()[:, None] + 2 * a * (r["sums"] * r["sign"][:, None]).abs()
    out["o"] = (signed if not diff else signed[:, 0::2] + signed[:, 1::2]) + u * r["o"].abs()
    e_kept = e_sum + 2 * a * r["sums"].abs()        # what the backward reads of the sums: unrounded
    if diff:
        out["parts"] = e_kept.view(r["parts"].shape)
    if "dp" not in r:
        return out
    e_delta = (r["d_full"].abs() * e_kept).sum(-1) + a * (D + 4) * (r["d_full"].abs() * r["sums"].abs()).sum(-1)
    e_dp = a * (D + 4) * (r["gper"].abs() * r["per"].abs()).sum(-1)
    mag = r["sign"].abs()
    eg = r["g"].abs() * (ep + 6 * a) + mag * p * (e_dp + e_delta[dst]) + tiny * (1 + mag * (r["dp"] - r["delta"][dst]).abs())
    gs, es_g = r["g"].abs(), eg + staged * r["g"].abs()
    add = lambda shape, idx, t: zeros(*shape).index_add(0, idx, t)  # noqa: E731
    out["dq"] = scale * (add(q.shape, dst, es_g[..., None] * r["ke"].abs())
                         + a * (deg[:, None, None] + 6) * add(q.shape, dst, gs[..., None] * r["ke"].abs())) + u * r["dq"].abs()
    out["dk"] = scale * (add(k.shape, src, es_g[..., None] * r["qe"].abs())
                         + a * (deg_t[:, None, None] + 6) * add(k.shape, src, gs[..., None] * r["qe"].abs())) + u * r["dk"].abs()
    ew, w = mag * (p * (ep + 4 * a + staged) + tiny), mag * p
    if diff:
        ew, w = ew[:, 0::2] + ew[:, 1::2], w[:, 0::2] + w[:, 1::2]
    out["dv"] = add(v.shape, src, ew[..., None] * r["ge"].abs()) + a * (deg_t[:, None, None] + 4) * \
        add(v.shape, src, w[..., None] * r["ge"].abs()) + u * r["dv"].abs()
    if diff:
        out["d_lam"] = e_delta[:, 1::2].sum(0) + a * n * r["delta"][:, 1::2].abs().sum(0) + u * r["d_lam"].abs()
    if table is not None:
        inside = (bucket >= 0) & (bucket < table.shape[0])
        b = bucket[inside].long()
        count = th.bincount(b, minlength=table.shape[0]).to(F64)[:, None]
        cut = 2.0 ** -15 if staged else 0.0
        out["d_table"] = add(table.shape, b, (eg + cut * gs)[inside]) + a * (count + 8) * add(table.shape, b, gs[inside]) \
            + u * r["d_table"].abs()
    return out


def assert_within(got, want, bound, what):
    """Every element of `got` within its bound of `want`; infinities have to be where they are."""
    got, want, bound = got.detach().to("cpu", F64), want.to("cpu"), bound.to("cpu")
    assert got.shape == want.shape, "%s: shape %s, not %s" % (what, tuple(got.shape), tuple(want.shape))
    fine = th.isfinite(want)
    assert bool((got[~fine] == want[~fine]).all()), "%s: other values where there is no finite one" % what
    over = ((got - want).abs() - bound)[fine]
    assert not bool(th.isnan(got[fine]).any()), "%s: NaN" % what
    if over.numel() and bool((over > 0).any()):
        i = int(over.argmax())
        raise AssertionError("%s: %d of %d elements out of bounds; worst |%g - %g| > %g" % (
            what, int((over > 0).sum()), over.numel(), got[fine][i], want[fine][i], bound[fine][i]))
