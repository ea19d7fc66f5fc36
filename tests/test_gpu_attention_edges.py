"""Attention at its edges: workgroups without work, rows of very different size within a head, positions of a batch's own,
streams shared between threads, graphs and growing workspaces."""
import numpy as np
import pytest

from oracle import transformer as T
from test_gpu_attention import K, U, arguments, case, close, dev, fetch, make, place, tolerances      # noqa: F401

pytestmark = pytest.mark.gpu


def test_bias_gradient_where_workgroups_have_nothing_to_do(K):
    # tiles behind the lengths, sequences of length 0, causal tiles that see nothing, pieces of a cut axis: what a workgroup
    # without a key leaves of the table's gradient is 0, whatever LDS held before it
    rs = np.random.RandomState(8)
    dirty = [dev(1e6 * rs.randn(8, 4, 256, 64)) for _ in range(4)]
    c = case(24, 4, 260, 300, 64, buckets=32, q_lengths=[0, 260, 5] * 8, k_lengths=[300, 0, 7] * 8)
    (q, k, v, table, go), att = make(c)
    for more in (dict(), dict(causal=True, q_offset=-200)):
        att = T.Attention(q, k, v, table, q_lengths=c["q_lengths"], k_lengths=c["k_lengths"], **more)
        want, tol = att.pullback(go)[3], tolerances(att, go)["gtable"]
        args = [dev(a) for a in (q, k, v, table)]
        more = dict(more, **{n: dev(c[n], np.int32) for n in ("q_lengths", "k_lengths")})
        o, lse = K.rel_attention_fwd(*args, **more)
        first = None
        for _ in range(8):
            o1, lse1 = K.rel_attention_fwd(*dirty[:3], args[3])
            K.rel_attention_bwd(*dirty[:3], args[3], o1, lse1, dirty[3])
            got = K.rel_attention_bwd(*args, o, lse, dev(go), **more)[3].get()
            close(got, want, tol, "gtable")
            first = got if first is None else first
            assert np.array_equal(got, first)
    none = dev(np.zeros((24, 4, 0, 64)))
    o, lse = K.rel_attention_fwd(args[0], none, none, args[3])
    gtable = K.rel_attention_bwd(args[0], none, none, args[3], o, lse, dev(go))[3]
    assert not gtable.get().any()


@pytest.mark.parametrize("p", [0.0, 0.25])
@pytest.mark.parametrize("Tq,Tk", [(40, 70), (150, 333)])
def test_gradients_of_rows_with_nothing_but_the_lowest_bias(K, Tq, Tk, p):
    # such a row weighs its keys equally; head 0 has rows of all kinds (keys before the query have the lowest bias, keys after it
    # -inf or an ordinary one), head 1 nothing else
    lowest = np.float32(-3.4028235e38)
    c = case(2, 2, Tq, Tk, 32, buckets=8, max_distance=16, p=p, k_lengths=[Tk, Tk - 37], q_lengths=[Tq, Tq - 5])
    (q, k, v, table, go), _ = make(c)
    table[:4, 0] = lowest
    table[4:7, 0] = -np.inf
    table[:, 1] = lowest
    keep = T.attention_keep(2, 2, Tq, Tk, p, 31337, 2) if p else 1.0
    # the same in float64: scores beside a bias that is 0 where it is the lowest, in rows that have no other key
    att = T.Attention(q, k, v, table, max_distance=16, q_lengths=c["q_lengths"], k_lengths=c["k_lengths"], keep=keep if p else None)
    bias = table[att.bucket].transpose(2, 0, 1)[None]
    seen = (np.arange(Tk)[None, :] < np.array(c["k_lengths"])[:, None])[:, None, None, :] & att.q_seen & (bias > -np.inf)
    alone = ~(seen & (bias > lowest)).any(-1, keepdims=True)
    assert alone[:, 0].any() and not alone[:, 0].all() and alone[:, 1].all()
    n = seen.sum(-1, keepdims=True)
    att.prob = np.where(alone, seen / np.maximum(n, 1), att.prob)
    att.o = np.einsum("bhij,bhjd->bhid", att.prob * att.keep, att.vm)
    att.lse = np.where((alone & (n > 0))[..., 0], 0.0, att.lse)      # (for the tolerances: these rows' probabilities are exact)
    tol = tolerances(att, go)
    more = arguments(c)
    o, lse = K.rel_attention_fwd(dev(q), dev(k), dev(v), dev(table), **more)
    close(o.get(), att.o, tol["o"], "o")
    assert np.array_equal(lse.get() == lowest, (alone & (n > 0))[..., 0])
    got = K.rel_attention_bwd(dev(q), dev(k), dev(v), dev(table), o, lse, dev(go), **more)
    for name, a, want in zip(("gq", "gk", "gv", "gtable"), got, att.pullback(go)):
        close(a.get(), want, tol[name], name)


@pytest.mark.parametrize("value", [-3e3, 7e5, -1.1e6, 2.9e6, -2.9e6, 1e8, -1e20])
def test_results_stay_within_the_values_whatever_the_bias(K, value):
    # scores whose whole digits leave no room for others: every probability is between 0 and 1, and they add up to 1
    c = case(1, 2, 70, 300, 64, buckets=8, max_distance=16)
    (q, k, v, table, go), _ = make(c)
    table[:, 1] = value * (1 + np.arange(8) * 2.0 ** -20)
    v = np.abs(v) + 1
    o, lse = K.rel_attention_fwd(dev(q), dev(k), dev(v), dev(table), max_distance=16)
    got = o.get()
    assert np.isfinite(got).all() and np.all(got <= v.max(2, keepdims=True) * (1 + 1e-5)) and np.all(got >= v.min(2, keepdims=True) * (1 - 1e-5))
    assert np.allclose(lse.get()[:, 1], value, rtol=1e-5, atol=20)


@pytest.mark.parametrize("value", [-1e7, -1e9, -1e30, -2e38, 1e9])
def test_rows_whose_lse_has_no_digits_contribute_to_no_gradient(K, value):
    # head 1 has such rows only, head 0 none
    c = case(1, 2, 70, 90, 64, buckets=8, max_distance=16)
    (q, k, v, table, go), _ = make(c)
    table[:, 1] = value
    o, lse = K.rel_attention_fwd(dev(q), dev(k), dev(v), dev(table), max_distance=16)
    assert np.isfinite(o.get()).all() and np.allclose(lse.get()[:, 1], value, rtol=1e-6, atol=0)
    got = K.rel_attention_bwd(dev(q), dev(k), dev(v), dev(table), o, lse, dev(go), max_distance=16)
    for a in got[:3]:
        assert not a.get()[:, 1].any()
    assert not got[3].get()[:, 1].any()
    table[:, 1] = 0
    att = T.Attention(q, k, v, table, max_distance=16)
    tol = tolerances(att, go)
    for name, a, want in zip(("gq", "gk", "gv"), got, att.pullback(go)):
        close(a.get()[:, 0], want[:, 0], tol[name][:, 0], name)


# ---------------------------------------------------------------- sequences at positions of their own

def by_sequence(c, arrays, offsets, go=None, keep=None):
    """Each sequence by itself in float64: (o, lse, tolerances of both, gradients, their tolerances)."""
    q, k, v, table = arrays
    parts = []
    for b, off in enumerate(offsets):
        more = {n: c[n] for n in ("causal", "bidirectional", "max_distance", "scale") if n in c}
        for n in ("q_lengths", "k_lengths"):
            if n in c:
                more[n] = c[n][b:b + 1]
        att = T.Attention(q[b:b + 1], k[b:b + 1], v[b:b + 1], table, q_offset=int(off), keep=None if keep is None else keep[b:b + 1], **more)
        tol = tolerances(att, None if go is None else go[b:b + 1])
        parts.append((att.o, att.lse, tol["o"], tol["lse"]) + (() if go is None else att.pullback(go[b:b + 1])[:3 + (table is not None)]
                                                               + tuple(tol[n] for n in ("gq", "gk", "gv", "gtable")[:3 + (table is not None)])))
    n = 4 + (0 if go is None else 2 * (3 + (table is not None)))
    out = [np.concatenate([p[i] for p in parts]) if not (go is not None and table is not None and i in (7, 11)) else sum(p[i] for p in parts)
           for i in range(n)]
    return out


OFFSETS = [
    (case(4, 2, 1, 500, 64, buckets=32, causal=True, k_lengths=[500, 1, 133, 0]), None),                 # one token each, sequences of different lengths
    (case(3, 2, 5, 1300, 40, buckets=16, causal=True, k_lengths=[1300, 700, 6]), None),
    (case(3, 2, 40, 700, 64, buckets=32, causal=True, k_lengths=[700, 333, 40], layout="bthd"), None),      # chunks of a prompt
    (case(2, 2, 150, 400, 128, buckets=32, causal=True, k_lengths=[400, 151], q_lengths=[150, 100]), None),
    (case(3, 1, 33, 90, 32, buckets=8, max_distance=9, p=0.2), [0, 57, -1000]),                            # positions without a mask
    (case(2, 2, 20, 60, 24, causal=True), [-5, 2 ** 31 - 1]),                                              # no bias; clamped
]


@pytest.mark.parametrize("c,offsets", OFFSETS, ids=["%dx%dx%dx%d" % (c["B"], c["H"], c["Tq"], c["Tk"]) for c, _ in OFFSETS])
def test_a_position_for_each_sequence(K, c, offsets):
    offsets = [n - c["Tq"] for n in c["k_lengths"]] if offsets is None else offsets
    (q, k, v, table, go), _ = make(dict(c, q_offset=0))
    keep = T.attention_keep(c["B"], c["H"], c["Tq"], c["Tk"], c["p"], 31337, 2) if c.get("p") else None
    want = by_sequence(c, (q, k, v, table), np.clip(offsets, -2 ** 20, 2 ** 20), go, keep)
    more = dict(arguments(c), q_offset=dev(np.array(offsets), np.int32))
    dt = None if table is None else dev(table)
    ins = [place(a, c) for a in (q, k, v)]
    o, lse = K.rel_attention_fwd(*ins, dt, **more)
    close(fetch(o, c), want[0], want[2], "o")
    close(lse.get(), want[1], want[3], "lse")
    got = K.rel_attention_bwd(*ins, dt, o, lse, place(go, c), **more)
    n = 3 + (table is not None)
    for name, a, w, t in zip(("gq", "gk", "gv", "gtable"), got, want[4:4 + n], want[4 + n:]):
        close(a.get() if name == "gtable" else fetch(a, c), w, t, name)
    # one number for all is the same as an array of it
    if len(set(offsets)) == 1 or c["Tk"] == 700:
        off = c["Tk"] - c["Tq"]
        more = arguments(c)
        a = K.rel_attention_fwd(*ins, dt, **dict(more, q_offset=off))
        b = K.rel_attention_fwd(*ins, dt, **dict(more, q_offset=dev(np.full(c["B"], off), np.int32)))
        assert all(np.array_equal(x.get(), y.get()) for x, y in zip(a, b))


@pytest.mark.parametrize("use_graph", [False, True])
def test_one_compiled_function_steps_through_a_cache(K, use_graph):
    # a new token of each sequence a step; lengths and positions are arguments
    import cgt_amd as cgt
    from cgt_amd import nn
    rs = np.random.RandomState(21)
    B, H, room, D = 3, 2, 300, 32
    c = case(B, H, 1, room, D, causal=True)
    k, v = (rs.randn(B, H, room, D).astype(np.float32) for _ in range(2))
    table = rs.randn(16, H).astype(np.float32)
    nq, nk, nv, lengths, offsets = (cgt.constant(a) for a in (rs.randn(B, H, 1, D).astype(np.float32), k, v, dev(np.ones(B), np.int32), dev(np.zeros(B), np.int32)))
    o = nn.relative_attention(nq, nk, nv, cgt.constant(table), causal=True, q_offset=offsets, k_lengths=lengths)
    f = cgt.function([nq, nk, nv, lengths, offsets], [o], use_graph=use_graph)
    for step in range(4):
        n = np.array([40 + step, 1 + step, 297 + step], np.int32)
        q = rs.randn(B, H, 1, D).astype(np.float32)
        want = by_sequence(dict(c, k_lengths=list(n)), (q, k, v, table), n - 1)
        close(f(q, k, v, n, (n - 1).astype(np.int32))[0], want[0], want[2], "step %d" % step)
    # whole numbers of any kind are one number
    a = nn.relative_attention(nq, nk, nv, causal=True, q_offset=7)
    for off in (np.int32(7), np.array(7), 7.0):
        assert np.array_equal(nn.relative_attention(nq, nk, nv, causal=True, q_offset=off).get(), a.get())
    # gradients through the op with such an input
    go = rs.randn(B, H, 1, D).astype(np.float32)
    off = [7, 0, 299]
    o = nn.relative_attention(nq, nk, nv, table, causal=True, q_offset=off)
    grads = cgt.grad(o, [nq, nk, nv], goutput=go)
    want = by_sequence(c, (nq.get(), k, v, table), off, go)
    for name, g, w, t in zip(("gq", "gk", "gv"), grads, want[4:7], want[8:11]):
        close(g.get(), w, t, name)
    with pytest.raises(ValueError):
        nn.relative_attention(nq, nk, nv, q_offset=[1, 2])
    with pytest.raises(TypeError):
        nn.relative_attention(nq, nk, nv, q_offset=np.zeros(B, np.float32))


def test_compiled_functions_follow_the_shapes_they_are_given(K):
    import cgt_amd as cgt
    from cgt_amd import nn
    rs = np.random.RandomState(22)
    draw = lambda *s: rs.randn(*s).astype(np.float32)      # noqa: E731
    nq, nk, nv, ngo = (cgt.constant(draw(1, 2, t, 16)) for t in (7, 20, 20, 7))
    o = nn.relative_attention(nq, nk, nv)
    f = cgt.function([nq, nk, nv, ngo], [o] + cgt.grad(cgt.sum(o * ngo), [nq, nk, nv]))
    for B, Tq, Tk, D in ((1, 7, 20, 16), (2, 5, 33, 64), (1, 9, 11, 20)):      # the scale is that of the head width at hand
        q, k, v, go = draw(B, 2, Tq, D), draw(B, 2, Tk, D), draw(B, 2, Tk, D), draw(B, 2, Tq, D)
        att = T.Attention(q, k, v)
        tol = tolerances(att, go)
        for name, a, want in zip(("o", "gq", "gk", "gv"), f(q, k, v, go), (att.o,) + att.pullback(go)[:3]):
            close(a, want, tol[name], name)
    # an offset computed from extents is a constant of the op: other shapes are refused, not answered with the old offset
    o = nn.relative_attention(nq, nk, nv, causal=True, q_offset=nk.shape[2] - nq.shape[2])
    f = cgt.function([nq, nk, nv], [o])
    q, k, v = nq.get(), nk.get(), nv.get()
    att = T.Attention(q, k, v, causal=True, q_offset=13)
    close(f(q, k, v)[0], att.o, tolerances(att)["o"], "o")
    with pytest.raises(ValueError, match="compiled for"):
        f(draw(1, 2, 7, 16), draw(1, 2, 30, 16), draw(1, 2, 30, 16))


# ---------------------------------------------------------------- rows of very different size within one head

def plain32(q, k, v, table, go, causal=False, max_distance=128, bidirectional=None, keep=1.0):
    """The composition of elementary operations in float32: (o, gq, gk, gv)."""
    f = np.float32
    Tq, Tk = q.shape[2], k.shape[2]
    scale = f(q.shape[3] ** -0.5)
    i, j = np.arange(Tq)[:, None], np.arange(Tk)[None, :]
    s = np.matmul(q * scale, k.transpose(0, 1, 3, 2))
    if table is not None:
        rel = np.arange(1 - Tq, Tk)
        by_rel = np.array([T.bucket(int(r), table.shape[0], max_distance, not causal if bidirectional is None else bidirectional) for r in rel])
        s = s + table.T[:, by_rel][:, j - i + Tq - 1]
    if causal:
        s = np.where(j <= i, s, f(-np.inf))
    p = np.exp(s - s.max(-1, keepdims=True))
    p /= p.sum(-1, keepdims=True)
    w = (p * keep).astype(f)
    o = np.matmul(w, v)
    gp = np.matmul(go, v.transpose(0, 1, 3, 2)) * keep
    ds = (p * (gp - (go * o).sum(-1, keepdims=True))).astype(f)
    return o, np.matmul(ds, k) * scale, np.matmul(ds.transpose(0, 1, 3, 2), q) * scale, np.matmul(w.transpose(0, 1, 3, 2), go)


def units(att, go):
    """For o, gq, gk and gv: what one rounding in every operation leaves in an element, errors of different operations added as
    a random walk.  Scores are off by a share of their largest products, of the largest score and of lse; that error of p,
    and those of go . v and go . o, go through the sums."""
    sq = np.square
    q, k, v, p, w = att.q, att.k, att.vm, att.prob, att.prob * att.keep
    root = lambda spec, *ops: np.sqrt(np.einsum(spec, *[sq(a) for a in ops]))      # noqa: E731
    s = att.scale * root("bhid,bhjd->bhij", q, k)
    es = U * (np.max(np.where(p > 0, s, 0.0), -1) + 2 * np.max(np.abs(np.where(p > 0, att.scores, 0.0)), -1) + 1)[..., None]     # of a row's scores
    gp = att.keep * np.einsum("bhid,bhjd->bhij", go, v)
    delta = (go * att.o).sum(-1, keepdims=True)
    egp, edelta = U * att.keep * root("bhid,bhjd->bhij", go, v), U * np.sqrt(sq(go * att.o).sum(-1, keepdims=True))
    eo = es * root("bhij,bhjd->bhid", w, v) + (es + U) * np.abs(att.o)
    ds = p * (gp - delta)
    # go . o carries what o is off by; it goes into all of a row's ds alike
    row = edelta + np.sqrt((sq(go * eo)).sum(-1, keepdims=True))
    eds = np.sqrt(sq(ds * es) + sq(p * egp) + sq(p * U * gp))
    gq = att.scale * (root("bhij,bhjd->bhid", eds, k) + row * np.abs(np.einsum("bhij,bhjd->bhid", p, k)) + es * np.abs(np.einsum("bhij,bhjd->bhid", ds, k)))
    gk = att.scale * root("bhij,bhid->bhjd", np.sqrt(sq(eds) + sq(p * row) + sq(ds * es)), q)
    gv = root("bhij,bhid->bhjd", w * (es + U), go)
    return eo, gq + U * np.abs(att.scale * np.einsum("bhij,bhjd->bhid", ds, k)), gk, gv


def rows_close(got, want, plain, unit, name):
    """Each row to float32 accuracy: within 8 times what float32 numpy is off by on that row, or (where it is lucky) a rounding
    in every operation would leave.  The operands of a score have 22 bits, so a product is off by up to 4 U where a
    rounding gives U, and a matrix instruction cuts its sum's last bits where numpy rounds them: 4 times 2."""
    norm = lambda a: np.sqrt((np.asarray(a, np.float64) ** 2).sum(-1))      # noqa: E731
    assert np.isfinite(got).all(), name
    off, allowed = norm(got - want), 8 * np.maximum(norm(plain - want), norm(unit)) + 1e-37
    worst = np.max(off / allowed)
    at = np.unravel_index(np.argmax(off / allowed), off.shape)
    size = np.maximum(norm(want)[at], 1e-300)
    said = "%s, row %s: off by %.3g of it, float32 numpy by %.3g, a rounding an operation %.3g" % (
        name, tuple(map(int, at)), off[at] / size, norm(plain - want)[at] / size, norm(unit)[at] / size)
    print("%.2f" % worst, said)
    assert worst <= 1, said


def spread(rs, n, low):
    """Factors from `low` to 1, one of them 1."""
    f = np.exp(rs.uniform(np.log(low), 0.0, n))
    f[rs.randint(n)] = 1.0
    return f[:, None]


SPREADS = {
    "normal": dict(),
    "small cotangents": dict(go=1e-6),
    "one large cotangent": dict(go=(7, 1e4)),
    "spread values": dict(v=1e-6),
    "one large value": dict(v=(300, 1e2)),
    "a huge value most queries do not see": dict(v=(690, 1e6), causal=True),
    "spread queries": dict(q=1e-4),
    "one large key": dict(k=(300, 30.0)),
    "a huge key most queries do not see": dict(k=(690, 1e4), causal=True),
    "garbage behind the causal horizon": dict(k=(690, 1e20), v=(690, 1e25), causal=True, Tq=600),
    "tiny values and cotangents": dict(scales=(1, 1, 1e-15, 1e-15)),
    "everything spread, dropout": dict(q=1e-3, k=1e-3, v=1e-5, go=1e-5, p=0.2),
    "sharp": dict(scales=(12, 1, 1, 1)),
    "a huge value among the first": dict(v=(3, 1e8), causal=True),
    "a huge key among the first": dict(k=(3, 1e3), causal=True),
    "blocks of values of very different size": dict(v=[1e-25, 1.0, 1e-12, 1e12], go=[1e-10, 1.0]),
    "blocks of keys of very different size": dict(k=[1e-20, 1.0, 1e-6], q=[1.0, 1e-15]),
    "rows of zeros": dict(k="zeros", v="zeros", q="zeros", go="zeros"),
}


@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("name", sorted(SPREADS))
def test_rows_of_any_size_keep_float32_accuracy(K, name, D):
    how = SPREADS[name]
    rs = np.random.RandomState(len(name) + D)
    H, Tq, Tk = 2, how.get("Tq", 700), 700
    arrays = {n: rs.randn(1, H, t, D) for n, t in (("q", Tq), ("k", Tk), ("v", Tk), ("go", Tq))}
    for n, f in zip(("q", "k", "v", "go"), how.get("scales", ())):
        arrays[n] *= f
    for n, a in arrays.items():
        f = how.get(n)
        if isinstance(f, tuple):
            a[:, 1, f[0]] *= f[1]          # the second head; the first stays as it is
        elif isinstance(f, list):          # runs of 96 rows
            a[:, 1] *= np.array(f)[np.arange(a.shape[2]) // 96 % len(f)][:, None]
        elif f == "zeros":                 # single ones, and whole tiles
            a[:, 1] *= spread(rs, a.shape[2], 1e-4)
            a[:, 1, 1::3] = 0.0
            a[:, 1, 64:130] = 0.0
        elif f:
            a[:, 1] *= spread(rs, a.shape[2], f)
    q, k, v, go = (arrays[n].astype(np.float32) for n in ("q", "k", "v", "go"))
    table = (0.5 * rs.randn(32, H)).astype(np.float32)
    causal, p = how.get("causal", False), how.get("p", 0.0)
    keep = T.attention_keep(1, H, Tq, Tk, p, 31337, 2) if p else None
    seen = slice(0, Tq if causal else Tk)      # (keys that no query sees do not count)
    att = T.Attention(q, k[:, :, seen], v[:, :, seen], table, causal=causal, keep=keep)
    att.scores = att.scale * np.matmul(att.q, att.k.transpose(0, 1, 3, 2)) + table.astype(np.float64)[att.bucket].transpose(2, 0, 1)
    plain = plain32(q, k[:, :, seen], v[:, :, seen], table, go, causal, keep=1.0 if keep is None else keep.astype(np.float32))
    more = dict(causal=causal)
    if p:
        more.update(p=p, rng=dev(np.array([31337, 2]), np.int64))
    ins = [dev(a) for a in (q, k, v, table)]
    o, lse = K.rel_attention_fwd(*ins, **more)
    unit = units(att, go.astype(np.float64))
    rows_close(o.get(), att.o, plain[0], unit[0], "o")
    gq, gk, gv, gtable = K.rel_attention_bwd(*ins, o, lse, dev(go), **more)
    want = att.pullback(go)
    for a, w, p32, u, n in zip((gq.get(), gk.get()[:, :, seen], gv.get()[:, :, seen]), want, plain[1:], unit[1:], ("gq", "gk", "gv")):
        rows_close(a, w, p32, u, n)
    # the table's gradient is a sum over all pairs: a random walk of their roundings, and a share of each pair's own error
    ds = att.prob * (np.matmul(go.astype(np.float64), att.v.transpose(0, 1, 3, 2)) * att.keep - (go * att.o).sum(-1, keepdims=True))
    allowed = 64 * U * np.sqrt((ds ** 2).sum((0, 2, 3))) + 8 * U * np.abs(ds).sum((0, 2, 3))
    assert np.all(np.abs(gtable.get() - want[3]).max(0) <= allowed)


@pytest.mark.parametrize("Tq,Tk", [(1, 6000), (5, 6000), (40, 6000), (6000, 40)])
def test_rows_of_any_size_on_long_axes(K, Tq, Tk):
    # cut axes and the sums of their pieces, at float32 accuracy
    rs = np.random.RandomState(Tq)
    H, D = 2, 64
    q, k, v, go = (rs.randn(1, H, t, D) for t in (Tq, Tk, Tk, Tq))
    v[:, 1] *= spread(rs, Tk, 1e-5)
    go[:, 1] *= spread(rs, Tq, 1e-5)
    q, k, v, go = (a.astype(np.float32) for a in (q, k, v, go))
    ins = [dev(a) for a in (q, k, v)]
    o, lse = K.rel_attention_fwd(*ins)
    att = T.Attention(q, k, v)
    att.scores = att.scale * np.matmul(att.q, att.k.transpose(0, 1, 3, 2))
    plain, unit = plain32(q, k, v, None, go), units(att, go.astype(np.float64))
    rows_close(o.get(), att.o, plain[0], unit[0], "o")
    assert np.abs(lse.get() - att.lse).max() <= 16 * U * np.abs(att.lse).max()
    got = K.rel_attention_bwd(*ins, None, o, lse, dev(go))
    for a, w, p32, u, n in zip(got, att.pullback(go), plain[1:], unit[1:], ("gq", "gk", "gv")):
        rows_close(a.get(), w, p32, u, n)
