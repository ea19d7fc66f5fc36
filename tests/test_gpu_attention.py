"""Attention with a relative position bias against the float64 formulas: odd sizes, both layouts, padded batches with
garbage behind the lengths, rows that see nothing, split keys, dropout, gradients, graphs, streams, and the Op API."""
import numpy as np
import pytest

from oracle import transformer as T

pytestmark = pytest.mark.gpu
U = 2.0 ** -24      # half a step of float32


@pytest.fixture(scope="module")
def K():
    from cgt_amd import capi, kernels
    capi.require_gpu()
    return kernels


def dev(a, dtype=np.float32, shift=0):
    from cgt_amd.gpuarray import GpuArray, empty
    a = np.ascontiguousarray(a, dtype)
    if not shift:
        return GpuArray(a.shape, dtype).set(a)
    whole = empty((a.size + shift,), dtype)
    return GpuArray(a.shape, dtype, _buffer=whole._buffer, _offset=shift * a.itemsize).set(a)


def tolerances(att, go=None):
    """What the roundings allow, element by element.  A score is a sum of D products (D + 4 roundings of its absolute
    terms) plus the bias; a probability is off by twice the worst score error of its row, a few roundings of the exponential and its
    argument, and the sum's; a sum over n terms by n roundings of its absolute terms at most."""
    q, k, v = np.abs(att.q), np.abs(att.k), np.abs(np.nan_to_num(att.vm))
    D, Tk, Tq = q.shape[3], k.shape[2], q.shape[2]
    s = att.scale * np.einsum("bhid,bhjd->bhij", q, k)
    seen = att.prob > 0
    es = U * np.max(np.where(seen, (D + 6) * s, 0.0), -1, initial=0.0) + 8 * U * (1 + np.abs(np.where(np.isfinite(att.lse), att.lse, 0.0)))
    rel = (2 * es + (Tk + 16) * U)[..., None]
    w = att.prob * att.keep
    tol = {"o": np.einsum("bhij,bhjd->bhid", w * (rel + (Tk + 4) * U), v) + 1e-37, "lse": es + (Tk + 16) * U + 2 * U * np.abs(np.nan_to_num(att.lse, neginf=0))}
    if go is None:
        return tol
    go = np.abs(np.where(att.q_seen, go, 0.0))
    gp = np.einsum("bhid,bhjd->bhij", go, v) * att.keep
    delta = (go * np.abs(att.o)).sum(-1, keepdims=True)
    edelta = (D + 4) * U * delta + (go * tol["o"]).sum(-1, keepdims=True)
    gs = att.prob * (gp + delta)                                            # absolute terms
    egs = gs * (rel + 4 * U) + att.prob * ((D + 6) * U * gp + edelta)
    tol["gq"] = att.scale * np.einsum("bhij,bhjd->bhid", egs + (Tk + 4) * U * gs, k) + 1e-37
    tol["gk"] = att.scale * np.einsum("bhij,bhid->bhjd", egs + (Tq + 4) * U * gs, q) + 1e-37
    tol["gv"] = np.einsum("bhij,bhid->bhjd", w * (rel + (Tq + 4) * U), go) + 1e-37
    if att.bucket is not None:
        n = gs.shape[0] * Tq * Tk
        total = (egs + min(n, 4000) * U * gs).sum(0)
        tol["gtable"] = np.stack([(total * (att.bucket == b)).sum((1, 2)) for b in range(att.buckets)]) + 1e-37
    return tol


def close(got, want, tol, name=""):
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    inf = ~np.isfinite(want)
    assert np.array_equal(got[inf], want[inf]), name
    got, want, tol = got[~inf], want[~inf], np.broadcast_to(tol, inf.shape)[~inf]
    worst = np.max(np.abs(got - want) - tol, initial=-1.0)
    assert worst <= 0, "%s: off by %g where %g is allowed" % (name, np.max(np.abs(got - want)), np.max(tol))


def case(B, H, Tq, Tk, D, **kw):
    return dict(kw, B=B, H=H, Tq=Tq, Tk=Tk, D=D)


CASES = [
    case(1, 1, 1, 1, 1, buckets=2, causal=True, max_distance=2),
    case(2, 3, 5, 7, 4, buckets=8, max_distance=5),
    case(1, 2, 33, 65, 20, buckets=32, causal=True, q_offset=32),
    case(2, 2, 128, 128, 64, buckets=32, layout="bthd"),
    case(1, 2, 129, 257, 64, buckets=32, causal=True, q_offset=128),
    case(2, 2, 40, 300, 63, buckets=16, shift=1),
    case(1, 1, 300, 40, 128, buckets=32),
    case(1, 2, 31, 32, 32, buckets=8, causal=True, bidirectional=True, max_distance=9),
    case(1, 3, 100, 100, 96, buckets=64, max_distance=200, layout="bthd", shift=1),
    case(3, 2, 70, 70, 64, buckets=32, k_lengths=[70, 33, 0], q_lengths=[70, 33, 0]),
    case(3, 2, 70, 90, 33, buckets=32, k_lengths=[1, 64, 95], q_lengths=[-3, 32, 70], layout="bthd"),
    case(2, 2, 66, 50, 40, buckets=8, causal=True, q_offset=-20),                       # the first queries see nothing
    case(1, 2, 200, 200, 80, causal=True),                                              # no bias
    case(2, 1, 97, 161, 64, buckets=256, max_distance=1024, bidirectional=True),
    case(1, 1, 600, 600, 16, buckets=32, max_distance=300, causal=True),
    case(1, 2, 45, 83, 64, buckets=32, scale=1.0),
    case(2, 3, 37, 61, 24, buckets=8, p=0.3, channel=5),
    case(1, 2, 130, 130, 64, buckets=32, p=0.1, causal=True, k_lengths=[101], layout="bthd"),
    case(1, 2, 64, 47, 128, buckets=32, p=0.5),
    case(2, 2, 3, 2000, 64, buckets=32, causal=True, q_offset=1997),                    # few queries: the keys are cut
    case(2, 1, 1, 5000, 40, buckets=32, causal=True, q_offset=4999, k_lengths=[5000, 4100]),
    case(1, 2, 130, 700, 128, buckets=32, k_lengths=[5]),
    case(1, 1, 2, 900, 128),
    case(2, 2, 4, 1100, 96, buckets=16, causal=True, q_offset=1096, p=0.2, layout="bthd"),
    case(1, 1, 5, 0, 8, buckets=8),
]
IDS = ["%dx%dx%dx%dx%d-%d" % (c["B"], c["H"], c["Tq"], c["Tk"], c["D"], n) for n, c in enumerate(CASES)]


def make(c, seed=0):
    rs = np.random.RandomState(seed + c["Tq"] * 31 + c["Tk"])
    B, H, Tq, Tk, D = (c[n] for n in ("B", "H", "Tq", "Tk", "D"))
    q, go = rs.randn(B, H, Tq, D).astype(np.float32), rs.randn(B, H, Tq, D).astype(np.float32)
    k, v = rs.randn(B, H, Tk, D).astype(np.float32), rs.randn(B, H, Tk, D).astype(np.float32)
    table = rs.randn(c["buckets"], H).astype(np.float32) if "buckets" in c else None
    keep = T.attention_keep(B, H, Tq, Tk, c["p"], 31337, 2, c.get("channel", 0)) if c.get("p") else None
    more = {n: c[n] for n in ("scale", "causal", "bidirectional", "max_distance", "q_offset", "q_lengths", "k_lengths") if n in c}
    att = T.Attention(q, k, v, table, keep=keep, **more)
    return (q, k, v, table, go), att


def arguments(c):
    more = {n: c[n] for n in ("scale", "causal", "bidirectional", "max_distance", "q_offset", "p", "channel", "layout") if n in c}
    for n in ("q_lengths", "k_lengths"):
        if n in c:
            more[n] = dev(c[n], np.int32)
    if c.get("p"):
        more["rng"] = dev(np.array([31337, 2]), np.int64)
    return more


def place(a, c):
    return dev(a if c.get("layout") != "bthd" else a.transpose(0, 2, 1, 3), shift=c.get("shift", 0))


def fetch(a, c):
    return a.get() if c.get("layout") != "bthd" else a.get().transpose(0, 2, 1, 3)


def spoil(a, lengths, T_):
    """NaN behind the lengths: nothing there may be read."""
    if lengths is not None:
        a = a.copy()
        for b, n in enumerate(np.clip(lengths, 0, T_)):
            a[b, :, n:] = np.nan
    return a


@pytest.mark.parametrize("c", CASES, ids=IDS)
def test_attention(K, c):
    (q, k, v, table, go), att = make(c)
    tol = tolerances(att, go)
    dq, dgo = (place(spoil(a, c.get("q_lengths"), c["Tq"]), c) for a in (q, go))
    dk, dv = (place(spoil(a, c.get("k_lengths"), c["Tk"]), c) for a in (k, v))
    dt = None if table is None else dev(table)
    more = arguments(c)
    o, lse = K.rel_attention_fwd(dq, dk, dv, dt, **more)
    close(fetch(o, c), att.o, tol["o"], "o")
    close(lse.get(), att.lse, tol["lse"], "lse")
    got = K.rel_attention_bwd(dq, dk, dv, dt, o, lse, dgo, **more)
    for name, a, want in zip(("gq", "gk", "gv"), got, att.pullback(go)):
        close(fetch(a, c), want, tol[name], name)
    if table is not None:
        close(got[3].get(), att.pullback(go)[3], tol["gtable"], "gtable")
    else:
        assert got[3] is None
    # same input, same bits, into results that held something else
    for r in [o, lse] + [g for g in got if g is not None]:
        r_bits = r.get()
        r.keep = r_bits
    again = K.rel_attention_fwd(dq, dk, dv, dt, **more)
    for a, b in zip(again, (o, lse)):
        assert np.array_equal(a.get(), b.keep)
    outs = [dev(np.full(g.shape, 7.0)) for g in got if g is not None]
    again = K.rel_attention_bwd(dq, dk, dv, dt, o, lse, dgo, out=outs, **more)
    for a, b in zip(again, got):
        assert a is b or np.array_equal(a.get(), b.keep)


def test_gradients_against_differences(K):
    # the kernels' own forward, differenced: o is rounded to float32, so a step of 2^-6 leaves about U * |o| * n / 2^-6
    # of noise in a sum of n terms, and the third derivative about 2^-12
    c = case(1, 2, 20, 36, 16, buckets=8, causal=True, q_offset=16, max_distance=20, p=0.2)
    (q, k, v, table, go), att = make(c)
    more = arguments(c)
    base = [q, k, v, table]
    o, lse = K.rel_attention_fwd(*[dev(a) for a in base], **more)
    grads = K.rel_attention_bwd(*[dev(a) for a in base], o, lse, dev(go), **more)
    rs = np.random.RandomState(9)
    for n in range(4):
        d = rs.randn(*base[n].shape)
        d /= np.linalg.norm(d)
        h = 2.0 ** -6
        ends = []
        for sign in (1, -1):
            moved = [a if m != n else (a + sign * h * d).astype(np.float32) for m, a in enumerate(base)]
            ends.append((K.rel_attention_fwd(*[dev(a) for a in moved], **more)[0].get().astype(np.float64) * go).sum())
        want = (grads[n].get() * d).sum()
        assert abs((ends[0] - ends[1]) / (2 * h) - want) <= 2e-3 * (1 + np.linalg.norm(grads[n].get()))


@pytest.mark.parametrize("value", [-np.inf, -3.4028235e38])
def test_bias_of_the_lowest_value(K, value):
    # a bucket that is switched off: -inf leaves its keys out, the lowest float loses against any other key
    c = case(1, 2, 40, 70, 32, buckets=8, max_distance=16)
    (q, k, v, table, go), _ = make(c)
    table[5:, 0] = value
    table[:, 1] = value          # a whole head: no key at all (-inf), or all of them equally
    att = T.Attention(q, k, v, table, max_distance=16)
    tol = tolerances(att, go)
    o, lse = K.rel_attention_fwd(dev(q), dev(k), dev(v), dev(table), max_distance=16)
    if value == -np.inf:
        assert not o.get()[:, 1].any() and np.all(lse.get()[:, 1] == -np.inf)
        close(o.get(), att.o, tol["o"], "o")
        got = K.rel_attention_bwd(dev(q), dev(k), dev(v), dev(table), o, lse, dev(go), max_distance=16)
        for name, a, want in zip(("gq", "gk", "gv", "gtable"), got, att.pullback(go)):
            close(a.get(), want, tol[name], name)
    else:
        close(o.get()[:, 0], att.o[:, 0], tol["o"][:, 0], "o")
        # next to 3.4e38 the scores vanish: every key weighs the same
        close(o.get()[:, 1], np.broadcast_to(v[:, 1].mean(1, dtype=np.float64)[:, None], att.o[:, 1].shape),
              np.full(att.o[:, 1].shape, 200 * U * np.abs(v).max()), "o")


def test_large_scores(K):
    # scores of some hundreds: the running maximum moves, and nothing overflows
    c = case(1, 1, 64, 400, 64, buckets=32)
    (q, k, v, table, go), _ = make(c)
    q = q * 30
    att = T.Attention(q, k, v, table)
    tol = tolerances(att, go)
    o, lse = K.rel_attention_fwd(dev(q), dev(k), dev(v), dev(table))
    close(o.get(), att.o, tol["o"], "o")
    close(lse.get(), att.lse, tol["lse"], "lse")


MORE = [
    case(2, 2, 5, 700, 64, buckets=32, causal=True, q_offset=695, k_lengths=[700, 133]),      # up to eight queries: vector units
    case(1, 3, 8, 1500, 128, buckets=16, layout="bthd", q_lengths=[6]),
    case(2, 1, 7, 90, 33, buckets=8, shift=1),
    case(1, 2, 8, 8, 96, causal=True),
    case(1, 1, 2, 300, 20, buckets=8),                                                     # two pieces: a team a row
    case(1, 2, 9, 1700, 64, buckets=32, causal=True, q_offset=1691),                        # nine: matrix cores, many pieces
    case(1, 1, 200, 1100, 64, buckets=32, k_lengths=[1050]),                               # few workgroups: short runs
    case(1, 2, 300, 300, 128, buckets=32, causal=True, p=0.2),
]


@pytest.mark.parametrize("c", MORE, ids=["%dx%dx%dx%dx%d-%d" % (c["B"], c["H"], c["Tq"], c["Tk"], c["D"], n) for n, c in enumerate(MORE)])
def test_attention_with_cut_keys(K, c):
    test_attention(K, c)


@pytest.mark.parametrize("sq,sk,sv,sg", [(1e-15, 1e15, 1, 1), (1e12, 1e-12, 1e-20, 1e15), (1, 1, 1e15, 1e-25), (1, 1, 1, 1e-25), (1, 1, 1e-12, 1e20)])
@pytest.mark.parametrize("Tq", [3, 70])
def test_heads_of_any_magnitude(K, Tq, sq, sk, sv, sg):
    # each array by a factor of its own: a power of two brings every head to the same range; squares leave float's
    c = case(1, 2, Tq, 130, 64, buckets=32)
    (q, k, v, table, go), _ = make(c)
    q, k, v, go = ((a * f).astype(np.float32) for a, f in ((q, sq), (k, sk), (v, sv), (go, sg)))
    att = T.Attention(q, k, v, table)
    tol = tolerances(att, go)
    o, lse = K.rel_attention_fwd(dev(q), dev(k), dev(v), dev(table))
    close(o.get(), att.o, tol["o"], "o")
    close(lse.get(), att.lse, tol["lse"], "lse")
    got = K.rel_attention_bwd(dev(q), dev(k), dev(v), dev(table), o, lse, dev(go))
    for name, a, want in zip(("gq", "gk", "gv", "gtable"), got, att.pullback(go)):
        close(a.get(), want, tol[name], name)


def test_values_that_are_no_numbers_stay_with_their_row_and_head(K):
    rs = np.random.RandomState(3)
    q, k, v = (rs.randn(2, 2, 50, 32).astype(np.float32) for _ in range(3))
    q[0, 1, 7, 3] = np.nan
    q[1, 0, 9, 0] = np.inf
    o, lse = K.rel_attention_fwd(dev(q), dev(k), dev(v))
    bad = np.zeros((2, 2, 50), bool)
    bad[0, 1, 7] = bad[1, 0, 9] = True
    assert np.isnan(o.get()[bad]).all() and np.isfinite(o.get()[~bad]).all()
    with np.errstate(invalid="ignore"):
        att = T.Attention(np.where(bad[..., None], 0, q), k, v)
    close(o.get()[~bad], att.o[~bad], tolerances(att)["o"][~bad], "o")


def test_no_queries_no_batch(K):
    from cgt_amd.gpuarray import empty
    table = dev(np.ones((8, 2)))
    q, k = dev(np.zeros((1, 2, 0, 8))), dev(np.ones((1, 2, 5, 8)))
    o, lse = K.rel_attention_fwd(q, k, k, table)
    assert o.shape == q.shape and lse.shape == (1, 2, 0)
    outs = [empty(q.shape), dev(np.ones((1, 2, 5, 8))), dev(np.ones((1, 2, 5, 8))), dev(np.ones((8, 2)))]
    K.rel_attention_bwd(q, k, k, table, o, lse, q, out=outs)
    assert not any(a.get().any() for a in outs[1:])
    none = dev(np.zeros((0, 2, 3, 8)))
    outs = [empty(none.shape), empty(none.shape), empty(none.shape), dev(np.ones((8, 2)))]
    K.rel_attention_bwd(none, none, none, table, none, empty((0, 2, 3)), none, out=outs)
    assert not outs[3].get().any()


def test_graphs_on_two_streams_replayed_with_new_inputs(K):
    from cgt_amd import capi
    from cgt_amd.gpuarray import empty
    c = case(2, 2, 3, 900, 64, buckets=32, causal=True, q_offset=897, p=0.2)
    more = arguments(c)
    (q, k, v, table, go), _ = make(c)
    ins = [dev(a) for a in (q, k, v, table, go)]

    def outs():
        return [empty(ins[0].shape), empty(ins[0].shape[:3])], [empty(a.shape) for a in ins[:4]]

    def step(o, stream):
        K.rel_attention_fwd(*ins[:4], out=o[0], stream=stream, **more)
        K.rel_attention_bwd(*ins[:4], o[0][0], o[0][1], ins[4], out=o[1], stream=stream, **more)
    streams, held, graphs = [capi.Stream(), capi.Stream()], [outs(), outs()], []
    for s, o in zip(streams, held):
        step(o, s.handle)
        s.synchronize()
        graphs.append(capi.Graph.capture(s, lambda: step(o, s.handle)))
    eager = outs()
    for n in range(4):
        more["rng"].set(np.array([31337, n], np.int64))
        ins[0].set(make(c, seed=n)[0][0])
        for g in graphs:
            g.launch()
        for s in streams:
            s.synchronize()
        step(eager, None)
        capi.synchronize()
        for o in held:
            assert all(np.array_equal(a.get(), b.get()) for a, b in zip(o[0] + o[1], eager[0] + eager[1])), "replay %d" % n


def test_first_call_inside_a_capture_is_refused_where_it_needs_a_workspace(K):
    from cgt_amd import capi
    q, k = dev(np.ones((1, 1, 1, 64))), dev(np.ones((1, 1, 4096, 64)))
    o, lse = K.rel_attention_fwd(q, k, k)
    s = capi.Stream()
    said = []

    def call():
        try:
            K.rel_attention_fwd(q, k, k, out=(o, lse), stream=s.handle)
        except capi.CgtAmdError as e:
            said.append(str(e))
    capi.Graph.capture(s, call)
    assert said and "captured" in said[0]


# ---------------------------------------------------------------- through the Op API

def test_ops_and_gradients(K):
    import cgt_amd as cgt
    from cgt_amd import nn
    for c in (case(2, 3, 21, 35, 24, buckets=8, max_distance=12, k_lengths=[35, 20], q_lengths=[21, 11], p=0.25, channel=4),
              case(1, 2, 20, 20, 16, causal=True, layout="bthd")):
        (q, k, v, table, go), att = make(c)
        tol = tolerances(att, go)
        flip = (lambda a: a) if c.get("layout") != "bthd" else (lambda a: a.transpose(0, 2, 1, 3))
        nodes = [cgt.constant(flip(a)) for a in (q, k, v)] + ([] if table is None else [cgt.constant(table)])
        more = {n: c[n] for n in ("causal", "max_distance", "q_lengths", "k_lengths", "p", "channel", "layout") if n in c}
        if c.get("p"):
            more["rng"] = nn.rng_state(31337, 2)
        o = nn.relative_attention(*nodes, **more)
        close(flip(o.get()), att.o, tol["o"], "o")
        grads = cgt.grad(o, nodes, goutput=flip(go))
        for name, g, want in zip(("gq", "gk", "gv", "gtable"), grads, att.pullback(go)):
            close(flip(g.get()) if name != "gtable" else g.get(), want, tol[name], name)
    q, k = nodes[0], cgt.constant(np.zeros((1, 2, 20, 17)))
    with pytest.raises(ValueError):
        nn.relative_attention(q, k, k)
    with pytest.raises(ValueError):
        nn.relative_attention(q, q, q, layout="btdh")
    with pytest.raises(ValueError):
        nn.relative_attention(q, q, q, p=0.5)
    with pytest.raises(ValueError):
        nn.relative_attention(q, q, q, k_lengths=[1, 2])


def test_no_gradients_through_what_is_kept_for_the_backward_pass(K):
    from cgt_amd import core
    from cgt_amd.nn_ops import attention, layer_norm
    x = core.constant(np.ones((1, 2, 3, 8), np.float32))
    info = attention.AttentionInfo(0.5, 0, 1, 128, 0, 0.0, 0, 0, 0, 0, 0)
    _o, lse = core.unpack(core.Result(attention.RelativeAttention(info), [x, x, x]))
    with pytest.raises(core.MethodNotDefined):
        core.grad(core.sum(lse), [x])
    w = core.constant(np.ones(8, np.float32))
    for op, inputs, n in ((layer_norm.LayerNorm(1e-5), [x, w, w], 1), (layer_norm.DropoutAddLayerNorm(0.0, 1e-5, 0), [x, x, w, w], 2)):
        with pytest.raises(core.MethodNotDefined):
            core.grad(core.sum(core.unpack(core.Result(op, inputs))[n]), [x])


def test_calls_from_two_threads_on_streams_of_their_own(K):
    import threading
    from cgt_amd import capi
    cases = [case(1, 2, 150, 300, 64, buckets=32, causal=True, q_offset=150), case(2, 3, 4, 2100, 32, buckets=8),
             case(1, 1, 520, 520, 128, buckets=16, p=0.2), case(3, 2, 30, 30, 40)]
    data = [([None if a is None else dev(a) for a in make(c)[0]], arguments(c)) for c in cases]

    def run(n, stream):
        (q, k, v, table, go), more = data[n]
        o, lse = K.rel_attention_fwd(q, k, v, table, stream=stream, **more)
        g = K.rel_attention_bwd(q, k, v, table, o, lse, go, stream=stream, **more)
        return [a for a in (o, lse) + tuple(g) if a is not None]
    want = [[a.get() for a in run(n, None)] for n in range(len(cases))]
    got, failed = [[], []], []

    def work(t):
        try:
            s = capi.Stream()
            for n in range(12):       # sizes rise and fall: workspaces grow under the calls in flight
                got[t].append(((n + t) % 4, run((n + t) % 4, s.handle)))
            s.synchronize()
        except Exception as e:      # noqa: BLE001
            failed.append(e)
    threads = [threading.Thread(target=work, args=(t,)) for t in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed
    for one in got:
        for n, results in one:
            assert all(np.array_equal(a.get(), b) for a, b in zip(results, want[n])), n


class Block(object):
    """A transformer encoder block as a user writes it: attention and feed-forward sub-layers, each ended by
    dropout + residual + layer norm."""

    def __init__(self, rs, width, heads, hidden, buckets):
        from cgt_amd import core, nn
        self.heads, self.width = heads, width
        init = lambda *s: (rs.randn(*s) / np.sqrt(s[0])).astype(np.float32)      # noqa: E731
        self.norm0 = nn.LayerNorm(width, weight_init=1 + 0.1 * rs.randn(width), bias_init=0.1 * rs.randn(width))
        self.q, self.k, self.v, self.out = (nn.Affine(width, width, weight_init=init(width, width), bias_init=0.1 * rs.randn(width)) for _ in range(4))
        self.table = core.constant(0.5 * rs.randn(buckets, heads))
        self.norm1 = nn.LayerNorm(width)
        self.up = nn.Affine(width, hidden, weight_init=init(width, hidden))
        self.down = nn.Affine(hidden, width, weight_init=init(hidden, width))
        self.params = [self.norm0.weight, self.norm0.bias, self.q.weight, self.k.weight, self.v.weight, self.out.weight, self.out.bias,
                       self.table, self.norm1.weight, self.norm1.bias, self.up.weight, self.down.weight, self.down.bias]

    def __call__(self, x, lengths, p, rng):
        """x [B, T, width] -> [B * T, width]"""
        from cgt_amd import nn
        B, T_, W = x.shape
        x = x.reshape([B * T_, W])
        h = self.norm0(x)
        q, k, v = (f(h).reshape([B, T_, self.heads, W // self.heads]) for f in (self.q, self.k, self.v))
        a = nn.relative_attention(q, k, v, self.table, q_lengths=lengths, k_lengths=lengths, max_distance=20, p=p, rng=rng, channel=0, layout="bthd")
        y, x = nn.dropout_add_layer_norm(self.out(a.reshape([B * T_, W])), x, self.norm1.weight, self.norm1.bias, p, rng, channel=1)
        return nn.dropout(self.down(nn.rectify(self.up(y))), p, rng, channel=2, residual=x) if p else self.down(nn.rectify(self.up(y))) + x

    def plain(self, x, lengths, p, seed, step, go):
        """The same in float64: (result, gradients of the parameters)."""
        val = lambda n: n.get().astype(np.float64)      # noqa: E731
        B, T_, W = x.shape
        H, D = self.heads, W // self.heads
        x = x.reshape(B * T_, W).astype(np.float64)
        g0, b0, g1, b1 = (val(n) for n in (self.norm0.weight, self.norm0.bias, self.norm1.weight, self.norm1.bias))
        h = T.layer_norm(x, g0, b0)[0]
        split = lambda f: (h @ val(f.weight) + val(f.bias)).reshape(B, T_, H, D).transpose(0, 2, 1, 3)      # noqa: E731
        att = T.Attention(split(self.q), split(self.k), split(self.v), val(self.table), max_distance=20, q_lengths=lengths, k_lengths=lengths,
                          keep=T.attention_keep(B, H, T_, T_, p, seed, step, 0) if p else None)
        a = att.o.transpose(0, 2, 1, 3).reshape(B * T_, W)
        f1 = T.keep_factors(x.shape, p, seed, step, 1) if p else 1.0
        f2 = T.keep_factors(x.shape, p, seed, step, 2) if p else 1.0
        x1 = (a @ val(self.out.weight) + val(self.out.bias)) * f1 + x
        y = T.layer_norm(x1, g1, b1)[0]
        u = y @ val(self.up.weight) + val(self.up.bias)
        r = u * (u >= 0)
        z = (r @ val(self.down.weight) + val(self.down.bias)) * f2 + x1
        gd = go * f2
        gu = (gd @ val(self.down.weight).T) * (u >= 0)
        gx1, gg1, gb1 = T.layer_norm_pullback(x1, g1, gu @ val(self.up.weight).T)
        gx1 = gx1 + go
        ga = gx1 * f1
        gq, gk, gv, gtable = att.pullback((ga @ val(self.out.weight).T).reshape(B, T_, H, D).transpose(0, 2, 1, 3))
        join = lambda t: t.transpose(0, 2, 1, 3).reshape(B * T_, W)      # noqa: E731
        gq, gk, gv = join(gq), join(gk), join(gv)
        gh = sum(g @ val(f.weight).T for g, f in ((gq, self.q), (gk, self.k), (gv, self.v)))
        _, gg0, gb0 = T.layer_norm_pullback(x, g0, gh)
        return z, [gg0, gb0, h.T @ gq, h.T @ gk, h.T @ gv, a.T @ ga, ga.sum(0, keepdims=True), gtable, gg1, gb1, y.T @ gu, r.T @ gd,
                   gd.sum(0, keepdims=True)]


@pytest.mark.parametrize("p,use_graph", [(0.0, False), (0.2, False), (0.2, True)])
def test_a_transformer_block(K, p, use_graph):
    # the operators together, as one compiled training function: values and every gradient against float64
    import cgt_amd as cgt
    rs = np.random.RandomState(12)
    B, T_, W = 3, 25, 48
    block = Block(rs, W, 4, 96, 8)
    x, go = rs.randn(B, T_, W).astype(np.float32), rs.randn(B * T_, W).astype(np.float32)
    lengths = np.array([25, 13, 4], np.int32)
    nx, ngo, nl, rng = cgt.constant(x), cgt.constant(go), cgt.constant(dev(lengths, np.int32)), cgt.constant(dev(np.array([6, 0]), np.int64))
    z = block(nx, nl, p, rng)
    grads = cgt.grad(cgt.sum(z * ngo), block.params)
    f = cgt.function([nx, ngo, nl] + ([rng] if p else []), [z] + grads, use_graph=use_graph)
    for step, lens in ((0, lengths), (3, lengths), (1, np.array([7, 0, 25], np.int32)), (3, lengths)):
        got = f(x, go, lens, *([np.array([6, step], np.int64)] if p else []))
        want = block.plain(x, lens, p, 6, step, go)
        # every stage is a float32 sum of some hundred terms: 2^-24 times about a hundred, through eight stages
        for name, a, b in zip(["z"] + ["gradient %d" % n for n in range(len(grads))], got, [want[0]] + want[1]):
            assert np.linalg.norm(a - b) <= 800 * U * np.linalg.norm(b), name
