"""Layer norm, dropout and the two fused, against the float64 formulas: odd widths, unaligned arrays, rows far from
zero, rows with NaN, no rows, graphs, streams, and the Op API."""
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
    """A device copy; shift = 1: at an address that is a multiple of 4 and of no more."""
    from cgt_amd.gpuarray import GpuArray, empty
    a = np.ascontiguousarray(a, dtype)
    if not shift:
        return GpuArray(a.shape, dtype).set(a)
    whole = empty((a.size + shift,), dtype)
    return GpuArray(a.shape, dtype, _buffer=whole._buffer, _offset=shift * a.itemsize).set(a)


def state(seed, step=0):
    return dev(np.array([seed, step]), np.int64)


def depth(cols):
    """Additions one value goes through in a row's sum: a lane's own, six between lanes, sixteen wavefronts."""
    return max(32, 8 * -(-cols // 8192)) + 6 + 16


def fwd_tolerance(x, gamma, beta, eps=1e-5):
    """Per element, from the roundings: the mean is off by depth * U times the mean of |x|; the squared distances' sum by
    depth relatively, half of that in rstd; a few products and the add of beta."""
    x = np.asarray(x, np.float64)
    _, mean, rstd = T.layer_norm(x, 1.0, 0.0, eps)
    d, L = np.abs(x - mean[..., None]), depth(x.shape[-1])
    off = L * np.abs(x).mean(-1)[..., None] + d
    # the mean's error shifts every distance: second order in the variance, except where the row is constant
    return U * (np.abs(gamma) * rstd[..., None] * (1.5 * off + (L / 2 + 8) * d) + 3 * np.abs(beta)) + 1e-37


def bwd_reference(x, gamma, mean, rstd, gy):
    x, gamma, mean, rstd, gy = (np.asarray(a, np.float64) for a in (x, gamma, mean, rstd, gy))
    xhat = (x - mean[..., None]) * rstd[..., None]
    g, L = gy * gamma, depth(x.shape[-1])
    gx = rstd[..., None] * (g - g.mean(-1, keepdims=True) - xhat * (g * xhat).mean(-1, keepdims=True))
    tol = U * rstd[..., None] * (6 * np.abs(g) + (L + 6) * np.abs(g).mean(-1, keepdims=True)
                                 + np.abs(xhat) * (L + 10) * np.abs(g * xhat).mean(-1, keepdims=True))
    rows = tuple(range(x.ndim - 1))
    # a column's sum: the rows of one wavefront, four of those, the partial rows of one of 32 groups, 32 groups
    n = x.size // x.shape[-1]
    down = min(n, -(-n // 512) + 64) + 40
    return (gx, tol), ((gy * xhat).sum(rows), U * (down + 4) * np.abs(gy * xhat).sum(rows)), (gy.sum(rows), U * down * np.abs(gy).sum(rows))


def close(got, want, tol):
    got = np.asarray(got, np.float64)
    worst = np.max(np.abs(got - want) - tol) if got.size else 0.0
    assert worst <= 0, "off by %g where %g is allowed" % (np.max(np.abs(got - want)), np.max(tol))


SHAPES = [(1, 1), (3, 1), (2, 2), (1, 5), (5, 63), (4, 64), (7, 255), (8, 256), (9, 257), (3, 511), (3, 513), (8, 768), (64, 1000),
          (5, 1024), (6, 1025), (2, 2049), (3, 4096), (2, 4100), (3, 8192), (2, 8193), (3, 20001), (300, 33), (2500, 96), (4099, 40)]


@pytest.mark.parametrize("shift", [0, 1])
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_layer_norm(K, rows, cols, shift):
    rs = np.random.RandomState(rows + cols)
    x = (rs.randn(rows, cols) + rs.randn(rows, 1)).astype(np.float32)
    gamma, beta, gy = (rs.randn(*s).astype(np.float32) for s in [(cols,), (cols,), (rows, cols)])
    dx, dg, db = dev(x, shift=shift), dev(gamma, shift=shift), dev(beta, shift=shift)
    y, mean, rstd = K.layer_norm_fwd(dx, dg, db)
    want, m, r = T.layer_norm(x, gamma, beta)
    close(y.get(), want, fwd_tolerance(x, gamma, beta))
    L = depth(cols)
    close(mean.get(), m, U * (L + 2) * np.abs(x).mean(-1))
    # a constant row's variance is what the mean's error leaves: next to eps it may count
    slack = U * L * np.abs(x).mean(-1)
    close(rstd.get(), r, r * (U * (L / 2 + 6) + 0.5 * r * r * (slack ** 2 + 2 * slack * U)))
    gx, ggamma, gbeta = K.layer_norm_bwd(dx, dg, mean, rstd, dev(gy, shift=shift))
    refs = bwd_reference(x, gamma, mean.get(), rstd.get(), gy)
    for got, (value, tol) in zip((gx, ggamma, gbeta), refs):
        close(got.get(), value, tol + 1e-37)
    # same input, same bits
    again = K.layer_norm_bwd(dx, dg, mean, rstd, dev(gy, shift=shift))
    assert all(np.array_equal(a.get(), b.get()) for a, b in zip(again, (gx, ggamma, gbeta)))


def test_layer_norm_rows_far_from_zero(K):
    # the distances from the mean are exact differences of floats: 1000 + noise keeps the noise's digits
    rs = np.random.RandomState(1)
    for cols in (100, 1000, 5000, 9000):
        x = (1000.0 + rs.randn(20, cols)).astype(np.float32)
        one = np.ones(cols, np.float32)
        y, _, _ = K.layer_norm_fwd(dev(x), dev(one), dev(0 * one))
        close(y.get(), T.layer_norm(x, one, 0 * one)[0], fwd_tolerance(x, one, 0 * one))


def test_layer_norm_values_that_are_no_numbers_stay_in_their_row(K):
    rs = np.random.RandomState(2)
    x = rs.randn(9, 300).astype(np.float32)
    x[3, 7], x[5, 0] = np.nan, np.inf
    gamma, beta = rs.randn(300).astype(np.float32), rs.randn(300).astype(np.float32)
    y, _, _ = K.layer_norm_fwd(dev(x), dev(gamma), dev(beta))
    fine = [0, 1, 2, 4, 6, 7, 8]
    close(y.get()[fine], T.layer_norm(x[fine], gamma, beta)[0], fwd_tolerance(x[fine], gamma, beta))
    assert np.isnan(y.get()[[3, 5]]).all()


def test_no_rows(K):
    gamma = dev(np.ones(7))
    x, stat = dev(np.zeros((0, 7))), dev(np.zeros(0))
    y, mean, rstd = K.layer_norm_fwd(x, gamma, gamma)
    assert y.shape == (0, 7) and mean.shape == (0,)
    gx, ggamma, gbeta = K.layer_norm_bwd(x, gamma, stat, stat, x, out=(x, dev(np.ones(7)), dev(np.ones(7))))
    assert not ggamma.get().any() and not gbeta.get().any()
    assert K.dropout(dev(np.zeros(0)), 0.5, state(1)).size == 0


@pytest.mark.parametrize("n", [1, 7, 8, 9, 255, 2049, 100003])
@pytest.mark.parametrize("residual", [False, True])
def test_dropout(K, n, residual):
    rs = np.random.RandomState(n)
    x, r = rs.randn(n).astype(np.float32), rs.randn(n).astype(np.float32)
    for p, shift, channel, step in [(0.1, 0, 0, 0), (0.5, 1, 3, 1), (0.9, 0, (1 << 32) - 1, (1 << 32) - 1), (0.0, 0, 0, 0)]:
        seed = -12345678901234567 if shift else 987654321
        y = K.dropout(dev(x, shift=shift), p, state(seed, step), channel, residual=dev(r, shift=shift) if residual else None).get()
        keep = T.keep_factors((n,), p, seed, step, channel)
        f = keep.astype(np.float32)
        # one product, one add, in float32: bit for bit up to a fused multiply-add
        want = x.astype(np.float64) * f + (r if residual else 0.0)
        close(y, want, U * (2 * np.abs(want) + np.abs(x * f)) * (1 if residual else 0.5) + 1e-40)
        if not residual:
            assert np.array_equal(y == 0, (f == 0) | (x == 0))


def test_dropout_share_and_expectation(K):
    n = 1 << 20
    x = dev(np.ones(n))
    for p in (0.1, 0.5):
        y = K.dropout(x, p, state(77)).get().astype(np.float64)
        t = T.threshold(p) / 65536.0
        assert abs((y == 0).mean() - t) < 5 * np.sqrt(t * (1 - t) / n)
        assert abs(y.mean() - 1) < 5 * np.sqrt(t / (1 - t) / n)


def test_dropped_elements_hide_what_they_held(K):
    x = np.full(4000, np.nan, np.float32)
    keep = T.keep_factors((4000,), 0.3, 5)
    x[keep > 0] = 1.0
    y = K.dropout(dev(x), 0.3, state(5)).get()
    assert np.isfinite(y).all() and np.array_equal(y == 0, keep == 0)


@pytest.mark.parametrize("with_gh", [False, True])
@pytest.mark.parametrize("p", [0.0, 0.2])
@pytest.mark.parametrize("rows,cols,shift", [(1, 1, 0), (3, 5, 0), (9, 64, 1), (5, 510, 0), (6, 512, 0), (4, 768, 0), (7, 1000, 1),
                                             (3, 1024, 0), (3, 1027, 0), (2, 4099, 1), (2, 8192, 0), (2, 9001, 0), (1500, 24, 0)])
def test_dropout_add_layer_norm(K, rows, cols, shift, p, with_gh):
    rs = np.random.RandomState(rows * 7 + cols)
    x, r, gy, gh = (rs.randn(rows, cols).astype(np.float32) for _ in range(4))
    gamma, beta = rs.randn(cols).astype(np.float32), rs.randn(cols).astype(np.float32)
    rng = state(4242, 9) if p else None
    f = T.keep_factors((rows, cols), p, 4242, 9, 2).astype(np.float32).astype(np.float64) if p else 1.0
    y, h, mean, rstd = K.dropout_add_layer_norm_fwd(dev(x, shift=shift), dev(r, shift=shift), dev(gamma), dev(beta), p, rng, channel=2)
    want_h = x * f + r
    close(h.get(), want_h, U * (np.abs(want_h) + np.abs(x * f)))
    hh = h.get()
    close(y.get(), T.layer_norm(hh, gamma, beta)[0], fwd_tolerance(hh, gamma, beta))
    gx, gres, ggamma, gbeta = K.dropout_add_layer_norm_bwd(h, dev(gamma), mean, rstd, dev(gy, shift=shift),
                                                           dev(gh, shift=shift) if with_gh else None, p, rng, channel=2)
    (value, tol), wg, wb = bwd_reference(hh, gamma, mean.get(), rstd.get(), gy)
    if with_gh:
        value, tol = value + gh, tol + U * (np.abs(value) + np.abs(gh))
    close(gres.get(), value, tol + 1e-37)
    close(gx.get(), gres.get().astype(np.float64) * f, U * np.abs(gres.get() * f) + 1e-40)
    close(ggamma.get(), wg[0], wg[1] + 1e-37)
    close(gbeta.get(), wb[0], wb[1] + 1e-37)


def test_replayed_graphs_draw_the_masks_of_the_step_they_find(K):
    from cgt_amd import capi
    from cgt_amd.gpuarray import empty
    rs = np.random.RandomState(3)
    rows, cols = 700, 200
    x, r, gy = (dev(rs.randn(rows, cols)) for _ in range(3))
    gamma, beta = dev(rs.randn(cols)), dev(rs.randn(cols))
    rng = state(11, 0)

    def outs():
        return [empty((rows, cols)), empty((rows, cols)), empty((rows,)), empty((rows,)), empty((rows, cols)), empty((rows, cols)),
                empty((cols,)), empty((cols,))]

    def step(o, stream):
        K.dropout_add_layer_norm_fwd(x, r, gamma, beta, 0.3, rng, out=o[:4], stream=stream)
        K.dropout_add_layer_norm_bwd(o[1], gamma, o[2], o[3], gy, None, 0.3, rng, out=o[4:], stream=stream)
    streams = [capi.Stream(), capi.Stream()]
    held, graphs = [outs(), outs()], []
    for s, o in zip(streams, held):       # two graphs, each with the workspace of its own stream
        step(o, s.handle)
        s.synchronize()
        graphs.append(capi.Graph.capture(s, lambda: step(o, s.handle)))
    eager = outs()
    for n in range(4):
        rng.set(np.array([11, n], np.int64))
        for g in graphs:
            g.launch()
        for s in streams:
            s.synchronize()
        step(eager, None)
        capi.synchronize()
        for o in held:
            assert all(np.array_equal(a.get(), b.get()) for a, b in zip(o, eager)), "replay %d" % n


def test_a_torch_tensor_is_used_in_place(K):
    # in a process of its own, where torch is imported before the library is loaded: both then use one HIP runtime
    import os
    import subprocess
    import sys
    code = """
import numpy as np
import torch
from cgt_amd import kernels as K
from cgt_amd.gpuarray import as_gpuarray
from oracle import transformer as T
t = torch.arange(24, dtype=torch.float32, device="cuda").reshape(4, 6)
y = K.layer_norm_fwd(as_gpuarray(t), as_gpuarray(torch.ones(6, device="cuda")), as_gpuarray(torch.zeros(6, device="cuda")))[0]
want = T.layer_norm(np.arange(24.0).reshape(4, 6), 1.0, 0.0)[0]
assert np.abs(y.get() - want).max() < 1e-5
back = torch.as_tensor(y, device="cuda")
assert back.data_ptr() == y.ptr and np.array_equal(back.cpu().numpy(), y.get())
try:
    as_gpuarray(t.t())
except ValueError:
    print("in place")
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    done = subprocess.run([sys.executable, "-c", code], cwd=root, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=100)
    assert done.returncode == 0 and "in place" in done.stdout, done.stdout


# ---------------------------------------------------------------- through the Op API

def test_ops_and_gradients(K):
    import cgt_amd as cgt
    from cgt_amd import nn
    rs = np.random.RandomState(4)
    x, r, gy = (rs.randn(4, 6, 50).astype(np.float32) for _ in range(3))
    gamma, beta = rs.randn(50).astype(np.float32), rs.randn(50).astype(np.float32)
    nx, nr, ng, nb = (cgt.constant(a) for a in (x, r, gamma, beta))
    y = nn.layer_norm(nx, ng, nb)
    close(y.get(), T.layer_norm(x, gamma, beta)[0], fwd_tolerance(x, gamma, beta))
    grads = [g.get() for g in cgt.grad(y, [nx, ng, nb], goutput=gy)]
    # here the statistics are the op's own: their relative error (depth / 2 + 6) U enters every term once or twice
    for got, want in zip(grads, T.layer_norm_pullback(x, gamma, gy)):
        assert np.linalg.norm(got - want) <= 2 * depth(50) * U * np.linalg.norm(want)
    rng = nn.rng_state(5, 1)
    z = nn.dropout(nx, 0.4, rng, channel=6, residual=nr)
    f = T.keep_factors(x.shape, 0.4, 5, 1, 6)
    assert np.allclose(z.get(), x * f + r, rtol=4 * U, atol=4 * U * 10)
    gx, gr = cgt.grad(z, [nx, nr], goutput=gy)
    assert np.allclose(gx.get(), gy * f, rtol=4 * U, atol=0) and np.array_equal(gr.get(), gy)
    assert nn.dropout(nx, 0.0, rng) is nx
    for p in (0.0, 0.4):
        f = T.keep_factors(x.shape, p, 5, 1, 0)
        y, h = nn.dropout_add_layer_norm(nx, nr, ng, nb, p, rng)
        out = y * 2.0 + h      # both results used
        got = [g.get() for g in cgt.grad(out, [nx, nr, ng, nb], goutput=gy)]
        gh, wg, wb = T.layer_norm_pullback(x * f + r, gamma, 2 * gy)
        for a, want in zip(got, ((gh + gy) * f, gh + gy, wg, wb)):
            assert np.linalg.norm(a - want) <= 2 * depth(50) * U * np.linalg.norm(want)
        gx, gr = cgt.grad(h, [nx, nr], goutput=gy)      # h alone
        assert np.allclose(gx.get(), gy * f, rtol=4 * U, atol=0) and np.array_equal(gr.get(), gy)
    with pytest.raises(ValueError):
        nn.layer_norm(nx, cgt.constant(np.ones(49)), nb)
    with pytest.raises(ValueError):
        nn.dropout(nx, 1.0, rng)
    with pytest.raises(ValueError):
        nn.dropout(nx, 0.5, None)
    with pytest.raises(ValueError):
        nn.dropout(nx, 0.5, np.zeros(3, np.int64))


@pytest.mark.parametrize("use_graph", [False, True])
def test_compiled_function_with_the_state_as_argument(K, use_graph):
    import cgt_amd as cgt
    from cgt_amd import nn
    rs = np.random.RandomState(5)
    x = rs.randn(33, 40).astype(np.float32)
    norm = nn.LayerNorm(40, weight_init=rs.randn(40), bias_init=rs.randn(40))
    nx, rng = cgt.constant(x), cgt.constant(nn.rng_state(3))
    y = norm(nn.dropout(nx, 0.25, rng))
    cost = cgt.sum(y * y)
    g = cgt.grad(cost, [norm.weight, norm.bias])
    f = cgt.function([nx, rng], [y] + g, use_graph=use_graph)
    for step in (0, 1, 5, 1):
        for rows in ((33,) if use_graph else (33, 7)):
            got = f(x[:rows], np.array([3, step], np.int64))
            dropped = (x[:rows] * T.keep_factors((rows, 40), 0.25, 3, step)).astype(np.float32)
            want = T.layer_norm(dropped, norm.weight.get(), norm.bias.get())[0]
            close(got[0], want, fwd_tolerance(dropped, norm.weight.get(), norm.bias.get()) * 2)
            _, wg, wb = T.layer_norm_pullback(dropped, norm.weight.get(), 2 * want)
            for a, w in zip(got[1:], (wg, wb)):
                assert np.linalg.norm(a - w) <= 2 * depth(40) * U * np.linalg.norm(w)
