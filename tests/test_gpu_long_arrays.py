"""Arrays of more than 2^31 elements: an attention's cache, the rows of a layer norm, a dropout."""
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


def filled(shape, value=0.0):
    from cgt_amd.gpuarray import empty
    return empty(shape).fill_u32(int(np.float32(value).view(np.uint32)))


def tail(a, rows):
    """The last `rows` rows (of elements, where there is one axis) as an array of its own."""
    from cgt_amd.gpuarray import GpuArray
    shape = (rows,) + a.shape[-1:] if a.ndim > 1 else (rows,)
    return GpuArray(shape, a.dtype, _buffer=a._buffer, _offset=a.nbytes - int(np.prod(shape)) * 4)


@pytest.mark.parametrize("Tq", [1, 9])
def test_attention_over_a_cache_of_2_to_the_31_elements(K, Tq):
    from cgt_amd.gpuarray import to_gpu
    rs = np.random.RandomState(Tq)
    n, D = (1 << 25) + 8, 64
    k, v = filled((1, 1, n, D)), filled((1, 1, n, D))
    last = rs.randn(1, D).astype(np.float32)
    tail(k, 1).set(np.full((1, D), 8, np.float32))
    tail(v, 1).set(last)
    q = to_gpu(np.ones((1, 1, Tq, D), np.float32))
    # the last key scores 8 * 64 / sqrt(64) = 64, every other one 0: n exp(-64) = 5.4e-21 of the sum is theirs
    o, lse = K.rel_attention_fwd(q, k, v)
    assert np.abs(o.get()[0, 0] - last).max() <= 300 * U * np.abs(last).max()
    assert np.abs(lse.get() - 64).max() <= 300 * U * 64
    if Tq == 1:
        return
    go = rs.randn(1, 1, Tq, D).astype(np.float32)
    gq, gk, gv, _ = K.rel_attention_bwd(q, k, v, None, o, lse, to_gpu(go))
    # p is 1 to within the roundings of a score of 64 and of lse; ds = p (go . v - go . o) is what the roundings of both leave
    want, size = go[0, 0].astype(np.float64).sum(0), np.abs(go[0, 0]).astype(np.float64)
    assert np.abs(tail(gv, 1).get()[0] - want).max() <= 400 * U * size.sum(0).max()
    ds = 800 * U * (size @ np.abs(last[0]))
    assert np.abs(tail(gk, 1).get()[0]).max() <= 0.125 * ds.sum()
    assert np.abs(gq.get()[0, 0]).max() <= 0.125 * 8 * ds.max()
    # a key in front of it has exp(-64) = 1.6e-28 of that
    assert np.abs(tail(gv, 2).get()[0]).max() <= 1e-26 and np.abs(tail(gk, 2).get()[0]).max() <= 1e-24


def test_layer_norm_of_2_to_the_31_elements(K):
    from cgt_amd.gpuarray import to_gpu
    rs = np.random.RandomState(0)
    rows, cols = (1 << 21) + 3, 1024
    x, g = rs.randn(1, cols).astype(np.float32), rs.randn(1, cols).astype(np.float32)
    gamma, beta = rs.rand(cols).astype(np.float32) + 0.5, rs.randn(cols).astype(np.float32)
    dx = filled((rows, cols))
    tail(dx, 1).set(x)
    y, mean, rstd = K.layer_norm_fwd(dx, to_gpu(gamma), to_gpu(beta))
    want, m, r = T.layer_norm(x, gamma, beta)
    # 38 additions of a row's sum and a few products, of values of size 8 at most
    assert np.abs(tail(y, 1).get() - want).max() <= 60 * U * 8
    assert np.abs(tail(mean, 1).get() - m).max() <= 60 * U and np.abs(tail(rstd, 1).get() / r - 1).max() <= 60 * U
    assert np.array_equal(tail(y, 2).get()[0], beta)
    dg = filled((rows, cols))
    tail(dg, 1).set(g)
    gx, ggamma, gbeta = K.layer_norm_bwd(dx, to_gpu(gamma), mean, rstd, dg, out=(y, to_gpu(beta), to_gpu(beta)))
    wx, wgamma, wbeta = T.layer_norm_pullback(x, gamma, g)
    assert np.abs(tail(gx, 1).get() - wx).max() <= 60 * U * 3 * np.abs(g * gamma).max() * 4
    assert np.abs(ggamma.get() - wgamma).max() <= 60 * U * np.abs(g).max() * 8 and np.array_equal(gbeta.get(), g[0])
    assert not tail(gx, 2).get()[0].any()


def test_dropout_of_2_to_the_31_elements(K):
    from cgt_amd.gpuarray import to_gpu
    n, p, seed, step = (1 << 31) + 4101, 0.3, 77, 5
    y = K.dropout(filled((n,), 1.0), p, to_gpu(np.array([seed, step], np.int64)), channel=9)
    first = (n - 20000) // 8
    u, t = T.random16(range(first, (n + 7) // 8), seed, step, 9).reshape(-1)[:n - first * 8], T.threshold(p)
    want = ((u >= t) * (65536.0 / (65536 - t))).astype(np.float32)
    assert np.array_equal(tail(y, want.size).get(), want)
