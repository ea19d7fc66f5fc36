"""Host threads that share a stream: calls of several kernels that hand data on through a workspace of the stream."""
import threading

import numpy as np
import pytest

from test_gpu_attention import arguments, case, dev, make

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def K():
    from cgt_amd import capi, kernels
    capi.require_gpu()
    return kernels


def attention(K, c):
    (q, k, v, table, go), _ = make(c)
    q, k, v, table, go = (None if a is None else dev(a) for a in (q, k, v, table, go))
    more = arguments(c)

    def call(stream):
        o, lse = K.rel_attention_fwd(q, k, v, table, stream=stream, **more)
        g = K.rel_attention_bwd(q, k, v, table, o, lse, go, stream=stream, **more)
        return [a for a in (o, lse) + tuple(g) if a is not None]
    return call


def norm(K, rows, cols):
    rs = np.random.RandomState(rows)
    x, gy, gamma, beta = dev(rs.randn(rows, cols)), dev(rs.randn(rows, cols)), dev(rs.randn(cols)), dev(rs.randn(cols))

    def call(stream):
        y, mean, rstd = K.layer_norm_fwd(x, gamma, beta, stream=stream)
        return [y, mean, rstd] + list(K.layer_norm_bwd(x, gamma, mean, rstd, gy, stream=stream))
    return call


def product(K, M, N, depth):
    rs = np.random.RandomState(M)
    a, b = dev(rs.randn(M, depth)), dev(rs.randn(depth, N))      # few tiles, long sums: cut along the depth
    return lambda stream: [K.mul22(a, b, stream=stream)]


@pytest.mark.parametrize("own_stream", [False, True])
def test_threads_that_share_a_stream(K, own_stream):
    from cgt_amd import capi
    calls = [attention(K, case(2, 2, 300, 500, 64, buckets=32)), attention(K, case(1, 2, 3, 3000, 32, buckets=8)),
             attention(K, case(1, 3, 150, 900, 128, buckets=16, causal=True, q_offset=750)), norm(K, 1500, 200), norm(K, 70, 9000),
             product(K, 64, 64, 20000), product(K, 32, 96, 9000)]
    want = [[a.get() for a in call(None)] for call in calls]
    stream = capi.Stream() if own_stream else None
    handle = stream.handle if own_stream else None
    got, failed, start = [[] for _ in range(4)], [], threading.Barrier(4)

    def work(t):
        try:
            start.wait()
            for n in range(30):
                i = (3 * n + t) % len(calls)
                got[t].append((i, calls[i](handle)))
        except Exception as e:      # noqa: BLE001
            failed.append(e)
    threads = [threading.Thread(target=work, args=(t,)) for t in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    stream.synchronize() if own_stream else capi.synchronize()
    assert not failed, failed
    for one in got:
        for i, results in one:
            assert all(np.array_equal(a.get(), b) for a, b in zip(results, want[i])), i
