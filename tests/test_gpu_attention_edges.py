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
