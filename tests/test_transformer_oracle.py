"""The float64 restatement of the transformer-layer operators against differences, the generator against its published
answers, and the entry points' refusals -- no GPU needed."""
import numpy as np
import pytest

from oracle import transformer as T


def _difference(f, x, direction, step=1e-5):
    return (f(x + step * direction) - f(x - step * direction)) / (2 * step)


@pytest.mark.parametrize("rows,cols", [(1, 2), (3, 7), (5, 16)])
def test_layer_norm_pullback_against_differences(rows, cols):
    rs = np.random.RandomState(rows * 100 + cols)
    x, gamma, beta, gy = rs.randn(rows, cols), rs.randn(cols), rs.randn(cols), rs.randn(rows, cols)
    gx, ggamma, gbeta = T.layer_norm_pullback(x, gamma, gy)
    for value, grad, f in [(x, gx, lambda v: (T.layer_norm(v, gamma, beta)[0] * gy).sum()),
                           (gamma, ggamma, lambda v: (T.layer_norm(x, v, beta)[0] * gy).sum()),
                           (beta, gbeta, lambda v: (T.layer_norm(x, gamma, v)[0] * gy).sum())]:
        for _ in range(3):
            d = rs.randn(*value.shape)
            # central differences of step h: error h^2 / 6 times a third derivative, and rounding over h
            assert abs(_difference(f, value, d) - (grad * d).sum()) <= 1e-6 * (1 + abs((grad * d).sum()))


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("drop", [False, True])
def test_attention_pullback_against_differences(causal, drop):
    rs = np.random.RandomState(7)
    B, H, Tq, Tk, D = 2, 3, 5, 7, 4
    q, k, v, table, go = rs.randn(B, H, Tq, D), rs.randn(B, H, Tk, D), rs.randn(B, H, Tk, D), rs.randn(8, H), rs.randn(B, H, Tq, D)
    more = dict(causal=causal, max_distance=5, q_offset=2 if causal else 0, q_lengths=[5, 3], k_lengths=[7, 0],
                keep=T.attention_keep(B, H, Tq, Tk, 0.3, 5) if drop else None)
    at = [q, k, v, table]
    grads = T.Attention(*at, **more).pullback(go)
    seen = (np.arange(Tq) < np.array([5, 3])[:, None])[:, None, :, None]
    for n in range(4):
        for _ in range(3):
            d = rs.randn(*at[n].shape)

            def f(value):
                return (T.Attention(*[value if m == n else at[m] for m in range(4)], **more).o * go * seen).sum()
            want = (grads[n] * d).sum()
            assert abs(_difference(f, at[n], d) - want) <= 1e-6 * (1 + abs(want))


def test_generator_known_answer():
    # Philox4x32 with 7 rounds of counter 0 and key 0, as its authors publish it
    words = T.random16([0], 0, 0, 0)[0].reshape(4, 2)
    assert [hex(lo | hi << 16) for lo, hi in words] == ["0x5f6fb709", "0xd893f64", "0x4f121f81", "0x4f730a48"]


def test_generator_is_uniform_and_its_uses_differ():
    n = 4000
    a = T.random16(range(n), 123456789012345, 3, 1)
    # mean of 8 n uniform 16-bit numbers: standard deviation 65536 / sqrt(12 * 8 n); five of them
    assert abs(a.mean() - 32767.5) < 5 * 65536 / np.sqrt(12 * 8 * n)
    for other in [T.random16(range(n), 123456789012346, 3, 1), T.random16(range(n), 123456789012345, 4, 1),
                  T.random16(range(n), 123456789012345, 3, 2), T.random16(range(n, 2 * n), 123456789012345, 3, 1)]:
        # equal numbers are chance hits: 8 n / 65536 expected
        assert (a == other).sum() < 10


def _fake(shape, dtype=np.float32):
    """A device array that no call may reach: refusals come before any launch."""
    from cgt_amd.gpuarray import GpuArray, _Borrowed
    return GpuArray(shape, dtype, _buffer=_Borrowed(4096, int(np.prod(shape)) * np.dtype(dtype).itemsize + 64, None))


def test_layer_norm_and_dropout_refusals():
    from cgt_amd import capi, kernels as K
    x, g, s, rng = _fake((4, 8)), _fake((8,)), _fake((4,)), _fake((2,), np.int64)
    with pytest.raises(ValueError):
        K.layer_norm_fwd(x, _fake((7,)), g)
    with pytest.raises(ValueError):
        K.layer_norm_fwd(x, g, _fake((9,)))
    with pytest.raises(ValueError):
        K.layer_norm_fwd(_fake(()), g, g)
    with pytest.raises(TypeError):
        K.layer_norm_fwd(_fake((4, 8), np.int32), g, g)
    with pytest.raises(capi.CgtAmdError, match="eps"):
        K.layer_norm_fwd(x, g, g, eps=-1.0, out=(x, s, s))
    with pytest.raises(ValueError):
        K.layer_norm_fwd(x, g, g, out=(x, s, _fake((5,))))
    with pytest.raises(ValueError):
        K.layer_norm_bwd(x, g, s, _fake((5,)), x)
    with pytest.raises(ValueError):
        K.layer_norm_bwd(x, g, s, s, _fake((8, 4)))
    for p in (-0.1, 1.0, 1.5, float("nan"), 1 - 2.0 ** -18):
        with pytest.raises(capi.CgtAmdError, match="probability"):
            K.dropout(x, p, rng, out=x)
        with pytest.raises(capi.CgtAmdError, match="probability"):
            K.dropout_add_layer_norm_fwd(x, x, g, g, p, rng, out=(x, x, s, s))
    with pytest.raises(ValueError):
        K.dropout(x, 0.1, None)
    with pytest.raises(TypeError):
        K.dropout(x, 0.1, _fake((2,), np.int32))
    with pytest.raises(TypeError):
        K.dropout(x, 0.1, _fake((3,), np.int64))
    with pytest.raises(ValueError):
        K.dropout(x, 0.1, rng, residual=_fake((8, 4)))
    with pytest.raises(ValueError):
        K.dropout(x, 0.1, rng, channel=-1, out=x)
    with pytest.raises(ValueError):
        K.dropout(x, 0.1, rng, channel=1 << 32, out=x)
    with pytest.raises(ValueError):
        K.dropout_add_layer_norm_fwd(x, x, g, g, 0.1)
    with pytest.raises(ValueError):
        K.dropout_add_layer_norm_bwd(x, g, s, s, x, _fake((4, 9)), 0.1, rng)
    lib = capi.lib()
    assert lib.cgt_amd_layer_norm_fwd_f32(None, 3, 4, None, None, 1e-5, None, None, None, None) == 1 and "null" in capi.last_error()
    assert lib.cgt_amd_layer_norm_fwd_f32(None, -1, 4, None, None, 1e-5, None, None, None, None) == 1
    assert lib.cgt_amd_layer_norm_fwd_f32(None, 1, 1 << 30, None, None, 1e-5, None, None, None, None) == 1
    assert lib.cgt_amd_layer_norm_fwd_f32(None, 0, 4, None, None, 1e-5, None, None, None, None) == 0
    assert lib.cgt_amd_dropout_f32(None, None, 0, 0.5, None, 0, None, None) == 0
    assert lib.cgt_amd_dropout_f32(None, None, 4, 0.5, None, 0, None, None) == 1 and "null" in capi.last_error()


def test_views_of_other_libraries_arrays_are_checked():
    from cgt_amd import gpuarray

    class Foreign(object):
        def __init__(self, **kw):
            self.__cuda_array_interface__ = dict(dict(shape=(3, 4), typestr="<f4", data=(4096, False), strides=None, version=2), **kw)
    a = gpuarray.as_gpuarray(Foreign())
    assert a.shape == (3, 4) and a.ptr == 4096 and a.__cuda_array_interface__["data"] == (4096, False)
    assert gpuarray.as_gpuarray(a) is a
    assert gpuarray.as_gpuarray(Foreign(strides=(16, 4))).shape == (3, 4)
    assert gpuarray.as_gpuarray(Foreign(shape=(1, 4), strides=(999, 4))).shape == (1, 4)
    assert gpuarray.as_gpuarray(Foreign(shape=(0, 4), data=(0, False))).size == 0
    with pytest.raises(ValueError):
        gpuarray.as_gpuarray(Foreign(strides=(4, 12)))
    with pytest.raises(TypeError):
        gpuarray.as_gpuarray(Foreign(typestr="<f2"))
    with pytest.raises(ValueError):
        gpuarray.as_gpuarray(Foreign(data=(0, False)))
    with pytest.raises(ValueError):
        gpuarray.as_gpuarray(Foreign(data=(4097, False)))


@pytest.mark.parametrize("bidirectional", [False, True])
def test_buckets_follow_the_rule_in_whole_numbers(bidirectional):
    from cgt_amd import kernels as K
    for buckets in (4, 6, 8, 16, 32, 64, 100, 256):
        for max_distance in (3, 5, 16, 20, 64, 100, 128, 200, 500, 1000, 1024):
            first = buckets // (4 if bidirectional else 2)
            if max_distance <= first:
                with pytest.raises(ValueError):
                    K.rel_bucket(0, buckets, bidirectional, max_distance)
                continue
            for rel in list(range(-140, 141, 1 if max_distance == 128 else 3)) + [-255, -256, -257, -511, -512, -513, -1024, -(10 ** 12), 999, 10 ** 12]:
                assert K.rel_bucket(rel, buckets, bidirectional, max_distance) == T.bucket(rel, buckets, max_distance, bidirectional), \
                    (rel, buckets, max_distance)
    for bad in ((1, False, 128), (2, True, 128), (7, True, 128), (258, False, 1024), (8, True, 1025), (8, True, 2)):
        with pytest.raises(ValueError):
            K.rel_bucket(0, *bad)


def test_attention_refusals():
    from cgt_amd import capi, kernels as K
    q, k, lse, table, rng = _fake((2, 3, 4, 8)), _fake((2, 3, 6, 8)), _fake((2, 3, 4)), _fake((8, 3)), _fake((2,), np.int64)
    out = (q, lse)
    for bad in [dict(k=_fake((2, 3, 6, 9))), dict(k=_fake((2, 4, 6, 8))), dict(k=_fake((1, 3, 6, 8))), dict(v=_fake((2, 3, 7, 8))),
                dict(q=_fake((2, 3, 8))), dict(table=_fake((8, 4))), dict(table=_fake((8,))), dict(q_lengths=_fake((3,), np.int32)),
                dict(k_lengths=_fake((2,), np.int64)), dict(layout="thbd"), dict(channel=-1), dict(p=0.5), dict(out=(q, _fake((2, 3, 5))))]:
        args = dict(dict(q=q, k=k, v=bad.get("k", k), table=table, out=out), **bad)
        with pytest.raises((ValueError, TypeError)):
            K.rel_attention_fwd(**args)
    with pytest.raises(TypeError):
        K.rel_attention_fwd(q, k, k, _fake((8, 3), np.int32), out=out)
    with pytest.raises(TypeError):
        K.rel_attention_fwd(q, k, k, table, p=0.5, rng=_fake((2,), np.int32), out=out)
    for bad in [dict(max_distance=2), dict(max_distance=1025), dict(table=_fake((7, 3))), dict(table=_fake((258, 3))), dict(p=1.0, rng=rng),
                dict(p=-0.5, rng=rng), dict(scale=float("nan")), dict(q_offset=1 << 30), dict(q_offset=-(1 << 40))]:
        args = dict(dict(q=q, k=k, v=k, table=table, out=out), **bad)
        with pytest.raises(capi.CgtAmdError):
            K.rel_attention_fwd(**args)
    wide = _fake((1, 1, 1, 129))
    with pytest.raises(capi.CgtAmdError, match="columns"):
        K.rel_attention_fwd(wide, wide, wide, out=(wide, _fake((1, 1, 1))))
    for bad in [dict(o=_fake((2, 3, 5, 8))), dict(lse=_fake((2, 3, 5))), dict(go=k)]:
        args = dict(dict(q=q, k=k, v=k, table=table, o=q, lse=lse, go=q), **bad)
        with pytest.raises(ValueError):
            K.rel_attention_bwd(**args)
    lib = capi.lib()
    rest = (0, 8, 1, 128, 0.5, 0, 0, None, None, 0.0, None, 0)
    assert lib.cgt_amd_rel_attention_fwd_f32(None, None, None, None, 1, 1, 4, 4, 8, *rest, None, None, None) == 1 and "null" in capi.last_error()
    assert lib.cgt_amd_rel_attention_fwd_f32(None, None, None, None, 1, 1, 0, 4, 8, *rest, None, None, None) == 0
    assert lib.cgt_amd_rel_attention_fwd_f32(None, None, None, None, 1, 1, -1, 4, 8, *rest, None, None, None) == 1
    assert lib.cgt_amd_rel_attention_fwd_f32(None, None, None, None, 1, 1, 1 << 29, 4, 8, *rest, None, None, None) == 1
    assert lib.cgt_amd_rel_attention_fwd_f32(None, None, None, None, 1 << 11, 1 << 11, 4, 4, 8, *rest, None, None, None) == 1
    assert lib.cgt_amd_rel_attention_bwd_f32(None, None, None, None, None, None, None, 1, 1, 4, 4, 8, *rest, None, None, None, None, None) == 1
