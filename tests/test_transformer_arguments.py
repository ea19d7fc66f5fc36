"""Refusals of the transformer operators and of views of other libraries' arrays; no call reaches a GPU."""
import numpy as np
import pytest

from test_transformer_oracle import _fake


def test_offsets_of_each_sequence_are_checked():
    from cgt_amd import capi, kernels as K
    q, k, lse, table = _fake((2, 3, 4, 8)), _fake((2, 3, 6, 8)), _fake((2, 3, 4)), _fake((8, 3))
    for bad in (_fake((3,), np.int32), _fake((2,), np.int64), _fake((2, 1), np.int32), _fake((2,), np.float32)):
        with pytest.raises(ValueError):
            K.rel_attention_fwd(q, k, k, table, q_offset=bad, out=(q, lse))
        with pytest.raises(ValueError):
            K.rel_attention_bwd(q, k, k, table, q, lse, q, q_offset=bad)
    lib = capi.lib()
    rest = (0, 8, 1, 128, 0.5, 0, None, None, None, 0.0, None, 0)
    assert lib.cgt_amd_rel_attention_at_fwd_f32(None, None, None, None, 1, 1, 4, 4, 8, *rest, None, None, None) == 1 and "offsets" in capi.last_error()
    assert lib.cgt_amd_rel_attention_at_bwd_f32(None, None, None, None, None, None, None, 1, 1, 4, 4, 8, *rest, None, None, None, None, None) == 1
    assert lib.cgt_amd_rel_attention_at_fwd_f32(None, None, None, None, 0, 1, 4, 4, 8, *rest, None, None, None) == 0


def test_read_only_arrays_of_other_libraries_are_inputs_only():
    import cgt_amd as cgt
    from cgt_amd import core, gpuarray, kernels as K

    class Foreign(object):
        def __init__(self, read_only):
            self.__cuda_array_interface__ = dict(shape=(4, 8), typestr="<f4", data=(4096, read_only), strides=None, version=2)
    free, fixed = gpuarray.as_gpuarray(Foreign(False)), gpuarray.as_gpuarray(Foreign(True))
    assert free.writeable and not fixed.writeable and not fixed.reshape(32).writeable and _fake((4,)).writeable
    assert fixed.__cuda_array_interface__["data"] == (4096, True)
    g, s = _fake((8,)), _fake((4,))
    for refused in (lambda: K.layer_norm_fwd(free, g, g, out=(fixed, s, s)), lambda: K.layer_norm_fwd(fixed, g, g, out=(fixed.reshape(4, 8), s, s)),
                    lambda: K.dropout(free, 0.5, _fake((2,), np.int64), out=fixed), lambda: K.mul22(free, _fake((8, 8)), out=fixed),
                    lambda: fixed.set(np.zeros((4, 8), np.float32)), lambda: fixed.fill_u32(0)):
        with pytest.raises(ValueError, match="read-only"):
            refused()
    param, new = core.constant(fixed), core.constant(free)
    with pytest.raises(ValueError, match="read-only"):
        cgt.function([], [new], updates=[(param, new)])


def test_rows_of_no_columns_have_no_statistics():
    from cgt_amd import capi, kernels as K
    x, g, s = _fake((5, 0)), _fake((0,)), _fake((5,))
    with pytest.raises(capi.CgtAmdError, match="no columns"):
        K.layer_norm_fwd(x, g, g, out=(x, s, s))
    with pytest.raises(capi.CgtAmdError, match="no columns"):
        K.dropout_add_layer_norm_fwd(x, x, g, g, out=(x, x, s, s))
    none = _fake((0, 0))
    assert K.layer_norm_fwd(none, g, g, out=(none, _fake((0,)), _fake((0,))))[0] is none
    assert capi.lib().cgt_amd_layer_norm_fwd_f32(None, 5, 0, None, None, 1e-5, None, None, None, None) == 0
