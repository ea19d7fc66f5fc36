"""Refusals of attention's entry points and of views of other libraries' arrays; no call reaches a GPU."""
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
