"""Layer norm of rows as wide as they may be, and of rows without columns."""
import numpy as np
import pytest

from test_gpu_layer_norm import K, U, close, dev      # noqa: F401

pytestmark = pytest.mark.gpu


def test_weight_gradients_of_a_row_of_more_than_2_to_the_26_columns(K):
    cols = (1 << 26) + 72
    rs = np.random.RandomState(1)
    x, gy = (rs.random_sample(cols).astype(np.float32).reshape(1, cols) for _ in range(2))
    one, mean, rstd = dev(np.ones(cols)), dev([0.5]), dev([3.5])
    _gx, ggamma, gbeta = K.layer_norm_bwd(dev(x), one, mean, rstd, dev(gy))
    assert np.array_equal(gbeta.get(), gy[0])
    # a difference, two products
    want = gy[0].astype(np.float64) * (x[0].astype(np.float64) - 0.5) * 3.5
    close(ggamma.get(), want, 4 * U * np.abs(want) + 1e-40)
