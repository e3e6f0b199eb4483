"""The transformer operators' results as near their definition as float32 arithmetic comes
(tests.attention_accuracy), where operands, weights or gradients are far apart in size."""
import numpy as np
import pytest

from tests.attention_accuracy import hold
from tests.test_gpu_transformer import _attention, _inputs

pytestmark = pytest.mark.gpu


def _both(dev, q, k, v, go, names=("out", "dq", "dk", "dv"), **kw):
    hold(_attention(dev, q, k, v, go, **kw), q, k, v, go, names=names, **kw)


@pytest.mark.parametrize("t,d", [(60, 64), (512, 64), (384, 128), (400, 40)])
@pytest.mark.parametrize("sizes", [(0, -55, -55), (0, -50, -50), (0, -58, -50), (-20, -58, -30), (0, -30, -58),
                                   (0, 40, 40), (0, 40, -40), (0, -40, 40)], ids=str)
def test_attention_gradients_of_small_and_large_operands(dev, t, d, sizes):
    """v and dout (and q, with k as much larger) times powers of two: products of them that reach
    2^-110 and 2^80 are still float32 numbers."""
    q, k, v, go = _inputs(1, t, t, 2, 1, d)
    q *= np.float32(2.0 ** sizes[0])
    k *= np.float32(2.0 ** -sizes[0])
    v *= np.float32(2.0 ** sizes[1])
    go *= np.float32(2.0 ** sizes[2])
    _both(dev, q, k, v, go)
