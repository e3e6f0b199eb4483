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


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("size", [1.0, 1e-6, 1e6])
@pytest.mark.parametrize("tile", [2.0 ** -10, 2.0 ** -20, 2.0 ** -40, 0.0])
@pytest.mark.parametrize("t,d", [(512, 64), (400, 128)])
def test_attention_gradients_where_a_run_of_values_is_small(dev, t, d, tile, size, causal):
    """128 keys whose v is small or 0: their dS is delta's, which the other keys' v make."""
    q, k, v, go = _inputs(1, t, t, 2, 1, d)
    v[:, 128:256] *= np.float32(tile)
    go *= np.float32(size)
    _both(dev, q, k, v, go, causal=causal)


@pytest.mark.parametrize("spread", [8, 13])
def test_attention_gradients_where_douts_rows_are_apart(dev, spread):
    """Rows of dout up to 2^spread apart, and last ones (which alone see the last keys) all small."""
    q, k, v, go = _inputs(1, 2048, 2048, 1, 1, 64)
    r = np.random.default_rng(6)
    go *= np.exp2(-r.integers(0, spread + 1, go.shape[:3] + (1,))).astype(np.float32)
    _both(dev, q, k, v, go)
    go[:, -40:] *= np.float32(2.0 ** -spread) / np.abs(go[:, -40:]).max(-1, keepdims=True)
    _both(dev, q, k, v, go, causal=True)


@pytest.mark.parametrize("spread", [8, 13])
def test_attention_gradients_where_values_rows_are_apart(dev, spread):
    q, k, v, go = _inputs(1, 1500, 1500, 1, 1, 128)
    r = np.random.default_rng(7)
    v *= np.exp2(-r.integers(0, spread + 1, v.shape[:3] + (1,))).astype(np.float32)
    _both(dev, q, k, v, go)


def _sink(t, n, h, d, above, small):
    """The first key's score lies `above` over the others' mean, its value 2^-small of theirs."""
    q, k, v, go = _inputs(1, t, n, h, 1, d)
    k[..., 0] = 0
    k[:, 0] = 0
    k[:, 0, :, 0] = 40
    q[..., 0] = above * np.sqrt(d) / 40
    v[:, 0] *= np.float32(2.0 ** -small)
    return q, k, v, go


@pytest.mark.parametrize("above", [16, 20])
@pytest.mark.parametrize("t,n,h,d", [(16, 300, 2, 64), (160, 2000, 2, 128), (700, 700, 4, 64)])
def test_attention_gradients_of_keys_of_little_weight(dev, t, n, h, d, above):
    """Weights of 2^-24 to 2^-34 for all keys but one: their dv is as small, with as many bits."""
    _both(dev, *_sink(t, n, h, d, above, 0), names=("dk", "dv"))


@pytest.mark.parametrize("above,small", [(16, 6), (20, 10)])
@pytest.mark.parametrize("t,n,h,d", [(16, 300, 2, 64), (160, 2000, 2, 128), (2048, 4096, 8, 64)])
def test_attention_where_one_key_takes_most(dev, t, n, h, d, above, small):
    """Results that are made of the small weights, which the first key's small value leaves over."""
    _both(dev, *_sink(t, n, h, d, above, small), names=("out", "dq", "dk", "dv"))


def test_attention_of_scores_near_the_limit(dev):
    """Scores up to 2^18 of either sign: what their rounding adds to a weight stays in float16, and
    results stay between the values."""
    q, k, v, go = _inputs(1, 300, 700, 2, 1, 64)
    q = np.float32(0.9 * 2.0 ** 8) * (1 + np.float32(0.01) * np.clip(q, -4, 4))
    k = np.float32(2.0 ** 7) * (1 + np.float32(0.01) * np.clip(k, -4, 4))
    k[:, ::2] *= -1
    for scale in (None, -0.125):
        got = _attention(dev, q, k, v, go, scale=scale)
        assert all(np.isfinite(got[x]).all() for x in got)
        assert np.abs(got["out"]).max() <= 1.00001 * np.abs(v).max()


@pytest.mark.parametrize("apart", [10, 20, 26])
@pytest.mark.parametrize("t,d", [(512, 64), (384, 80)])
def test_attention_where_features_are_apart(dev, t, d, apart):
    """Features of an operand 2^apart below its others: they keep the accuracy of their own size."""
    small = np.array([1, 17, d - 1])
    for which in range(4):
        x = list(_inputs(1, t, t, 2, 1, d))
        x[which][..., small] *= np.float32(2.0 ** -apart)
        got = _attention(dev, *x)
        hold(got, *x)
        name = ("dk", "dq", "out", "dv")[which]             # the result whose features are the operand's
        pick = {y: got[y][..., small] if y == name else got[y] for y in got}
        hold(pick, *x, names=(name,), features={name: small})
