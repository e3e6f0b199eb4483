"""The transformer operators' results as near their definition as float32 arithmetic comes
(tests.attention_accuracy), where operands, weights or gradients are far apart in size."""
import ctypes

import numpy as np
import pytest

from directcompute_torch_b200 import _abi
from oracle import transformer as T
from tests.attention_accuracy import hold
from tests.test_gpu_transformer import _attention, _inputs, _muon

pytestmark = pytest.mark.gpu


def _both(dev, q, k, v, go, names=("out", "dq", "dk", "dv"), **kw):
    hold(_attention(dev, q, k, v, go, **kw), q, k, v, go, names=names, **kw)


@pytest.mark.parametrize("mask", [{}, {"causal": True}, {"causal": True, "window": 200}], ids=str)
@pytest.mark.parametrize("shape", [(2, 70, 70, 4, 2, 64), (1, 300, 300, 2, 2, 96), (3, 16, 1500, 16, 4, 128),
                                   (1, 400, 400, 4, 1, 128), (2, 385, 385, 4, 4, 112), (1, 1500, 1500, 2, 1, 64),
                                   (4, 260, 260, 8, 1, 33), (1, 700, 900, 6, 6, 72)], ids=str)
def test_attention_as_near_as_float32(dev, shape, mask):
    """Ordinary inputs, on the CUDA cores and the tensor cores."""
    _both(dev, *_inputs(*shape), **mask)


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


def _newton_schulz(x, dtype, steps=5, coefficients=T.COEFFICIENTS, eps=1e-7):
    """The definition in one type (the norm in float64, as everywhere here)."""
    a, b, c = (dtype(v) for v in coefficients)
    tall = x.shape[0] > x.shape[1]
    x = x.astype(np.float64)
    x = ((x.T if tall else x) / (np.linalg.norm(x) + eps)).astype(dtype)
    for _ in range(steps):
        g = x @ x.T
        x = a * x + (b * g + c * (g @ g)) @ x
    return (x.T if tall else x).astype(np.float64)


def _near(got, x, **kw):
    """got is off by at most 8 times what float32 is (see tests.attention_accuracy), or what roundings of
    x alone become in these steps."""
    want, own = _newton_schulz(x, np.float64, **kw), _newton_schulz(x, np.float32, **kw)
    r = np.random.default_rng(1)
    moved = _newton_schulz(x * (1 + T.U * r.choice([-1.0, 1.0], x.shape)), np.float64, **kw)
    off, own, moved = (np.linalg.norm(y - want) for y in (got, own, moved))
    assert off <= 8 * own + 8 * moved + 4 * T.U * np.linalg.norm(want), (off, own, moved)


@pytest.mark.parametrize("kind", ["even", "few", "falling"])
@pytest.mark.parametrize("steps", [1, 2, 3, 5])
@pytest.mark.parametrize("shape", [(40, 24), (128, 128), (333, 127), (60, 2500), (130, 257), (300, 300), (700, 520),
                                   (1100, 1300), (150, 4000)], ids=str)
def test_orthogonalize_as_near_as_float32(dev, shape, steps, kind):
    """Matrices of even, of few and of steadily falling singular values, through each way and the steps between."""
    r = np.random.default_rng(4)
    x = r.normal(size=shape)
    if kind != "even":
        n = min(shape)
        u, s, v = np.linalg.svd(x, full_matrices=False)
        s = np.where(np.arange(n) < max(1, n // 8), 1.0, 1e-3) if kind == "few" else 10.0 ** -np.linspace(0, 4, n)
        x = (u * s) @ v
    x = x.astype(np.float32)
    h, y = dev.buf(x), dev.empty(x.size)
    try:
        _abi.check(dev.lib, dev.lib.dct_orthogonalize(ctypes.byref(_muon((1, *shape), steps=steps)), h, y))
        _near(dev.read(y).reshape(shape), x, steps=steps)
    finally:
        dev.free(h, y)


@pytest.mark.parametrize("shape", [(90, 200), (400, 260)], ids=str)
@pytest.mark.parametrize("coefficients", [(1.5, -0.5, 0.0), (2.0, -1.5, 0.5)], ids=str)
def test_orthogonalize_other_polynomials_as_near_as_float32(dev, shape, coefficients):
    x = np.random.default_rng(5).normal(size=shape).astype(np.float32)
    a, b, c = coefficients
    h, y = dev.buf(x), dev.empty(x.size)
    try:
        p = _muon((1, *shape), steps=12, a=a, b=b, c=c)
        _abi.check(dev.lib, dev.lib.dct_orthogonalize(ctypes.byref(p), h, y))
        _near(dev.read(y).reshape(shape), x, steps=12, coefficients=coefficients)
    finally:
        dev.free(h, y)


@pytest.mark.parametrize("shape", [(2, 130, 257), (3, 128, 128)], ids=str)
def test_muon_step_as_near_as_float32(dev, shape):
    r = np.random.default_rng(6)
    w, m, g = (f * r.normal(size=shape).astype(np.float32) for f in (np.float32(0.01), 1, 1))
    hs = [dev.buf(x) for x in (w, m, g)]
    try:
        p = _muon(shape, lr=0.5, momentum=0.9, weight_decay=0.5, nesterov=1, scale=2.0)
        _abi.check(dev.lib, dev.lib.dct_muon(ctypes.byref(p), *hs))
        got = dev.read(hs[0]).reshape(shape)
    finally:
        dev.free(*hs)
    for i in range(shape[0]):
        u = g[i] + np.float32(0.9) * (np.float32(0.9) * m[i] + g[i])
        _near(0.75 * w[i].astype(np.float64) - got[i], u)        # w is small, its roundings too: lr scale is 1
