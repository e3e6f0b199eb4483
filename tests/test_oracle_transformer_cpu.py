"""The float64 oracle of the transformer operators, held to their definitions: gradients
against differences, rotations against complex products, the orthogonalisation against
the polynomial of the singular values."""
import numpy as np
import pytest

from oracle import transformer as T


@pytest.mark.parametrize("causal,window,q_lens,kv_lens", [
    (False, 0, None, None), (True, 0, None, None), (True, 3, None, None), (False, 2, None, None),
    (True, 0, [4, 2], [3, 6]), (False, 0, [0, 4], [6, 0])])
def test_attention_gradients_match_differences(causal, window, q_lens, kv_lens):
    r = np.random.default_rng(1)
    q, k, v = r.normal(size=(2, 4, 4, 5)), r.normal(size=(2, 6, 2, 5)), r.normal(size=(2, 6, 2, 5))
    go = r.normal(size=q.shape)
    kw = dict(causal=causal, window=window, q_lens=q_lens, kv_lens=kv_lens)
    got = T.attention(q, k, v, go, **kw)
    step = 1e-5
    for name, x in (("dq", q), ("dk", k), ("dv", v)):
        for at in r.integers(0, x.size, 25):
            old = x.flat[at]
            x.flat[at] = old + step
            up = (T.attention(q, k, v, **kw)["out"] * go).sum()
            x.flat[at] = old - step
            down = (T.attention(q, k, v, **kw)["out"] * go).sum()
            x.flat[at] = old
            # third derivatives of order 1 times step^2, and 2^-52 of sums of order 100 over the step
            assert abs((up - down) / (2 * step) - got[name].flat[at]) < 1e-7


def test_attention_rows_that_see_nothing():
    r = np.random.default_rng(2)
    q, k = r.normal(size=(1, 5, 1, 4)), r.normal(size=(1, 3, 1, 4))
    got = T.attention(q, k, k, np.ones_like(q), causal=True)
    assert np.array_equal(np.isneginf(got["lse"][0, 0]), [True, True, False, False, False])
    assert not got["out"][0, :2].any() and not got["dq"][0, :2].any()


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_is_a_complex_product_and_inverts(interleaved):
    r = np.random.default_rng(3)
    x = r.normal(size=(2, 3, 2, 10))
    pos = r.integers(-5, 1000, (2, 3))
    y, _ = T.rotary(x, pos, 8, interleaved)
    for j in range(4):
        one, two = (2 * j, 2 * j + 1) if interleaved else (j, j + 4)
        z = (x[..., one] + 1j * x[..., two]) * np.exp(1j * pos * 10000.0 ** (-2 * j / 8))[..., None]
        assert np.allclose(y[..., one], z.real) and np.allclose(y[..., two], z.imag)
    assert np.array_equal(y[..., 8:], x[..., 8:])
    assert np.allclose(T.rotary(y, pos, 8, interleaved, inverse=True)[0], x)


@pytest.mark.parametrize("shape", [(5, 9), (9, 5), (6, 6), (1, 4)])
def test_orthogonalize_moves_the_singular_values(shape):
    x = np.random.default_rng(4).normal(size=shape)
    u, s, vt = np.linalg.svd(x, full_matrices=False)
    s = s / (np.linalg.norm(x) + 1e-7)
    for _ in range(5):
        a, b, c = T.COEFFICIENTS
        s = a * s + b * s ** 3 + c * s ** 5
    assert np.allclose(T.orthogonalize(x)[0], u @ np.diag(s) @ vt)
