"""The measure of attention's accuracy itself: float32 arithmetic passes it, fewer bits do not."""
import numpy as np
import pytest

from oracle import transformer as T
from tests import attention_accuracy as A


def _inputs(t, n, h, hk, d):
    r = np.random.default_rng(2)
    return tuple(r.normal(size=s).astype(np.float32) for s in ((1, t, h, d), (1, n, hk, d), (1, n, hk, d), (1, t, h, d)))


def _run(q, k, v, go, causal, dtype=np.float32):
    """Every head by the formulas in one type."""
    t, h, d = q.shape[1:]
    n, hk = k.shape[1:3]
    got = {"out": np.zeros(q.shape), "dq": np.zeros(q.shape), "dk": np.zeros(k.shape), "dv": np.zeros(k.shape)}
    for i in range(h):
        g = i // (h // hk)
        r = A._head(q[0, :, i], k[0, :, g], v[0, :, g], go[0, :, i], T.visible(t, n, t, n, causal, 0), 1 / np.sqrt(d), dtype)
        got["out"][0, :, i], got["dq"][0, :, i] = r["out"], r["dq"]
        got["dk"][0, :, g] += r["dk"]
        got["dv"][0, :, g] += r["dv"]
    return got


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("shape", [(60, 90, 4, 2, 64), (200, 200, 2, 2, 33), (1, 300, 2, 1, 128)], ids=str)
def test_float32_passes_and_float16_operands_fail(shape, causal):
    x = _inputs(*shape)
    A.hold(_run(*x, causal), *x, causal=causal)
    for which, off in enumerate(("dq", "dk", "out", "dv")):       # of q, k, v, dout: a result that each reaches
        y = list(x)
        y[which] = y[which].astype(np.float16).astype(np.float32)
        worst = A.compare(_run(*y, causal), *x, causal=causal)
        assert max(worst[off]) > 4, (which, worst)


def test_a_small_row_is_held_to_its_own_size():
    """Rows of dout 2^-13 of the others, whose dS has lost its last ten bits."""
    q, k, v, go = _inputs(200, 200, 1, 1, 64)
    go[:, ::3] *= np.float32(2.0 ** -13)
    got = _run(q, k, v, go, False)
    A.hold(got, q, k, v, go)
    got["dq"][:, ::3] *= 1 + 2.0 ** -13
    worst = A.compare(got, q, k, v, go)
    assert worst["dq"][1] > 4 and worst["dq"][0] < 1


def test_a_result_that_is_not_finite_fails():
    x = _inputs(20, 20, 1, 1, 16)
    got = _run(*x, False)
    got["dk"][0, 3, 0, 2] = np.nan
    assert max(A.compare(got, *x)["dk"]) == np.inf
