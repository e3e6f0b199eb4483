"""Refusals of the transformer ops that come before any call of the library: values that a
32-bit field of its structs would change without a word."""
import numpy as np
import pytest

ops = pytest.importorskip("directcompute_torch_b200.ops")


class Shape:
    def __init__(self, *shape):
        self.shape = shape


@pytest.mark.parametrize("positions", [2 ** 31, -2 ** 31 - 1, 2 ** 32 + 5], ids=str)
def test_positions_beyond_32_bits(positions):
    with pytest.raises(ValueError):
        ops.rotary(Shape(1, 2, 1, 8), positions=np.array([[0, positions]], np.int64))
    with pytest.raises(ValueError):
        ops.rotary(Shape(1, 2, 1, 8), start=positions)
    with pytest.raises(ValueError):
        ops.attention(*(Shape(1, 2, 1, 8),) * 3, kv_lens=[positions])
    with pytest.raises(ValueError):
        ops.attention(*(Shape(1, 2, 1, 8),) * 3, q_lens=np.array([positions]))


@pytest.mark.parametrize("rotated", [-2, 2 ** 32 + 8, 2.5])
def test_rotated(rotated):
    with pytest.raises(ValueError):
        ops.rotary(Shape(1, 2, 1, 8), rotated=rotated)


@pytest.mark.parametrize("window", [-1, 2 ** 32, 2 ** 32 + 5, 1.5])
def test_window(window):
    with pytest.raises(ValueError):
        ops.attention(*(Shape(1, 2, 1, 8),) * 3, window=window)


@pytest.mark.parametrize("scale", [0.0, -0.0, 1e-60, np.float32(0)])
def test_scale_of_zero_is_not_the_default(scale):
    with pytest.raises(ValueError):
        ops.attention(*(Shape(1, 2, 1, 8),) * 3, scale=scale)


@pytest.mark.parametrize("steps", [-1, 17, 2 ** 32 + 5, 0.5])
def test_steps(steps):
    with pytest.raises(ValueError):
        ops.orthogonalize(Shape(8, 8), steps=steps)
