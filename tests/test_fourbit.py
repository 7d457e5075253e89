"""The four-bit format on the CPU: the library's size helpers, and the plain quantiser the GPU tests compare with."""
import numpy as np
import pytest

from conftest import tcu
import fourbit_plain as plain


def test_sizes():
    for w, p, g, h in [(128, 64, 32, 8), (32, 16, 32, 1), (256, 256, 128, 3), (64, 128, 64, 5)]:
        assert tcu.Kv4Cache.page_bytes(h, w, p, g) == h * p * (w + 8 * (w // g))
    for n, k, g in [(1, 1, 32), (7, 128, 64), (5, 129, 128)]:
        blocks = -(-k // 128)
        assert tcu.W4.code_bytes(n, k) == n * blocks * 64
        assert tcu.W4.scale_bytes(n, k, g) == n * blocks * (128 // g) * 4


@pytest.mark.parametrize("heads,width,page,group", [(0, 128, 64, 32), (8, 96, 64, 32), (8, 128, 48, 32), (8, 128, 8, 32),
                                                    (8, 128, 64, 16), (8, 32, 64, 64), (1025, 128, 64, 32), (8, 512, 64, 32)])
def test_sizes_not_taken(heads, width, page, group):
    assert tcu.Kv4Cache.page_bytes(heads, width, page, group) == 0


def test_weight_sizes_not_taken():
    assert tcu.W4.code_bytes(0, 5) == 0 and tcu.W4.scale_bytes(4, 0, 32) == 0 and tcu.W4.scale_bytes(4, 5, 48) == 0


@pytest.mark.parametrize("width", [32, 64, 128, 256])
def test_every_nibble_has_one_place(width):
    for values in (False, True):
        assert sorted(plain.places(width, values)) == list(range(width))


@pytest.mark.parametrize("group", [32, 64, 128])
def test_quantised_values_are_within_a_step(group):
    # a value is at most half a step from what it stands for, plus what rounding step and low to f16 moved the ends: low by
    # 2^-11 of its size, step by 2^-11 of 15 steps
    x = np.random.default_rng(group).normal(3, 5, (50, 256)).astype(np.float32)
    code, step, low = plain.quantise(x, group)
    got = plain.value(code, step, low, group)
    rep = lambda a: np.repeat(np.abs(a.astype(np.float64)), group, -1)  # noqa: E731
    assert (np.abs(got - x) <= 0.5 * rep(step) + rep(low) * 2.0**-11 + 15 * rep(step) * 2.0**-10 + 1e-6).all()
    assert code.max() == 15 and code.min() == 0
