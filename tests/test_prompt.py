"""The four-bit floating-point format on the CPU: the library's size helpers, and the plain quantiser the GPU tests compare with."""
import numpy as np
import pytest

from conftest import tcu
import prompt_plain as plain


def test_sizes():
    for rows, k in [(1, 1), (7, 128), (130, 129), (300, 4096)]:
        kp = -(-k // 128) * 128
        assert tcu.Fp4.code_bytes(rows, k) == rows * kp // 2
        for fmt in (plain.MX, plain.NV):
            assert tcu.Fp4.scale_bytes(rows, k, fmt) == -(-rows // 128) * 128 * kp // plain.BLOCK[fmt]


@pytest.mark.parametrize("rows,k,fmt", [(0, 5, 0), (5, 0, 0), (-1, 5, 1), (5, 2**24 + 1, 1), (2**24, 4096, 0), (5, 5, 2), (5, 5, -1)])
def test_sizes_not_taken(rows, k, fmt):
    assert tcu.Fp4.scale_bytes(rows, k, fmt) == 0
    if fmt in (0, 1):
        assert tcu.Fp4.code_bytes(rows, k) == 0


def test_every_scale_has_one_place():
    for rows, k, fmt in [(130, 300, plain.NV), (128, 128, plain.MX), (5, 1000, plain.MX)]:
        count = plain.padded(k) // plain.BLOCK[fmt]
        _, place = plain.stored(np.zeros((rows, plain.padded(k)), np.uint8), np.zeros((rows, count), np.uint8))
        assert len(np.unique(place)) == place.size and place.max() < tcu.Fp4.scale_bytes(rows, k, fmt)


@pytest.mark.parametrize("fmt", [plain.MX, plain.NV])
def test_quantised_values_are_within_half_a_number(fmt):
    # between two numbers at most 2 apart (1 scale of 4 to 6), or held at 6: an MX block's largest may be just below 8 scales; an
    # e4m3 scale is off by 2^-4 of itself, which 6 numbers feel
    x = np.random.default_rng(fmt).normal(0, 3, (50, 256))
    unit = 0.01 if fmt == plain.NV else 1.0
    code, byte = plain.quantise(x, fmt, unit)
    got = plain.values(code, byte, fmt, unit, 256)
    by = np.repeat(plain.scales(byte, fmt) * float(np.float32(unit)), plain.BLOCK[fmt], -1)
    assert (np.abs(got - x) <= by * (2.0 if fmt == plain.MX else 1.0)).all()
    # what the format holds stays as it is
    again, byte2 = plain.quantise(got, plain.MX) if fmt == plain.MX else (code, byte)
    assert np.array_equal(plain.values(again, byte2, fmt, unit, 256), got)


def test_plain_attention_by_hand():
    q, k, v = np.ones((2, 1, 1)), np.array([0.0, np.log(3), np.nan]).reshape(3, 1, 1), np.array([1.0, 5.0, np.inf]).reshape(3, 1, 1)
    out, lse = plain.attend(q, k, v, [2], [2], 1, 1.0, True, 0)  # row 0 sees key 0, row 1 both; the third is behind the end
    assert np.allclose(out.ravel(), [1, (1 + 3 * 5) / 4]) and np.allclose(lse.ravel(), [0, np.log(4)])
    out, lse = plain.attend(q, k, v, [2], [1], 1, 1.0, True, 0)  # row 0 sees nothing
    assert np.array_equal(out.ravel(), [0, 1]) and lse[0, 0] == -np.inf
