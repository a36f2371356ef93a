"""The series of csrc/verify.cu are as exact as their comments say: their numbers, as they stand in the source, in extended precision."""
import re
from pathlib import Path

import numpy as np
import pytest

TEXT = (Path(__file__).resolve().parent.parent / "turbo_fieldfare_b200" / "csrc" / "verify.cu").read_text()
L = np.longdouble
NUMBER = r"-?\d+\.\d+(?:e-?\d+)?"
pytestmark = pytest.mark.skipif(np.finfo(L).eps > 1e-18, reason="no extended precision here")


def function(start):
    body = TEXT[TEXT.index(start):]
    return body[:body.index("\n}")]


def horner(coefficients, z):
    r = np.zeros_like(z) + coefficients[-1]
    for c in coefficients[-2::-1]:
        r = r * z + c
    return r


def test_capped_logits_of_32_bits():
    """x + x z R(z), z = u^2, beside tanh(u) / u on (0, 1]: numbers rounded to 32 bits are what the compiler takes."""
    body = function("__device__ __forceinline__ float capped_near(")
    first = re.findall(rf"float r = ({NUMBER})f;", body)
    c = [L(np.float32(v)) for v in (first + re.findall(rf"r = fmaf\(r, z, ({NUMBER})f\);", body))[::-1]]
    assert len(c) == 7
    u = np.arange(1, 100001, dtype=L) / 100000
    off = np.abs((1 + u * u * horner(c, u * u)) * u / np.tanh(u) - 1)
    assert off.max() < 5.5e-9
    assert "5.5e-9 of it off" in TEXT


def test_capped_logits_of_64_bits():
    body = function("__device__ __forceinline__ void near_capped(")
    c = [L(float(v)) for v in re.findall(NUMBER, re.search(r"c\[13\] = {(.*?)};", body, re.S).group(1))]
    assert len(c) == 13
    u = np.arange(1, 100001, dtype=L) / 100000
    off = np.abs(horner(c, u * u) * u / np.tanh(u) - 1)
    assert off.max() < 2.05e-14
    assert "2e-14 of it off" in TEXT


def test_powers_of_two():
    table = [float(v) for v in re.findall(NUMBER, re.search(r"kPowers\[32\] = {(.*?)};", TEXT, re.S).group(1).split("2^(j / 32)")[1])]
    assert table == [float(L(2) ** (L(j) / 32)) for j in range(32)]
    c = L(float("0.69314718055994530942")) / 32
    fifth = c ** 5 / 120
    poly = [L(1), c - fifth * 5 / 256, c * c / 2, c ** 3 / 6 + fifth * 5 / 16, c ** 4 / 24]
    assert "poly[4] = {c - fifth * 5 / 256, c * c / 2, c * c * c / 6 + fifth * 5 / 16, c * c * c * c / 24}" in TEXT
    r = (np.arange(200001, dtype=L) - 100000) / 200000
    assert np.abs(horner(poly, r) / L(2) ** (r / 32) - 1).max() < 8e-14
