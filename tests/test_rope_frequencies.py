"""The frequency table of scaled rotary positions, against its definition in float64; host only."""
import math

import numpy as np
import pytest

from llm_rs_b200 import BackendError, DType, RopeScaling, rope_frequencies


@pytest.fixture(autouse=True)
def _lib(cuda_lib):
    return cuda_lib


def plain(dim, theta):
    return theta ** (-2.0 * np.arange(dim // 2, dtype=np.float64) / dim)


def close(got, want):
    assert got.dtype == np.float32
    # one rounding to float32 (2^-24) and float32 arguments held as doubles
    assert np.all(np.abs(got - want) <= 2.0 ** -24 * want + 1e-45)


@pytest.mark.parametrize("dim", [2, 16, 64, 128, 256])
@pytest.mark.parametrize("theta", [10000.0, 500000.0])
def test_none_and_linear(dim, theta):
    got, mag = rope_frequencies(dim, theta)
    close(got, plain(dim, theta))
    assert mag == 1.0
    got, mag = rope_frequencies(dim, theta, RopeScaling.LINEAR, factor=4.0)
    close(got, plain(dim, theta) / 4.0)
    assert mag == 1.0


def test_by_wavelength():
    f = plain(128, 500000.0)
    got, mag = rope_frequencies(128, 500000.0, RopeScaling.WAVELENGTH, 8.0, 8192, 1.0, 4.0)
    want = np.empty_like(f)
    for i, x in enumerate(f):
        turns = 8192 * x / (2 * math.pi)
        share = (turns - 1.0) / 3.0
        want[i] = x if turns > 4 else x / 8 if turns < 1 else share * x + (1 - share) * x / 8
    close(got, want)
    assert mag == 1.0 and got[0] == 1.0 and got[-1] == np.float32(f[-1] / 8)


def test_yarn():
    f = plain(64, 10000.0)
    got, mag = rope_frequencies(64, 10000.0, RopeScaling.YARN, 16.0, 4096, 1.0, 32.0)
    at = lambda turns: 64 * math.log(4096 / (turns * 2 * math.pi)) / (2 * math.log(10000.0))  # noqa: E731
    lo, hi = max(math.floor(at(32.0)), 0), min(math.ceil(at(1.0)), 63)
    ramp = np.clip((np.arange(32) - lo) / (hi - lo), 0, 1)
    close(got, f * (1 - ramp) + f / 16 * ramp)
    assert abs(mag - (0.1 * math.log(16.0) + 1.0)) <= 2.0 ** -23


def test_factors_divide():
    fac = np.linspace(1.0, 9.0, 32).astype(np.float32)
    got, _ = rope_frequencies(64, 10000.0, factors=fac)
    close(got, plain(64, 10000.0) / fac.astype(np.float64))


@pytest.mark.parametrize("kw,code", [
    (dict(rotary_dim=0), -2), (dict(rotary_dim=3), -2), (dict(rotary_dim=258), -2),
    (dict(rope_theta=1.0), -4), (dict(rope_theta=float("nan")), -4), (dict(rope_theta=float("inf")), -4),
    (dict(kind=RopeScaling.LINEAR, factor=0.5), -4), (dict(kind=RopeScaling.LINEAR, factor=float("nan")), -4),
    (dict(kind=7), -4),
    (dict(kind=RopeScaling.YARN, factor=2.0, original_context=0, low=1.0, high=32.0), -4),
    (dict(kind=RopeScaling.WAVELENGTH, factor=2.0, original_context=100, low=4.0, high=4.0), -4),
    (dict(factors=[0.0] * 32), -4), (dict(factors=[float("nan")] * 32), -4),
])
def test_refusals(kw, code):
    args = dict(rotary_dim=64, rope_theta=10000.0) | kw
    with pytest.raises(BackendError) as e:
        rope_frequencies(**args)
    assert e.value.code == code and "rope_frequencies" in str(e.value)


def test_factor_count_is_checked():
    with pytest.raises(ValueError):
        rope_frequencies(64, 10000.0, factors=[1.0] * 31)


def test_e4m3_is_not_a_weight_type():
    assert DType.E4M3.storage_size(7) == 7 and DType.E4M3.block_elems() == 1
