"""float32 matrix products of the operators, one product a result: what splitting the operands may cost."""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def _operands(rng, count):
    """Values whose upper eight bits are followed by ones, by a one and zeros, by random bits; small and large."""
    bits = rng.integers(0, 2 ** 23, count, dtype=np.uint32)
    kind = np.arange(count) % 5
    bits[kind == 0] |= 0xFFFF
    bits[kind == 1] = (bits[kind == 1] & ~np.uint32(0xFFFF)) | 0x80FF
    bits[kind == 2] = (bits[kind == 2] & ~np.uint32(0xFFFF)) | 0x7F80
    bits[kind == 3] = (bits[kind == 3] & ~np.uint32(0x1FF)) | 0x100
    exponent = rng.integers(100, 150, count).astype(np.uint32)
    sign = rng.integers(0, 2, count).astype(np.uint32)
    values = (sign << 31 | exponent << 23 | bits).view(np.float32)
    values[0], values[1] = np.uint32(0x3F80FFFF).view(np.float32), 0.0
    return values


def _product(capi, x, w):
    d_x, d_w = capi.DeviceArray.from_host(x[:, None]), capi.DeviceArray.from_host(w[:, None])
    out = capi.DeviceArray((x.size, w.size), np.float32)
    capi.adapted_projection(capi.adapted_desc(d_x, x.size, 1, d_w, w.size, capi.F32), out, capi.F32, None, 0)
    capi.synchronize()
    return out.to_host().astype(np.float64), np.outer(x.astype(np.float64), w.astype(np.float64))


# the products left out, the last addition (of any rounding), and those of the small parts
TOLERANCE = 2.0 ** -24 * (1 + 2.0 ** -8) + 2.0 ** -23 + 2.0 ** -28


@pytest.mark.parametrize("rows,columns", [(70, 50), (4100, 4099)])  # tiles of 64 and of 128
def test_single_products(gpu, rows, columns):
    rng = np.random.default_rng(51)
    got, expected = _product(gpu, _operands(rng, rows), _operands(rng, columns))
    assert np.all(np.abs(got - expected) <= TOLERANCE * np.abs(expected))
    # what is left out has no preferred sign: of so many products it cancels. The last addition may be cut off
    # (up to 2^-24 of a product in the mean), so the bound is on what lies beyond that
    wanted = expected != 0
    assert abs(np.mean((got[wanted] - expected[wanted]) / expected[wanted])) <= 1.1 * 2.0 ** -24


@pytest.mark.parametrize("rows,columns", [(70, 50), (4100, 4099)])
def test_largest_values(gpu, rows, columns):
    """float32 values beyond bf16's largest have finite parts."""
    rng = np.random.default_rng(52)
    x = np.full(rows, np.finfo(np.float32).max, np.float32)
    x[::2] = -x[::2]
    x[1::7] = np.uint32(0x7F7F8000).view(np.float32)
    w = (_operands(rng, columns).view(np.uint32) & np.uint32(0x807FFFFF) | np.uint32(100 << 23)).view(np.float32)
    got, expected = _product(gpu, x, w)
    assert np.all(np.abs(got - expected) <= TOLERANCE * np.abs(expected))
