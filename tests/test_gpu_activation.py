"""The activations and their slopes over the whole range of their argument, against 64 bits, to a few float32 roundings."""

import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

ACTS = ["silu", "gelu", "gelu_tanh"]
_erfc = np.vectorize(math.erfc)


def activation(name, g):
    """Value and slope in 64 bits, without differences of nearly equal numbers."""
    with np.errstate(over="ignore", under="ignore"):
        if name == "gelu":
            y = 0.5 * _erfc(-g / math.sqrt(2.0))
            return g * y, y + g * np.exp(-0.5 * g * g) / math.sqrt(2.0 * math.pi)
        if name == "silu":
            z, dz = g, np.ones_like(g)
        else:
            c = 2.0 * math.sqrt(2.0 / math.pi)
            z, dz = c * (g + 0.044715 * g ** 3), c * (1.0 + 3.0 * 0.044715 * g * g)
        y = 1.0 / (1.0 + np.exp(-z))
        rest = 1.0 / (1.0 + np.exp(z))  # 1 - y
        inner = np.where(y * rest == 0.0, 0.0, g * y * rest * dz)
        return g * y, y + inner


def run(capi, act, g):
    """The library's value and slope at float32 arguments: g = 1 * gate, u = 1 * up with up = 1, so that
    out = act(g), up_gradient = act(g) and gate_gradient = act'(g)."""
    n = g.size
    arrays = [capi.DeviceArray.from_host(a) for a in (np.ones((1, 1), np.float32), g[:, None], np.ones((n, 1), np.float32),
                                                      np.ones((1, n), np.float32))]
    code = {"silu": capi.ACT_SILU, "gelu": capi.ACT_GELU, "gelu_tanh": capi.ACT_GELU_TANH}[act]
    desc = capi.gated_desc(arrays[0], 1, 1, arrays[1], arrays[2], n, capi.F32, code)
    out, gate, up = (capi.DeviceArray(n, np.float32) for _ in range(3))
    size = capi.gated_gradient_workspace_bytes(desc)
    workspace = capi.DeviceArray(size, np.uint8)
    capi.gated_projection(desc, out)
    capi.gated_gradient(desc, arrays[3], None, gate, up, workspace, size)
    capi.synchronize()
    return [a.to_host().astype(np.float64) for a in (out, up, gate)]


@pytest.mark.parametrize("act", ACTS)
def test_large_arguments(gpu, act):
    """Far from 0 the value is g or 0 and the slope 1 or 0, for every finite g."""
    g = np.array([s * m for s in (1, -1) for m in (50.0, 300.0, 1e4, 1e10, 1.5e19, 1e20, 3e25, 1e38)], np.float32)
    out, up, slope = run(gpu, act, g)
    # a single product of 1 is within 2^-23 (1.5 times with the last addition), and passes twice
    positive = g > 0
    for value in (out, up):
        assert np.all(np.abs(value - g)[positive] <= 4 * 2.0 ** -23 * g[positive]) and np.all(np.abs(value[~positive]) < 1e-19)
    assert np.all(np.abs(slope[positive] - 1.0) <= 4 * 2.0 ** -23) and np.all(np.abs(slope[~positive]) < 1e-18)


@pytest.mark.parametrize("act", ACTS)
def test_values_and_slopes(gpu, act):
    """Errors by what the formulas round: with eps = 2^-24, the argument z of the logistic function (two or six
    roundings and its constants, 3 eps |z| or 8 eps |z|, with those of g itself), its exponential and reciprocal (6 eps), a few
    products; the error function's within 4 eps of 1 and its Gaussian's exponent."""
    rng = np.random.default_rng(71)
    g = np.concatenate([np.linspace(-12, 12, 4801), rng.standard_normal(4000), 2.0 ** rng.uniform(-20, 0, 500)]).astype(np.float32)
    out, up, slope = run(gpu, act, g)
    g = g.astype(np.float64)
    value, exact_slope = activation(act, g)
    eps, size = 2.0 ** -24, np.abs(g)
    if act == "gelu":
        # g (1 + erf): absolute in 1 + erf; products 8 eps of the value
        value_error = size * (4 * eps + 3 * eps * size * np.exp(-0.5 * g * g)) + 8 * eps * np.abs(value)
        slope_error = 4 * eps + (8 + 4 * g * g) * eps * size * np.exp(-0.5 * g * g) + 8 * eps
    else:
        z = size if act == "silu" else 1.5957691 * (size + 0.044715 * size ** 3)
        dz = 1.0 if act == "silu" else 1.5957691 * (1 + 0.134145 * size ** 2)
        with np.errstate(over="ignore", under="ignore"):
            rest = 1.0 / (1.0 + np.exp(z))  # the smaller of y and 1 - y
        # y moves by y (1 - y) times z's error; relative to y that is at most z's error
        z_error = (4 if act == "silu" else 10) * eps * z
        bent = np.minimum(1.0, np.where(g > 0, rest, 1.0)) * z_error + 6 * eps  # of y, relative
        value_error = np.abs(value) * (bent + 6 * eps)
        y = np.where(g > 0, 1.0 - rest, rest)
        # y + g y (1 - y) dz: 1 - y is taken from 1, eps in y's own size there
        slope_error = y * bent + size * dz * y * ((1 - y) * (2 * bent + 8 * eps) + y * bent + 2 * eps) + 8 * eps * np.abs(exact_slope)
    floor = 2.0 ** -120
    for got in (out, up):
        # u is a product of 1, and one of g and of the result's
        assert np.all(np.abs(got - value) <= value_error + 8 * eps * np.abs(value) + floor)
    # gate_gradient contracts one row: another product of 1
    assert np.all(np.abs(slope - exact_slope) <= slope_error + 8 * eps * np.abs(exact_slope) + floor)
