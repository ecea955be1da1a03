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
