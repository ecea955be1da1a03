"""The gated projection and its gradient against the formulas in 64 bits, and the gradient against
differences, at odd sizes, strides and alignments."""

import math

import numpy as np
import pytest

from operator_helpers import FLOOR, UNIT, Output, kind_code, strided

pytestmark = pytest.mark.gpu

# one float32 addition of the matrix cores, whose rounding need not be to nearest
STEP = 2.0 ** -23

_erf = np.vectorize(math.erf)


def activation(name, g):
    """Value and slope in 64 bits."""
    if name == "silu":
        y = 1.0 / (1.0 + np.exp(-g))
        return g * y, y * (1.0 + g * (1.0 - y))
    if name == "gelu":
        y = 0.5 * (1.0 + _erf(g / math.sqrt(2.0)))
        return g * y, y + g * np.exp(-0.5 * g * g) / math.sqrt(2.0 * math.pi)
    c = math.sqrt(2.0 / math.pi)
    t = np.tanh(c * (g + 0.044715 * g ** 3))
    return 0.5 * g * (1.0 + t), 0.5 * (1.0 + t) + 0.5 * g * (1.0 - t * t) * c * (1.0 + 3.0 * 0.044715 * g * g)


def act_code(capi, name):
    return {"silu": capi.ACT_SILU, "gelu": capi.ACT_GELU, "gelu_tanh": capi.ACT_GELU_TANH}[name]


class Case:
    def __init__(self, capi, kind, rows, dim, hidden, act, pad=0, shift=0, seed=1):
        rng = np.random.default_rng(seed)
        self.capi, self.kind, self.rows, self.dim, self.hidden, self.act = capi, kind, rows, dim, hidden, act
        self.x_owner, x_ptr, x_stride, self.x = strided(capi, rng.standard_normal((rows, dim)), kind, pad, shift)
        scale = 1.0 / math.sqrt(dim)
        weights = rng.standard_normal((2 * hidden, dim)) * scale
        self.w_owner, w_ptr, w_stride, w = strided(capi, weights, kind, pad, shift)
        size = 4 if kind == "f32" else 2
        self.gate, self.up = w[:hidden], w[hidden:]
        self.desc = capi.gated_desc(x_ptr, rows, dim, w_ptr, w_ptr + hidden * w_stride * size, hidden,
                                    kind_code(capi, kind), act_code(capi, act), x_stride=x_stride, weight_stride=w_stride)
        self.g, self.u = self.x @ self.gate.T, self.x @ self.up.T
        # errors of the float32 sums, and of the activation's value and slope: a few roundings, of
        # which the exponent's argument (up to about 3 |g|, cubed terms included) counts by its size
        sums = (dim + 2) * STEP
        self.g_error = sums * (np.abs(self.x) @ np.abs(self.gate).T)
        self.u_error = sums * (np.abs(self.x) @ np.abs(self.up).T)
        self.value, self.slope = activation(act, self.g)
        own = 2.0 ** -20 * (1.0 + np.abs(self.g)) ** 3
        # |act'| < 1.13 and |act''| < 1.2 for all three
        self.value_error = 1.13 * self.g_error + own * np.abs(self.value)
        self.slope_error = 1.2 * self.g_error + own

    def forward_tolerance(self):
        h = np.abs(self.value * self.u)
        return (np.abs(self.u) * self.value_error + np.abs(self.value) * self.u_error + self.value_error * self.u_error
                + 2 * STEP * h + UNIT[self.kind] * h + FLOOR[self.kind])


CASES = [
    # kind, rows, dim, hidden, act, pad, shift
    ("f32", 1, 1, 1, "silu", 0, 0),
    ("f16", 1, 768, 512, "silu", 0, 0),
    ("bf16", 2, 33, 40, "gelu", 0, 0),
    ("f16", 17, 64, 64, "gelu_tanh", 8, 0),
    ("bf16", 16, 1000, 130, "silu", 24, 8),
    ("f32", 31, 100, 72, "gelu", 0, 0),
    ("f32", 65, 130, 67, "gelu_tanh", 1, 1),
    ("f16", 33, 200, 1001, "silu", 3, 1),
    ("bf16", 130, 72, 65, "gelu_tanh", 0, 4),
    ("f16", 500, 384, 264, "gelu", 0, 0),
    ("bf16", 1100, 136, 2050, "silu", 0, 0),
    ("f16", 1100, 72, 2051, "silu", 1, 0),
    ("f32", 1025, 36, 2048, "silu", 4, 0),
    ("bf16", 64, 520, 4096, "silu", 0, 0),
]


@pytest.mark.parametrize("case", CASES, ids=str)
def test_projection(gpu, case):
    capi = gpu
    kind, rows, dim, hidden, act, pad, shift = case
    c = Case(capi, *case)
    got = Output(capi, rows, hidden, kind, pad, shift)
    capi.gated_projection(c.desc, got.ptr, out_stride=got.stride)
    capi.synchronize()
    assert np.all(np.abs(got.read() - c.value * c.u) <= c.forward_tolerance())


def gradients(c, d):
    dg, du = d * c.u * c.slope, d * c.value
    return dg @ c.gate + du @ c.up, dg.T @ c.x, du.T @ c.x


def gradient_tolerances(c, d):
    unit, floor = UNIT[c.kind], FLOOR[c.kind]
    ad = np.abs(d)
    dg, du = ad * np.abs(c.u * c.slope), ad * np.abs(c.value)
    dg_error = ad * (c.u_error * np.abs(c.slope) + np.abs(c.u) * c.slope_error + c.u_error * c.slope_error)
    dg_error += (unit + 4 * STEP) * (dg + dg_error) + floor
    du_error = ad * c.value_error
    du_error += (unit + 4 * STEP) * (du + du_error) + floor
    gate, up, x = np.abs(c.gate), np.abs(c.up), np.abs(c.x)
    x_mass, x_error = dg @ gate + du @ up, dg_error @ gate + du_error @ up
    tolerances = [x_error + (2 * c.hidden + 2) * STEP * (x_mass + x_error)]
    for one, error in ((dg, dg_error), (du, du_error)):
        mass, slack = one.T @ x, error.T @ x
        tolerances.append(slack + (c.rows + 2) * STEP * (mass + slack))
    return [t + unit * (np.abs(e) + t) + floor for t, e in zip(tolerances, gradients(c, d))]


@pytest.mark.parametrize("case", CASES, ids=str)
def test_gradient(gpu, case):
    capi = gpu
    kind, rows, dim, hidden, act, pad, shift = case
    c = Case(capi, *case)
    values = np.random.default_rng(2).standard_normal((rows, hidden)) * 0.1
    owner, d_ptr, d_stride, d = strided(capi, values, kind, pad, shift)
    size = capi.gated_gradient_workspace_bytes(c.desc)
    workspace = capi.DeviceArray.from_host(np.full(size, 0xFF, np.uint8))  # NaN everywhere
    outs = [Output(capi, rows, dim, kind, pad, shift), Output(capi, hidden, dim, kind, pad, shift),
            Output(capi, hidden, dim, kind, pad, shift)]
    capi.gated_gradient(c.desc, d_ptr, outs[0].ptr, outs[1].ptr, outs[2].ptr, workspace, size,
                        out_gradient_stride=d_stride, x_gradient_stride=outs[0].stride,
                        weight_gradient_stride=outs[1].stride)
    capi.synchronize()
    first = [o.read() for o in outs]
    for name, got, expected, tolerance in zip(("x", "gate", "up"), first, gradients(c, d), gradient_tolerances(c, d)):
        assert np.all(np.abs(got - expected) <= tolerance), name
    # once more, and each part alone: the same bits
    capi.gated_gradient(c.desc, d_ptr, outs[0].ptr, None, None, workspace, size, out_gradient_stride=d_stride,
                        x_gradient_stride=outs[0].stride)
    capi.gated_gradient(c.desc, d_ptr, None, outs[1].ptr, outs[2].ptr, workspace, size, out_gradient_stride=d_stride,
                        weight_gradient_stride=outs[1].stride)
    capi.synchronize()
    assert all(np.array_equal(o.read(), f) for o, f in zip(outs, first))


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
def test_gradient_is_the_difference_of_the_formula(gpu, act):
    capi = gpu
    c = Case(capi, "f32", 9, 20, 24, act, seed=3)
    d = np.random.default_rng(4).standard_normal((9, 24)).astype(np.float32).astype(np.float64)
    d_from = capi.DeviceArray.from_host(d.astype(np.float32))
    outs = [capi.DeviceArray(s, np.float32) for s in ((9, 20), (24, 20), (24, 20))]
    size = capi.gated_gradient_workspace_bytes(c.desc)
    workspace = capi.DeviceArray(size, np.uint8)
    capi.gated_gradient(c.desc, d_from, *outs, workspace, size)
    capi.synchronize()
    operands = [c.x, c.gate, c.up]

    def loss(x, gate, up):
        return float((activation(act, x @ gate.T)[0] * (x @ up.T) * d).sum())

    # central differences with a step of 2^-13: the third derivative's part is below 1e-6 of the sums'
    # size of about 10, the rounding of the losses below 1e-10
    for which, (out, tolerance) in enumerate(zip(outs, gradient_tolerances(c, d))):
        got = out.to_host()
        for i, j in [(0, 0), (3, 7), (8, 19)]:
            step = 2.0 ** -13
            ends = []
            for sign in (1, -1):
                moved = [o.copy() for o in operands]
                moved[which][i, j] += sign * step
                ends.append(loss(*moved))
            assert abs((ends[0] - ends[1]) / (2 * step) - got[i, j]) <= tolerance[i, j] + 1e-5


def test_no_rows(gpu):
    capi = gpu
    weight = capi.DeviceArray.from_host(np.ones((8, 6), np.float16))
    desc = capi.gated_desc(None, 0, 6, weight, weight, 8, capi.F16, capi.ACT_SILU)
    capi.gated_projection(desc, None)
    grads = [capi.DeviceArray.from_host(np.ones((8, 6), np.float16)) for _ in range(2)]
    capi.gated_gradient(desc, None, None, grads[0], grads[1], None, 0)
    capi.synchronize()
    assert all(np.all(g.to_host() == 0) for g in grads)


def test_infinite_rows_stay_in_their_rows(gpu):
    """Rows with infinities and NaN, among them the one that stands in for rows past the end."""
    capi = gpu
    rng = np.random.default_rng(5)
    x = rng.standard_normal((70, 96)).astype(np.float16)
    x[3, 5], x[69, 0] = np.inf, np.nan
    w = (rng.standard_normal((80, 96)) * 0.1).astype(np.float16)
    arrays = [capi.DeviceArray.from_host(a) for a in (x, w)]
    out = capi.DeviceArray((70, 40), np.float16)
    desc = capi.gated_desc(arrays[0], 70, 96, arrays[1], arrays[1].ptr + 40 * 96 * 2, 40, capi.F16, capi.ACT_SILU)
    capi.gated_projection(desc, out)
    capi.synchronize()
    got = out.to_host()
    ok = np.ones(70, bool)
    ok[[3, 69]] = False
    assert np.all(np.isfinite(got[ok])) and not np.any(np.isfinite(got[69]))
