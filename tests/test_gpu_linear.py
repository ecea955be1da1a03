"""The linear projection with its epilogue, on float and int8 operands, and its gradient against the formulas in 64
bits and against differences, at odd sizes, strides and alignments."""

import math

import numpy as np
import pytest

from operator_helpers import FLOOR, UNIT, Output, from_bits, kind_code, storage, strided, to_bits

pytestmark = pytest.mark.gpu

# one float32 addition of the matrix cores, whose rounding need not be to nearest
STEP = 2.0 ** -23

_erf = np.vectorize(math.erf)


def activation(name, g):
    """Value and slope in 64 bits."""
    if name == "none":
        return g, np.ones_like(g)
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
    return {"none": capi.ACT_NONE, "silu": capi.ACT_SILU, "gelu": capi.ACT_GELU, "gelu_tanh": capi.ACT_GELU_TANH}[name]


def vector(capi, values, kind):
    stored = to_bits(values, kind)
    return capi.DeviceArray.from_host(stored), from_bits(stored, kind)


class Case:
    def __init__(self, capi, kind, rows, dim, width, act, pad=0, shift=0, bias=True, residual=True, seed=1):
        rng = np.random.default_rng(seed)
        self.capi, self.kind, self.rows, self.dim, self.width, self.act = capi, kind, rows, dim, width, act
        self.x_owner, x_ptr, x_stride, self.x = strided(capi, rng.standard_normal((rows, dim)), kind, pad, shift)
        self.w_owner, w_ptr, w_stride, self.weight = strided(capi, rng.standard_normal((width, dim)) / math.sqrt(dim), kind,
                                                             pad, shift)
        self.b_owner, self.bias = vector(capi, 0.5 * rng.standard_normal(width), kind)
        self.r_owner, r_ptr, r_stride, self.residual = strided(capi, rng.standard_normal((rows, width)), kind, pad + 1)
        if not bias:
            self.bias = np.zeros(width)
        if not residual:
            self.residual = np.zeros((rows, width))
        self.desc = capi.linear_desc(x_ptr, rows, dim, w_ptr, width, kind_code(capi, kind),
                                     bias=self.b_owner if bias else None, activation=act_code(capi, act),
                                     residual=r_ptr if residual else None, x_stride=x_stride, weight_stride=w_stride,
                                     residual_stride=r_stride)
        self.z = self.x @ self.weight.T + self.bias
        # errors of the float32 sums, and of the activation's value and slope: a few roundings, of which the
        # exponent's argument (up to about 3 |z|, cubed terms included) counts by its size
        self.z_error = (dim + 3) * STEP * (np.abs(self.x) @ np.abs(self.weight).T + np.abs(self.bias))
        self.value, self.slope = activation(act, self.z)
        own = 2.0 ** -20 * (1.0 + np.abs(self.z)) ** 3 if act != "none" else np.zeros_like(self.z)
        # |act'| < 1.13 and |act''| < 1.2 for all of them
        self.value_error = 1.13 * self.z_error + own * np.abs(self.value)
        self.slope_error = (1.2 * self.z_error + own) if act != "none" else np.zeros_like(self.z)

    def check(self, got, kind):
        expected = self.value + self.residual
        tolerance = self.value_error + STEP * (np.abs(expected) + self.value_error)
        tolerance = tolerance + UNIT[kind] * (np.abs(expected) + tolerance) + FLOOR[kind]
        assert np.all(np.abs(got - expected) <= tolerance)


CASES = [
    # kind, rows, dim, width, act, pad, shift
    ("f32", 1, 1, 1, "none", 0, 0),
    ("f16", 1, 768, 512, "none", 0, 0),
    ("bf16", 2, 33, 40, "gelu", 0, 0),
    ("f16", 17, 64, 64, "gelu_tanh", 8, 0),
    ("bf16", 16, 1000, 130, "silu", 24, 8),
    ("f32", 31, 100, 72, "gelu", 0, 0),
    ("f32", 64, 515, 67, "gelu_tanh", 1, 1),
    ("f16", 33, 200, 1001, "silu", 3, 1),
    ("bf16", 65, 4100, 36, "none", 0, 0),
    ("bf16", 130, 72, 65, "gelu_tanh", 0, 4),
    ("f16", 500, 384, 264, "gelu", 0, 0),
    ("f32", 257, 70, 129, "none", 2, 0),
    ("bf16", 1100, 136, 4100, "silu", 0, 0),
    ("bf16", 1100, 136, 4100, "gelu", 0, 0),
    ("f16", 1100, 72, 2051, "none", 1, 0),
    ("f32", 1025, 36, 2048, "silu", 4, 0),
    ("bf16", 2050, 64, 4096, "none", 0, 0),
    ("f16", 64, 520, 4096, "gelu_tanh", 0, 0),
]


@pytest.mark.parametrize("case", CASES, ids=str)
@pytest.mark.parametrize("wide", [False, True], ids=["", "f32out"])
def test_projection(gpu, case, wide):
    kind, rows, dim, width, act, pad, shift = case
    c = Case(gpu, *case)
    out_kind = "f32" if wide else kind
    got = Output(gpu, rows, width, out_kind, pad, shift)
    gpu.linear(c.desc, got.ptr, kind_code(gpu, out_kind), out_stride=got.stride)
    gpu.synchronize()
    c.check(got.read(), out_kind)


@pytest.mark.parametrize("bias,residual", [(False, False), (True, False), (False, True)])
@pytest.mark.parametrize("rows", [3, 90, 700])
def test_parts_of_the_epilogue(gpu, bias, residual, rows):
    c = Case(gpu, "bf16", rows, 96, 200, "silu", bias=bias, residual=residual)
    got = Output(gpu, rows, 200, "bf16")
    gpu.linear(c.desc, got.ptr, gpu.BF16)
    gpu.synchronize()
    c.check(got.read(), "bf16")


@pytest.mark.parametrize("rows", [5, 300])
def test_output_over_the_residual(gpu, rows):
    c = Case(gpu, "f16", rows, 128, 384, "none")
    apart = Output(gpu, rows, 384, "f16", 1)
    gpu.linear(c.desc, apart.ptr, gpu.F16, out_stride=apart.stride)
    gpu.linear(c.desc, c.desc.residual, gpu.F16, out_stride=c.desc.residual_stride)
    gpu.synchronize()
    flat = c.r_owner.to_host().reshape(rows, 385)
    assert np.array_equal(from_bits(np.ascontiguousarray(flat[:, :384]), "f16"), apart.read())
    assert np.isnan(flat[:, 384]).all()


INT8 = [
    # rows, dim, width, act, epilogue, out, pad, shift
    (1, 1, 1, "none", "f32", "f32", 0, 0),
    (1, 768, 384, "silu", "f16", "f16", 0, 0),
    (7, 100, 33, "gelu", "bf16", "f32", 3, 1),
    (40, 1024, 130, "none", "f32", "f32", 0, 0),
    (64, 129, 64, "gelu_tanh", "f16", "f32", 0, 16),
    (65, 64, 100, "none", "bf16", "bf16", 16, 0),
    (300, 1000, 260, "silu", "f16", "f16", 24, 8),
    (1030, 144, 4100, "gelu_tanh", "bf16", "bf16", 0, 0),
    (1030, 145, 2050, "gelu", "f32", "f32", 0, 0),
    (3, 131072, 5, "none", "f32", "f32", 0, 0),
]


@pytest.mark.parametrize("case", INT8, ids=str)
def test_int8_operands(gpu, case):
    capi = gpu
    rows, dim, width, act, epilogue, out_kind, pad, shift = case
    rng = np.random.default_rng(11)

    def codes(n):
        values = rng.integers(-127, 128, (n, dim)).astype(np.int8)
        if dim == 131072:
            values[:] = 127  # the largest sum there is
        wide = np.full(shift + n * (dim + pad), 99, np.int8)
        wide[shift:].reshape(n, dim + pad)[:, :dim] = values
        owner = capi.DeviceArray.from_host(wide)
        return owner, owner.ptr + shift, values.astype(np.float64)

    x_owner, x_ptr, x = codes(rows)
    w_owner, w_ptr, w = codes(width)
    sx, sw = ((0.5 + rng.random(n)).astype(np.float32) / 127 for n in (rows, width))
    sw /= np.float32(math.sqrt(dim))
    d_sx, d_sw = map(capi.DeviceArray.from_host, (sx, sw))
    b_owner, bias = vector(capi, rng.standard_normal(width), epilogue)
    r_owner, r_ptr, r_stride, residual = strided(capi, rng.standard_normal((rows, width)), epilogue, pad)
    desc = capi.linear_desc(x_ptr, rows, dim, w_ptr, width, capi.I8, bias=b_owner, activation=act_code(capi, act),
                            residual=r_ptr, epilogue_dtype=kind_code(capi, epilogue), x_scales=d_sx, weight_scales=d_sw,
                            x_stride=dim + pad, weight_stride=dim + pad, residual_stride=r_stride)
    got = Output(capi, rows, width, out_kind, pad, shift)
    capi.linear(desc, got.ptr, kind_code(capi, out_kind), out_stride=got.stride)
    capi.synchronize()
    product = (x @ w.T) * sx[:, None].astype(np.float64) * sw
    z = product + bias
    value, _ = activation(act, z)
    # the sum is exact; it, the scales' product, theirs and the bias's addition round to nearest
    z_error = 2.0 ** -24 * (3 * np.abs(product) + np.abs(z)) * 1.001
    error = 1.13 * z_error + (2.0 ** -20 * (1 + np.abs(z)) ** 3 * np.abs(value) if act != "none" else 0.0)
    expected = value + residual
    error = error + 2.0 ** -24 * (np.abs(expected) + error)
    assert np.all(np.abs(got.read() - expected) <= error + UNIT[out_kind] * (np.abs(expected) + error) + FLOOR[out_kind])


def gradients(c, d):
    dz = d * c.slope
    return dz @ c.weight, dz.T @ c.x, dz.sum(0)


def gradient_tolerances(c, d):
    unit, floor = UNIT[c.kind], FLOOR[c.kind]
    ad = np.abs(d)
    dz = ad * np.abs(c.slope)
    unrounded = ad * c.slope_error + (STEP * (dz + ad * c.slope_error) if c.act != "none" else 0.0)
    dz_error = unrounded + (unit * (dz + unrounded) + floor if c.act != "none" else 0.0)
    weight, x = np.abs(c.weight), np.abs(c.x)
    tolerances = []
    for mass, slack, terms in ((dz @ weight, dz_error @ weight, c.width), (dz.T @ x, dz_error.T @ x, c.rows)):
        tolerances.append(slack + (terms + 2) * STEP * (mass + slack))
    tolerances.append(unrounded.sum(0) + (c.rows + 2) * STEP * (dz + unrounded).sum(0))
    return [t + unit * (np.abs(e) + t) + floor for t, e in zip(tolerances, gradients(c, d))]


@pytest.mark.parametrize("case", CASES, ids=str)
def test_gradient(gpu, case):
    capi = gpu
    kind, rows, dim, width, act, pad, shift = case
    c = Case(capi, *case)
    values = np.random.default_rng(2).standard_normal((rows, width)) * 0.1
    owner, d_ptr, d_stride, d = strided(capi, values, kind, pad, shift)
    size = capi.linear_gradient_workspace_bytes(c.desc)
    workspace = capi.DeviceArray.from_host(np.full(size, 0xFF, np.uint8))  # NaN everywhere
    outs = [Output(capi, rows, dim, kind, pad, shift), Output(capi, width, dim, kind, pad, shift),
            Output(capi, 1, width, kind, 3, 1)]
    strides = dict(out_gradient_stride=d_stride, x_gradient_stride=outs[0].stride, weight_gradient_stride=outs[1].stride)
    capi.linear_gradient(c.desc, d_ptr, outs[0].ptr, outs[1].ptr, outs[2].ptr, workspace, size, **strides)
    capi.synchronize()
    first = [o.read() for o in outs]
    for name, got, expected, tolerance in zip(("x", "weight", "bias"), first, gradients(c, d), gradient_tolerances(c, d)):
        assert np.all(np.abs(got - expected) <= tolerance), name
    # each alone: the same bits
    for i in range(3):
        wanted = [o.ptr if i == j else None for j, o in enumerate(outs)]
        capi.linear_gradient(c.desc, d_ptr, *wanted, workspace, size, **strides)
    capi.synchronize()
    assert all(np.array_equal(a, o.read()) for a, o in zip(first, outs))


@pytest.mark.parametrize("act", ["none", "silu", "gelu", "gelu_tanh"])
def test_gradient_against_differences(gpu, act):
    capi = gpu
    c = Case(capi, "f32", 4, 9, 7, act, residual=False)
    d = np.random.default_rng(6).standard_normal((4, 7)).astype(np.float32)
    size = capi.linear_gradient_workspace_bytes(c.desc)
    workspace, d_d = capi.DeviceArray(size, np.uint8), capi.DeviceArray.from_host(d)
    outs = [Output(capi, 4, 9, "f32"), Output(capi, 7, 9, "f32"), Output(capi, 1, 7, "f32")]
    capi.linear_gradient(c.desc, d_d, *(o.ptr for o in outs), workspace, size)
    capi.synchronize()
    operands = [c.x, c.weight, c.bias[None, :]]

    def loss(x, weight, bias):
        return (activation(act, x @ weight.T + bias)[0] * d).sum()

    # central differences with a step of 1e-5 in 64 bits: off by about 1e-9
    for which, out in enumerate(outs):
        got = out.read()
        for i in range(operands[which].shape[0]):
            for j in range(operands[which].shape[1]):
                moved = [[o.copy() for o in operands] for _ in range(2)]
                moved[0][which][i, j] += 1e-5
                moved[1][which][i, j] -= 1e-5
                slope = (loss(*moved[0]) - loss(*moved[1])) / 2e-5
                assert abs(slope - got[i, j]) <= 2e-5 * (1 + abs(slope))


def test_no_rows(gpu):
    capi = gpu
    outs = [Output(capi, 6, 10, "bf16", 2), Output(capi, 1, 6, "bf16", 2)]
    desc = capi.linear_desc(None, 0, 10, None, 6, capi.BF16, bias=1 << 20)
    capi.linear_gradient(desc, None, None, outs[0].ptr, outs[1].ptr, None, 0, weight_gradient_stride=outs[0].stride)
    capi.synchronize()
    assert not outs[0].read().any() and not outs[1].read().any()


@pytest.mark.parametrize("rows", [9, 200])
def test_non_finite_rows_stay_apart(gpu, rows):
    """A row of infinities or NaN changes no other row."""
    capi = gpu
    rng = np.random.default_rng(3)
    x = to_bits(rng.standard_normal((rows, 72)), "f16")
    w = capi.DeviceArray.from_host(to_bits(rng.standard_normal((40, 72)), "f16"))
    outs = []
    for bad in (False, True):
        if bad:
            x[rows // 2] = np.inf
            x[rows - 1] = np.nan
        d_x, out = capi.DeviceArray.from_host(x), capi.DeviceArray((rows, 40), np.float16)
        capi.linear(capi.linear_desc(d_x, rows, 72, w, 40, capi.F16), out, capi.F16)
        capi.synchronize()
        outs.append(out.to_host())
    rest = [r for r in range(rows) if r not in (rows // 2, rows - 1)]
    assert np.array_equal(outs[0][rest], outs[1][rest])
    assert np.isnan(outs[1][rows - 1]).all()


def test_graph_replays(gpu):
    capi = gpu
    c = Case(capi, "f16", 130, 384, 520, "gelu_tanh")
    out = capi.DeviceArray((130, 520), np.float16)
    grads = [capi.DeviceArray(s, np.float16) for s in ((130, 384), (520, 384), (520,))]
    size = capi.linear_gradient_workspace_bytes(c.desc)
    workspace = capi.DeviceArray(size, np.uint8)

    def step(stream):
        capi.linear(c.desc, out, capi.F16, stream=stream)
        capi.linear_gradient(c.desc, out, *grads, workspace, size, stream=stream)

    results = (out, *grads)
    step(None)
    capi.synchronize()
    eager = [a.to_host() for a in results]
    stream = capi.Stream()
    graph = capi.Graph(stream, lambda: step(stream))
    for replay in range(3):
        for a in results:
            fill = capi.DeviceArray.from_host(np.full(a.nbytes, 0xEE, np.uint8))
            capi.call("zcgvs_memcpy_d2d", a.ptr, fill.ptr, a.nbytes, None)
        capi.synchronize()
        graph.launch(stream)
        capi.synchronize()
        assert all(np.array_equal(a.to_host(), e) for a, e in zip(results, eager)), replay
