"""The residual norm, its int8 rows and its gradient against the formulas in 64 bits, at odd sizes, strides and
alignments, in place, on streams and in a graph."""

import numpy as np
import pytest

from operator_helpers import FLOOR, UNIT, Output, from_bits, kind_code, storage, strided, to_bits

pytestmark = pytest.mark.gpu

ULP = 2.0 ** -24
# A row's squares: at most 64 terms a thread one after the other, then 9 additions of a tree: 74 roundings of a sum
# of positive terms, half of them in its root; mean, root, reciprocal, the sum of both rows, weight and two products
# are 8 more.
ROW = (37 + 8) * ULP


class Case:
    def __init__(self, capi, kind, rows, dim, *, residual=True, weight=True, offset=0.0, pad=0, shift=0, scale=1.0, seed=3):
        rng = np.random.default_rng(seed)
        self.capi, self.kind, self.rows, self.dim, self.eps = capi, kind, rows, dim, 1e-5
        self.x_owner, x_ptr, stride, self.x = strided(capi, rng.standard_normal((rows, dim)) * scale, kind, pad, shift)
        self.r_owner, r_ptr, r_stride, r = strided(capi, rng.standard_normal((rows, dim)) * scale, kind, pad + 2, shift)
        self.residual = r if residual else np.zeros_like(r)
        stored = to_bits(1.0 - offset + 0.3 * rng.standard_normal(dim), kind)
        self.w_owner = capi.DeviceArray.from_host(stored)
        self.weight = (from_bits(stored, kind) if weight else np.ones(dim)) + offset
        self.desc = capi.norm_desc(x_ptr, rows, dim, kind_code(capi, kind), weight=self.w_owner if weight else None,
                                   weight_offset=offset, residual=r_ptr if residual else None, eps=self.eps,
                                   x_stride=stride, residual_stride=r_stride)
        self.s = self.x + self.residual
        self.factor = 1.0 / np.sqrt((self.s ** 2).mean(1, keepdims=True) + self.eps)
        self.y = self.s * self.factor * self.weight

    def tolerance(self, values, kind, own):
        return own + UNIT[kind] * (np.abs(values) + own) + FLOOR[kind]


CASES = [
    # kind, rows, dim, more
    ("f32", 1, 1, dict()),
    ("f16", 3, 7, dict(pad=1, shift=1)),
    ("bf16", 1, 8, dict(residual=False)),
    ("f32", 5, 33, dict(pad=3)),
    ("f16", 24, 768, dict()),
    ("bf16", 700, 384, dict(offset=1.0)),
    ("f32", 1001, 384, dict(pad=4)),
    ("bf16", 9, 1024, dict(pad=8)),
    ("f16", 6, 1543, dict(pad=5, shift=3)),
    ("f32", 4, 1024, dict(weight=False, offset=0.25)),
    ("f32", 7, 1025, dict()),
    ("bf16", 5, 2048, dict(weight=False)),
    ("f16", 4, 2050, dict(shift=1)),
    ("bf16", 3, 5000, dict(pad=1)),
    ("f32", 3, 5000, dict(residual=False)),
    ("f16", 2, 16384, dict()),
    ("f32", 2, 16384, dict()),
    ("f32", 2, 16381, dict(pad=1)),
    ("bf16", 5003, 65, dict()),
    ("f16", 1200, 2100, dict()),
]
IDS = [f"{k}-{r}x{d}-{'-'.join(f'{a}{b}' for a, b in m.items())}" for k, r, d, m in CASES]


@pytest.mark.parametrize("kind,rows,dim,more", CASES, ids=IDS)
@pytest.mark.parametrize("wide", [False, True], ids=["", "f32out"])
def test_rows_and_sum(gpu, kind, rows, dim, more, wide):
    c = Case(gpu, kind, rows, dim, **more)
    out_kind = "f32" if wide else kind
    out = Output(gpu, rows, dim, out_kind, more.get("pad", 0), more.get("shift", 0))
    total = Output(gpu, rows, dim, kind, 3, 1)
    gpu.residual_norm(c.desc, out.ptr, kind_code(gpu, out_kind), sum_out=total.ptr, out_stride=out.stride,
                      sum_stride=total.stride)
    gpu.synchronize()
    assert np.all(np.abs(out.read() - c.y) <= c.tolerance(c.y, out_kind, ROW * np.abs(c.y)))
    # both operands are float32 values, so their float32 sum has one rounding, its storage another
    assert np.all(np.abs(total.read() - c.s) <= c.tolerance(c.s, kind, ULP * np.abs(c.s)))


@pytest.mark.parametrize("kind,rows,dim,more", CASES, ids=IDS)
def test_int8_rows(gpu, kind, rows, dim, more):
    capi = gpu
    c = Case(capi, kind, rows, dim, **more)
    pad = more.get("pad", 0)
    guard = np.full((rows, dim + pad), 77, np.int8)
    codes, scales = capi.DeviceArray.from_host(guard), capi.DeviceArray((rows,), np.float32)
    capi.residual_norm(c.desc, codes, capi.I8, out_scales=scales, out_stride=dim + pad)
    wide = capi.DeviceArray((rows, dim), np.float32)
    capi.residual_norm(c.desc, wide, capi.F32)
    # the library's quantizer over the float32 rows: the same codes and scales
    again, again_scales = capi.DeviceArray((rows, dim), np.int8), capi.DeviceArray((rows,), np.float32)
    capi.launch_quantize_rows_i8(wide, rows, dim, again, again_scales)
    capi.synchronize()
    got = codes.to_host()
    assert np.array_equal(got[:, :dim], again.to_host())
    assert np.array_equal(scales.to_host(), again_scales.to_host())
    assert np.all(got[:, dim:] == 77)
    step = np.abs(c.y).max(1, keepdims=True) / 127.0
    # the step's error, and of the rounded quotient's that of both
    assert np.all(np.abs(scales.to_host()[:, None] - step) <= (ROW + 2 * ULP) * step)
    assert np.all(np.abs(got[:, :dim] - c.y / step) <= 0.5 + 127 * (2 * ROW + 6 * ULP))


def test_rows_of_zeros_and_extremes(gpu):
    capi = gpu
    x = np.zeros((4, 96), np.float32)
    x[1] = 3e19  # squares beyond float32
    x[2, 5] = 1e-30
    x[3] = 1.0
    x[3, 7] = np.nan
    d_x, out, total = capi.DeviceArray.from_host(x), capi.DeviceArray((4, 96), np.float32), capi.DeviceArray((4, 96), np.float32)
    capi.residual_norm(capi.norm_desc(d_x, 4, 96, capi.F32, eps=1e-6), out, capi.F32, sum_out=total)
    codes, scales = capi.DeviceArray((3, 96), np.int8), capi.DeviceArray((3,), np.float32)
    capi.residual_norm(capi.norm_desc(d_x, 3, 96, capi.F32, eps=1e-6), codes, capi.I8, out_scales=scales)
    capi.synchronize()
    got = out.to_host()
    assert not got[0].any() and not got[1].any()
    assert abs(got[2, 5] - 1e-27) <= 1e-32 and np.count_nonzero(got[2]) == 1
    assert np.isnan(got[3]).all()
    assert np.array_equal(total.to_host(), x, equal_nan=True)
    assert scales.to_host()[0] == 1.0 and not codes.to_host()[0].any()
    assert codes.to_host()[2, 5] == 127


def gradients(c, d, through):
    u, g = c.s * c.factor, d * c.weight
    mean = (g * u).mean(1, keepdims=True)
    return c.factor * (g - u * mean) + through, (d * u).sum(0)


def gradient_tolerances(c, d, through):
    u, g = np.abs(c.s * c.factor), np.abs(d * c.weight)
    # the mean's sum has 74 roundings like the squares', the factor enters u, the mean and the result
    own = c.factor * ((ROW + 4 * ULP) * g + (3 * ROW + 84 * ULP) * u * (g * u).mean(1, keepdims=True))
    dx = own + ULP * (np.abs(through) + own)
    dw = ((ROW + (c.rows + 40) * ULP) * (np.abs(d) * u)).sum(0)
    return dx, dw


@pytest.mark.parametrize("kind,rows,dim,more", CASES, ids=IDS)
@pytest.mark.parametrize("with_sum", [True, False], ids=["through", ""])
def test_gradient(gpu, kind, rows, dim, more, with_sum):
    capi = gpu
    c = Case(capi, kind, rows, dim, **more)
    rng = np.random.default_rng(8)
    d_owner, d_ptr, d_stride, d = strided(capi, rng.standard_normal((rows, dim)) * 0.1, kind, 6)
    t_owner, t_ptr, t_stride, t = strided(capi, rng.standard_normal((rows, dim)) * 0.1, kind, 1)
    t = t if with_sum else np.zeros_like(t)
    size = capi.residual_norm_gradient_workspace_bytes(c.desc)
    workspace = capi.DeviceArray.from_host(np.full(size, 0xFF, np.uint8))  # NaN everywhere
    dx, dw = Output(capi, rows, dim, kind, 4, 1), Output(capi, 1, dim, kind, 3)
    more_args = dict(sum_gradient=t_ptr if with_sum else None, out_gradient_stride=d_stride, sum_gradient_stride=t_stride,
                     x_gradient_stride=dx.stride)
    capi.residual_norm_gradient(c.desc, d_ptr, dx.ptr, dw.ptr, workspace, size, **more_args)
    capi.synchronize()
    first = dx.read(), dw.read()[0]
    for got, expected, own in zip(first, gradients(c, d, t), gradient_tolerances(c, d, t)):
        assert np.all(np.abs(got - expected) <= c.tolerance(expected, kind, own))
    # each alone: the same bits
    capi.residual_norm_gradient(c.desc, d_ptr, dx.ptr, None, None, 0, **more_args)
    capi.residual_norm_gradient(c.desc, d_ptr, None, dw.ptr, workspace, size, **more_args)
    capi.synchronize()
    assert np.array_equal(first[0], dx.read()) and np.array_equal(first[1], dw.read()[0])


def test_gradient_against_differences(gpu):
    capi = gpu
    c = Case(capi, "f32", 3, 20)
    rng = np.random.default_rng(4)
    d, t = (rng.standard_normal((3, 20)).astype(np.float32).astype(np.float64) for _ in range(2))
    size = capi.residual_norm_gradient_workspace_bytes(c.desc)
    workspace = capi.DeviceArray(size, np.uint8)
    d_d, d_t = capi.DeviceArray.from_host(d.astype(np.float32)), capi.DeviceArray.from_host(t.astype(np.float32))
    dx, dw = Output(capi, 3, 20, "f32"), Output(capi, 1, 20, "f32")
    capi.residual_norm_gradient(c.desc, d_d, dx.ptr, dw.ptr, workspace, size, sum_gradient=d_t)
    capi.synchronize()

    def loss(s, weight):
        y = s / np.sqrt((s ** 2).mean(1, keepdims=True) + c.eps) * weight
        return (y * d).sum() + (s * t).sum()

    # central differences with a step of 1e-5 in 64 bits: off by about 1e-9
    step = 1e-5
    for i in range(3):
        for j in range(0, 20, 3):
            bump = np.zeros_like(c.s)
            bump[i, j] = step
            slope = (loss(c.s + bump, c.weight) - loss(c.s - bump, c.weight)) / (2 * step)
            assert abs(slope - dx.read()[i, j]) <= 1e-5 * (1 + abs(slope))
    for j in range(20):
        bump = np.zeros(20)
        bump[j] = step
        slope = (loss(c.s, c.weight + bump) - loss(c.s, c.weight - bump)) / (2 * step)
        assert abs(slope - dw.read()[0, j]) <= 1e-5 * (1 + abs(slope))


@pytest.mark.parametrize("dim", [100, 768, 3000])
def test_in_place(gpu, dim):
    """The sum over the residual, the rows over x, the gradient over that of the rows."""
    capi = gpu
    rng = np.random.default_rng(5)
    x, r, d = (to_bits(rng.standard_normal((37, dim)), "bf16") for _ in range(3))
    d_x, d_r, d_d = map(capi.DeviceArray.from_host, (x, r, d))
    desc = capi.norm_desc(d_x, 37, dim, capi.BF16, residual=d_r)
    out, total, dx = (capi.DeviceArray((37, dim), np.uint16) for _ in range(3))
    dw, dw2 = capi.DeviceArray((dim,), np.uint16), capi.DeviceArray((dim,), np.uint16)
    size = capi.residual_norm_gradient_workspace_bytes(desc)
    workspace = capi.DeviceArray(size, np.uint8)
    capi.residual_norm(desc, out, capi.BF16, sum_out=total)
    capi.residual_norm_gradient(desc, d_d, dx, dw, workspace, size)
    capi.residual_norm_gradient(desc, d_d, d_d, dw2, workspace, size)
    capi.residual_norm(desc, d_x, capi.BF16, sum_out=d_r)
    capi.synchronize()
    assert np.array_equal(d_x.to_host(), out.to_host()) and np.array_equal(d_r.to_host(), total.to_host())
    assert np.array_equal(d_d.to_host(), dx.to_host()) and np.array_equal(dw.to_host(), dw2.to_host())


def test_no_rows(gpu):
    capi = gpu
    dw = Output(capi, 1, 50, "f16", 3)
    desc = capi.norm_desc(None, 0, 50, capi.F16)
    size = capi.residual_norm_gradient_workspace_bytes(desc)
    capi.residual_norm_gradient(desc, None, None, dw.ptr, None, size)
    capi.synchronize()
    assert not dw.read().any()


def test_graph_replays(gpu):
    capi = gpu
    c = Case(capi, "f16", 50, 384)
    out, total = capi.DeviceArray((50, 384), np.float16), capi.DeviceArray((50, 384), np.float16)
    dx, dw = capi.DeviceArray((50, 384), np.float16), capi.DeviceArray((384,), np.float16)
    size = capi.residual_norm_gradient_workspace_bytes(c.desc)
    workspace = capi.DeviceArray(size, np.uint8)

    def step(stream):
        capi.residual_norm(c.desc, out, capi.F16, sum_out=total, stream=stream)
        capi.residual_norm_gradient(c.desc, out, dx, dw, workspace, size, sum_gradient=total, stream=stream)

    results = (out, total, dx, dw)
    step(None)
    capi.synchronize()
    eager = [a.to_host() for a in results]
    stream = capi.Stream()
    graph = capi.Graph(stream, lambda: step(stream))
    for replay in range(3):
        for a in results:
            call = capi.DeviceArray.from_host(np.full(a.nbytes, 0xEE, np.uint8))
            capi.call("zcgvs_memcpy_d2d", a.ptr, call.ptr, a.nbytes, None)
        capi.synchronize()
        graph.launch(stream)
        capi.synchronize()
        assert all(np.array_equal(a.to_host(), e) for a, e in zip(results, eager)), replay
