"""The gated projection and its gradient at sizes that take the large tiles, several tiles a workgroup and
products split over k, against the formulas in 64 bits (computed on the GPU)."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

STEP = 2.0 ** -23  # one float32 addition of the matrix cores, whose rounding need not be to nearest
UNIT = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
FLOOR = {"f32": 0.0, "f16": 2.0 ** -25, "bf16": 0.0}
TYPE = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def activation(name, g):
    if name == "silu":
        y = torch.sigmoid(g)
        return g * y, y * (1.0 + g * (1.0 - y))
    if name == "gelu":
        y = 0.5 * (1.0 + torch.erf(g / math.sqrt(2.0)))
        return g * y, y + g * torch.exp(-0.5 * g * g) / math.sqrt(2.0 * math.pi)
    c = math.sqrt(2.0 / math.pi)
    t = torch.tanh(c * (g + 0.044715 * g ** 3))
    return 0.5 * g * (1.0 + t), 0.5 * (1.0 + t) + 0.5 * g * (1.0 - t * t) * c * (1.0 + 3.0 * 0.044715 * g * g)


# float16 and bfloat16 on all tiles and on rows that are no whole chunks; float32; one and several splits
@pytest.mark.parametrize("kind,rows,dim,hidden,act", [
    ("bf16", 2048, 64, 3000, "silu"),
    ("f16", 2048, 72, 3000, "gelu"),
    ("f16", 4100, 64, 4096, "silu"),
    ("f32", 4096, 96, 4000, "gelu"),
    ("bf16", 16384, 768, 2048, "silu"),
    ("bf16", 9000, 1024, 2000, "gelu_tanh"),
    ("f16", 16385, 201, 1031, "gelu_tanh"),
    ("f32", 6001, 384, 2500, "silu"),
    ("bf16", 20, 768, 4096, "silu"),
    ("f32", 30000, 60, 300, "gelu"),
])
def test_large(gpu, kind, rows, dim, hidden, act):
    capi = gpu
    rng = torch.Generator(device="cuda")
    rng.manual_seed(rows + dim)

    def normal(*shape, std=1.0):
        return (torch.randn(*shape, generator=rng, device="cuda") * std).to(TYPE[kind])

    x, d = normal(rows, dim), normal(rows, hidden, std=0.1)
    gate, up = normal(hidden, dim, std=dim ** -0.5), normal(hidden, dim, std=dim ** -0.5)
    code = {"f32": capi.F32, "f16": capi.F16, "bf16": capi.BF16}[kind]
    desc = capi.gated_desc(x.data_ptr(), rows, dim, gate.data_ptr(), up.data_ptr(), hidden, code,
                           {"silu": capi.ACT_SILU, "gelu": capi.ACT_GELU, "gelu_tanh": capi.ACT_GELU_TANH}[act])
    size = capi.gated_gradient_workspace_bytes(desc)
    workspace = torch.full((size,), 255, dtype=torch.uint8, device="cuda")  # NaN everywhere
    out, dx = torch.empty_like(d), torch.empty_like(x)
    dgate, dup = torch.empty_like(gate), torch.empty_like(up)
    capi.gated_projection(desc, out.data_ptr())
    capi.gated_gradient(desc, d.data_ptr(), dx.data_ptr(), dgate.data_ptr(), dup.data_ptr(), workspace.data_ptr(), size)
    torch.cuda.synchronize()

    unit, floor = UNIT[kind], FLOOR[kind]
    x, d, gate, up = x.double(), d.double(), gate.double(), up.double()
    g, u = x @ gate.T, x @ up.T
    g_error = (dim + 2) * STEP * (x.abs() @ gate.abs().T)
    u_error = (dim + 2) * STEP * (x.abs() @ up.abs().T)
    value, slope = activation(act, g)
    own = 2.0 ** -20 * (1.0 + g.abs()) ** 3  # roundings of the activation and of its argument
    value_error = 1.13 * g_error + own * value.abs()  # |act'| < 1.13 and |act''| < 1.2
    slope_error = 1.2 * g_error + own
    h = value * u
    tolerance = u.abs() * value_error + value.abs() * u_error + value_error * u_error
    tolerance += (2 * STEP + unit) * h.abs() + floor
    assert torch.all((out.double() - h).abs() <= tolerance)

    dg, du = d * u * slope, d * value
    dg_error = d.abs() * (u_error * slope.abs() + u.abs() * slope_error + u_error * slope_error)
    dg_error += (unit + 4 * STEP) * (dg.abs() + dg_error) + floor
    du_error = d.abs() * value_error
    du_error += (unit + 4 * STEP) * (du.abs() + du_error) + floor

    def check(got, expected, error, mass, terms):
        error = error + (terms + 2) * STEP * (mass + error)
        assert torch.all((got.double() - expected).abs() <= error + unit * (expected.abs() + error) + floor)

    check(dx, dg @ gate + du @ up, dg_error @ gate.abs() + du_error @ up.abs(), dg.abs() @ gate.abs() + du.abs() @ up.abs(),
          2 * hidden)
    check(dgate, dg.T @ x, dg_error.T @ x.abs(), dg.abs().T @ x.abs(), rows)
    check(dup, du.T @ x, du_error.T @ x.abs(), du.abs().T @ x.abs(), rows)
