"""The projection on its largest tiles (256 rows by 192 or 256 columns), each activation and operand type: what stands in
registers there does not all fit."""

import pytest

import test_gpu_linear as linear

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("act", ["none", "silu", "gelu", "gelu_tanh"])
def test_int8(gpu, act):
    linear.test_int8_operands(gpu, (2050, 128, 4096, act, "bf16", "bf16", 0, 0))


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
def test_projection_and_gradient(gpu, kind, act):
    linear.test_projection(gpu, (kind, 2050, 64, 4096, act, 0, 0), False)
    linear.test_gradient(gpu, (kind, 2050, 64, 4096, act, 0, 0))


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
def test_gradient_on_the_widest(gpu, kind, act):
    linear.test_gradient(gpu, (kind, 4200, 64, 3000, act, 0, 0))
