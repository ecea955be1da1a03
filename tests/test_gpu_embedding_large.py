"""Lookups whose bags take a wavefront each and gradients of more tokens than one workgroup sorts, against the formulas:
invalid and padding ids, bags, types, strides, several slices of columns and passes of the sort."""

import pytest

from test_gpu_embedding import test_gradient as check_gradient
from test_gpu_embedding import test_lookup as check_lookup

pytestmark = pytest.mark.gpu

# kind, out, vocab, dim, tokens, bags, mean, padding_id, pad, shift, scale: 4096 slices of 64 packs and more (on 256 compute
# units), numbers of them that leave a workgroup of four partly filled, bags of none to some hundred tokens
LOOKUPS = [
    ("f32", "f32", 3000, 384, 60_000, 5003, True, 0, 0, 0, 1.0),
    ("f16", "f16", 700, 64, 400_000, 4099, True, 5, 4, 0, 2.0),
    ("bf16", "f32", 1000, 33, 50_000, 6001, False, -1, 1, 1, 0.5),
    ("bf16", "bf16", 1000, 132, 300_000, 4101, False, 0, 8, 0, 1.0),
    ("f16", "f32", 300, 1028, 20_000, 1001, True, 2, 3, 1, 1.0),
    ("f32", "f32", 90, 3, 30_000, 4097, False, 7, 0, 0, 1.0),
    ("f32", "f32", 500, 260, 100, 8001, True, 0, 1, 2, 1.0),  # most bags are empty
]


@pytest.mark.parametrize("case", LOOKUPS, ids=str)
def test_lookup_of_many_bags(gpu, case):
    kind, out, vocab, dim, tokens, bags, *_ = case
    packs = dim // 4 + (dim % 4 > 0) if dim >= 4 else dim
    assert bags * -(-packs // 64) >= 16 * gpu.device_info().compute_units
    check_lookup(gpu, case)


GRADIENTS = [
    ("bf16", "f32", 300, 260, 10_007, 0, False, 0, 4, 0, 1.0),
    ("f16", "f16", 70_000, 100, 100_003, 0, False, 3, 3, 1, 0.5),
    ("f32", "f32", 300_000, 12, 9_000, 700, True, 0, 0, 0, 1.0),  # three passes of the sort
    ("bf16", "f32", 128_000, 64, 100_001, 4000, True, 0, 0, 0, 8.0),
    ("f16", "f32", 2_200_000, 8, 20_000, 0, False, -1, 0, 0, 1.0),
    ("bf16", "bf16", 5, 516, 70_001, 333, False, 1, 8, 0, 1.0),
    ("f32", "f32", 40_000, 3, 262_145, 262_145, True, 0, 1, 0, 1.0),
    ("f16", "f32", 513, 1025, 8_193, 50, True, 0, 0, 0, 1.0),
]


@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("case", GRADIENTS, ids=str)
def test_gradient_of_many_tokens(gpu, case, accumulate):
    check_gradient(gpu, case, accumulate)
