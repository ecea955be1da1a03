"""Attention where its calls reach what ordinary batches do not: keys that no query row stands before."""

import numpy as np
import pytest

from attention_helpers import Batch
from test_gpu_attention_gradient import check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("far", [30, 300])
@pytest.mark.parametrize("q_lens,k_lens,room", [([70], [200], None), ([0, 0], [130, 64], None), ([33, 0, 1], [900, 300, 700], None),
                                                ([5, 0, 40], [5, 300, 77], 320)], ids=str)
def test_bias_gradient_of_keys_without_queries(gpu, kind, far, q_lens, k_lens, room):
    """Tiles of keys that no query row sees add nothing to the bias's gradient, whatever the workgroup that ran on their CU
    before left in its tables."""
    before = Batch(gpu, kind, [300, 200, 90, 70], heads=8, kv_heads=2, head_dim=32, bias="table", far=far, spread=3.0)
    batch = Batch(gpu, kind, q_lens, k_lens=k_lens, heads=8, kv_heads=2, head_dim=32, mask="causal", bias="table", far=far, room=room)
    check(before)
    grad, got = check(batch)
    first = {name: values.copy() for name, values in got.items()}
    for _ in range(3):
        check(before)
        grad.call()
        gpu.synchronize()
        assert all(np.array_equal(first[name], values) for name, values in grad.read().items())
