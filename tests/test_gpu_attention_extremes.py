"""Attention where its calls reach what ordinary batches do not: keys that no query row stands before, caps far above and
below the scores."""

import numpy as np
import pytest

from attention_helpers import STEP, Batch
from operator_helpers import UNIT, from_bits, kind_code, to_bits
from test_gpu_attention import check as forward
from test_gpu_attention_gradient import Gradient, check

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


class Capped(Batch):
    """A batch whose allowance goes by the scores, not by their cap, where the cap is large."""

    def scores(self, q, k, distance, table=None):
        x = q @ k.transpose(0, 2, 1) * self.scale
        error = (self.head_dim + 4) * STEP * abs(self.scale) * (np.abs(q) @ np.abs(k).transpose(0, 2, 1))
        t = np.tanh(x / self.cap)
        c = self.cap * t
        # the tangent is within 2^-20 of its value (float32: two units in the last place, 2^-22; 16-bit under caps of up to 64
        # off by 2^-21); its argument takes three roundings of 2^-24, log2(e) cap two and the product one: 2^-19 in all
        error = error * (1.0 - t * t) + 2.0 ** -19 * np.abs(c)
        if self.kind != "f32" and self.cap <= 64.0:
            error = error + 2.0 ** -21 * self.cap
        if self.slopes is not None:
            c = c - self.slopes.astype(np.float64)[:, None, None] * np.abs(distance)
        table = self.table if table is None else table
        if table is not None:
            c = c + table[:, np.clip(distance, -self.far, self.far) + self.far]
        size = np.abs(c)
        return c, 1.0 - t * t, error + 2.0 ** -21 * (size + (size.max(2, keepdims=True) if size.shape[2] else 0.0))


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("cap", [1e-39, 1e-7, 0.5, 5.0, 50.0, 1e4, 1e6, 1e8, 3e38])
@pytest.mark.parametrize("bias", [None, "slopes", "table"])
def test_caps_of_any_size(gpu, kind, cap, bias):
    """Scores of some units under caps far above them are the scores themselves, under caps far below their signs."""
    cap = float(np.float32(cap))
    b = Capped(gpu, kind, [130, 1, 45], heads=4, kv_heads=2, head_dim=64, mask="causal", bias=bias, far=7 if bias == "table" else 0,
               cap=cap, spread=1.5)
    forward(b)
    if cap >= 50.0:
        # a score's error of up to 1.5e-4 (68 additions over products of up to 19) changes its slope by 0.77 / cap of that,
        # below the 2^-18 that a slope is allowed
        check(b)
    else:
        grad = Gradient(b)
        grad.call()
        gpu.synchronize()
        assert all(np.all(np.isfinite(values)) for values in grad.read().values())


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("cap", [3.0, 1e5])
def test_caps_over_split_keys(gpu, kind, cap):
    """One query row over long keys, split over workgroups."""
    forward(Capped(gpu, kind, [1], k_lens=[5000], heads=8, kv_heads=2, head_dim=128, last=True, cap=cap))


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("cap", [1e-39, 1e6, 3e38])
def test_scores_of_zero_under_any_cap(gpu, kind, cap):
    """Keys of zeros: every key counts the same, and no NaN comes of 0 times an infinity."""
    capi = gpu
    rows, width = 40, 16
    rng = np.random.default_rng(3)
    q, v = (to_bits(rng.standard_normal((rows, width)), kind) for _ in range(2))
    d_q, d_k, d_v = map(capi.DeviceArray.from_host, (q, np.zeros_like(q), v))
    out, lse = capi.DeviceArray((rows, width), q.dtype), capi.DeviceArray((rows, 1), np.float32)
    desc = capi.attention_desc(d_q, d_k, d_v, 1, rows, rows, 1, width, kind_code(capi, kind), cap=cap)
    size = capi.attention_workspace_bytes(desc)
    capi.attention(desc, out, capi.DeviceArray(size, np.uint8), size, lse=lse)
    capi.synchronize()
    mean = from_bits(v, kind).mean(0)
    # rows of equal weights: sums of 40 values, the weights' and the results' roundings
    allowed = 2 * (UNIT[kind] + 48 * STEP) * np.abs(from_bits(v, kind)).mean(0)
    assert np.all(np.abs(from_bits(out.to_host(), kind) - mean) <= allowed)
    assert np.allclose(lse.to_host(), np.log(rows), rtol=2.0 ** -20)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("mask", ["full", "causal"])
def test_one_long_text_among_short_ones(gpu, kind, mask):
    """The kernel for few rows is chosen by the mean of a text's rows: it takes a long text as well."""
    b = Batch(gpu, kind, [1] * 40 + [700] + [0, 2] * 30, heads=2, head_dim=64, mask=mask, bias="table", far=9)
    assert b.q_rows / b.texts <= 16
    forward(b)
    check(b)
