"""The same rows in different batches: among few and many others, of few and many adapters, some of which hold NaN and
infinities. A row's result stays within the formula's error in each of them."""

import pytest
import torch

from test_gpu_adapted_large import Case

pytestmark = pytest.mark.gpu

ROWS, DIM, WIDTH, RANK, SHARED = 40, 64, 96, 16, 3
# rows, adapters, rows after each other with one adapter: one launch for low, sorted with one adapter after the other,
# sorted and row by row
BATCHES = [(300, 5, 1), (6000, 5, 300), (6000, 600, 1)]
SPOILED = {3: float("nan"), 4: float("inf")}


def _alone(kind):
    c = Case(kind, ROWS, DIM, WIDTH, SHARED, RANK, 1, seed=81)
    c.ranks[0] = RANK
    c.ids.clamp_(max=SHARED - 1)
    return c


def _among(alone, kind, rows, adapters, run):
    """The rows of `alone` at random places of another batch -> (batch, places)."""
    c = Case(kind, rows, DIM, WIDTH, adapters, RANK, run, seed=82)
    c.weight = alone.weight
    c.down[:SHARED], c.up[:SHARED] = alone.down, alone.up
    c.ranks[:SHARED], c.scales[:SHARED] = alone.ranks, alone.scales
    for adapter, value in SPOILED.items():
        c.ranks[adapter] = RANK
        c.down[adapter, 0], c.up[adapter, :, 1] = value, value
    rng = torch.Generator().manual_seed(83)
    order = torch.randperm(rows, generator=rng).cuda()
    at = order[:ROWS]
    c.x[order[ROWS:ROWS + 20]] = float("nan")
    c.x[at], c.ids[at] = alone.x, alone.ids
    return c, at


@pytest.mark.parametrize("kind,out", [("f32", "f32"), ("f16", "f32"), ("bf16", "f32"), ("bf16", "bf16")])
def test_rows_in_different_batches(gpu, kind, out):
    alone = _alone(kind)
    expected, tolerance = alone.expected(out)
    assert torch.all((alone.run(gpu, out).double() - expected).abs() <= tolerance)
    for batch in BATCHES:
        c, at = _among(alone, kind, *batch)
        got = c.run(gpu, out)
        assert torch.isnan(got).any(), batch  # the spoiled rows are there
        assert torch.all((got[at].double() - expected).abs() <= tolerance), batch
        assert torch.equal(got[at], c.run(gpu, out)[at]), batch
