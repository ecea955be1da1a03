"""The shared projection with per-row low-rank adapters against the formula in 64 bits: orders of the
rows, ranks, rows without an adapter, odd sizes, strides and alignments."""

import math

import numpy as np
import pytest

from operator_helpers import FLOOR, UNIT, Output, kind_code, strided, to_bits

pytestmark = pytest.mark.gpu

STEP = 2.0 ** -23  # one float32 addition of the matrix cores, whose rounding need not be to nearest


class Case:
    def __init__(self, capi, kind, out, rows, dim, width, adapters, rank, order, pad=0, shift=0, seed=1, with_ranks=True,
                 spoil=None):
        rng = np.random.default_rng(seed)
        self.capi, self.kind, self.rows, self.width = capi, kind, rows, width
        size = 4 if kind == "f32" else 2
        self.keep = []

        def put(values):
            owner, address, stride, stored = strided(capi, values, kind, pad, shift)
            self.keep.append(owner)
            return address, stride, stored

        x_ptr, x_stride, x = put(rng.standard_normal((rows, dim)))
        w_ptr, w_stride, w = put(rng.standard_normal((width, dim)) / math.sqrt(dim))
        if order == "mixed":
            ids = rng.integers(-1, adapters + 1, rows)
        elif order == "runs":
            ids = np.repeat(rng.integers(-1, adapters, rows), 37)[:rows]
        elif order == "one":
            ids = np.full(rows, adapters - 1)
        else:
            ids = np.full(rows, -1)
        self.ids = ids = ids.astype(np.int32)
        ranks = rng.integers(0, rank + 1, adapters).astype(np.int32)
        ranks[-1] = rank
        scales = (0.25 + rng.random(adapters)).astype(np.float32)
        if not with_ranks:
            ranks[:], scales[:] = rank, 1.0
        down = rng.standard_normal((adapters, rank, dim)) / math.sqrt(dim)
        up = rng.standard_normal((adapters, width, rank)) / math.sqrt(rank)
        if spoil:
            spoil(down, up)
        for a in range(adapters):  # what lies past an adapter's rank is not used
            down[a, ranks[a]:] = np.nan
            up[a, :, ranks[a]:] = np.nan
        d_down, d_up = (np.concatenate([np.zeros(shift, to_bits(v[:0], kind).dtype), to_bits(v, kind).ravel()])
                        for v in (down, up))
        arrays = [capi.DeviceArray.from_host(a) for a in (d_down, d_up, ids, ranks, scales)]
        self.keep += arrays
        self.desc = capi.adapted_desc(x_ptr, rows, dim, w_ptr, width, kind_code(capi, kind), x_stride=x_stride,
                                      weight_stride=w_stride, down=arrays[0].ptr + shift * size,
                                      up=arrays[1].ptr + shift * size, adapter_count=adapters, max_rank=rank,
                                      ranks=arrays[3] if with_ranks else None, scales=arrays[4] if with_ranks else None,
                                      adapter_ids=arrays[2])
        from operator_helpers import from_bits
        down, up = (from_bits(to_bits(v, kind), kind) for v in (down, up))
        self.expected = x @ w.T
        mass = np.abs(x) @ np.abs(w).T
        extra = np.zeros_like(mass)
        split = {"f32": 0.0, "f16": 2.0 ** -22, "bf16": 2.0 ** -16}[kind]
        for a in range(adapters):
            at = np.nonzero(ids == a)[0]
            if at.size == 0 or ranks[a] == 0:
                continue
            low_down, low_up = down[a, :ranks[a]], up[a, :, :ranks[a]]
            low = float(scales[a]) * (x[at] @ low_down.T)
            low_mass = float(scales[a]) * (np.abs(x[at]) @ np.abs(low_down).T)
            low_error = (dim + 6) * STEP * low_mass + split * np.abs(low)
            low_error += 2.0 ** -38 * np.abs(low).max(axis=1, keepdims=True)
            self.expected[at] += low @ low_up.T
            part = (np.abs(low) + low_error) @ np.abs(low_up).T
            mass[at] += part
            extra[at] += low_error @ np.abs(low_up).T + 2 * (ranks[a] + 2) * STEP * part
        # the tile's sums start with the adapter's part and add the dim products to it
        error = extra + (dim + 2) * STEP * mass
        self.tolerance = error + UNIT[out] * (np.abs(self.expected) + error) + FLOOR[out]

    def run(self, out, pad=0, shift=0):
        capi = self.capi
        got = Output(capi, self.rows, self.width, out, pad, shift)
        size = capi.adapted_projection_workspace_bytes(self.desc)
        workspace = capi.DeviceArray.from_host(np.full(size, 0xFF, np.uint8))
        capi.adapted_projection(self.desc, got.ptr, kind_code(capi, out), workspace, size, out_stride=got.stride)
        capi.synchronize()
        return got.read()


CASES = [
    # kind, out, rows, dim, width, adapters, rank, order, pad, shift
    ("f32", "f32", 1, 1, 1, 1, 1, "one", 0, 0),
    ("f16", "f32", 1, 768, 384, 3, 16, "one", 0, 0),
    ("f16", "f32", 8, 768, 384, 64, 16, "mixed", 0, 0),
    ("bf16", "bf16", 16, 100, 33, 4, 8, "mixed", 0, 0),
    ("bf16", "f32", 17, 96, 130, 5, 64, "mixed", 8, 0),
    ("f32", "f32", 33, 72, 65, 6, 20, "mixed", 1, 1),
    ("f16", "f16", 65, 200, 128, 1, 128, "mixed", 0, 8),
    ("f16", "f32", 300, 136, 260, 200, 8, "mixed", 3, 1),
    ("bf16", "bf16", 500, 64, 128, 7, 33, "runs", 0, 0),
    ("f32", "f32", 129, 256, 100, 2, 100, "runs", 0, 0),
    ("f16", "f16", 70, 64, 64, 3, 4, "none", 0, 0),
    ("bf16", "f32", 2100, 72, 2050, 40, 32, "mixed", 0, 0),
    ("f16", "f16", 2100, 70, 2051, 600, 16, "mixed", 1, 0),
    ("f32", "f32", 2100, 36, 2048, 12, 12, "runs", 4, 0),
    ("f16", "f32", 9001, 64, 64, 1000, 8, "mixed", 0, 0),
]


@pytest.mark.parametrize("case", CASES, ids=str)
def test_projection(gpu, case):
    kind, out, rows, dim, width, adapters, rank, order, pad, shift = case
    c = Case(gpu, *case)
    first = c.run(out, pad, shift)
    assert np.all(np.abs(first - c.expected) <= c.tolerance)
    assert np.array_equal(first, c.run(out, pad, shift))


def test_no_ranks_and_no_scales(gpu):
    c = Case(gpu, "f16", "f32", 50, 80, 90, 5, 12, "mixed", with_ranks=False)
    assert np.all(np.abs(c.run("f32") - c.expected) <= c.tolerance)


def test_no_adapters(gpu):
    """Without adapter ids the projection alone, and no workspace."""
    capi = gpu
    rng = np.random.default_rng(3)
    x, w = rng.standard_normal((77, 64)).astype(np.float32), rng.standard_normal((50, 64)).astype(np.float32)
    d_x, d_w = capi.DeviceArray.from_host(x), capi.DeviceArray.from_host(w)
    out = capi.DeviceArray((77, 50), np.float32)
    desc = capi.adapted_desc(d_x, 77, 64, d_w, 50, capi.F32)
    capi.adapted_projection(desc, out, capi.F32, None, 0)
    capi.synchronize()
    x, w = x.astype(np.float64), w.astype(np.float64)
    assert np.all(np.abs(out.to_host() - x @ w.T) <= 68 * STEP * (np.abs(x) @ np.abs(w).T))


def test_large_low_rank_values(gpu):
    """x down^T far beyond float16's range, brought back by small values of up."""

    def spoil(down, up):
        down *= 2.0 ** 12
        up *= 2.0 ** -12

    c = Case(gpu, "f16", "f32", 40, 512, 64, 2, 16, "mixed", spoil=spoil)
    got = c.run("f32")
    assert np.all(np.isfinite(got)) and np.all(np.abs(got - c.expected) <= c.tolerance)


def test_spoiled_adapters_stay_in_their_rows(gpu):
    """Infinities and NaN in one adapter reach the rows that name it and no others."""

    def spoil(down, up):
        down[1, 0, 0] = np.nan
        up[2, :, 0] = np.inf

    c = Case(gpu, "f16", "f32", 200, 64, 96, 5, 8, "mixed", with_ranks=False, spoil=spoil)
    got = c.run("f32")
    bad = (c.ids == 1) | (c.ids == 2)
    assert bad.any() and (~bad).any()
    assert np.all(np.abs(got[~bad] - c.expected[~bad]) <= c.tolerance[~bad])
    assert not np.any(np.isfinite(got[bad]))


@pytest.mark.parametrize("kind,out", [("f32", "f32"), ("f16", "f32"), ("bf16", "bf16")])
def test_a_row_does_not_depend_on_its_batch(gpu, kind, out):
    """The result of a row is within its own error wherever it stands among other rows."""
    c = Case(gpu, kind, out, 190, 128, 64, 9, 16, "mixed")
    order = np.argsort(c.ids, kind="stable")
    got = c.run(out)
    for rows in (order[:5], order[-64:]):
        assert np.all(np.abs(got[rows] - c.expected[rows]) <= c.tolerance[rows])
