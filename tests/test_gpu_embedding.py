"""Token-table lookup and its gradient against the formulas in 64 bits, at the sizes, ids, bags and
strides where they can go wrong."""

import numpy as np
import pytest

from operator_helpers import FLOOR, UNIT, Output, kind_code, strided

pytestmark = pytest.mark.gpu

def make_ids(rng, vocab, tokens, padding_id):
    ids = np.minimum((rng.pareto(0.6, tokens)).astype(np.int64), vocab - 1).astype(np.int32)
    if tokens > 4:
        ids[rng.integers(0, tokens, max(1, tokens // 20))] = -1
        ids[rng.integers(0, tokens, max(1, tokens // 20))] = vocab  # one past the table
        ids[rng.integers(0, tokens, max(1, tokens // 20))] = padding_id
        ids[1], ids[3] = -2 ** 31, 2 ** 31 - 1
    return ids


def make_offsets(rng, tokens, bags):
    if bags == 0:
        return None
    cuts = np.sort(rng.integers(0, tokens + 1, bags + 1))
    cuts[0], cuts[-1] = 0, tokens
    if bags > 2:
        cuts[1] = 0  # an empty first bag
        cuts[-2] = tokens  # and an empty last one
    return cuts.astype(np.int64)


def weights_of(ids, offsets, vocab, padding_id, mean, scale):
    """Per token: whether it counts, its output row, its weight."""
    ok = (ids >= 0) & (ids < vocab) & (ids != padding_id)
    if offsets is None:
        return ok, np.arange(ids.size), np.full(ids.size, scale)
    row = np.searchsorted(offsets, np.arange(ids.size), side="right") - 1
    inside = (row >= 0) & (row < offsets.size - 1)
    ok = ok & inside
    row = np.where(inside, row, 0)
    count = np.bincount(row[ok], minlength=offsets.size - 1)
    return ok, row, scale / np.maximum(count[row], 1) if mean else np.full(ids.size, scale)


CASES = [
    # kind, out, vocab, dim, tokens, bags, mean, padding_id, pad, shift, scale
    ("f32", "f32", 10, 1, 1, 0, False, -1, 0, 0, 1.0),
    ("f16", "f16", 100, 64, 24, 0, False, 0, 0, 0, 8.0),
    ("bf16", "bf16", 1000, 96, 513, 0, False, 3, 8, 0, 0.5),
    ("f16", "f32", 1000, 100, 300, 0, False, -1, 4, 0, 1.0),
    ("bf16", "f32", 511, 33, 1025, 0, False, 0, 1, 1, 3.0),
    ("f32", "f32", 513, 260, 700, 0, False, 0, 3, 2, 1.0),
    ("f32", "f32", 300, 384, 2000, 40, True, 0, 0, 0, 1.0),
    ("f16", "f16", 300, 130, 900, 1, True, 5, 2, 0, 2.0),
    ("bf16", "f32", 262_144, 12, 5000, 333, False, 0, 0, 0, 1.0),
    ("f16", "f32", 70_000, 1028, 700, 64, True, -1, 0, 0, 1.0),
    ("f32", "f32", 5, 7, 3000, 3000, True, 1, 1, 1, 1.0),
    ("bf16", "bf16", 2, 2048, 66, 0, False, -1, 0, 0, 1.0),
]


def _setup(capi, case, seed):
    kind, out, vocab, dim, tokens, bags, mean, padding_id, pad, shift, scale = case
    rng = np.random.default_rng(seed)
    ids = make_ids(rng, vocab, tokens, padding_id)
    offsets = make_offsets(rng, tokens, bags)
    return rng, ids, offsets, weights_of(ids, offsets, vocab, padding_id, mean, float(np.float32(scale)))


def _desc(capi, case, table, table_stride, ids, offsets):
    kind, out, vocab, dim, tokens, bags, mean, padding_id, pad, shift, scale = case
    d_ids = capi.DeviceArray.from_host(ids)
    d_offsets = None if offsets is None else capi.DeviceArray.from_host(offsets)
    desc = capi.embedding_desc(table, vocab, dim, kind_code(capi, kind), d_ids, tokens, bag_offsets=d_offsets,
                               bag_count=bags, reduce=capi.EMBEDDING_MEAN if mean else capi.EMBEDDING_SUM,
                               padding_id=padding_id, scale=scale, table_stride=table_stride)
    return desc


@pytest.mark.parametrize("case", CASES, ids=str)
def test_lookup(gpu, case):
    capi = gpu
    kind, out, vocab, dim, tokens, bags, mean, padding_id, pad, shift, scale = case
    rng, ids, offsets, (ok, row, weight) = _setup(capi, case, 11)
    values = rng.standard_normal((vocab, dim))
    if 0 <= padding_id < vocab:
        values[padding_id] = np.inf  # never read
    owner, address, stride, table = strided(capi, values, kind, pad, shift)
    desc = _desc(capi, case, address, stride, ids, offsets)
    rows = bags or tokens
    got = Output(capi, rows, dim, out, pad, shift)
    capi.embedding_lookup(desc, got.ptr, kind_code(capi, out), out_stride=got.stride)
    capi.synchronize()
    expected, mass = np.zeros((rows, dim)), np.zeros((rows, dim))
    np.add.at(expected, row[ok], table[ids[ok]] * weight[ok, None])
    np.add.at(mass, row[ok], np.abs(table[ids[ok]] * weight[ok, None]))
    # n float32 additions and two products, then the rounding of the result
    n = np.zeros(rows)
    np.add.at(n, row[ok], 1)
    tolerance = (n[:, None] + 4) * 2.0 ** -24 * mass + UNIT[out] * np.abs(expected) + FLOOR[out]
    result = got.read()
    assert np.all(np.abs(result - expected) <= tolerance)
    assert np.all(result[n == 0] == 0.0)


@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("case", CASES, ids=str)
def test_gradient(gpu, case, accumulate):
    capi = gpu
    kind, out, vocab, dim, tokens, bags, mean, padding_id, pad, shift, scale = case
    rng, ids, offsets, (ok, row, weight) = _setup(capi, case, 12)
    rows = bags or tokens
    values = rng.standard_normal((rows, dim))
    none = np.ones(rows, bool)
    none[row[ok]] = False
    values[none] = np.nan  # gradients of rows of zeros are never read
    owner, address, stride, d_out = strided(capi, values, kind, pad, shift)
    desc = _desc(capi, case, None, 0, ids, offsets)
    start = rng.standard_normal((vocab, dim)) if accumulate else None
    got = Output(capi, vocab, dim, out, pad, shift, fill=start)
    before = got.read()
    size = capi.embedding_gradient_workspace_bytes(desc)
    results = []
    for _ in range(1 if accumulate else 2):
        # a workspace of all ones: nothing may rely on its contents
        workspace = capi.DeviceArray.from_host(np.full(size, 0xFF, np.uint8))
        capi.embedding_gradient(desc, address, kind_code(capi, kind), got.ptr, kind_code(capi, out), workspace, size,
                                out_gradient_stride=stride, table_gradient_stride=got.stride, accumulate=accumulate)
        capi.synchronize()
        results.append(got.read())
    result = results[-1]
    assert all(np.array_equal(result, r) for r in results)
    expected, mass, n = np.zeros((vocab, dim)), np.zeros((vocab, dim)), np.zeros(vocab)
    np.add.at(expected, ids[ok], d_out[row[ok]] * weight[ok, None])
    np.add.at(mass, ids[ok], np.abs(d_out[row[ok]] * weight[ok, None]))
    np.add.at(n, ids[ok], 1)
    if accumulate:
        expected += before
        mass += np.abs(before)
        assert np.array_equal(result[n == 0], before[n == 0]), "rows of absent tokens are not touched"
    else:
        assert np.all(result[n == 0] == 0.0)
    # n additions, the mean's reciprocal and product, the scale, the addition to what was there
    tolerance = (n[:, None] + 6) * 2.0 ** -24 * mass + UNIT[out] * np.abs(expected) + FLOOR[out]
    assert np.all(np.abs(result - expected) <= tolerance)


FEW_CASES = [
    ("f32", "f32", 40, 5, 2, 2, True, -1, 0, 0, 1.0),
    ("f16", "f32", 300, 130, 60, 7, True, 5, 2, 0, 2.0),
    ("bf16", "bf16", 2, 1028, 511, 0, False, -1, 0, 0, 1.0),
    ("f32", "f32", 7, 384, 512, 40, True, 0, 3, 1, 1.0),
    ("bf16", "f32", 30_000, 260, 512, 1, False, 0, 0, 0, 0.5),
    ("f32", "f32", 2_200_001, 4, 100, 0, False, -1, 0, 0, 1.0),
    ("f16", "f16", 5000, 2051, 9, 0, False, 0, 3, 0, 1.0),
]


@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("case", FEW_CASES, ids=str)
def test_gradient_of_few_tokens(gpu, case, accumulate):
    """Up to 512 tokens are not sorted: bags, one id at nearly all positions, several slices of columns."""
    test_gradient(gpu, case, accumulate)


def test_gradient_is_the_difference_of_the_lookup(gpu):
    """A step in one table entry changes the weighted sum of the outputs by the gradient's entry."""
    capi = gpu
    case = ("f32", "f32", 40, 20, 200, 17, True, 0, 0, 0, 2.0)
    kind, out, vocab, dim, tokens, bags, mean, padding_id, pad, shift, scale = case
    rng, ids, offsets, _ = _setup(capi, case, 13)
    table = rng.integers(-8, 9, (vocab, dim)).astype(np.float32)
    weight = rng.integers(-4, 5, (bags, dim)).astype(np.float32)
    d_weight = capi.DeviceArray.from_host(weight)
    grad, rows = capi.DeviceArray((vocab, dim), np.float32), capi.DeviceArray((bags, dim), np.float32)
    desc = _desc(capi, case, None, 0, ids, offsets)
    size = capi.embedding_gradient_workspace_bytes(desc)
    workspace = capi.DeviceArray(size, np.uint8)
    capi.embedding_gradient(desc, d_weight, capi.F32, grad, capi.F32, workspace, size)

    def loss(t):
        d_table = capi.DeviceArray.from_host(t)
        capi.embedding_lookup(_desc(capi, case, d_table, 0, ids, offsets), rows, capi.F32)
        capi.synchronize()
        return float((rows.to_host().astype(np.float64) * weight).sum())

    base, gradient = loss(table), grad.to_host()
    for v, c in [(0, 0), (1, 3), (2, 19), (3, 7), (39, 5)]:
        stepped = table.copy()
        stepped[v, c] += 16.0  # the lookup is linear: any step will do
        # the loss is a sum of about 340 products of size below 100, each to 2^-22 of its size
        assert abs((loss(stepped) - base) / 16.0 - gradient[v, c]) <= 340 * 100 * 2.0 ** -22 / 16.0 * 2


@pytest.mark.parametrize("tokens", [4096 * 3 + 1, 300_001])
def test_gradient_of_one_frequent_token(gpu, tokens):
    """One token at almost all positions: its run crosses every chunk and every sorting tile."""
    capi = gpu
    vocab, dim = 600, 8
    rng = np.random.default_rng(14)
    ids = np.full(tokens, 517, np.int32)
    ids[rng.integers(0, tokens, tokens // 100)] = 5
    ids[-1] = 599
    # whole numbers: float32 sums are exact, whatever their order
    d_out = rng.integers(-3, 4, (tokens, dim)).astype(np.float32)
    d_ids, d_from = capi.DeviceArray.from_host(ids), capi.DeviceArray.from_host(d_out)
    desc = capi.embedding_desc(None, vocab, dim, capi.F32, d_ids, tokens)
    size = capi.embedding_gradient_workspace_bytes(desc)
    workspace, got = capi.DeviceArray(size, np.uint8), capi.DeviceArray((vocab, dim), np.float32)
    capi.embedding_gradient(desc, d_from, capi.F32, got, capi.F32, workspace, size)
    capi.synchronize()
    expected = np.zeros((vocab, dim))
    np.add.at(expected, ids, d_out)
    assert np.array_equal(got.to_host(), expected)


def test_no_tokens(gpu):
    capi = gpu
    offsets = capi.DeviceArray.from_host(np.zeros(4, np.int64))
    table = capi.DeviceArray.from_host(np.ones((5, 6), np.float32))
    desc = capi.embedding_desc(table, 5, 6, capi.F32, None, 0, bag_offsets=offsets, bag_count=3)
    out = capi.DeviceArray.from_host(np.ones((3, 6), np.float32))
    capi.embedding_lookup(desc, out, capi.F32)
    grad = capi.DeviceArray.from_host(np.ones((5, 6), np.float32))
    desc = capi.embedding_desc(None, 5, 6, capi.F32, None, 0)
    capi.embedding_gradient(desc, None, capi.F32, grad, capi.F32, None, 0, accumulate=True)
    capi.synchronize()
    assert np.all(out.to_host() == 0.0) and np.all(grad.to_host() == 1.0)
    capi.embedding_gradient(desc, None, capi.F32, grad, capi.F32, None, 0)
    capi.synchronize()
    assert np.all(grad.to_host() == 0.0)


def test_tokens_of_no_bag(gpu):
    """Without bags no token counts, and every row of the gradient is zeros."""
    capi = gpu
    ids = capi.DeviceArray.from_host(np.arange(4, dtype=np.int32))
    offsets = capi.DeviceArray.from_host(np.zeros(1, np.int64))
    grad = capi.DeviceArray.from_host(np.ones((5, 6), np.float32))
    desc = capi.embedding_desc(None, 5, 6, capi.F32, ids, 4, bag_offsets=offsets, bag_count=0)
    capi.embedding_gradient(desc, None, capi.F32, grad, capi.F32, None, 0, accumulate=True)
    capi.synchronize()
    assert np.all(grad.to_host() == 1.0)
    capi.embedding_gradient(desc, None, capi.F32, grad, capi.F32, None, 0)
    capi.synchronize()
    assert np.all(grad.to_host() == 0.0)


def test_offsets_outside_the_tokens(gpu):
    """Bags that reach past the token list are cut to it, and tokens before the first bag are in none."""
    capi = gpu
    ids = np.arange(10, dtype=np.int32)
    offsets = np.array([3, 5, 5, 40], np.int64)
    table = np.arange(10, dtype=np.float32)[:, None] * np.ones(4, np.float32)
    d_ids, d_offsets, d_table = (capi.DeviceArray.from_host(a) for a in (ids, offsets, table))
    out = capi.DeviceArray((3, 4), np.float32)
    desc = capi.embedding_desc(d_table, 10, 4, capi.F32, d_ids, 10, bag_offsets=d_offsets, bag_count=3)
    capi.embedding_lookup(desc, out, capi.F32)
    grad, d_from = capi.DeviceArray((10, 4), np.float32), capi.DeviceArray.from_host(np.ones((3, 4), np.float32))
    size = capi.embedding_gradient_workspace_bytes(desc)
    workspace = capi.DeviceArray(size, np.uint8)
    capi.embedding_gradient(desc, d_from, capi.F32, grad, capi.F32, workspace, size)
    capi.synchronize()
    assert out.to_host()[:, 0].tolist() == [7.0, 0.0, 35.0]
    assert grad.to_host()[:, 0].tolist() == [0.0] * 3 + [1.0] * 7


def test_table_beyond_32_bit_offsets(gpu):
    """Rows of a table of more than 2^32 bytes and 2^31 elements."""
    capi = gpu
    vocab, dim = 2_200_003, 1024
    table = capi.DeviceArray((vocab, dim), np.uint16)
    ids = np.array([0, 1_100_000, 2_097_153, vocab - 1], np.int32)
    for i, v in enumerate(ids):
        row = np.full(dim, i + 1, np.float16)
        capi.call("zcgvs_memcpy_h2d", table.ptr + int(v) * dim * 2, row.ctypes.data, row.nbytes, None)
    capi.synchronize()
    d_ids, out = capi.DeviceArray.from_host(ids), capi.DeviceArray((4, dim), np.float16)
    capi.embedding_lookup(capi.embedding_desc(table, vocab, dim, capi.F16, d_ids, 4), out, capi.F16)
    capi.synchronize()
    assert np.array_equal(out.to_host(), np.repeat(np.arange(1, 5, dtype=np.float16), dim).reshape(4, dim))
