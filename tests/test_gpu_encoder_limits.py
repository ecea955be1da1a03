"""The encoder block's operators at the ends of what their calls allow: rows billions of values apart, many texts, calls
at once on two streams, biases that leave keys out, int8 rows from the norm to the product."""

import numpy as np
import pytest

from attention_helpers import Batch
from operator_helpers import from_bits, kind_code, to_bits
from test_gpu_attention_gradient import check

pytestmark = pytest.mark.gpu

FAR = ((1 << 31) // 100 // 8 + 1) * 8  # elements from row to row: a hundred rows pass 2^31


def spread_out(capi, rows, stride):
    """float16 rows `stride` elements apart; nothing is read or written between them."""
    count, width = rows.shape
    array = capi.DeviceArray(((count - 1) * stride + width,), np.float16)
    for r in range(count):
        row = np.ascontiguousarray(rows[r])
        capi.call("zcgvs_memcpy_h2d", array.ptr + 2 * r * stride, row.ctypes.data, row.nbytes, None)
    capi.synchronize()
    return array


def gather(capi, array, count, width, stride):
    out = np.empty((count, width), np.float16)
    capi.synchronize()
    for r in range(count):
        capi.call("zcgvs_memcpy_d2h", out[r].ctypes.data, array.ptr + 2 * r * stride, 2 * width, None)
    capi.synchronize()
    return out


def workspace(capi, size):
    return capi.DeviceArray(max(size, 1), np.uint8)


def test_linear_rows_far_apart(gpu):
    """The same bits as from packed rows: which kernel runs goes by sizes and alignment, and both are the same."""
    capi = gpu
    rng = np.random.default_rng(1)
    rows, dim, width = 130, 64, 72
    x, w, dy = (to_bits(rng.standard_normal(s), "f16") for s in ((rows, dim), (width, dim), (rows, width)))
    results = []
    for stride_x, stride_y in ((dim, width), (FAR, FAR)):
        d_x, d_w, d_dy = spread_out(capi, x, stride_x), capi.DeviceArray.from_host(w), spread_out(capi, dy, stride_y)
        desc = capi.linear_desc(d_x, rows, dim, d_w, width, capi.F16, activation=capi.ACT_SILU, residual=d_dy,
                                x_stride=stride_x, residual_stride=stride_y)
        out = capi.DeviceArray(((rows - 1) * stride_y + width,), np.float16)
        capi.linear(desc, out, capi.F16, out_stride=stride_y)
        got = [gather(capi, out, rows, width, stride_y)]
        dx = capi.DeviceArray(((rows - 1) * stride_x + dim,), np.float16)
        dw = capi.DeviceArray((width, dim), np.float16)
        size = capi.linear_gradient_workspace_bytes(desc)
        capi.linear_gradient(desc, d_dy, dx, dw, None, workspace(capi, size), size, out_gradient_stride=stride_y,
                             x_gradient_stride=stride_x)
        got += [gather(capi, dx, rows, dim, stride_x), dw.to_host()]
        results.append(got)
    for near, far in zip(*results):
        assert np.array_equal(near, far)
    z = x.astype(np.float64) @ w.astype(np.float64).T
    assert np.allclose(results[1][0], z / (1 + np.exp(-z)) + dy, rtol=2.0 ** -9, atol=2.0 ** -9)


def test_norm_rows_far_apart(gpu):
    capi = gpu
    rng = np.random.default_rng(2)
    rows, dim = 130, 72
    x, more, dy = (to_bits(rng.standard_normal((rows, dim)), "f16") for _ in range(3))
    weight = capi.DeviceArray.from_host(to_bits(rng.standard_normal(dim), "f16"))
    results = []
    for stride in (dim, FAR):
        d_x, d_more, d_dy = (spread_out(capi, a, stride) for a in (x, more, dy))
        desc = capi.norm_desc(d_x, rows, dim, capi.F16, weight=weight, residual=d_more, x_stride=stride, residual_stride=stride)
        out, total, dx = (capi.DeviceArray(((rows - 1) * stride + dim,), np.float16) for _ in range(3))
        capi.residual_norm(desc, out, capi.F16, sum_out=total, out_stride=stride, sum_stride=stride)
        dw = capi.DeviceArray((dim,), np.float16)
        size = capi.residual_norm_gradient_workspace_bytes(desc)
        capi.residual_norm_gradient(desc, d_dy, dx, dw, workspace(capi, size), size, out_gradient_stride=stride,
                                    x_gradient_stride=stride)
        results.append([gather(capi, a, rows, dim, stride) for a in (out, total, dx)] + [dw.to_host()])
    for near, far in zip(*results):
        assert np.array_equal(near, far)


@pytest.mark.parametrize("lens", [[130], [1, 100, 29]], ids=str)
def test_attention_rows_far_apart(gpu, lens):
    capi = gpu
    rng = np.random.default_rng(3)
    rows, heads, head_dim = 130, 2, 32
    width = heads * head_dim
    q, k, v, dy = (to_bits(rng.standard_normal((rows, width)), "f16") for _ in range(4))
    offsets = capi.DeviceArray.from_host(np.concatenate([[0], np.cumsum(lens)]).astype(np.int64))
    results = []
    for stride in (width, FAR):
        d_q, d_k, d_v, d_dy = (spread_out(capi, a, stride) for a in (q, k, v, dy))
        desc = capi.attention_desc(d_q, d_k, d_v, len(lens), rows, rows, heads, head_dim, capi.F16, q_offsets=offsets,
                                   k_offsets=offsets, causal=True, q_stride=stride, k_stride=stride, v_stride=stride)
        out, dq, dk, dv = (capi.DeviceArray(((rows - 1) * stride + width,), np.float16) for _ in range(4))
        lse = capi.DeviceArray((rows, heads), np.float32)
        size = capi.attention_workspace_bytes(desc)
        capi.attention(desc, out, workspace(capi, size), size, lse=lse, out_stride=stride)
        size = capi.attention_gradient_workspace_bytes(desc)
        capi.attention_gradient(desc, out, lse, d_dy, dq, dk, dv, workspace(capi, size), size, out_stride=stride,
                                out_gradient_stride=stride, q_gradient_stride=stride, k_gradient_stride=stride,
                                v_gradient_stride=stride)
        results.append([gather(capi, a, rows, width, stride) for a in (out, dq, dk, dv)] + [lse.to_host()])
    for near, far in zip(*results):
        assert np.array_equal(near, far)


def test_more_texts_than_blocks_of_a_smaller_launch(gpu):
    """400,000 texts of one row and 16 heads: a row that sees itself alone gives its value."""
    capi = gpu
    texts, heads, head_dim = 400_000, 16, 8
    rng = np.random.default_rng(4)
    q, k, v = (to_bits(rng.standard_normal((texts, heads * head_dim)), "f16") for _ in range(3))
    d_q, d_k, d_v = map(capi.DeviceArray.from_host, (q, k, v))
    desc = capi.attention_desc(d_q, d_k, d_v, texts, texts, texts, heads, head_dim, capi.F16)
    out, dq, dk, dv = (capi.DeviceArray((texts, heads * head_dim), np.float16) for _ in range(4))
    lse = capi.DeviceArray((texts, heads), np.float32)
    size = capi.attention_workspace_bytes(desc)
    capi.attention(desc, out, workspace(capi, size), size, lse=lse)
    size = capi.attention_gradient_workspace_bytes(desc)
    capi.attention_gradient(desc, out, lse, d_q, dq, dk, dv, workspace(capi, size), size)
    capi.synchronize()
    # one key: its probability is exp(0) to 2^-22, before and after rounding to float16
    assert np.allclose(out.to_host().astype(np.float64), v, rtol=2.0 ** -10, atol=2.0 ** -24)
    assert np.allclose(dv.to_host().astype(np.float64), q, rtol=2.0 ** -10, atol=2.0 ** -24)


def block_call(capi, rng, kind, lens):
    """One block's operators over texts with everything they need: functions that enqueue the calls, and the results."""
    code, element = kind_code(capi, kind), to_bits(np.zeros(1), kind).dtype
    rows, heads, head_dim, hidden = sum(lens), 4, 16, 96
    dim = heads * head_dim
    keep = capi.DeviceArray.from_host
    x, w_qkv, w_out, w_norm, dy = (keep(to_bits(rng.standard_normal(s) * f, kind)) for s, f in
                                   (((rows, dim), 1.0), ((3 * dim, dim), 0.2), ((dim, dim), 0.2), (dim, 1.0), ((rows, dim), 1.0)))
    offsets = keep(np.concatenate([[0], np.cumsum(lens)]).astype(np.int64))
    made = {name: capi.DeviceArray((rows, width), element) for name, width in
            dict(h=dim, qkv=3 * dim, mixed=dim, out=dim, d_mixed=dim, d_qkv=3 * dim, d_h=dim, dx=dim).items()}
    lse = capi.DeviceArray((rows, heads), np.float32)
    d_w = {name: capi.DeviceArray(shape, element) for name, shape in
           dict(out=(dim, dim), qkv=(3 * dim, dim), norm=(dim,)).items()}
    item = element.itemsize
    norm = capi.norm_desc(x, rows, dim, code, weight=w_norm)
    qkv = capi.linear_desc(made["h"], rows, dim, w_qkv, 3 * dim, code)
    attention = capi.attention_desc(made["qkv"], made["qkv"].ptr + dim * item, made["qkv"].ptr + 2 * dim * item, len(lens), rows,
                                    rows, heads, head_dim, code, q_offsets=offsets, k_offsets=offsets, q_stride=3 * dim,
                                    k_stride=3 * dim, v_stride=3 * dim)
    out = capi.linear_desc(made["mixed"], rows, dim, w_out, dim, code, residual=x)
    sizes = dict(attention=capi.attention_workspace_bytes(attention), attention_gradient=capi.attention_gradient_workspace_bytes(attention),
                 out=capi.linear_gradient_workspace_bytes(out), qkv=capi.linear_gradient_workspace_bytes(qkv),
                 norm=capi.residual_norm_gradient_workspace_bytes(norm))
    space = {name: workspace(capi, size) for name, size in sizes.items()}

    def call(stream):
        capi.residual_norm(norm, made["h"], code, stream=stream)
        capi.linear(qkv, made["qkv"], code, stream=stream)
        capi.attention(attention, made["mixed"], space["attention"], sizes["attention"], lse=lse, stream=stream)
        capi.linear(out, made["out"], code, stream=stream)
        capi.linear_gradient(out, dy, made["d_mixed"], d_w["out"], None, space["out"], sizes["out"], stream=stream)
        d_qkv = made["d_qkv"].ptr
        capi.attention_gradient(attention, made["mixed"], lse, made["d_mixed"], d_qkv, d_qkv + dim * item, d_qkv + 2 * dim * item,
                                space["attention_gradient"], sizes["attention_gradient"], q_gradient_stride=3 * dim,
                                k_gradient_stride=3 * dim, v_gradient_stride=3 * dim, stream=stream)
        capi.linear_gradient(qkv, made["d_qkv"], made["d_h"], d_w["qkv"], None, space["qkv"], sizes["qkv"], stream=stream)
        capi.residual_norm_gradient(norm, made["d_h"], made["dx"], d_w["norm"], space["norm"], sizes["norm"], sum_gradient=dy,
                                    stream=stream)

    def results():
        return [a.to_host().copy() for a in (*made.values(), lse, *d_w.values())]

    def clear():
        for a in (*made.values(), lse, *d_w.values()):
            capi.call("zcgvs_memset", a.ptr, 0xFF, a.nbytes, None)
        capi.synchronize()

    return call, results, clear


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
def test_two_streams_at_once(gpu, kind):
    """Two blocks, forward and backward, on two streams at once: each has the bits of a call of its own."""
    capi = gpu
    rng = np.random.default_rng(5)
    blocks = [block_call(capi, rng, kind, lens) for lens in ([700, 3, 90], [40, 500, 260])]
    alone = []
    for call, results, _ in blocks:
        call(None)
        capi.synchronize()
        alone.append(results())
    streams = [capi.Stream(), capi.Stream()]
    for _, _, clear in blocks:
        clear()
    for _ in range(3):
        for (call, _, _), stream in zip(blocks, streams):
            call(stream)
    for stream in streams:
        stream.synchronize()
    for (_, results, _), want in zip(blocks, alone):
        assert all(np.array_equal(a.view(np.uint8), b.view(np.uint8)) for a, b in zip(results(), want))


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_block_replays_from_graphs(gpu, kind):
    """Two graphs of whole blocks replayed in turn, with eager calls between: the eager call's bits each time."""
    capi = gpu
    rng = np.random.default_rng(6)
    blocks = [block_call(capi, rng, kind, lens) for lens in ([130, 1, 64], [20, 9])]
    stream = capi.Stream()
    want, graphs = [], []
    for call, results, _ in blocks:
        call(stream)
        stream.synchronize()
        want.append(results())
        graphs.append(capi.Graph(stream, lambda call=call: call(stream)))
    for _ in range(3):
        for (call, results, clear), graph, expected in zip(blocks, graphs, want):
            clear()
            graph.launch(stream)
            stream.synchronize()
            assert all(np.array_equal(a.view(np.uint8), b.view(np.uint8)) for a, b in zip(results(), expected))
            call(None)
            capi.synchronize()


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
def test_biases_that_leave_keys_out(gpu, kind):
    """A window by distance: biases of the type's lowest value (float16: minus infinity, its lowest is a finite bias) hide
    keys, in the softmax and in every gradient; a text of one row that may not see itself gives zeros."""
    capi = gpu
    rng = np.random.default_rng(7)
    window, far, head_dim, lens = 3, 5, 16, [60, 1, 33]
    rows = sum(lens)
    lowest = {"f32": np.finfo(np.float32).min, "f16": -np.inf, "bf16": np.float32(-3.3895314e38)}[kind]
    table = np.zeros((1, 2 * far + 1))
    table[0, np.abs(np.arange(-far, far + 1)) > window] = lowest
    table[0, far] = lowest  # not itself either
    q, k, v, dy = (to_bits(rng.standard_normal((rows, head_dim)), kind) for _ in range(4))
    keep = capi.DeviceArray.from_host
    d_q, d_k, d_v, d_dy, d_table = map(keep, (q, k, v, dy, to_bits(table, kind)))
    offsets = keep(np.concatenate([[0], np.cumsum(lens)]).astype(np.int64))
    desc = capi.attention_desc(d_q, d_k, d_v, len(lens), rows, rows, 1, head_dim, kind_code(capi, kind), q_offsets=offsets,
                               k_offsets=offsets, distance_bias=d_table, max_distance=far)
    out, dq, dk, dv = (capi.DeviceArray((rows, head_dim), q.dtype) for _ in range(4))
    lse, d_bias = capi.DeviceArray((rows, 1), np.float32), capi.DeviceArray((1, 2 * far + 1), q.dtype)
    size = capi.attention_workspace_bytes(desc)
    capi.attention(desc, out, workspace(capi, size), size, lse=lse)
    size = capi.attention_gradient_workspace_bytes(desc)
    capi.attention_gradient(desc, out, lse, d_dy, dq, dk, dv, workspace(capi, size), size, distance_bias_gradient=d_bias)
    capi.synchronize()
    got = [from_bits(a.to_host(), kind) for a in (out, dq, dk, dv)]
    q, k, v, dy = (from_bits(a, kind) for a in (q, k, v, dy))
    want = [np.zeros((rows, head_dim)) for _ in range(4)]
    want_bias = np.zeros(2 * far + 1)
    start, largest = 0, 0.0
    for n in lens:
        s = slice(start, start + n)
        start += n
        apart = np.arange(n)[None, :] - np.arange(n)[:, None]
        seen = (np.abs(apart) <= window) & (apart != 0)
        scores = np.where(seen, q[s] @ k[s].T / 4.0, -np.inf)
        top = np.where(seen.any(1), scores.max(1), 0.0)[:, None]
        p = np.exp(scores - top)
        p = p / np.where(seen.any(1), p.sum(1), 1.0)[:, None]
        dp = dy[s] @ v[s].T
        delta = (p * dp).sum(1, keepdims=True)
        ds = p * (dp - delta)
        largest = max(largest, (p * (np.abs(dp) + np.abs(delta))).max())
        for to, value in zip(want, (p @ v[s], ds @ k[s] / 4.0, ds.T @ q[s] / 4.0, p.T @ dy[s])):
            to[s] = value
        for a in range(-far, far + 1):
            want_bias[a + far] += ds[apart == a].sum() if abs(a) < far else ds[(apart <= a) if a < 0 else (apart >= a)].sum()
    # at most seven keys of each row: p and ds rounded once, the rows stored once, and delta from the stored rows;
    # sums of 16 products of values up to 5
    unit = {"f32": 2.0 ** -19, "f16": 2.0 ** -10, "bf16": 2.0 ** -7}[kind]
    for have, expected in zip(got, want):
        assert np.abs(have - expected).max() <= 8 * unit * np.abs(expected).max()
    bias = from_bits(d_bias.to_host(), kind)[0]
    hidden = table[0] < 0
    assert np.all(bias[hidden] == 0.0)
    # a sum of at most `rows` terms, each off by p's and its difference's roundings
    assert np.abs(bias - want_bias).max() <= 2 * rows * unit * largest
    assert np.all(got[0][60] == 0.0) and np.all(got[3][60] == 0.0) and lse.to_host()[60, 0] == -np.inf


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows", [1, 40, 700])
def test_int8_rows_into_the_product(gpu, kind, rows):
    """residual_norm's codes and scales are linear's operands: the product of what they stand for, and its epilogue."""
    capi = gpu
    rng = np.random.default_rng(rows)
    dim, width, code = 200, 136, kind_code(capi, kind)
    keep = capi.DeviceArray.from_host
    x, bias, residual = (to_bits(rng.standard_normal(s), kind) for s in ((rows, dim), width, (rows, width)))
    d_x, d_bias, d_residual = map(keep, (x, bias, residual))
    w, w_scales = rng.integers(-127, 128, (width, dim)).astype(np.int8), rng.random(width).astype(np.float32) / 400
    d_w, d_w_scales = keep(w), keep(w_scales)
    codes, scales = capi.DeviceArray((rows, dim), np.int8), capi.DeviceArray((rows,), np.float32)
    capi.residual_norm(capi.norm_desc(d_x, rows, dim, code), codes, capi.I8, out_scales=scales)
    out = capi.DeviceArray((rows, width), np.float32)
    capi.linear(capi.linear_desc(codes, rows, dim, d_w, width, capi.I8, bias=d_bias, residual=d_residual, epilogue_dtype=code,
                                 x_scales=scales, weight_scales=d_w_scales), out, capi.F32)
    capi.synchronize()
    h, s = codes.to_host().astype(np.float64), scales.to_host().astype(np.float64)
    y = from_bits(x, kind)
    y = y / np.sqrt((y * y).mean(1, keepdims=True) + 1e-6)
    assert np.abs(h * s[:, None] - y).max() <= 0.51 * s.max()  # a code is half a step off at most
    product = (h @ w.astype(np.float64).T) * (s[:, None] * w_scales)
    want = product + from_bits(bias, kind) + from_bits(residual, kind)
    # the scales' product, the sum's conversion and product, two additions: a float32 rounding each
    allowed = 5 * 2.0 ** -24 * (np.abs(product) + np.abs(from_bits(bias, kind)) + np.abs(from_bits(residual, kind)))
    assert np.all(np.abs(out.to_host() - want) <= allowed)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,head_dim", [(3, 1, 33), (16, 2, 64), (7, 1, 20), (6, 2, 1), (5, 5, 40)])
def test_key_heads_of_many_query_heads(gpu, kind, heads, kv_heads, head_dim):
    """Few keys under many query heads, whose parts are formed apart and added: the formula's gradients, and rows of no
    text left as they were."""
    batch = Batch(gpu, kind, [30, 0, 77, 1], heads=heads, kv_heads=kv_heads, head_dim=head_dim, mask="causal", bias="table", far=4,
                  lead=5, tail=3, pad=1)
    grad, got = check(batch, pad=3, shift=1)
    for name in ("q", "k", "v"):
        assert np.all(got[name][:5] == 7.0) and np.all(got[name][-3:] == 7.0), name
    first = {name: values.copy() for name, values in got.items()}
    grad.call()
    gpu.synchronize()
    assert all(np.array_equal(first[name], values) for name, values in grad.read().items())
