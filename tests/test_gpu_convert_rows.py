"""Row quantization and synthetic rows beyond what one launch's workgroups can take."""

import numpy as np
import pytest

import oracle

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim,rows", [(1, (1 << 26) + 5), (4, (1 << 26) + 9)])  # four rows to a workgroup, and sixteen
def test_quantized_rows(gpu, dim, rows):
    capi = gpu
    src = np.random.default_rng(1).standard_normal((rows, dim), dtype=np.float32)
    d_src = capi.DeviceArray.from_host(src)
    codes, scales = capi.DeviceArray((rows, dim), np.int8), capi.DeviceArray((rows,), np.float32)
    capi.call("zcgvs_memset", codes.ptr, 0x80, codes.nbytes, None)  # no code
    capi.launch_quantize_rows_i8(d_src, rows, dim, codes, scales)
    capi.synchronize()
    got, got_scales = codes.to_host(), scales.to_host()
    assert not np.any(got == -128)
    for part in (slice(0, 1000), slice((1 << 26) - 500, rows)):
        want, want_scales = oracle.quantize_rows_i8(src[part])
        assert np.array_equal(got[part], want) and np.array_equal(got_scales[part], want_scales)


def test_generated_rows(gpu):
    """Rows of one call are those of calls for parts of them."""
    capi = gpu
    rows, dim, few = (1 << 26) + 5, 2, 64
    out, part = capi.DeviceArray((rows, dim), np.float32), capi.DeviceArray((few, dim), np.float32)
    capi.call("zcgvs_memset", out.ptr, 0xFF, out.nbytes, None)
    capi.generate_normalized(out, rows, dim, 7)
    capi.synchronize()
    got = out.to_host()
    assert np.all(np.abs(np.square(got).sum(1) - 1.0) <= 1e-5)  # squares, their sum, root and quotients: a few 2^-24
    for first in (0, 1 << 20, rows - few):
        capi.generate_normalized(part, few, dim, 7, row_offset=first)
        capi.synchronize()
        assert np.array_equal(part.to_host(), got[first:first + few])
