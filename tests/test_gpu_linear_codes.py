"""The int8 projection's sums at the most codes a row may hold."""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

CODES = 131072


@pytest.mark.parametrize("rows", [3, 4100])  # the kernel for few rows, tiles
def test_lowest_codes(gpu, rows):
    """Rows of -128 throughout: a product of 2^31 with rows of -128, exact with others (scales are powers of two)."""
    capi = gpu
    width = 20
    w = np.random.default_rng(1).integers(-128, 128, (width, CODES)).astype(np.int8)
    w[0] = w[5] = w[19] = -128
    w[1] = 127
    w[2, :-1], w[2, -1] = -128, -127
    x = capi.DeviceArray((rows, CODES), np.int8)
    capi.call("zcgvs_memset", x.ptr, 0x80, x.nbytes, None)
    d_w = capi.DeviceArray.from_host(w)
    x_scales = capi.DeviceArray.from_host(np.full(rows, 2.0 ** -20, np.float32))
    w_scales = capi.DeviceArray.from_host(np.full(width, 2.0 ** -3, np.float32))
    out = capi.DeviceArray((rows, width), np.float32)
    capi.linear(capi.linear_desc(x, rows, CODES, d_w, width, capi.I8, epilogue_dtype=capi.F32, x_scales=x_scales,
                                 weight_scales=w_scales), out, capi.F32)
    capi.synchronize()
    sums = -128 * w.astype(np.int64).sum(1)
    assert sums[0] == 2 ** 31
    assert np.array_equal(out.to_host(), np.broadcast_to(sums.astype(np.float32) * np.float32(2.0 ** -23), (rows, width)))
