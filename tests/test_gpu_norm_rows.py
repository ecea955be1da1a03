"""The residual norm over more rows than one launch's workgroups can take."""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def test_rows_of_a_wavefront(gpu):
    """2^26 rows and some of one value each, four rows to a workgroup."""
    capi = gpu
    rows = (1 << 26) + 5
    x = np.random.default_rng(1).standard_normal(rows, dtype=np.float32).astype(np.float16)
    d_x, out = capi.DeviceArray.from_host(x), capi.DeviceArray((rows,), np.float16)
    capi.call("zcgvs_memset", out.ptr, 0xFF, out.nbytes, None)
    capi.residual_norm(capi.norm_desc(d_x, rows, 1, capi.F16, eps=1.0), out, capi.F16)
    capi.synchronize()
    got = out.to_host()
    for part in np.array_split(np.arange(rows), 16):
        want = x[part].astype(np.float64)
        want /= np.sqrt(want * want + 1.0)
        # the float32 result is within 8 roundings, the float16 one half a step of what that is
        assert np.all(np.abs(got[part] - want) <= 2.0 ** -11 * 1.001 * np.abs(want) + 2.0 ** -25)


def test_rows_of_a_workgroup(gpu):
    """2^24 rows and some, a workgroup each, in place: rows of one value become rows of ones."""
    capi = gpu
    rows, dim = (1 << 24) + 3, 2049
    x = capi.DeviceArray((rows, dim), np.float16)
    capi.call("zcgvs_memset", x.ptr, 0x3E, x.nbytes, None)  # 1.56
    capi.residual_norm(capi.norm_desc(x, rows, dim, capi.F16, eps=0.0), x, capi.F16)
    capi.synchronize()
    row = np.empty(dim, np.float16)
    for r in (0, 1, (1 << 24) - 2, (1 << 24) - 1, 1 << 24, rows - 1):
        capi.call("zcgvs_memcpy_d2h", row.ctypes.data, x.ptr + 2 * dim * r, row.nbytes, None)
        capi.synchronize()
        assert np.all(np.abs(row.astype(np.float64) - 1.0) <= 2.0 ** -11), r  # the float32 results are within 2^-19
