"""Element types, strided inputs and guarded outputs shared by the operators' tests."""

import numpy as np

UNIT = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
# float16 values below its smallest normal number are rounded to multiples of 2^-24
FLOOR = {"f32": 0.0, "f16": 2.0 ** -25, "bf16": 0.0}


def to_bits(x, kind):
    """float64 values rounded to `kind`, as the array that goes to the device."""
    x = np.asarray(x, dtype=np.float32)
    if kind == "f32":
        return x
    if kind == "f16":
        return x.astype(np.float16)
    bits = x.view(np.uint32).astype(np.uint64)
    bits = (bits + 0x7FFF + ((bits >> 16) & 1)) >> 16
    return bits.astype(np.uint16)


def from_bits(x, kind):
    if kind == "bf16":
        return (x.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return x.astype(np.float64)


def kind_code(capi, kind):
    return {"f32": capi.F32, "f16": capi.F16, "bf16": capi.BF16}[kind]


def storage(kind):
    return {"f32": np.float32, "f16": np.float16, "bf16": np.uint16}[kind]


def strided(capi, values, kind, pad, shift=0):
    """A matrix whose rows are `pad` elements longer and filled with NaN there, `shift` elements into
    its allocation -> (owner, address, stride, the values as stored in float64)."""
    rows, cols = values.shape
    stored = to_bits(values, kind)
    wide = np.empty(shift + rows * (cols + pad), dtype=storage(kind))
    wide[:] = to_bits(np.full(1, np.nan), kind)[0] if kind != "bf16" else 0x7FC0
    wide[shift:].reshape(rows, cols + pad)[:, :cols] = stored
    owner = capi.DeviceArray.from_host(wide)
    return owner, owner.ptr + shift * wide.itemsize, cols + pad, from_bits(stored, kind)


class Output:
    """An output matrix with `pad` guarded elements after each row."""

    def __init__(self, capi, rows, cols, kind, pad=0, shift=0, fill=None):
        self.rows, self.cols, self.kind, self.pad, self.shift = rows, cols, kind, pad, shift
        self.host = np.full(shift + rows * (cols + pad), 7.0).astype(np.float32)
        if fill is not None:
            self.host[shift:].reshape(rows, cols + pad)[:, :cols] = fill
        self.host = to_bits(self.host, kind)
        self.array = capi.DeviceArray.from_host(self.host)
        self.ptr = self.array.ptr + shift * self.host.itemsize
        self.stride = cols + pad

    def read(self):
        flat = self.array.to_host()
        view = flat[self.shift:].reshape(self.rows, self.stride)
        guard = self.host[self.shift:].reshape(self.rows, self.stride)
        assert np.array_equal(flat[:self.shift], self.host[:self.shift]), "wrote before the output"
        assert np.array_equal(view[:, self.cols:], guard[:, self.cols:]), "wrote past a row's end"
        return from_bits(np.ascontiguousarray(view[:, :self.cols]), self.kind)
