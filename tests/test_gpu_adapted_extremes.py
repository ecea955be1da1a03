"""Infinities and very large values in adapters, on every path that the adapted projection takes: few rows (one launch and
two), sorted rows whose tiles take one adapter after the other, and those whose tiles go row by row."""

import pytest
import torch

pytestmark = pytest.mark.gpu

TYPE = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
INF = float("inf")
# rows, adapters, rows after each other with one adapter, rank
PATHS = {"one launch": (9, 3, 1, 8), "few rows": (200, 3, 1, 16), "by adapter": (6000, 3, 300, 16), "by row": (6000, 600, 1, 8)}
# operands and output; rounding of the output; what is left out of x down^T between the products
KINDS = {("f16", "f32"): (2.0 ** -24, 2.0 ** -22), ("bf16", "f32"): (2.0 ** -24, 2.0 ** -23),
         ("bf16", "bf16"): (2.0 ** -8, 2.0 ** -16), ("f16", "f16"): (2.0 ** -11, 2.0 ** -22)}


def _code(capi, kind):
    return {"f32": capi.F32, "f16": capi.F16, "bf16": capi.BF16}[kind]


class Case:
    """Whole numbers in x (of which x[:, 0] is 1 or -1) and small ones elsewhere, so that signs are certain."""

    def __init__(self, kind, path, seed=61):
        self.kind = kind
        self.rows, self.adapters, run, self.rank = PATHS[path]
        self.dim, self.width = 64, 96
        rng = torch.Generator(device="cuda")
        rng.manual_seed(seed)
        self.x = torch.randint(-4, 5, (self.rows, self.dim), generator=rng, device="cuda").to(TYPE[kind])
        self.x[:, 0] = torch.where(self.x[:, 0] > 0, 1.0, -1.0).to(TYPE[kind])
        self.weight = torch.randint(-4, 5, (self.width, self.dim), generator=rng, device="cuda").to(TYPE[kind]) / 64
        self.down = torch.randint(-4, 5, (self.adapters, self.rank, self.dim), generator=rng, device="cuda").to(TYPE[kind]) / 4
        self.up = torch.randint(-4, 5, (self.adapters, self.width, self.rank), generator=rng, device="cuda").to(TYPE[kind]) / 4
        ids = torch.randint(0, self.adapters, (-(-self.rows // run),), generator=rng, device="cuda")
        self.ids = ids.repeat_interleave(run)[:self.rows].to(torch.int32)

    def run(self, capi, out_kind):
        desc = capi.adapted_desc(self.x.data_ptr(), self.rows, self.dim, self.weight.data_ptr(), self.width,
                                 _code(capi, self.kind), down=self.down.data_ptr(), up=self.up.data_ptr(),
                                 adapter_count=self.adapters, max_rank=self.rank, adapter_ids=self.ids.data_ptr())
        size = capi.adapted_projection_workspace_bytes(desc)
        workspace = torch.full((size,), 255, dtype=torch.uint8, device="cuda")
        out = torch.empty(self.rows, self.width, dtype=TYPE[out_kind], device="cuda")
        capi.adapted_projection(desc, out.data_ptr(), _code(capi, out_kind), workspace.data_ptr(), size)
        torch.cuda.synchronize()
        return out.double()

    def low(self):
        return torch.bmm(self.down.double()[self.ids.long()], self.x.double()[:, :, None])[:, :, 0]

    def check(self, got, where, unit, left_out):
        """Rows and columns `where` against the formula; additions of 64 + 16 terms, each of any rounding."""
        up = torch.nan_to_num(self.up.double(), nan=0.0, posinf=0.0, neginf=0.0)[self.ids.long()]
        low = torch.nan_to_num(self.low(), nan=0.0, posinf=0.0, neginf=0.0)
        part, mass = torch.bmm(up, low[:, :, None])[:, :, 0], torch.bmm(up.abs(), low.abs()[:, :, None])[:, :, 0]
        x, weight = self.x.double(), self.weight.double()
        expected, mass = x @ weight.T + part, x.abs() @ weight.abs().T + mass
        tolerance = (left_out + (self.dim + self.rank + 8) * 2.0 ** -23) * mass
        tolerance += unit * (expected.abs() + tolerance)
        assert torch.all(((got - expected).abs() <= tolerance)[where])


@pytest.mark.parametrize("path", PATHS)
@pytest.mark.parametrize("kind,out", KINDS)
def test_infinite_up(gpu, kind, out, path):
    """An infinity in up makes its column of its adapter's rows infinite, with the sign of x down^T."""
    c = Case(kind, path)
    c.up[1, 5, 2], c.up[1, 70, 7] = INF, -INF
    c.down[1, 2] *= 1.0 + 2.0 ** -7  # values that the operands' type does not hold: the rest is not zero
    c.down[1, 7, 3] = 2.0 ** -6
    low = c.low()
    got = c.run(gpu, out)
    named = c.ids == 1
    assert named.any() and not named.all()
    rest = torch.ones_like(got, dtype=torch.bool)
    for column, rank, sign in ((5, 2, 1.0), (70, 7, -1.0)):
        rest[named, column] = False
        sure = named & (low[:, rank] != 0.0)
        assert sure.any()
        assert torch.all(got[sure, column] == sign * torch.sign(low[sure, rank]) * INF)
    c.check(got, rest, *KINDS[kind, out])


@pytest.mark.parametrize("path", PATHS)
@pytest.mark.parametrize("kind,out", KINDS)
def test_infinite_down(gpu, kind, out, path):
    """An infinite value of x down^T makes its row infinite, whatever the size of the row's other values."""
    c = Case(kind, path)
    c.down[1] *= 2.0 ** 13  # x down^T up to 2^19, beyond float16's range
    c.down[1, 3, 0] = INF  # x[:, 0] is 1 or -1
    c.up[1, :, 3] = torch.where(c.up[1, :, 3] > 0, 1.0, -1.0).to(TYPE[kind])
    got = c.run(gpu, out)
    named = c.ids == 1
    sign = torch.sign(c.x[named, 0].double())[:, None] * torch.sign(c.up[1, :, 3].double())[None, :]
    assert torch.all(got[named] == sign * INF)
    c.check(got, (~named)[:, None].expand_as(got), *KINDS[kind, out])


@pytest.mark.parametrize("path", PATHS)
@pytest.mark.parametrize("kind,out", [k for k in KINDS if k[0] == "bf16"])
@pytest.mark.parametrize("down_by,up_by", [(-40, 118), (115, -100), (60, 60)])
def test_far_ends_of_bfloat16(gpu, kind, out, path, down_by, up_by):
    """Values near float32's largest in up, or in x down^T, whose products are in its range."""
    c = Case(kind, path)
    c.down, c.up = c.down * 2.0 ** down_by, c.up * 2.0 ** up_by
    got = c.run(gpu, out)
    c.check(got, torch.ones_like(got, dtype=torch.bool), *KINDS[kind, out])
