"""The adapted projection at sizes whose rows are sorted by adapter, on both tiles, with few and with many
adapters a tile, against the formula in 64 bits (computed on the GPU)."""

import pytest
import torch

pytestmark = pytest.mark.gpu

STEP = 2.0 ** -23  # one float32 addition of the matrix cores, whose rounding need not be to nearest
UNIT = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
FLOOR = {"f32": 0.0, "f16": 2.0 ** -25, "bf16": 0.0}
TYPE = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _code(capi, kind):
    return {"f32": capi.F32, "f16": capi.F16, "bf16": capi.BF16}[kind]


class Case:
    def __init__(self, kind, rows, dim, width, adapters, rank, run, pad=0, seed=5):
        rng = torch.Generator(device="cuda")
        rng.manual_seed(seed)

        def normal(*shape, std=1.0):
            return (torch.randn(*shape, generator=rng, device="cuda") * std).to(TYPE[kind])

        self.kind, self.rows, self.dim, self.width, self.rank = kind, rows, dim, width, rank
        self.x = normal(rows, dim + pad)[:, :dim]
        self.weight = normal(width, dim, std=dim ** -0.5)
        self.down, self.up = normal(adapters, rank, dim, std=dim ** -0.5), normal(adapters, width, rank, std=rank ** -0.5)
        ids = torch.randint(-1, adapters + 1, (-(-rows // run),), generator=rng, device="cuda")
        self.ids = ids.repeat_interleave(run)[:rows].to(torch.int32)
        self.ranks = torch.randint(0, rank + 1, (adapters,), generator=rng, device="cuda").to(torch.int32)
        self.scales = 0.25 + torch.rand(adapters, generator=rng, device="cuda")

    def run(self, capi, out_kind):
        desc = capi.adapted_desc(self.x.data_ptr(), self.rows, self.dim, self.weight.data_ptr(), self.width,
                                 _code(capi, self.kind), x_stride=self.x.stride(0), down=self.down.data_ptr(),
                                 up=self.up.data_ptr(), adapter_count=self.down.shape[0], max_rank=self.rank,
                                 ranks=self.ranks.data_ptr(), scales=self.scales.data_ptr(),
                                 adapter_ids=self.ids.data_ptr())
        size = capi.adapted_projection_workspace_bytes(desc)
        workspace = torch.full((size,), 255, dtype=torch.uint8, device="cuda")  # NaN everywhere
        out = torch.empty(self.rows, self.width, dtype=TYPE[out_kind], device="cuda")
        capi.adapted_projection(desc, out.data_ptr(), _code(capi, out_kind), workspace.data_ptr(), size)
        torch.cuda.synchronize()
        return out

    def expected(self, out_kind):
        """The formula and the error that the kernel's sums and roundings may have."""
        x, weight = self.x.double(), self.weight.double()
        out, mass = x @ weight.T, x.abs() @ weight.abs().T
        extra = torch.zeros_like(mass)
        split = {"f32": 0.0, "f16": 2.0 ** -22, "bf16": 2.0 ** -16}[self.kind]
        for a, (rank, scale) in enumerate(zip(self.ranks.tolist(), self.scales.double().tolist())):
            at = torch.nonzero(self.ids == a).flatten()
            if at.numel() == 0 or rank == 0:
                continue
            down, up = self.down[a, :rank].double(), self.up[a, :, :rank].double()
            low, low_mass = scale * (x[at] @ down.T), scale * (x[at].abs() @ down.abs().T)
            error = (self.dim + 6) * STEP * low_mass + split * low.abs() + 2.0 ** -38 * low.abs().amax(1, keepdim=True)
            out[at] += low @ up.T
            part = (low.abs() + error) @ up.abs().T
            mass[at] += part
            extra[at] += error @ up.abs().T + 2 * (rank + 2) * STEP * part
        error = extra + (self.dim + 2) * STEP * mass
        return out, error + UNIT[out_kind] * (out.abs() + error) + FLOOR[out_kind]


# both tiles of every type; runs (few adapters a tile) and mixed rows (many, and few of large rank); rows that
# are no whole chunks; more rows than one workgroup sorts
@pytest.mark.parametrize("kind,out,rows,dim,width,adapters,rank,run,pad", [
    ("f16", "f32", 4200, 72, 130, 7, 64, 1, 0),
    ("f16", "f16", 5000, 136, 260, 300, 8, 1, 0),
    ("bf16", "bf16", 4097, 200, 600, 40, 32, 250, 0),
    ("bf16", "f32", 6001, 256, 2050, 32, 33, 100, 0),
    ("f16", "f32", 9000, 96, 2048, 1000, 4, 1, 0),
    ("bf16", "bf16", 8193, 1000, 128, 1, 128, 1, 0),
    ("f32", "f32", 4500, 100, 300, 50, 20, 1, 0),
    ("f32", "f32", 8200, 64, 2050, 6, 70, 300, 0),
    ("f16", "f32", 5003, 101, 333, 20, 13, 1, 3),
    ("bf16", "f32", 7000, 77, 2049, 90, 9, 30, 1),
    ("f32", "f32", 4200, 33, 65, 400, 5, 1, 2),
    ("f16", "f16", 1500, 768, 768, 30, 16, 40, 0),
])
def test_large(gpu, kind, out, rows, dim, width, adapters, rank, run, pad):
    c = Case(kind, rows, dim, width, adapters, rank, run, pad)
    got = c.run(gpu, out)
    expected, tolerance = c.expected(out)
    assert torch.all((got.double() - expected).abs() <= tolerance)
    assert torch.equal(got, c.run(gpu, out))


@pytest.mark.parametrize("run", [1, 200])
def test_spoiled_adapters_stay_in_their_rows(gpu, run):
    """Infinities and NaN in adapters reach the rows that name them and no others; NaN past the ranks none."""
    c = Case("f16", 6000, 128, 192, 12, 16, run)
    for a in range(12):
        rank = int(c.ranks[a])
        c.down[a, rank:], c.up[a, :, rank:] = float("nan"), float("nan")
    c.ranks[1], c.ranks[2] = 16, 16
    c.down[1], c.up[2] = float("nan"), float("inf")
    got = c.run(gpu, "f32")
    bad = (c.ids == 1) | (c.ids == 2)
    assert bad.any()
    c.down[1], c.up[2] = 0.0, 0.0
    expected, tolerance = c.expected("f32")
    assert torch.all((got.double() - expected).abs()[~bad] <= tolerance[~bad])
    assert not torch.isfinite(got[bad]).any()
