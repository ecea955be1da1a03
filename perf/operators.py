"""Performance cases of the embedding-model operators, from token ids to query vectors.

A text-embedding model in front of the search turns token ids into query vectors on the device:
`embedding_lookup` reads (and pools) rows of the token table, `gated_projection` is the first half of
a gated feed-forward block, and `adapted_projection` takes the hidden rows to the width of the store,
each row through the low-rank adapter of its tenant or collection. Training the model adds
`embedding_gradient` and `gated_gradient`.

A pass is one call of one operator. With `own` false it is the operator's plain form, elementary
torch operations in float32; with `own` true it is the call of the library's entry point.
"""

from __future__ import annotations

import importlib.util
import math
import sys
from pathlib import Path

import torch

own = False

ROOT = Path(__file__).resolve().parent.parent
PKG = ROOT / "zero-copy-gpu-vector-search-re-ranking-engine_amd"

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_BYTES = {"f32": 4, "f16": 2, "bf16": 2}


# ---- the cases ------------------------------------------------------------------------------

_LOOKUP = dict(op="lookup", bags=0, scale=1.0, pad=0)
_TABLE_GRADIENT = dict(op="table_gradient", bags=0, scale=1.0, pad=0, accumulate=False)
_GATED = dict(op="gated", act="silu", pad=0)
_GATED_GRADIENT = dict(op="gated_gradient", act="silu", pad=0)
_ADAPTED = dict(op="adapted", pad=0, run=1)


def listed():
    return [
        # One query of two dozen tokens, its rows scaled by the square root of the width: latency.
        dict(_LOOKUP, name="lookup-24", type="f16", out="f16", vocab=30_000, dim=768, tokens=24, scale=27.712812921102035),
        # Passages mean-pooled straight from a token table (a static embedding model building its
        # corpus): ragged token lists, a few of them empty, float32 rows of the store's width.
        dict(_LOOKUP, name="lookup-pooled-16k", type="f32", out="f32", vocab=30_000, dim=384, tokens=1_000_003, bags=16_384),
        # The gradient of a small fine-tuning step: most rows of the table stay zero.
        dict(_TABLE_GRADIENT, name="table-gradient-2k", type="f32", out="f32", vocab=30_000, dim=384, tokens=2_051),
        # The gradient of a full training step with a large vocabulary: the most frequent token
        # holds several percent of the positions.
        dict(_TABLE_GRADIENT, name="table-gradient-256k", type="bf16", out="f32", vocab=128_000, dim=768, tokens=262_144, scale=27.712812921102035),
        # One pooled row through the gated block, the quickest request of a service.
        dict(_GATED, name="gated-1", type="f16", rows=1, dim=768, hidden=2048),
        # All tokens of a batch of passages while a corpus is encoded.
        dict(_GATED, name="gated-8k", type="bf16", rows=8192, dim=1024, hidden=4096),
        # Full-precision encoding of an odd number of rows that are slices of wider ones.
        dict(_GATED, name="gated-f32-1001", type="f32", rows=1001, dim=384, hidden=1536, act="gelu", pad=384),
        # A short fine-tuning batch.
        dict(_GATED_GRADIENT, name="gated-gradient-500", type="f16", rows=500, dim=384, hidden=1024, act="gelu_tanh"),
        # A full training batch.
        dict(_GATED_GRADIENT, name="gated-gradient-16k", type="bf16", rows=16_384, dim=768, hidden=2048),
        # Eight queries of eight tenants, float32 query vectors for the search.
        dict(_ADAPTED, name="adapted-8", type="f16", out="f32", rows=8, dim=768, width=384, adapters=64, rank=16),
        # A service's larger batch of queries, in no order, over a few hundred adapters' worth of tenants.
        dict(_ADAPTED, name="adapted-300", type="f16", out="f32", rows=300, dim=768, width=768, adapters=200, rank=8),
        # Token rows of many requests at once, each request's tokens next to each other.
        dict(_ADAPTED, name="adapted-8k", type="bf16", out="bf16", rows=8192, dim=1024, width=1024, adapters=32, rank=32, run=250),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


# Multiply-adds of the largest listed gated gradient.
_MOST_MACS = 6 * 16_384 * 768 * 2048


def draw(rng):
    """One more case of the ranges the listed ones stand for."""
    op = rng.choice(["lookup", "table_gradient", "gated", "gated", "gated_gradient", "adapted", "adapted"])
    kind = rng.choice(["f32", "f16", "bf16"])
    dim = rng.choice([64, 96, 128, 200, 256, 384, 512, 640, 768, 1024, rng.randrange(33, 1025)])
    pad = rng.choice([0, 0, 0, 8, 64, rng.randrange(1, 100)])
    if op in ("lookup", "table_gradient"):
        tokens = _log_int(rng, 1, 500_000)
        bags = rng.choice([0, 0, max(1, tokens // rng.randrange(2, 200))])
        case = dict(_LOOKUP if op == "lookup" else _TABLE_GRADIENT, type=kind, out=rng.choice([kind, "f32"]), dim=dim,
                    vocab=_log_int(rng, 1000, 128_000), tokens=tokens, bags=bags, pad=pad,
                    scale=rng.choice([1.0, math.sqrt(dim)]))
        if op == "table_gradient" and case["out"] == "f32":
            case["accumulate"] = rng.choice([False, True])
        return case
    act = rng.choice(["silu", "gelu", "gelu_tanh"])
    hidden = rng.choice([256, 512, 1000, 1024, 1536, 2048, 2730, 4096, rng.randrange(100, 4097)])
    # float32 products cost about eight times as much as 16-bit ones
    most = _MOST_MACS // (8 if kind == "f32" else 1)
    if op == "gated":
        rows = min(_log_int(rng, 1, 16_384), most // (2 * dim * hidden))
        return dict(_GATED, type=kind, rows=rows, dim=dim, hidden=hidden, act=act, pad=pad)
    if op == "gated_gradient":
        rows = min(_log_int(rng, 1, 16_384), most // (6 * dim * hidden))
        return dict(_GATED_GRADIENT, type=kind, rows=rows, dim=dim, hidden=hidden, act=act, pad=pad)
    rank = rng.choice([4, 8, 16, 32, 64, rng.randrange(1, 65)])
    return dict(_ADAPTED, type=kind, out=rng.choice([kind, "f32"]), rows=_log_int(rng, 1, 8192), dim=dim,
                width=rng.choice([128, 256, 384, 768, 1024, rng.randrange(33, 1025)]),
                adapters=min(_log_int(rng, 1, 200), 4096 // rank), rank=rank, run=rng.choice([1, 1, rng.randrange(2, 300)]),
                pad=pad)


# ---- inputs ---------------------------------------------------------------------------------


class _Maker:
    def __init__(self, case, seed):
        self.type = _TYPES[case["type"]]
        self.rng = torch.Generator(device="cuda")
        self.rng.manual_seed(seed)

    def normal(self, *shape, std=1.0, dtype=None):
        return (torch.randn(*shape, generator=self.rng, device="cuda") * std).to(dtype or self.type)

    def uniform(self, *shape):
        return torch.rand(*shape, generator=self.rng, device="cuda")

    def integers(self, low, high, count):
        return torch.randint(low, high, (count,), generator=self.rng, device="cuda")

    def rows_of(self, rows, dim, pad, std=1.0):
        """[rows, dim] as a slice of rows that are `pad` wider."""
        return self.normal(rows, dim + pad, std=std)[:, :dim]


def _inputs(case, seed):
    make = _Maker(case, seed)
    op, s = case["op"], {}
    if op in ("lookup", "table_gradient"):
        vocab, dim, tokens, bags = case["vocab"], case["dim"], case["tokens"], case["bags"]
        # Zipf-distributed token ids; id 0 is the padding and stands for one position in fifty
        weight = torch.arange(1, vocab, device="cuda", dtype=torch.float64).pow(-1.05)
        cdf = torch.cumsum(weight / weight.sum(), 0).float()
        ids = torch.searchsorted(cdf, make.uniform(tokens)).clamp_(max=vocab - 2) + 1
        s["ids"] = torch.where(make.uniform(tokens) < 0.02, torch.zeros_like(ids), ids).to(torch.int32)
        s["offsets"] = None
        if bags:
            cuts = torch.sort(make.integers(0, tokens + 1, bags - 1)).values
            s["offsets"] = torch.cat([cuts.new_zeros(1), cuts, cuts.new_full((1,), tokens)])
        if op == "lookup":
            s["table"] = make.rows_of(vocab, dim, case["pad"], std=0.05)
        else:
            s["out_gradient"] = make.rows_of(bags or tokens, dim, case["pad"], std=0.01)
            if case["accumulate"]:
                s["gradient"] = make.normal(vocab, dim, std=0.01, dtype=torch.float32)
        return s
    rows, dim = case["rows"], case["dim"]
    s["x"] = make.rows_of(rows, dim, case["pad"])
    if op in ("gated", "gated_gradient"):
        hidden = case["hidden"]
        s["gate"] = make.normal(hidden, dim, std=dim ** -0.5)
        s["up"] = make.normal(hidden, dim, std=dim ** -0.5)
        if op == "gated_gradient":
            s["out_gradient"] = make.normal(rows, hidden, std=0.1)
        return s
    width, adapters, rank = case["width"], case["adapters"], case["rank"]
    s["weight"] = make.normal(width, dim, std=dim ** -0.5)
    s["down"] = make.normal(adapters, rank, dim, std=dim ** -0.5)
    s["up"] = make.normal(adapters, width, rank, std=rank ** -0.5)
    s["ranks"] = make.integers((rank + 1) // 2, rank + 1, adapters).to(torch.int32)
    s["scales"] = 0.25 + 0.5 * make.uniform(adapters)
    # one adapter for `run` rows after each other; every tenth request has none
    requests = -(-rows // case["run"])
    ids = torch.where(make.uniform(requests) < 0.1, -1, make.integers(0, adapters, requests))
    s["adapter_ids"] = ids.repeat_interleave(case["run"])[:rows].to(torch.int32)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    return s


# ---- the plain forms ------------------------------------------------------------------------


def _bag_of(offsets, tokens):
    """The bag of every token position."""
    return torch.repeat_interleave(torch.arange(offsets.numel() - 1, device="cuda"), offsets.diff(), output_size=tokens)


def _token_weights(s):
    """What each position's row counts for (0 at the padding), and the position's output row."""
    case, ids = s["case"], s["ids"]
    valid = (ids > 0).float()
    if s["offsets"] is None:
        return valid * case["scale"], torch.arange(case["tokens"], device="cuda")
    bag = _bag_of(s["offsets"], case["tokens"])
    count = torch.zeros(case["bags"], device="cuda").index_add_(0, bag, valid)
    return valid * (case["scale"] / count.clamp(min=1.0))[bag], bag


def _plain_lookup(s):
    case = s["case"]
    weight, row = _token_weights(s)
    values = s["table"][s["ids"].long()].float() * weight[:, None]
    if s["offsets"] is not None:
        values = torch.zeros(case["bags"], case["dim"], device="cuda").index_add_(0, row, values)
    return {"rows": values.to(_TYPES[case["out"]])}


def _plain_table_gradient(s):
    case = s["case"]
    weight, row = _token_weights(s)
    out = s["gradient"].clone() if case["accumulate"] else torch.zeros(case["vocab"], case["dim"], device="cuda")
    out.index_add_(0, s["ids"].long(), s["out_gradient"].float()[row] * weight[:, None])
    return {"table_gradient": out.to(_TYPES[case["out"]])}


def _activation(name, g):
    """The activation of g and its derivative."""
    if name == "silu":
        y = torch.sigmoid(g)
        return g * y, y * (1.0 + g * (1.0 - y))
    if name == "gelu":
        y = 0.5 * (1.0 + torch.erf(g * math.sqrt(0.5)))
        return g * y, y + g * torch.exp(-0.5 * g * g) * (1.0 / math.sqrt(2.0 * math.pi))
    c = math.sqrt(2.0 / math.pi)
    t = torch.tanh(c * (g + 0.044715 * g * g * g))
    return 0.5 * g * (1.0 + t), 0.5 * (1.0 + t) + 0.5 * g * (1.0 - t * t) * c * (1.0 + 3.0 * 0.044715 * g * g)


def _plain_gated(s):
    x = s["x"].float()
    a, _ = _activation(s["case"]["act"], x @ s["gate"].float().T)
    return {"hidden": (a * (x @ s["up"].float().T)).to(s["x"].dtype)}


def _plain_gated_gradient(s):
    kind = s["x"].dtype
    x, gate, up, d = s["x"].float(), s["gate"].float(), s["up"].float(), s["out_gradient"].float()
    a, slope = _activation(s["case"]["act"], x @ gate.T)
    dg, du = d * (x @ up.T) * slope, d * a
    return {"x_gradient": (dg @ gate + du @ up).to(kind), "gate_gradient": (dg.T @ x).to(kind),
            "up_gradient": (du.T @ x).to(kind)}


def _plain_adapted(s):
    case = s["case"]
    n, r, width = case["adapters"], case["rank"], case["width"]
    x = s["x"].float()
    # the products with every adapter's rows, of which each row keeps those of its own adapter
    keep = (s["adapter_ids"][:, None] == torch.arange(n, device="cuda")) * s["scales"]
    rank_ok = torch.arange(r, device="cuda") < s["ranks"][:, None]
    low = (x @ s["down"].float().reshape(n * r, -1).T).view(-1, n, r) * keep[:, :, None] * rank_ok
    delta = low.view(-1, n * r) @ s["up"].float().permute(0, 2, 1).reshape(n * r, width)
    return {"rows": (x @ s["weight"].float().T + delta).to(_TYPES[case["out"]])}


# ---- the library's operators ----------------------------------------------------------------


def _capi():
    """The package directory, whose name is not an identifier, imported as `zcgvs_amd`."""
    if "zcgvs_amd" not in sys.modules:
        spec = importlib.util.spec_from_file_location("zcgvs_amd", PKG / "__init__.py",
                                                      submodule_search_locations=[str(PKG)])
        module = importlib.util.module_from_spec(spec)
        sys.modules["zcgvs_amd"] = module
        spec.loader.exec_module(module)
    from zcgvs_amd import capi

    return capi


def _plan(s):
    """The descriptor, workspace and outputs that a program keeps for calls of one shape."""
    capi, case = _capi(), s["case"]
    kinds = {"f32": capi.F32, "f16": capi.F16, "bf16": capi.BF16}
    kind, out_kind = kinds[case["type"]], kinds[case.get("out", case["type"])]
    empty = lambda *shape: torch.empty(*shape, dtype=_TYPES[case.get("out", case["type"])], device="cuda")  # noqa: E731
    workspace = lambda size: torch.empty(size, dtype=torch.uint8, device="cuda")  # noqa: E731
    op = case["op"]
    if op in ("lookup", "table_gradient"):
        source = s["table"] if op == "lookup" else None
        offsets = s["offsets"].data_ptr() if case["bags"] else None
        desc = capi.embedding_desc(source.data_ptr() if op == "lookup" else None, case["vocab"], case["dim"], kind,
                                   s["ids"].data_ptr(), case["tokens"], bag_offsets=offsets, bag_count=case["bags"],
                                   reduce=capi.EMBEDDING_MEAN if case["bags"] else capi.EMBEDDING_SUM, padding_id=0,
                                   scale=case["scale"], table_stride=source.stride(0) if op == "lookup" else 0)
        if op == "lookup":
            out = empty(case["bags"] or case["tokens"], case["dim"])
            return lambda stream: capi.embedding_lookup(desc, out.data_ptr(), out_kind, stream=stream), {"rows": out}
        size = capi.embedding_gradient_workspace_bytes(desc)
        d, space = s["out_gradient"], workspace(size)
        out = empty(case["vocab"], case["dim"])

        def gradient(stream):
            if case["accumulate"]:
                out.copy_(s["gradient"])
            capi.embedding_gradient(desc, d.data_ptr(), kind, out.data_ptr(), out_kind, space.data_ptr(), size,
                                    out_gradient_stride=d.stride(0), accumulate=case["accumulate"], stream=stream)

        return gradient, {"table_gradient": out}
    x, rows, dim = s["x"], case["rows"], case["dim"]
    if op in ("gated", "gated_gradient"):
        act = {"silu": capi.ACT_SILU, "gelu": capi.ACT_GELU, "gelu_tanh": capi.ACT_GELU_TANH}[case["act"]]
        desc = capi.gated_desc(x.data_ptr(), rows, dim, s["gate"].data_ptr(), s["up"].data_ptr(), case["hidden"], kind,
                               act, x_stride=x.stride(0))
        if op == "gated":
            out = empty(rows, case["hidden"])
            return lambda stream: capi.gated_projection(desc, out.data_ptr(), stream=stream), {"hidden": out}
        size = capi.gated_gradient_workspace_bytes(desc)
        d, space = s["out_gradient"], workspace(size)
        dx, dgate, dup = empty(rows, dim), empty(case["hidden"], dim), empty(case["hidden"], dim)
        return lambda stream: capi.gated_gradient(desc, d.data_ptr(), dx.data_ptr(), dgate.data_ptr(), dup.data_ptr(),
                                                  space.data_ptr(), size, stream=stream), {
            "x_gradient": dx, "gate_gradient": dgate, "up_gradient": dup}
    desc = capi.adapted_desc(x.data_ptr(), rows, dim, s["weight"].data_ptr(), case["width"], kind, x_stride=x.stride(0),
                             down=s["down"].data_ptr(), up=s["up"].data_ptr(), adapter_count=case["adapters"],
                             max_rank=case["rank"], ranks=s["ranks"].data_ptr(), scales=s["scales"].data_ptr(),
                             adapter_ids=s["adapter_ids"].data_ptr())
    size = capi.adapted_projection_workspace_bytes(desc)
    space, out = workspace(size), empty(rows, case["width"])
    return lambda stream: capi.adapted_projection(desc, out.data_ptr(), out_kind, space.data_ptr(), size,
                                                  stream=stream), {"rows": out}


# ---- one pass -------------------------------------------------------------------------------

_PLAIN = {"lookup": _plain_lookup, "table_gradient": _plain_table_gradient, "gated": _plain_gated,
          "gated_gradient": _plain_gated_gradient, "adapted": _plain_adapted}


def run(state):
    if not own:
        return _PLAIN[state["case"]["op"]](state)
    if "plan" not in state:
        state["plan"] = _plan(state)
    call, outputs = state["plan"]
    call(torch.cuda.current_stream().cuda_stream)
    return outputs


# ---- what a pass needs at least ----------------------------------------------------------------


def _distinct(draws, vocab):
    """Expected number of distinct ids among `draws` Zipf ones."""
    weights = [(i + 1) ** -1.05 for i in range(vocab - 1)]
    total = sum(weights)
    return sum(-math.expm1(draws * math.log1p(-w / total)) if w < total else 1.0 for w in weights)


def work(case):
    e, o = _BYTES[case["type"]], _BYTES[case.get("out", case["type"])]
    if case["op"] in ("lookup", "table_gradient"):
        vocab, dim, tokens = case["vocab"], case["dim"], case["tokens"]
        out_rows = case["bags"] or tokens
        index = 4 * tokens + (8 * (case["bags"] + 1) if case["bags"] else 0)
        if case["op"] == "lookup":
            return {"bytes": int(_distinct(tokens, vocab) * dim * e + out_rows * dim * o + index), "flops": tokens * dim}
        table = 2 * _distinct(tokens, vocab) * dim * o if case["accumulate"] else vocab * dim * o
        if case["accumulate"]:
            table += 2 * vocab * dim * o  # the pass starts from a copy of the gradient so far
        return {"bytes": int(out_rows * dim * e + table + index), "flops": 2 * tokens * dim}
    rows, dim = case["rows"], case["dim"]
    if case["op"] in ("gated", "gated_gradient"):
        hidden = case["hidden"]
        bytes_ = e * (rows * dim + 2 * hidden * dim + rows * hidden)
        flops = 4 * rows * dim * hidden
        if case["op"] == "gated_gradient":
            bytes_, flops = bytes_ + e * (rows * dim + 2 * hidden * dim), 3 * flops
        return {"bytes": bytes_, "flops": flops}
    width, rank = case["width"], case["rank"]
    requests = -(-rows // case["run"])
    used = case["adapters"] * -math.expm1(0.9 * requests * math.log1p(-1.0 / case["adapters"])) if case["adapters"] > 1 else 1
    # ranks are spread evenly over the upper half of [1, rank]
    mean_rank = ((rank + 1) // 2 + rank) / 2
    return {"bytes": int(e * (rows * dim + width * dim + used * mean_rank * (dim + width)) + o * rows * width + 4 * rows),
            "flops": int(2 * rows * dim * width + 0.9 * 2 * rows * mean_rank * (dim + width))}


# ---- 64-bit results --------------------------------------------------------------------------


def exact(case, seed):
    s = _inputs(case, seed)
    op = case["op"]
    if op in ("lookup", "table_gradient"):
        ids = s["ids"].long()
        valid = ids != 0
        # the one-hot matrix of output rows by tokens, as its non-zero entries
        row = torch.arange(case["tokens"], device="cuda")
        share = valid.double() * case["scale"]
        rows = case["tokens"]
        if case["bags"]:
            rows = case["bags"]
            row = torch.searchsorted(s["offsets"], row, right=True) - 1
            count = torch.bincount(row, weights=valid.double(), minlength=rows)
            share = share / count.clamp(min=1.0)[row]
        chunk = 1 << 17
        if op == "lookup":
            out = torch.zeros(rows, case["dim"], dtype=torch.float64, device="cuda")
            for i in range(0, case["tokens"], chunk):
                part = slice(i, i + chunk)
                out.index_put_((row[part],), s["table"][ids[part]].double() * share[part, None], accumulate=True)
            return {"rows": out}
        out = torch.zeros(case["vocab"], case["dim"], dtype=torch.float64, device="cuda")
        if case["accumulate"]:
            out += s["gradient"].double()
        for i in range(0, case["tokens"], chunk):
            part = slice(i, i + chunk)
            out.index_put_((ids[part],), s["out_gradient"][row[part]].double() * share[part, None], accumulate=True)
        return {"table_gradient": out}
    x = s["x"].double()
    if op in ("gated", "gated_gradient"):
        act = {"silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu,
               "gelu_tanh": lambda g: torch.nn.functional.gelu(g, approximate="tanh")}[case["act"]]
        gate, up = s["gate"].double(), s["up"].double()
        if op == "gated":
            return {"hidden": act(x @ gate.T) * (x @ up.T)}
        leaves = [t.requires_grad_() for t in (x.clone(), gate, up)]
        with torch.enable_grad():
            hidden = act(leaves[0] @ leaves[1].T) * (leaves[0] @ leaves[2].T)
            dx, dgate, dup = torch.autograd.grad(hidden, leaves, s["out_gradient"].double())
        return {"x_gradient": dx, "gate_gradient": dgate, "up_gradient": dup}
    out = x @ s["weight"].double().T
    for a, (rank, scale) in enumerate(zip(s["ranks"].tolist(), s["scales"].double().tolist())):
        at = torch.nonzero(s["adapter_ids"] == a).flatten()
        if at.numel():
            low = x[at] @ s["down"][a, :rank].double().T
            out[at] += scale * (low @ s["up"][a, :, :rank].double().T)
    return {"rows": out}
