"""Performance cases of the operators of an encoder block, forward and backward.

A text-embedding model puts encoder blocks between its token rows and the pooled row: `residual_norm`
adds a block's output to the running rows and normalises them (to the operands' type, or to int8 codes with
a scale a row, which are what the int8 product and a per-vector int8 store take), `linear` is a projection
with its bias, activation and residual in one pass (float operands or int8 codes), and `attention` lets the
tokens of each text of a packed batch see each other, with a bias by distance, a cap on the scores, a causal or
a prefix mask. Training adds the gradients of the three.

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

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "i8": torch.int8}
_BYTES = {"f32": 4, "f16": 2, "bf16": 2, "i8": 1}
# what the values that int8 codes stand for come back in
_DECODED = {"f32": torch.float16, "f16": torch.float16, "bf16": torch.bfloat16}
_EPS = 1e-6


# ---- the cases ------------------------------------------------------------------------------

_NORM = dict(op="norm", residual=True, offset=0.0, pad=0)
_NORM_GRADIENT = dict(op="norm_gradient", offset=0.0, through=False, pad=0)
_LINEAR = dict(op="linear", act="none", bias=True, residual=False, pad=0)
_LINEAR_GRADIENT = dict(op="linear_gradient", act="none", bias=True, pad=0)
_ATTENTION = dict(op="attention", query="all", mask="full", cap=0.0, bias="none", far=0, padded=False)


def listed():
    return [
        # One query's tokens on their way into an int8 product: latency.
        dict(_NORM, name="norm-24-i8", type="f16", out="i8", rows=24, dim=768),
        # All tokens of a batch of passages between two blocks; the running rows are written as well.
        dict(_NORM, name="norm-16k", type="bf16", out="bf16", rows=16_384, dim=1024),
        # The last norm of a full-precision fine-tuning step, rows that are slices of wider ones.
        dict(_NORM_GRADIENT, name="norm-gradient-1001", type="f32", rows=1001, dim=384, pad=384),
        # A norm within a block of a training batch: the running rows bring a gradient of their own.
        dict(_NORM_GRADIENT, name="norm-gradient-16k", type="bf16", rows=16_384, dim=1024, through=True),
        # The projection behind the attention for the one row of a query that is pooled.
        dict(_LINEAR, name="linear-1", type="f16", out="f16", rows=1, dim=768, width=768, residual=True),
        # A feed-forward block's first product on int8 codes while a corpus is encoded.
        dict(_LINEAR, name="linear-8k-i8", type="i8", out="bf16", rows=8192, dim=1024, width=4096, act="gelu_tanh"),
        # A short full-precision fine-tuning batch.
        dict(_LINEAR_GRADIENT, name="linear-gradient-500", type="f32", rows=500, dim=384, width=1536, act="gelu"),
        # A full training batch.
        dict(_LINEAR_GRADIENT, name="linear-gradient-16k", type="bf16", rows=16_384, dim=768, width=2048, act="gelu_tanh"),
        # The last block of a model that pools the last token: one query row over a long text's keys,
        # four query heads to a key head, scores capped.
        dict(_ATTENTION, name="attention-pooled-1", type="f16", texts=1, short=8193, long=8193, query="last", mask="causal",
             heads=16, kv_heads=4, head_dim=128, cap=50.0),
        # A batch of passages of 64 to 1024 tokens, a learned bias by distance.
        dict(_ATTENTION, name="attention-passages", type="bf16", texts=128, short=64, long=1024, heads=12, kv_heads=12,
             head_dim=64, bias="table", far=128),
        # A few short texts in full precision: an instruction that all its tokens see, the rest causal.
        dict(_ATTENTION, op="attention_gradient", name="attention-gradient-77", type="f32", texts=3, short=20, long=77,
             heads=6, kv_heads=2, head_dim=32, mask="prefix", cap=30.0),
        # A training batch of passages of 64 to 512 tokens, the bias by distance trained too.
        dict(_ATTENTION, op="attention_gradient", name="attention-gradient-passages", type="bf16", texts=128, short=64,
             long=512, heads=12, kv_heads=12, head_dim=64, bias="table", far=128),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


# Multiply-adds of the largest listed cases: a linear gradient's, an attention's and its gradient's.
_MOST_LINEAR = 3 * 16_384 * 768 * 2048
_MOST_ATTENTION = 2 * 768 * 128 * 370_000


def draw(rng):
    """One more case of the ranges the listed ones stand for."""
    op = rng.choice(["norm", "norm_gradient", "linear", "linear", "linear_gradient", "attention", "attention", "attention",
                     "attention_gradient", "attention_gradient"])
    kind = rng.choice(["f32", "f16", "bf16"])
    pad = rng.choice([0, 0, 0, 8, 64, rng.randrange(1, 100)])
    if op in ("norm", "norm_gradient"):
        dim = rng.choice([64, 128, 200, 256, 384, 512, 768, 1024, 2048, rng.randrange(33, 2049)])
        rows = min(_log_int(rng, 1, 30_000), 16_384 * 1024 * 2 // (dim * _BYTES[kind]))
        offset = rng.choice([0.0, 1.0])
        if op == "norm":
            return dict(_NORM, type=kind, out=rng.choice([kind, "f32", "i8"]), rows=rows, dim=dim, pad=pad, offset=offset,
                        residual=rng.choice([True, True, False]))
        return dict(_NORM_GRADIENT, type=kind, rows=rows, dim=dim, pad=pad, offset=offset, through=rng.choice([True, False]))
    if op in ("linear", "linear_gradient"):
        dim = rng.choice([64, 128, 200, 256, 384, 512, 768, 1024, 2048, rng.randrange(33, 2049)])
        width = rng.choice([128, 256, 384, 768, 1000, 1024, 2048, 2304, 4096, rng.randrange(33, 4097)])
        act = rng.choice(["none", "silu", "gelu", "gelu_tanh"])
        bias = rng.choice([True, False])
        # float32 products cost about eight times as much as 16-bit ones
        most = _MOST_LINEAR // (8 if kind == "f32" else 1)
        if op == "linear":
            kind = rng.choice([kind, kind, "i8"])
            out = rng.choice(["f16", "bf16", "f32"]) if kind == "i8" else rng.choice([kind, kind, "f32"])
            return dict(_LINEAR, type=kind, out=out, rows=min(_log_int(rng, 1, 16_384), most // (dim * width)), dim=dim,
                        width=width, act=act, bias=bias, residual=rng.choice([True, False]), pad=pad)
        return dict(_LINEAR_GRADIENT, type=kind, rows=min(_log_int(rng, 1, 16_384), most // (3 * dim * width)), dim=dim,
                    width=width, act=act, bias=bias, pad=pad)
    kv_heads = rng.choice([1, 2, 3, 4, 6, 8, 12])
    heads = kv_heads * rng.choice([1, 1, 1, 2, 4])
    head_dim = rng.choice([32, 64, 64, 96, 128, rng.randrange(8, 129)])
    bias = rng.choice(["none", "slopes", "table"])
    case = dict(_ATTENTION, op=op, type=kind, heads=heads, kv_heads=kv_heads, head_dim=head_dim,
                mask=rng.choice(["full", "full", "causal", "prefix"]), cap=rng.choice([0.0, 0.0, 20.0, 50.0]), bias=bias,
                far=rng.choice([16, 64, 128, rng.randrange(2, 300)]) if bias == "table" else 0,
                padded=rng.choice([False, False, True]))
    case["long"] = _log_int(rng, 2, 8192)
    case["short"] = max(1, case["long"] // rng.randrange(1, 12))
    if op == "attention" and rng.random() < 0.3:
        case["query"] = rng.choice(["first", "last"])
        if case["query"] == "first":
            case["mask"] = "full"  # causal, it would see itself alone
    # keys of the whole batch, and the scores of it
    pairs = case["long"] * (case["long"] if case["query"] == "all" else 1) * heads * head_dim
    pairs *= (8 if kind == "f32" else 1) * (2 if op == "attention_gradient" else 1)
    case["texts"] = max(1, min(_log_int(rng, 1, 512), 65_536 // case["long"], _MOST_ATTENTION // (2 * pairs)))
    if case["texts"] * 2 * pairs > _MOST_ATTENTION:
        case["long"] = max(2, case["long"] // 8)
        case["short"] = min(case["short"], case["long"])
    return case


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

    def codes(self, rows, cols):
        """int8 codes of normal rows, the largest of each row 127."""
        values = torch.randn(rows, cols, generator=self.rng, device="cuda")
        return torch.round(values * (127.0 / values.abs().amax(1, keepdim=True))).to(torch.int8)

    def rows_of(self, rows, dim, pad, std=1.0, dtype=None):
        """[rows, dim] as a slice of rows that are `pad` wider."""
        return self.normal(rows, dim + pad, std=std, dtype=dtype)[:, :dim]


def _lengths(case):
    """The texts' lengths in ascending order, spread evenly over the range."""
    n, low, high = case["texts"], case["short"], case["long"]
    return [high if n == 1 else low + (high - low) * i // (n - 1) for i in range(n)]


def _attention_inputs(case, seed, make):
    s = {}
    lengths = _lengths(case)
    order = torch.randperm(case["texts"], generator=torch.Generator().manual_seed(seed)).tolist()
    lens = [lengths[i] for i in order]
    # padded: every text has as many rows as the longest, packed: one behind the other
    starts = [t * case["long"] for t in range(len(lens))] if case["padded"] else [sum(lens[:t]) for t in range(len(lens))]
    rows = case["texts"] * case["long"] if case["padded"] else sum(lens)
    s["lens"], s["starts"] = lens, starts
    s["offsets"] = None if case["padded"] else torch.tensor(starts + [rows], dtype=torch.int64, device="cuda")
    s["lengths"] = torch.tensor(lens, dtype=torch.int32, device="cuda") if case["padded"] else None
    heads, kv_heads, d = case["heads"], case["kv_heads"], case["head_dim"]
    # query and key heads of a trained model have scores of a few units, more for related tokens
    if case["query"] == "all":
        both = make.normal(rows, (heads + 2 * kv_heads) * d)
        s["q"], s["k"], s["v"] = both.split([heads * d, kv_heads * d, kv_heads * d], dim=1)
    else:
        s["q"] = make.normal(case["texts"], heads * d)
        s["k"], s["v"] = make.normal(rows, 2 * kv_heads * d).split([kv_heads * d, kv_heads * d], dim=1)
    s["prefix"] = None
    if case["mask"] == "prefix":
        s["prefix"] = (make.uniform(case["texts"]) * torch.tensor(lens, device="cuda")).to(torch.int32)
    if case["bias"] == "slopes":
        s["slopes"] = torch.pow(2.0, -8.0 * torch.arange(1, heads + 1, device="cuda") / heads)
    if case["bias"] == "table":
        s["table"] = make.normal(heads, 2 * case["far"] + 1)
    if case["op"] == "attention_gradient":
        s["out_gradient"] = make.normal(rows, heads * d, std=0.1)
    return s


def _inputs(case, seed):
    make = _Maker(case, seed)
    op, s = case["op"], {}
    if op.startswith("attention"):
        return _attention_inputs(case, seed, make)
    rows, dim, pad = case["rows"], case["dim"], case["pad"]
    if op in ("norm", "norm_gradient"):
        s["x"] = make.rows_of(rows, dim, pad, std=2.0)
        s["weight"] = make.normal(dim, std=0.2) + (1.0 - case["offset"])
        if op == "norm":
            s["residual"] = make.rows_of(rows, dim, pad, std=0.5) if case["residual"] else None
        else:
            s["out_gradient"] = make.rows_of(rows, dim, pad, std=0.1)
            s["sum_gradient"] = make.rows_of(rows, dim, pad, std=0.1) if case["through"] else None
        return s
    width = case["width"]
    if case["type"] == "i8":
        s["x"], s["weight"] = make.codes(rows, dim), make.codes(width, dim)
        s["x_scales"] = (0.5 + make.uniform(rows)) / 40.0
        s["weight_scales"] = (0.5 + make.uniform(width)) / 40.0 * dim ** -0.5
        kind = _TYPES[case["out"]]
    else:
        s["x"], kind = make.rows_of(rows, dim, pad), make.type
        s["weight"] = make.normal(width, dim, std=dim ** -0.5)
    s["bias"] = make.normal(width, std=0.5, dtype=kind) if case["bias"] else None
    if op == "linear":
        s["residual"] = make.rows_of(rows, width, pad, dtype=kind) if case["residual"] else None
    else:
        s["out_gradient"] = make.rows_of(rows, width, pad, std=0.1)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if case["op"] == "attention_gradient":
        # what the forward pass has left: its rows, and the logarithm of each row's sum of exponentials
        s["out"], s["lse"] = _attention_rows(s)
    return s


# ---- the plain forms ------------------------------------------------------------------------


def _activation(name, g):
    """The activation of g and its derivative."""
    if name == "none":
        return g, torch.ones_like(g)
    if name == "silu":
        y = torch.sigmoid(g)
        return g * y, y * (1.0 + g * (1.0 - y))
    if name == "gelu":
        y = 0.5 * (1.0 + torch.erf(g * math.sqrt(0.5)))
        return g * y, y + g * torch.exp(-0.5 * g * g) * (1.0 / math.sqrt(2.0 * math.pi))
    c = math.sqrt(2.0 / math.pi)
    t = torch.tanh(c * (g + 0.044715 * g * g * g))
    return 0.5 * g * (1.0 + t), 0.5 * (1.0 + t) + 0.5 * g * (1.0 - t * t) * c * (1.0 + 3.0 * 0.044715 * g * g)


def _plain_norm(s):
    case = s["case"]
    total = s["x"].float()
    if case["residual"]:
        total = total + s["residual"].float()
    y = total * torch.rsqrt((total * total).mean(1, keepdim=True) + _EPS) * (s["weight"].float() + case["offset"])
    out = {}
    if case["out"] == "i8":
        scale = y.abs().amax(1, keepdim=True) / 127.0
        scale = torch.where(scale > 0, scale, torch.ones_like(scale))
        out["rows"] = (torch.clamp(torch.round(y * (1.0 / scale)), -127, 127) * scale).to(_DECODED[case["type"]])
    else:
        out["rows"] = y.to(_TYPES[case["out"]])
    if case["residual"]:
        out["sum"] = total.to(s["x"].dtype)
    return out


def _plain_norm_gradient(s):
    case, kind = s["case"], s["x"].dtype
    x, d = s["x"].float(), s["out_gradient"].float()
    r = torch.rsqrt((x * x).mean(1, keepdim=True) + _EPS)
    unit = x * r
    wd = d * (s["weight"].float() + case["offset"])
    dx = r * (wd - unit * (wd * unit).mean(1, keepdim=True))
    if case["through"]:
        dx = dx + s["sum_gradient"].float()
    return {"x_gradient": dx.to(kind), "weight_gradient": (d * unit).sum(0).to(kind)}


def _plain_linear(s):
    case = s["case"]
    z = s["x"].float() @ s["weight"].float().T
    if case["type"] == "i8":
        z = z * (s["x_scales"][:, None] * s["weight_scales"])
    if case["bias"]:
        z = z + s["bias"].float()
    z, _ = _activation(case["act"], z)
    if case["residual"]:
        z = z + s["residual"].float()
    return {"rows": z.to(_TYPES[case["out"]])}


def _plain_linear_gradient(s):
    case, kind = s["case"], s["x"].dtype
    x, weight, d = s["x"].float(), s["weight"].float(), s["out_gradient"].float()
    if case["act"] != "none":
        z = x @ weight.T
        d = d * _activation(case["act"], z + s["bias"].float() if case["bias"] else z)[1]
    out = {"x_gradient": (d @ weight).to(kind), "weight_gradient": (d.T @ x).to(kind)}
    if case["bias"]:
        out["bias_gradient"] = d.sum(0).to(kind)
    return out


def _groups(s):
    """Texts of similar length, as many at a time as 2^29 scores allow."""
    case = s["case"]
    order = sorted(range(len(s["lens"])), key=lambda t: -s["lens"][t])
    i = 0
    while i < len(order):
        most = s["lens"][order[i]]
        count = max(1, (1 << 29) // (case["heads"] * most * (most if case["query"] == "all" else 1)))
        yield most, order[i:i + count]
        i += count


def _padded_group(s, most, texts):
    """Queries, keys and values [texts, heads, rows, head_dim] in float32, the scores before the softmax, the cap's
    derivative, the query rows and which of them exist."""
    case = s["case"]
    heads, kv_heads, d = case["heads"], case["kv_heads"], case["head_dim"]
    lens = torch.tensor([s["lens"][t] for t in texts], device="cuda")
    starts = torch.tensor([s["starts"][t] for t in texts], device="cuda")
    place = torch.arange(most, device="cuda")
    there = place < lens[:, None]
    rows = torch.where(there, starts[:, None] + place, starts[:, None])
    k = s["k"][rows].float().view(len(texts), most, kv_heads, 1, d).expand(-1, -1, -1, heads // kv_heads, -1)
    v = s["v"][rows].float().view(len(texts), most, kv_heads, 1, d).expand(-1, -1, -1, heads // kv_heads, -1)
    k, v = (x.reshape(len(texts), most, heads, d).transpose(1, 2).contiguous() for x in (k, v))
    if case["query"] == "all":
        q_rows, q_place = rows, place.expand(len(texts), -1)
    else:
        q_rows = torch.tensor(texts, device="cuda")[:, None]
        q_place = torch.zeros_like(q_rows) if case["query"] == "first" else lens[:, None] - 1
    q = s["q"][q_rows].float().view(len(texts), -1, heads, d).transpose(1, 2).contiguous()
    raw = torch.matmul(q, k.transpose(2, 3).contiguous()) * d ** -0.5
    slope = None
    if case["cap"]:
        t = torch.tanh(raw / case["cap"])
        raw, slope = case["cap"] * t, 1.0 - t * t
    distance = place - q_place[:, :, None]
    if case["bias"] == "slopes":
        raw = raw - s["slopes"][:, None, None] * distance.abs()[:, None]
    if case["bias"] == "table":
        bins = distance.clamp(-case["far"], case["far"]) + case["far"]
        raw = raw + s["table"].float()[:, bins].transpose(0, 1)
    seen = there[:, None, :].expand_as(distance)
    if case["mask"] != "full":
        ahead = distance <= 0
        if case["mask"] == "prefix":
            ahead = ahead | (place < s["prefix"][texts][:, None, None])
        seen = seen & ahead
    scores = raw.masked_fill_(~seen[:, None], -math.inf)
    q_there = there if case["query"] == "all" else torch.ones_like(q_rows, dtype=torch.bool)
    return q, k, v, scores, slope, q_rows, q_there


def _attention_rows(s):
    """The attention's rows, and the logarithm of each row's sum of exponentials [rows, heads]."""
    case = s["case"]
    out = torch.zeros_like(s["q"], memory_format=torch.contiguous_format)
    lse = torch.full((out.shape[0], case["heads"]), -math.inf, device="cuda")
    for most, texts in _groups(s):
        _, _, v, scores, _, q_rows, q_there = _padded_group(s, most, texts)
        top = scores.amax(3, keepdim=True)
        p = torch.exp(scores - top)
        total = p.sum(3, keepdim=True)
        rows = (torch.matmul(p, v) / total).transpose(1, 2).flatten(2)
        out[q_rows[q_there]] = rows[q_there].to(out.dtype)
        lse[q_rows[q_there]] = (top + torch.log(total))[..., 0].transpose(1, 2)[q_there]
    return out, lse


def _plain_attention(s):
    return {"rows": _attention_rows(s)[0]}


def _plain_attention_gradient(s):
    case, kind = s["case"], s["q"].dtype
    heads, kv_heads, d = case["heads"], case["kv_heads"], case["head_dim"]
    out = {name: torch.zeros(s[of].shape, dtype=kind, device="cuda")
           for name, of in (("q_gradient", "q"), ("k_gradient", "k"), ("v_gradient", "v"))}
    table = torch.zeros(heads, 2 * case["far"] + 1, device="cuda")
    for most, texts in _groups(s):
        q, k, v, scores, slope, rows, there = _padded_group(s, most, texts)
        p = torch.exp(scores - scores.amax(3, keepdim=True))
        p = p / p.sum(3, keepdim=True) * there[:, None, :, None]
        g = s["out_gradient"][rows].float().view(len(texts), most, heads, d).transpose(1, 2).contiguous()
        dp = torch.matmul(g, v.transpose(2, 3).contiguous())
        ds = p * (dp - (p * dp).sum(3, keepdim=True))
        if case["bias"] == "table":
            # rows moved along by their number: a column is then one distance
            wide = torch.nn.functional.pad(ds.sum(0).flip(1), (0, most)).flatten(1)[:, :most * (2 * most - 1)]
            by_distance = wide.view(heads, most, 2 * most - 1).sum(1)
            table.index_add_(1, torch.arange(1 - most, most, device="cuda").clamp(-case["far"], case["far"]) + case["far"],
                             by_distance)
        if slope is not None:
            ds = ds * slope
        ds = ds * d ** -0.5
        dq = torch.matmul(ds, k)
        dk = torch.matmul(ds.transpose(2, 3).contiguous(), q)
        dv = torch.matmul(p.transpose(2, 3).contiguous(), g)
        dk, dv = (x.view(len(texts), kv_heads, heads // kv_heads, most, d).sum(2) for x in (dk, dv))
        for name, grad in (("q_gradient", dq), ("k_gradient", dk), ("v_gradient", dv)):
            out[name][rows[there]] = grad.transpose(1, 2).flatten(2)[there].to(kind)
    if case["bias"] == "table":
        out["table_gradient"] = table.to(kind)
    return out


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


def _address(t):
    return None if t is None else t.data_ptr()


def _stride(t):
    return 0 if t is None else t.stride(0)


def _empty(kind, *shape):
    return torch.empty(*shape, dtype=_TYPES[kind], device="cuda")


def _norm_plan(capi, s, code):
    case = s["case"]
    kind, rows, dim = case["type"], case["rows"], case["dim"]
    x, residual = s["x"], s.get("residual")
    desc = capi.norm_desc(x.data_ptr(), rows, dim, code[kind], weight=s["weight"].data_ptr(), weight_offset=case["offset"],
                          residual=_address(residual), eps=_EPS, x_stride=x.stride(0), residual_stride=_stride(residual))
    if case["op"] == "norm":
        out = _empty(case["out"], rows, dim)
        outputs = {"rows": out}
        scales = None
        if case["out"] == "i8":
            scales = _empty("f32", rows, 1)
            outputs["rows"] = torch.empty(rows, dim, dtype=_DECODED[kind], device="cuda")
        if case["residual"]:
            outputs["sum"] = _empty(kind, rows, dim)

        def norm(stream):
            capi.residual_norm(desc, out.data_ptr(), code[case["out"]], out_scales=_address(scales),
                               sum_out=_address(outputs.get("sum")), stream=stream)
            if scales is not None:
                torch.mul(out, scales, out=outputs["rows"])

        return norm, outputs
    size = capi.residual_norm_gradient_workspace_bytes(desc)
    space, d, through = _empty("i8", size), s["out_gradient"], s["sum_gradient"]
    dx, dw = _empty(kind, rows, dim), _empty(kind, dim)
    return lambda stream: capi.residual_norm_gradient(
        desc, d.data_ptr(), dx.data_ptr(), dw.data_ptr(), space.data_ptr(), size, sum_gradient=_address(through),
        out_gradient_stride=d.stride(0), sum_gradient_stride=_stride(through), stream=stream), {
            "x_gradient": dx, "weight_gradient": dw}


def _linear_plan(capi, s, code):
    case = s["case"]
    kind, rows, dim, width = case["type"], case["rows"], case["dim"], case["width"]
    x, residual = s["x"], s.get("residual")
    act = {"none": capi.ACT_NONE, "silu": capi.ACT_SILU, "gelu": capi.ACT_GELU, "gelu_tanh": capi.ACT_GELU_TANH}[case["act"]]
    more = code[case["out"] if kind == "i8" else kind]
    desc = capi.linear_desc(x.data_ptr(), rows, dim, s["weight"].data_ptr(), width, code[kind], bias=_address(s["bias"]),
                            activation=act, residual=_address(residual), epilogue_dtype=more,
                            x_scales=_address(s.get("x_scales")), weight_scales=_address(s.get("weight_scales")),
                            x_stride=x.stride(0), residual_stride=_stride(residual))
    if case["op"] == "linear":
        out = _empty(case["out"], rows, width)
        return lambda stream: capi.linear(desc, out.data_ptr(), code[case["out"]], stream=stream), {"rows": out}
    size = capi.linear_gradient_workspace_bytes(desc)
    space, d = _empty("i8", size), s["out_gradient"]
    outputs = {"x_gradient": _empty(kind, rows, dim), "weight_gradient": _empty(kind, width, dim)}
    if case["bias"]:
        outputs["bias_gradient"] = _empty(kind, width)
    return lambda stream: capi.linear_gradient(
        desc, d.data_ptr(), outputs["x_gradient"].data_ptr(), outputs["weight_gradient"].data_ptr(),
        _address(outputs.get("bias_gradient")), space.data_ptr(), size, out_gradient_stride=d.stride(0),
        stream=stream), outputs


def _attention_plan(capi, s, code):
    case = s["case"]
    kind, heads, kv_heads, d = case["type"], case["heads"], case["kv_heads"], case["head_dim"]
    q, k, v = s["q"], s["k"], s["v"]
    every = case["query"] == "all"
    desc = capi.attention_desc(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), case["texts"], q.shape[0], k.shape[0], heads, d, code[kind],
        kv_heads=kv_heads, q_offsets=_address(s["offsets"]) if every else None, k_offsets=_address(s["offsets"]),
        q_lengths=_address(s["lengths"]) if every else None, k_lengths=_address(s["lengths"]),
        q_align=capi.ATTENTION_LAST if case["query"] == "last" else capi.ATTENTION_FIRST, causal=case["mask"] != "full",
        prefix_lengths=_address(s["prefix"]), cap=case["cap"], slopes=_address(s.get("slopes")),
        distance_bias=_address(s.get("table")), max_distance=case["far"], q_stride=q.stride(0), k_stride=k.stride(0),
        v_stride=v.stride(0))
    if case["op"] == "attention":
        size = capi.attention_workspace_bytes(desc)
        space, out = _empty("i8", size), _empty(kind, *q.shape)
        return lambda stream: capi.attention(desc, out.data_ptr(), space.data_ptr(), size, stream=stream), {"rows": out}
    size = capi.attention_gradient_workspace_bytes(desc)
    space, out, lse, g = _empty("i8", size), s["out"], s["lse"], s["out_gradient"]
    outputs = {"q_gradient": _empty(kind, *q.shape), "k_gradient": _empty(kind, *k.shape), "v_gradient": _empty(kind, *v.shape)}
    if case["bias"] == "table":
        outputs["table_gradient"] = _empty(kind, heads, 2 * case["far"] + 1)
    return lambda stream: capi.attention_gradient(
        desc, out.data_ptr(), lse.data_ptr(), g.data_ptr(), outputs["q_gradient"].data_ptr(),
        outputs["k_gradient"].data_ptr(), outputs["v_gradient"].data_ptr(), space.data_ptr(), size,
        distance_bias_gradient=_address(outputs.get("table_gradient")), stream=stream), outputs


def _plan(s):
    """The descriptor, workspace and outputs that a program keeps for calls of one shape."""
    capi = _capi()
    code = {"f32": capi.F32, "f16": capi.F16, "bf16": capi.BF16, "i8": capi.I8}
    op = s["case"]["op"]
    make = _norm_plan if op.startswith("norm") else _linear_plan if op.startswith("linear") else _attention_plan
    return make(capi, s, code)


# ---- one pass -------------------------------------------------------------------------------

_PLAIN = {"norm": _plain_norm, "norm_gradient": _plain_norm_gradient, "linear": _plain_linear,
          "linear_gradient": _plain_linear_gradient, "attention": _plain_attention,
          "attention_gradient": _plain_attention_gradient}


def run(state):
    if not own:
        return _PLAIN[state["case"]["op"]](state)
    if "plan" not in state:
        state["plan"] = _plan(state)
    call, outputs = state["plan"]
    call(torch.cuda.current_stream().cuda_stream)
    return outputs


# ---- what a pass needs at least ----------------------------------------------------------------


def work(case):
    op, e = case["op"], _BYTES[case["type"]]
    if op.startswith("norm"):
        rows, dim = case["rows"], case["dim"]
        if op == "norm":
            moved = (1 + 2 * case["residual"]) * e + _BYTES[case["out"]]
            return {"bytes": rows * dim * moved + dim * e + (4 * rows if case["out"] == "i8" else 0), "flops": 5 * rows * dim}
        return {"bytes": rows * dim * (3 + case["through"]) * e + 2 * dim * e, "flops": 10 * rows * dim}
    if op.startswith("linear"):
        rows, dim, width = case["rows"], case["dim"], case["width"]
        products = 2 * rows * dim * width
        if op == "linear":
            o = _BYTES[case["out"]]
            bytes_ = e * (rows + width) * dim + rows * width * (o + (o if case["type"] == "i8" else e) * case["residual"])
            return {"bytes": bytes_, "flops": products}
        # with an activation its slope needs the product once more
        return {"bytes": e * (rows * width + 2 * rows * dim + 2 * width * dim), "flops": (2 + (case["act"] != "none")) * products}
    lengths = _lengths(case)
    heads, d = case["heads"], case["head_dim"]
    if case["query"] != "all":
        pairs, q_rows = sum(lengths), len(lengths)
    else:
        # a prefix of any length: two thirds of all pairs on average
        pairs = sum({"full": n * n, "causal": n * (n + 1) // 2, "prefix": 2 * n * n // 3}[case["mask"]] for n in lengths)
        q_rows = sum(lengths)
    q, k = q_rows * heads * d * e, sum(lengths) * case["kv_heads"] * d * e
    if op == "attention":
        return {"bytes": 2 * q + 2 * k, "flops": 4 * pairs * heads * d}
    return {"bytes": 4 * q + 4 * k + 4 * q_rows * heads, "flops": 10 * pairs * heads * d}


# ---- 64-bit results --------------------------------------------------------------------------


def _exact_attention(case, s):
    heads, kv_heads, d = case["heads"], case["kv_heads"], case["head_dim"]
    gradient = case["op"] == "attention_gradient"
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    dq, dk, dv = (torch.zeros(s[n].shape, dtype=torch.float64, device="cuda") for n in "qkv")
    table = s["table"].double() if case["bias"] == "table" else None
    d_table = torch.zeros_like(table) if gradient and table is not None else None
    for t, (start, n) in enumerate(zip(s["starts"], s["lens"])):
        own_keys = slice(start, start + n)
        own_queries = own_keys if case["query"] == "all" else slice(t, t + 1)
        place = torch.arange(n, device="cuda")
        q_place = place if case["query"] == "all" else place[:1] if case["query"] == "first" else place[-1:]
        leaves = [s["q"][own_queries].double(), s["k"][own_keys].double(), s["v"][own_keys].double()]
        leaves += [table] if table is not None else []
        if gradient:
            leaves = [x.clone().requires_grad_() for x in leaves]
        with torch.set_grad_enabled(gradient):
            q = leaves[0].view(-1, heads, d).permute(1, 0, 2)
            k, v = (x.view(n, kv_heads, d).permute(1, 0, 2).repeat_interleave(heads // kv_heads, 0) for x in leaves[1:3])
            scores = torch.bmm(q.contiguous(), k.transpose(1, 2).contiguous()) / math.sqrt(d)
            if case["cap"]:
                scores = case["cap"] * torch.tanh(scores / case["cap"])
            gap = place[None, :] - q_place[:, None]
            if case["bias"] == "slopes":
                scores = scores - s["slopes"].double()[:, None, None] * gap.abs()
            if table is not None:
                scores = scores + leaves[3][:, gap.clamp(-case["far"], case["far"]) + case["far"]]
            if case["mask"] != "full":
                hidden = gap > 0
                if s["prefix"] is not None:
                    hidden &= place[None, :] >= s["prefix"][t]
                scores = scores.masked_fill(hidden, -math.inf)
            rows = torch.bmm(torch.softmax(scores, 2), v.contiguous()).permute(1, 0, 2).reshape(-1, heads * d)
            if gradient:
                grads = torch.autograd.grad(rows, leaves, s["out_gradient"][own_queries].double())
                dq[own_queries], dk[own_keys], dv[own_keys] = grads[:3]
                if d_table is not None:
                    d_table += grads[3]
            else:
                out[own_queries] = rows
    if not gradient:
        return {"rows": out}
    result = {"q_gradient": dq, "k_gradient": dk, "v_gradient": dv}
    if d_table is not None:
        result["table_gradient"] = d_table
    return result


def exact(case, seed):
    s = _inputs(case, seed)
    op = case["op"]
    if op.startswith("attention"):
        return _exact_attention(case, s)
    x = s["x"].double()
    if op.startswith("norm"):
        weight = s["weight"].double() + case["offset"]
        if op == "norm":
            total = x + s["residual"].double() if case["residual"] else x
            y = total / (total.square().mean(1, keepdim=True) + _EPS).sqrt() * weight
            if case["out"] == "i8":
                step = y.abs().amax(1, keepdim=True) / 127
                step = step.masked_fill(step == 0, 1.0)
                y = (y / step).round().clamp(-127, 127) * step
            return {"rows": y, "sum": total} if case["residual"] else {"rows": y}
        leaves = [x.clone().requires_grad_(), weight.requires_grad_()]
        with torch.enable_grad():
            y = leaves[0] / (leaves[0].square().mean(1, keepdim=True) + _EPS).sqrt() * leaves[1]
            dx, dw = torch.autograd.grad(y, leaves, s["out_gradient"].double())
        return {"x_gradient": dx + s["sum_gradient"].double() if case["through"] else dx, "weight_gradient": dw}
    act = {"none": lambda g: g, "silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu,
           "gelu_tanh": lambda g: torch.nn.functional.gelu(g, approximate="tanh")}[case["act"]]
    weight = s["weight"].double()
    if case["type"] == "i8":
        x, weight = x * s["x_scales"].double()[:, None], weight * s["weight_scales"].double()[:, None]
    bias = s["bias"].double() if case["bias"] else torch.zeros(case["width"], dtype=torch.float64, device="cuda")
    if op == "linear":
        z = act(torch.nn.functional.linear(x, weight, bias))
        return {"rows": z + s["residual"].double() if case["residual"] else z}
    leaves = [t.clone().requires_grad_() for t in (x, weight, bias)]
    with torch.enable_grad():
        z = act(torch.nn.functional.linear(*leaves))
        dx, dw, db = torch.autograd.grad(z, leaves, s["out_gradient"].double())
    return {"x_gradient": dx, "weight_gradient": dw, "bias_gradient": db} if case["bias"] else {
        "x_gradient": dx, "weight_gradient": dw}
