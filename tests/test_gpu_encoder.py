"""An embedding model with encoder blocks: the operators of a block one behind the other, forward and backward, against
the formulas in 64 bits."""

import math

import numpy as np
import pytest
import torch

from operator_helpers import from_bits, kind_code, to_bits

pytestmark = pytest.mark.gpu

TYPES = dict(f32=torch.float32, f16=torch.float16, bf16=torch.bfloat16)
VOCAB, DIM, HIDDEN, WIDTH = 300, 48, 72, 40


class Round(torch.autograd.Function):
    """Rounds a stored tensor, and its gradient, to a type."""

    @staticmethod
    def forward(ctx, x, kind):
        ctx.kind = kind
        return x.to(kind).to(x.dtype)

    @staticmethod
    def backward(ctx, g):
        return g.to(ctx.kind).to(g.dtype), None


def weights(rng, kind, heads, kv_heads, head_dim, *, blocks=2, far=0, bias=False):
    def draw(*shape, size=None):
        return to_bits((size or shape[-1] ** -0.5) * rng.standard_normal(shape), kind)

    wide = (heads + 2 * kv_heads) * head_dim
    made = []
    for _ in range(blocks):
        block = dict(norm1=draw(DIM, size=1.0), qkv=draw(wide, DIM), out=draw(DIM, heads * head_dim),
                     norm2=draw(DIM, size=1.0), gate=draw(56, DIM), up=draw(56, DIM), down=draw(DIM, 56))
        if bias:
            block["qkv_bias"] = draw(wide, size=0.5)
        if far:
            block["distance_bias"] = draw(heads, 2 * far + 1, size=1.0)
        made.append(block)
    return dict(blocks=made, final_norm=draw(DIM, size=1.0), table=draw(VOCAB, DIM, size=1.0), gate=draw(HIDDEN, DIM),
                up=draw(HIDDEN, DIM), projection=draw(WIDTH, HIDDEN))


def as_tensors(w, kind, dtype):
    def one(bits):
        return torch.tensor(from_bits(bits, kind), dtype=dtype, requires_grad=True)

    return {name: [{n: one(b) for n, b in block.items()} for block in held] if name == "blocks" else one(held)
            for name, held in w.items()}


def chain(p, texts, heads, kv_heads, head_dim, *, causal=False, cap=0.0, slopes=None, rounded=lambda x: x):
    """The hidden rows; `rounded` is applied to what the operators store."""
    silu = torch.nn.functional.silu

    def norm(x, weight):
        return rounded(x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6) * weight)

    def attended(qkv, block):
        n = len(qkv)
        q, k, v = (part.reshape(n, -1, head_dim).transpose(0, 1) for part in
                   qkv.split([heads * head_dim, kv_heads * head_dim, kv_heads * head_dim], 1))
        k, v = (part.repeat_interleave(heads // kv_heads, 0) for part in (k, v))
        s = q @ k.transpose(1, 2) / math.sqrt(head_dim)
        if cap:
            s = cap * torch.tanh(s / cap)
        apart = torch.arange(n)[None, :] - torch.arange(n)[:, None]
        if slopes is not None:
            s = s - torch.tensor(slopes, dtype=s.dtype)[:, None, None] * apart.abs()
        if "distance_bias" in block:
            far = block["distance_bias"].shape[1] // 2
            s = s + block["distance_bias"][:, apart.clamp(-far, far) + far]
        if causal:
            s = s.masked_fill(apart > 0, -math.inf)
        return rounded((rounded(s.softmax(-1)) @ v).transpose(0, 1).reshape(n, -1))

    out = []
    for ids in texts:
        if len(ids) == 0:
            out.append(torch.zeros(DIM, dtype=p["table"].dtype))
            continue
        x = rounded(p["table"][torch.tensor(ids, dtype=torch.int64)])
        for block in p["blocks"]:
            qkv = norm(x, block["norm1"]) @ block["qkv"].T
            qkv = rounded(qkv + block["qkv_bias"] if "qkv_bias" in block else qkv)
            x = rounded(attended(qkv, block) @ block["out"].T + x)
            h = norm(x, block["norm2"])
            x = rounded(rounded(silu(h @ block["gate"].T) * (h @ block["up"].T)) @ block["down"].T + x)
        out.append(rounded(norm(x, p["final_norm"]).mean(0)))
    rows = torch.stack(out)
    return rounded(silu(rows @ p["gate"].T) * (rows @ p["up"].T))


def flat(grads):
    """Gradients by name, a block's under its number."""
    named = {}
    for name, held in grads.items():
        if name == "blocks":
            named.update({f"{i} {n}": g for i, block in enumerate(held) for n, g in block.items()})
        else:
            named[name] = held
    return named


def batch(rng, lengths):
    """Tokens and offsets with rows of no text at both ends, padding and ids out of range; and the texts' own ids."""
    texts = [rng.integers(1, VOCAB, n) for n in lengths]
    ids, offsets = [7, 9], [2]
    for t, text in enumerate(texts):
        mixed = list(text)
        for extra in (0, VOCAB, -1)[:t % 4]:
            mixed.insert(int(rng.integers(0, len(mixed) + 1)), extra)
        ids += mixed
        offsets.append(len(ids))
    return np.array(ids + [3, 4], np.int32), np.array(offsets, np.int64), texts


def embedder(capi, kind, w, heads, kv_heads, **more):
    from zcgvs_amd.embedder import DeviceEmbedder
    from zcgvs_amd.encoder import EncoderBlocks
    code = kind_code(capi, kind)
    encoder = EncoderBlocks(w["blocks"], w["final_norm"], heads=heads, kv_heads=kv_heads, dtype=code, **more)
    return DeviceEmbedder(w["table"], w["gate"], w["up"], w["projection"], dtype=code, padding_id=0, encoder=encoder)


CASES = {
    "plain": (dict(heads=3, kv_heads=3, head_dim=16), dict(), {}, [0, 1, 17, 40, 2, 130, 0]),
    "shared-heads": (dict(heads=4, kv_heads=2, head_dim=24), dict(bias=True), dict(causal=True), [33, 1, 64, 5]),
    "distances": (dict(heads=2, kv_heads=1, head_dim=32), dict(far=9, blocks=3), dict(cap=4.0), [70, 3, 20, 0]),
    "slopes": (dict(heads=2, kv_heads=2, head_dim=8), dict(bias=True, blocks=1), dict(slopes=[0.5, 0.25]), [18, 90]),
}


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("case", CASES)
def test_rows_and_gradients(gpu, case, kind):
    """Forward and backward against the formulas. The tolerance is what rounding does to the formulas themselves: the
    chain is evaluated once more with every stored tensor and its gradient rounded to the type, as the operators round
    (in 32 bits throughout for float32). The kernels' roundings are another draw of the same size, so that the norm of
    their error is near that of this one; four times it leaves room for the roundings that the chain does not have
    (the softmax's gradient, float32 sums)."""
    capi = gpu
    heads, sizes, options, lengths = CASES[case]
    rng = np.random.default_rng(len(case))
    w = weights(rng, kind, **heads, **sizes)
    ids, offsets, texts = batch(rng, lengths)
    upstream = to_bits(rng.standard_normal((len(texts), HIDDEN)), kind)
    slopes = options.get("slopes")
    model = embedder(capi, kind, w, heads["heads"], heads["kv_heads"],
                     **dict(options, slopes=None if slopes is None else np.array(slopes, np.float32)))

    def formulas(dtype, rounded):
        p = as_tensors(w, kind, dtype)
        rows = chain(p, texts, **heads, **options, rounded=rounded)
        rows.backward(torch.tensor(from_bits(upstream, kind), dtype=dtype))
        grads = {n: v for n, v in p.items() if n != "projection"}
        grads = flat(dict(grads, blocks=[{n: g.grad for n, g in b.items()} for b in p["blocks"]],
                          **{n: v.grad for n, v in grads.items() if n != "blocks"}))
        return rows.detach().double().numpy(), {n: g.double().numpy() for n, g in grads.items()}

    stored = TYPES[kind]
    rows, grads = formulas(torch.float64, lambda x: x)
    if kind == "f32":
        rough, rough_grads = formulas(torch.float32, lambda x: x)
    else:
        rough, rough_grads = formulas(torch.float64, lambda x: Round.apply(x, stored))
    half_step = torch.finfo(stored).eps / 2

    hidden = from_bits(model.hidden_rows(ids, offsets), kind)
    found = model.gradient(ids, offsets, upstream)
    capi.synchronize()
    encoder = found.pop("encoder")
    got = flat(dict(found, blocks=encoder["blocks"], final_norm=encoder["final_norm"]))
    assert set(got) == set(grads)

    def near(name, have, want, roughly):
        error = np.linalg.norm(have - want)
        allowed = 4 * np.linalg.norm(roughly - want) + half_step * np.linalg.norm(want)  # and its own rounding
        print(f"{name}: {error:.3g} of {allowed:.3g}, size {np.linalg.norm(want):.3g}")
        assert error <= allowed, name

    near("rows", hidden, rows, rough)
    for name, want in grads.items():
        have = got[name].to_host()
        have = have.astype(np.float64) if name == "table" else from_bits(have, kind)
        near(name, have, want, rough_grads[name])
    outside = np.setdiff1d(np.arange(VOCAB), np.concatenate(texts).astype(int))
    assert np.all(got["table"].to_host()[outside] == 0.0)


def test_queries_and_calls_that_follow(gpu):
    """Queries of calls of growing and shrinking sizes, on changing streams, are those of a fresh model."""
    capi = gpu
    rng = np.random.default_rng(5)
    w = weights(rng, "f16", 2, 2, 32, far=3)
    model = embedder(capi, "f16", w, 2, 2)
    streams = [capi.Stream(), None, capi.Stream()]
    for i, lengths in enumerate(([4, 9], [200, 0, 31], [1], [300, 300], [0, 0], [5, 77, 2])):
        ids, offsets, texts = batch(rng, lengths)
        stream = streams[i % 3]
        queries = model.embed(ids, offsets, stream=stream)
        (stream or capi).synchronize()
        fresh = embedder(capi, "f16", w, 2, 2)
        want = fresh.embed(ids, offsets)
        capi.synchronize()
        assert np.array_equal(queries.to_host(), want.to_host())
        assert np.array_equal(model.hidden_rows(ids, offsets), fresh.hidden_rows(ids, offsets))
    empty = model.gradient(np.zeros(0, np.int32), np.zeros(1, np.int64), np.zeros((0, HIDDEN), np.float16))
    assert empty["encoder"] is None
    assert np.all(empty["table"].to_host() == 0.0)


def test_gradient_against_differences(gpu):
    """A step along the gradient changes the loss by what it promises (central differences of the formulas in 64 bits:
    their third order and the gradient's float32 sums stay below a thousandth of the slope)."""
    capi = gpu
    rng = np.random.default_rng(6)
    heads = dict(heads=2, kv_heads=1, head_dim=16)
    w = weights(rng, "f32", **heads, far=4, bias=True)
    ids, offsets, texts = batch(rng, [12, 30, 1])
    target = rng.standard_normal((3, HIDDEN))
    model = embedder(capi, "f32", w, 2, 1, cap=5.0)

    def loss(p):
        with torch.no_grad():
            rows = chain(p, texts, **heads, cap=5.0).numpy()
        return 0.5 * ((rows - target) ** 2).sum()

    hidden = model.hidden_rows(ids, offsets).astype(np.float64)
    found = model.gradient(ids, offsets, (hidden - target).astype(np.float32))
    capi.synchronize()
    encoder = found.pop("encoder")
    grads = {n: torch.tensor(g.to_host().astype(np.float64)) for n, g in
             flat(dict(found, blocks=encoder["blocks"], final_norm=encoder["final_norm"])).items()}
    slope = sum(float((g ** 2).sum()) for g in grads.values())
    step = 1e-4 / math.sqrt(slope)

    def moved(sign):
        p = as_tensors(w, "f32", torch.float64)
        return {name: [{n: b + sign * step * grads[f"{i} {n}"] for n, b in block.items()} for i, block in enumerate(held)]
                if name == "blocks" else held + sign * step * grads[name] if name in grads else held
                for name, held in p.items()}

    change = (loss(moved(1)) - loss(moved(-1))) / (2 * step)
    assert abs(change - slope) <= 1e-3 * slope
