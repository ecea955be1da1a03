"""Encoder blocks between the token rows of a DeviceEmbedder and the mean over each text.

    h = norm(x);    x = x + attention(h qkv^T + qkv_bias) out^T       (residual_norm, linear, attention, linear)
    h = norm(x);    x = x + (act(h gate^T) * (h up^T)) down^T         (residual_norm, gated_projection, linear)

block after block, and a last norm of x. The texts stay packed: attention finds them by their offsets, and no row
of padding is computed. The residual rows x are of the model's type, rounded once a sublayer.

    encoder = EncoderBlocks(blocks, final_norm, heads=12, dtype=capi.F16)
    model = DeviceEmbedder(table, gate, up, projection, dtype=capi.F16, encoder=encoder)
"""

from __future__ import annotations

import numpy as np

from . import capi
from .embedder import _STORAGE, _matrix, _refuse


class EncoderBlocks:
    """Weights of the blocks (host arrays of `dtype`, bfloat16 as uint16 bit patterns).

    Each block is a dict: norm1 and norm2 [dim], qkv [(heads + 2 kv_heads) head_dim, dim], out [dim, heads head_dim],
    gate and up [hidden, dim], down [dim, hidden], and optionally qkv_bias and distance_bias
    [heads, 2 max_distance + 1]. slopes [heads] (float32) serve all blocks."""

    REQUIRED = ("norm1", "qkv", "out", "norm2", "gate", "up", "down")
    OPTIONAL = ("qkv_bias", "distance_bias")

    def __init__(self, blocks, final_norm, *, heads, kv_heads=0, dtype, activation=capi.ACT_SILU, eps=1e-6, causal=False,
                 cap=0.0, slopes=None):
        if dtype not in _STORAGE:
            _refuse("dtype must be F32, F16 or BF16")
        element = _STORAGE[dtype]
        final_norm = _matrix("final_norm", final_norm, (None,), element)
        self.dim, self.heads, self.kv_heads = final_norm.shape[0], heads, kv_heads or heads
        self.dtype, self.activation, self.eps, self.causal, self.cap = dtype, activation, eps, causal, cap
        if not 1 <= self.heads <= 1024 or self.kv_heads < 1 or self.heads % self.kv_heads:
            _refuse("heads must lie in [1, 1024] and be a multiple of kv_heads")
        limits = capi.library()
        self._limits = dict(dim=limits.zcgvs_residual_norm_max_dim(), head_dim=limits.zcgvs_attention_max_head_dim(),
                            max_distance=limits.zcgvs_attention_max_distance())
        if not 1 <= self.dim <= self._limits["dim"]:
            _refuse(f"final_norm must have 1 to {self._limits['dim']} values")
        if not (np.isfinite(eps) and eps >= 0 and np.isfinite(cap) and cap >= 0):
            _refuse("eps and cap must be finite and at least 0")
        if activation not in (capi.ACT_SILU, capi.ACT_GELU, capi.ACT_GELU_TANH):
            _refuse("unknown activation")
        self.head_dim = 0
        self.blocks = [self._block(block, element) for block in blocks]
        self.final_norm = capi.DeviceArray.from_host(final_norm)
        self.slopes = None
        if slopes is not None:
            self.slopes = capi.DeviceArray.from_host(_matrix("slopes", slopes, (heads,), np.dtype(np.float32)))
        self.element = element

    def _block(self, block, element):
        missing = [name for name in self.REQUIRED if block.get(name) is None]
        unknown = set(block) - set(self.REQUIRED) - set(self.OPTIONAL)
        if missing or unknown:
            _refuse(f"a block without {missing}" if missing else f"a block's {sorted(unknown)}")
        out = _matrix("out", block["out"], (self.dim, None), element)
        if out.shape[1] == 0 or out.shape[1] % self.heads:
            _refuse("out must have heads * head_dim columns")
        if self.head_dim and out.shape[1] != self.heads * self.head_dim:
            _refuse("all blocks must have one head_dim")
        self.head_dim = out.shape[1] // self.heads
        if self.head_dim > self._limits["head_dim"]:
            _refuse(f"heads hold at most {self._limits['head_dim']} values, not {self.head_dim}")
        wide = (self.heads + 2 * self.kv_heads) * self.head_dim
        hidden = _matrix("a block's gate", block["gate"], (None, self.dim), element).shape[0]
        shapes = dict(norm1=(self.dim,), norm2=(self.dim,), qkv=(wide, self.dim), out=out.shape, gate=(hidden, self.dim),
                      up=(hidden, self.dim), down=(self.dim, hidden), qkv_bias=(wide,), distance_bias=(self.heads, None))
        held = {name: _matrix(f"a block's {name}", values, shapes[name], element)
                for name, values in block.items() if values is not None}
        if "distance_bias" in held and held["distance_bias"].shape[1] % 2 == 0:
            _refuse("distance_bias must have 2 max_distance + 1 columns")
        if "distance_bias" in held and held["distance_bias"].shape[1] // 2 > self._limits["max_distance"]:
            _refuse(f"distance_bias reaches to distances of at most {self._limits['max_distance']}")
        return {name: capi.DeviceArray.from_host(values) for name, values in held.items()}

    def _attention_desc(self, block, qkv, offsets, texts, tokens):
        wide = (self.heads + 2 * self.kv_heads) * self.head_dim
        start = qkv.ptr
        key = start + self.heads * self.head_dim * self.element.itemsize
        value = key + self.kv_heads * self.head_dim * self.element.itemsize
        bias = block.get("distance_bias")
        return capi.attention_desc(start, key, value, texts, tokens, tokens, self.heads, self.head_dim, self.dtype,
                                   kv_heads=self.kv_heads, q_offsets=offsets, k_offsets=offsets, causal=self.causal,
                                   cap=self.cap, slopes=self.slopes, distance_bias=bias,
                                   max_distance=0 if bias is None else bias.shape[1] // 2,
                                   q_stride=wide, k_stride=wide, v_stride=wide)

    def forward(self, buffer, x, offsets, texts, tokens, stream, keep=False):
        """The last norm's rows [tokens, dim] from x (its rows are left as they were) and, with `keep`, each
        block's rows for gradient(). `buffer(name, shape, kind)` gives work buffers."""
        kept = []

        def rows(name, width, kind=None):
            index = len(kept) if keep else (len(kept) & 1 if name.startswith("x") else 0)
            return buffer(f"block {index} {name}", (tokens, width), kind or self.element)

        wide = (self.heads + 2 * self.kv_heads) * self.head_dim
        for block in self.blocks:
            h1, qkv, mixed = rows("h1", self.dim), rows("qkv", wide), rows("mixed", self.heads * self.head_dim)
            lse = rows("lse", self.heads, np.float32) if keep else None
            x1, h2, x2 = rows("x1", self.dim), rows("h2", self.dim), rows("x2", self.dim)
            hidden = rows("hidden", block["gate"].shape[0])
            descs = dict(
                norm1=capi.norm_desc(x, tokens, self.dim, self.dtype, weight=block["norm1"], eps=self.eps),
                qkv=capi.linear_desc(h1, tokens, self.dim, block["qkv"], wide, self.dtype, bias=block.get("qkv_bias")),
                attention=self._attention_desc(block, qkv, offsets, texts, tokens),
                out=capi.linear_desc(mixed, tokens, self.heads * self.head_dim, block["out"], self.dim, self.dtype,
                                     residual=x),
                norm2=capi.norm_desc(x1, tokens, self.dim, self.dtype, weight=block["norm2"], eps=self.eps),
                gated=capi.gated_desc(h2, tokens, self.dim, block["gate"], block["up"], hidden.shape[1], self.dtype,
                                      self.activation),
                down=capi.linear_desc(hidden, tokens, hidden.shape[1], block["down"], self.dim, self.dtype, residual=x1))
            size = capi.attention_workspace_bytes(descs["attention"])
            capi.residual_norm(descs["norm1"], h1, self.dtype, stream=stream)
            capi.linear(descs["qkv"], qkv, self.dtype, stream=stream)
            capi.attention(descs["attention"], mixed, buffer("attention workspace", (size,), np.uint8), size, lse=lse,
                           stream=stream)
            capi.linear(descs["out"], x1, self.dtype, stream=stream)
            capi.residual_norm(descs["norm2"], h2, self.dtype, stream=stream)
            capi.gated_projection(descs["gated"], hidden, stream=stream)
            capi.linear(descs["down"], x2, self.dtype, stream=stream)
            kept.append(dict(descs, mixed=mixed, lse=lse))
            x = x2
        final = capi.norm_desc(x, tokens, self.dim, self.dtype, weight=self.final_norm, eps=self.eps)
        out = buffer("encoded", (tokens, self.dim), self.element)
        capi.residual_norm(final, out, self.dtype, stream=stream)
        return out, dict(blocks=kept, final=final)

    def gradient(self, buffer, kept, out_gradient, tokens, stream):
        """From the gradient of forward()'s rows: that of x, and those of the weights as device arrays of their
        type, dict(blocks=[{name: array}], final_norm=array). `kept`: what forward(keep=True) gave."""

        def like(array):
            return capi.DeviceArray(array.shape, self.element)

        def norm(desc, dy, weight, name, sum_gradient=None):
            dx, dw = buffer(name, (tokens, self.dim), self.element), like(weight)
            size = capi.residual_norm_gradient_workspace_bytes(desc)
            capi.residual_norm_gradient(desc, dy, dx, dw, buffer("norm workspace", (size,), np.uint8), size,
                                        sum_gradient=sum_gradient, stream=stream)
            return dx, dw

        def linear(desc, dy, weight, name, bias=None):
            dx, dw = buffer(name, (tokens, desc.dim), self.element), like(weight)
            db = None if bias is None else like(bias)
            size = capi.linear_gradient_workspace_bytes(desc)
            capi.linear_gradient(desc, dy, dx, dw, db, buffer("linear workspace", (size,), np.uint8), size, stream=stream)
            return dx, dw, db

        wide = (self.heads + 2 * self.kv_heads) * self.head_dim
        dx, final_norm = norm(kept["final"], out_gradient, self.final_norm, "x gradient")
        blocks = []
        for block, saved in zip(reversed(self.blocks), reversed(kept["blocks"])):
            grads = {}
            d_hidden, grads["down"], _ = linear(saved["down"], dx, block["down"], "hidden gradient")
            d_h = buffer("h gradient", (tokens, self.dim), self.element)
            grads["gate"], grads["up"] = like(block["gate"]), like(block["up"])
            size = capi.gated_gradient_workspace_bytes(saved["gated"])
            capi.gated_gradient(saved["gated"], d_hidden, d_h, grads["gate"], grads["up"],
                                buffer("block gated workspace", (size,), np.uint8), size, stream=stream)
            dx1, grads["norm2"] = norm(saved["norm2"], d_h, block["norm2"], "x1 gradient", dx)
            d_mixed, grads["out"], _ = linear(saved["out"], dx1, block["out"], "mixed gradient")
            d_qkv = buffer("qkv gradient", (tokens, wide), self.element)
            key = d_qkv.ptr + self.heads * self.head_dim * self.element.itemsize
            value = key + self.kv_heads * self.head_dim * self.element.itemsize
            if "distance_bias" in block:
                grads["distance_bias"] = like(block["distance_bias"])
            size = capi.attention_gradient_workspace_bytes(saved["attention"])
            capi.attention_gradient(saved["attention"], saved["mixed"], saved["lse"], d_mixed, d_qkv, key, value,
                                    buffer("attention gradient workspace", (size,), np.uint8), size,
                                    distance_bias_gradient=grads.get("distance_bias"), q_gradient_stride=wide,
                                    k_gradient_stride=wide, v_gradient_stride=wide, stream=stream)
            d_h, grads["qkv"], bias = linear(saved["qkv"], d_qkv, block["qkv"], "h gradient", block.get("qkv_bias"))
            if bias is not None:
                grads["qkv_bias"] = bias
            dx, grads["norm1"] = norm(saved["norm1"], d_h, block["norm1"], "x gradient", dx1)
            blocks.append(grads)
        return dx, dict(blocks=blocks[::-1], final_norm=final_norm)
