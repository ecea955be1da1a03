"""Refusals of the operators of an encoder block and what they answer without touching a GPU."""

import pytest

A = 1 << 20  # an address that nothing reads here
NAN, INF = float("nan"), float("inf")


def _norm(capi, **kw):
    return capi.norm_desc(**dict(dict(x=A, rows=4, dim=8, dtype=capi.F32, weight=A, residual=A), **kw))


@pytest.mark.parametrize("kw,match", [
    (dict(dtype=2), "float32, float16 or bfloat16"),
    (dict(dtype=5), "float32, float16 or bfloat16"),
    (dict(dim=0), "dim must lie"),
    (dict(dim=16385), "dim must lie"),
    (dict(rows=-1), "rows must lie"),
    (dict(rows=2**30 + 1), "rows must lie"),
    (dict(x_stride=7), "smaller than dim"),
    (dict(residual_stride=7), "smaller than dim"),
    (dict(x_stride=-8), "smaller than dim"),
    (dict(eps=-1e-6), "eps must be finite"),
    (dict(eps=NAN), "eps must be finite"),
    (dict(eps=INF), "eps must be finite"),
    (dict(weight_offset=INF), "weight_offset finite"),
    (dict(x=None), "null device pointer"),
])
def test_norm_descriptor(capi, kw, match):
    with pytest.raises(ValueError, match=match):
        capi.residual_norm(_norm(capi, **kw), A, capi.F32)
    with pytest.raises(ValueError, match=match):
        capi.residual_norm_gradient_workspace_bytes(_norm(capi, **kw))
    with pytest.raises(ValueError, match=match):
        capi.residual_norm_gradient(_norm(capi, **kw), A, A, A, A, 1 << 30)


def test_norm_operands(capi):
    assert capi.library().zcgvs_residual_norm_max_dim() == 16384
    with pytest.raises(ValueError, match="float32 or int8"):
        capi.residual_norm(_norm(capi, dtype=capi.F16), A, capi.BF16)
    with pytest.raises(ValueError, match="float32 or int8"):
        capi.residual_norm(_norm(capi), A, capi.BINARY)
    with pytest.raises(ValueError, match="smaller than dim"):
        capi.residual_norm(_norm(capi), A, capi.F32, out_stride=7)
    with pytest.raises(ValueError, match="smaller than dim"):
        capi.residual_norm(_norm(capi), A, capi.F32, sum_out=A, sum_stride=7)
    with pytest.raises(ValueError, match="null device pointer"):
        capi.residual_norm(_norm(capi), None, capi.F32)
    with pytest.raises(ValueError, match="null device pointer"):
        capi.residual_norm(_norm(capi), A, capi.I8)  # codes without scales
    with pytest.raises(ValueError, match="null device pointer"):
        capi.residual_norm_gradient(_norm(capi), None, A, A, A, 1 << 30)
    for name in ("out_gradient_stride", "sum_gradient_stride", "x_gradient_stride"):
        with pytest.raises(ValueError, match="smaller than dim"):
            capi.residual_norm_gradient(_norm(capi), A, A, A, A, 1 << 30, **{name: 7})
    need = capi.residual_norm_gradient_workspace_bytes(_norm(capi))
    with pytest.raises(ValueError, match="too small"):
        capi.residual_norm_gradient(_norm(capi), A, A, A, A, need - 1)
    with pytest.raises(ValueError, match="too small"):
        capi.residual_norm_gradient(_norm(capi), A, A, A, None, need)
    with pytest.raises(ValueError, match="16 bytes"):
        capi.residual_norm_gradient(_norm(capi), A, A, A, A + 4, need)


def _linear(capi, **kw):
    return capi.linear_desc(**dict(dict(x=A, rows=4, dim=8, weight=A, out_dim=6, dtype=capi.F32, bias=A, residual=A), **kw))


@pytest.mark.parametrize("kw,match", [
    (dict(dtype=3), "float16, bfloat16 or int8"),
    (dict(dtype=-1), "float16, bfloat16 or int8"),
    (dict(epilogue_dtype=1), "the operands' type"),
    (dict(dtype=2), "the operands' type"),  # int8 codes with int8 biases
    (dict(activation=4), "unknown activation"),
    (dict(activation=-1), "unknown activation"),
    (dict(dim=0), "must be positive"),
    (dict(out_dim=-1), "must be positive"),
    (dict(dim=2**24 + 1), "at most 2\\^24"),
    (dict(out_dim=2**24 + 1), "at most 2\\^24"),
    (dict(rows=-1), "rows must lie"),
    (dict(rows=2**30 + 1), "rows must lie"),
    (dict(x_stride=7), "smaller than dim"),
    (dict(weight_stride=7), "smaller than dim"),
    (dict(residual_stride=5), "smaller than out_dim"),
    (dict(x=None), "null device pointer"),
    (dict(weight=None), "null device pointer"),
])
def test_linear_descriptor(capi, kw, match):
    with pytest.raises(ValueError, match=match):
        capi.linear(_linear(capi, **kw), A, capi.F32)
    with pytest.raises(ValueError, match=match):
        capi.linear_gradient_workspace_bytes(_linear(capi, **kw))
    with pytest.raises(ValueError, match=match):
        capi.linear_gradient(_linear(capi, **kw), A, A, A, A, A, 1 << 30)


def test_linear_int8(capi):
    codes = dict(dtype=capi.I8, epilogue_dtype=capi.F16, x_scales=A, weight_scales=A)
    with pytest.raises(ValueError, match="131072 codes"):
        capi.linear(_linear(capi, **dict(codes, dim=131073)), A, capi.F16)
    for name in ("x_scales", "weight_scales"):
        with pytest.raises(ValueError, match="need the scales"):
            capi.linear(_linear(capi, **dict(codes, **{name: None})), A, capi.F16)
    with pytest.raises(ValueError, match="the bias's type or float32"):
        capi.linear(_linear(capi, **codes), A, capi.BF16)
    with pytest.raises(ValueError, match="the bias's type or float32"):
        capi.linear(_linear(capi, **codes), A, capi.I8)
    with pytest.raises(ValueError, match="takes float operands"):
        capi.linear_gradient_workspace_bytes(_linear(capi, **codes))
    with pytest.raises(ValueError, match="takes float operands"):
        capi.linear_gradient(_linear(capi, **codes), A, A, A, A, A, 1 << 30)


def test_linear_operands(capi):
    with pytest.raises(ValueError, match="the bias's type or float32"):
        capi.linear(_linear(capi, dtype=capi.F16), A, capi.BF16)
    with pytest.raises(ValueError, match="smaller than out_dim"):
        capi.linear(_linear(capi), A, capi.F32, out_stride=5)
    with pytest.raises(ValueError, match="null device pointer"):
        capi.linear(_linear(capi), None, capi.F32)
    with pytest.raises(ValueError, match="null device pointer"):
        capi.linear_gradient(_linear(capi), None, A, A, A, A, 1 << 30)
    for name, short in (("out_gradient_stride", 5), ("x_gradient_stride", 7), ("weight_gradient_stride", 7)):
        with pytest.raises(ValueError, match="smaller than its row"):
            capi.linear_gradient(_linear(capi), A, A, A, A, A, 1 << 30, **{name: short})
    need = capi.linear_gradient_workspace_bytes(_linear(capi))
    with pytest.raises(ValueError, match="too small"):
        capi.linear_gradient(_linear(capi), A, A, A, A, A, need - 1)
    with pytest.raises(ValueError, match="too small"):
        capi.linear_gradient(_linear(capi), A, A, A, A, None, need)
    with pytest.raises(ValueError, match="16 bytes"):
        capi.linear_gradient(_linear(capi), A, A, A, A, A + 8, need)


def _attention(capi, **kw):
    args = dict(q=A, k=A, v=A, texts=2, q_rows=6, k_rows=6, heads=4, head_dim=8, dtype=capi.F32, kv_heads=2)
    return capi.attention_desc(**dict(args, **kw))


ATTENTION_REFUSALS = [
    (dict(dtype=2), "float32, float16 or bfloat16"),
    (dict(heads=0), "multiple of kv_heads"),
    (dict(heads=5), "multiple of kv_heads"),
    (dict(heads=1026), "multiple of kv_heads"),
    (dict(kv_heads=-1), "multiple of kv_heads"),
    (dict(head_dim=0), "head_dim must lie"),
    (dict(head_dim=129), "head_dim must lie"),
    (dict(q_rows=-2), "must lie in \\[0, 2\\^28\\]"),
    (dict(k_rows=2**28 + 2), "must lie in \\[0, 2\\^28\\]"),
    (dict(texts=-1), "texts must lie"),
    (dict(texts=2**24 + 1, q_offsets=A, k_offsets=A), "texts must lie"),
    (dict(q_rows=7), "multiple of texts"),
    (dict(k_rows=7), "multiple of texts"),
    (dict(q_stride=31), "smaller than its heads"),
    (dict(k_stride=15), "smaller than its heads"),
    (dict(v_stride=15), "smaller than its heads"),
    (dict(q_align=2), "unknown alignment"),
    (dict(prefix_lengths=A), "need the causal mask"),
    (dict(scale=NAN), "must be finite"),
    (dict(scale=INF), "must be finite"),
    (dict(cap=-1.0), "cap at least 0"),
    (dict(cap=NAN), "must be finite"),
    (dict(distance_bias=A, max_distance=-1), "max_distance must lie"),
    (dict(distance_bias=A, max_distance=513), "max_distance must lie"),
    (dict(q=None), "null device pointer"),
    (dict(k=None), "null device pointer"),
    (dict(v=None), "null device pointer"),
]


@pytest.mark.parametrize("kw,match", ATTENTION_REFUSALS)
def test_attention_descriptor(capi, kw, match):
    with pytest.raises(ValueError, match=match):
        capi.attention_workspace_bytes(_attention(capi, **kw))
    with pytest.raises(ValueError, match=match):
        capi.attention(_attention(capi, **kw), A, A, 1 << 30)
    with pytest.raises(ValueError, match=match):
        capi.attention_gradient_workspace_bytes(_attention(capi, **kw))
    with pytest.raises(ValueError, match=match):
        capi.attention_gradient(_attention(capi, **kw), A, A, A, A, A, A, A, 1 << 30)


def test_attention_gradient_operands(capi):
    for name in ("out_stride", "out_gradient_stride", "q_gradient_stride", "k_gradient_stride", "v_gradient_stride"):
        with pytest.raises(ValueError, match="smaller than its heads"):
            capi.attention_gradient(_attention(capi), A, A, A, A, A, A, A, 1 << 30, **{name: 15})
    for i in range(6):
        with pytest.raises(ValueError, match="null device pointer"):
            capi.attention_gradient(_attention(capi), *(None if i == j else A for j in range(6)), A, 1 << 30)
    with pytest.raises(ValueError, match="needs the distance bias"):
        capi.attention_gradient(_attention(capi), A, A, A, A, A, A, A, 1 << 30, distance_bias_gradient=A)
    need = capi.attention_gradient_workspace_bytes(_attention(capi))
    with pytest.raises(ValueError, match="too small"):
        capi.attention_gradient(_attention(capi), A, A, A, A, A, A, A, need - 1)
    with pytest.raises(ValueError, match="too small"):
        capi.attention_gradient(_attention(capi), A, A, A, A, A, A, None, need)
    with pytest.raises(ValueError, match="16 bytes"):
        capi.attention_gradient(_attention(capi), A, A, A, A, A, A, A + 4, need)
    biased = _attention(capi, distance_bias=A, max_distance=100)
    assert capi.attention_gradient_workspace_bytes(biased) > need


def test_attention_operands(capi):
    assert capi.library().zcgvs_attention_max_head_dim() == 128
    assert capi.library().zcgvs_attention_max_distance() == 512
    with pytest.raises(ValueError, match="smaller than its heads"):
        capi.attention(_attention(capi), A, A, 1 << 30, out_stride=31)
    with pytest.raises(ValueError, match="null device pointer"):
        capi.attention(_attention(capi), None, A, 1 << 30)
    long = _attention(capi, q_rows=2, k_rows=100_000)  # split keys
    need = capi.attention_workspace_bytes(long)
    assert need > 256
    with pytest.raises(ValueError, match="too small"):
        capi.attention(long, A, A, need - 1)
    with pytest.raises(ValueError, match="too small"):
        capi.attention(long, A, None, need)
    with pytest.raises(ValueError, match="16 bytes"):
        capi.attention(long, A, A + 4, need)


def test_null_descriptors(capi):
    lib = capi.library()
    assert lib.zcgvs_attention(None, A, 0, None, A, 0, None) == capi.ERR_INVALID_ARGUMENT
    assert lib.zcgvs_linear(None, A, 0, capi.F32, None) == capi.ERR_INVALID_ARGUMENT
    assert lib.zcgvs_linear_gradient_workspace_bytes(None) == 0 and "null descriptor" in capi.last_error()
    assert lib.zcgvs_residual_norm(None, A, 0, capi.F32, None, None, 0, None) == capi.ERR_INVALID_ARGUMENT
    assert lib.zcgvs_residual_norm_gradient_workspace_bytes(None) == 0 and "null descriptor" in capi.last_error()


def test_empty_work_returns_ok(capi):
    capi.residual_norm(_norm(capi, rows=0, x=None, residual=None), None, capi.F32)
    capi.residual_norm_gradient(_norm(capi), None, None, None, None, 0)  # no gradient is wanted
    capi.residual_norm_gradient(_norm(capi, rows=0, x=None), None, A, None, None, 0)
    capi.linear(_linear(capi, rows=0, x=None, weight=None), None, capi.F32)
    capi.linear_gradient(_linear(capi), None, None, None, None, None, 0)  # no gradient is wanted
    capi.linear_gradient(_linear(capi, rows=0, x=None, weight=None), None, A, None, None, None, 0)
    for kw in (dict(texts=0), dict(q_rows=0), dict(texts=0, q_rows=0, k_rows=0, q=None, k=None, v=None)):
        capi.attention(_attention(capi, **kw), None, None, 0)
    capi.attention_gradient(_attention(capi, texts=0, q_rows=0, k_rows=0), *(None,) * 6, None, 0)
