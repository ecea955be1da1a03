"""Refusals of the embedding-model operators and what they answer without touching a GPU."""

import pytest

A = 1 << 20  # an address that nothing reads here


def _embedding(capi, **kw):
    args = dict(table=A, vocab=10, dim=8, dtype=capi.F32, ids=A, token_count=5)
    return capi.embedding_desc(**dict(args, **kw))


def _gated(capi, **kw):
    args = dict(x=A, rows=4, dim=8, gate=A, up=A, hidden=6, dtype=capi.F32, activation=capi.ACT_SILU)
    return capi.gated_desc(**dict(args, **kw))


def _adapted(capi, **kw):
    args = dict(x=A, rows=4, dim=8, weight=A, out_dim=6, dtype=capi.F32, down=A, up=A, adapter_count=3, max_rank=4,
                adapter_ids=A)
    return capi.adapted_desc(**dict(args, **kw))


@pytest.mark.parametrize("kw,match", [
    (dict(vocab=0), "must be positive"),
    (dict(dim=-1), "must be positive"),
    (dict(vocab=2**31 - 1), "below 2\\^31 - 1"),
    (dict(token_count=-1), "token_count"),
    (dict(token_count=2**28 + 1), "token_count"),
    (dict(bag_offsets=A, bag_count=-1), "bag_count"),
    (dict(bag_count=3), "needs bag_offsets"),
    (dict(reduce=2), "unknown reduction"),
    (dict(ids=None), "null token ids"),
])
def test_embedding_descriptor(capi, kw, match):
    with pytest.raises(ValueError, match=match):
        capi.embedding_lookup(_embedding(capi, **kw), A, capi.F32)
    with pytest.raises(ValueError, match=match):
        capi.embedding_gradient_workspace_bytes(_embedding(capi, **kw))
    with pytest.raises(ValueError, match=match):
        capi.embedding_gradient(_embedding(capi, **kw), A, capi.F32, A, capi.F32, A, 1 << 30)


def test_embedding_operands(capi):
    for dtype in (capi.I8, capi.BINARY, 5, -1):
        with pytest.raises(ValueError, match="float32, float16 or bfloat16"):
            capi.embedding_lookup(_embedding(capi, dtype=dtype), A, capi.F32)
        with pytest.raises(ValueError, match="float32, float16 or bfloat16"):
            capi.embedding_gradient(_embedding(capi), A, dtype, A, capi.F32, A, 1 << 30)
    with pytest.raises(ValueError, match="the table's or float32"):
        capi.embedding_lookup(_embedding(capi, dtype=capi.F16), A, capi.BF16)
    with pytest.raises(ValueError, match="the output gradient's or float32"):
        capi.embedding_gradient(_embedding(capi), A, capi.F32, A, capi.F16, A, 1 << 30)
    with pytest.raises(ValueError, match="row stride"):
        capi.embedding_lookup(_embedding(capi, table_stride=7), A, capi.F32)
    with pytest.raises(ValueError, match="row stride"):
        capi.embedding_lookup(_embedding(capi), A, capi.F32, out_stride=7)
    with pytest.raises(ValueError, match="row stride"):
        capi.embedding_gradient(_embedding(capi), A, capi.F32, A, capi.F32, A, 1 << 30, table_gradient_stride=7)
    with pytest.raises(ValueError, match="null device pointer"):
        capi.embedding_lookup(_embedding(capi, table=None), A, capi.F32)
    with pytest.raises(ValueError, match="null device pointer"):
        capi.embedding_gradient(_embedding(capi), None, capi.F32, A, capi.F32, A, 1 << 30)
    need = capi.embedding_gradient_workspace_bytes(_embedding(capi))
    with pytest.raises(ValueError, match="too small"):
        capi.embedding_gradient(_embedding(capi), A, capi.F32, A, capi.F32, A, need - 1)
    with pytest.raises(ValueError, match="16 bytes"):
        capi.embedding_gradient(_embedding(capi), A, capi.F32, A, capi.F32, A + 4, need)


@pytest.mark.parametrize("kw,match", [
    (dict(dtype=2), "float32, float16 or bfloat16"),
    (dict(dtype=7), "float32, float16 or bfloat16"),
    (dict(activation=3), "unknown activation"),
    (dict(activation=-1), "unknown activation"),
    (dict(dim=0), "must be positive"),
    (dict(hidden=0), "must be positive"),
    (dict(hidden=2**24 + 1), "at most 2\\^24"),
    (dict(rows=-1), "rows must lie"),
    (dict(rows=2**30 + 1), "rows must lie"),
    (dict(x_stride=7), "smaller than dim"),
    (dict(weight_stride=7), "smaller than dim"),
    (dict(x=None), "null device pointer"),
    (dict(up=None), "null device pointer"),
])
def test_gated_descriptor(capi, kw, match):
    with pytest.raises(ValueError, match=match):
        capi.gated_projection(_gated(capi, **kw), A)
    with pytest.raises(ValueError, match=match):
        capi.gated_gradient_workspace_bytes(_gated(capi, **kw))
    with pytest.raises(ValueError, match=match):
        capi.gated_gradient(_gated(capi, **kw), A, A, A, A, A, 1 << 30)


def test_gated_operands(capi):
    with pytest.raises(ValueError, match="smaller than hidden"):
        capi.gated_projection(_gated(capi), A, out_stride=5)
    with pytest.raises(ValueError, match="null device pointer"):
        capi.gated_projection(_gated(capi), None)
    with pytest.raises(ValueError, match="smaller than its row"):
        capi.gated_gradient(_gated(capi), A, A, A, A, A, 1 << 30, weight_gradient_stride=7)
    with pytest.raises(ValueError, match="both or neither"):
        capi.gated_gradient(_gated(capi), A, A, A, None, A, 1 << 30)
    with pytest.raises(ValueError, match="null device pointer"):
        capi.gated_gradient(_gated(capi), None, A, A, A, A, 1 << 30)
    need = capi.gated_gradient_workspace_bytes(_gated(capi))
    with pytest.raises(ValueError, match="too small"):
        capi.gated_gradient(_gated(capi), A, A, A, A, A, need - 1)
    with pytest.raises(ValueError, match="too small"):
        capi.gated_gradient(_gated(capi), A, A, A, A, None, need)
    with pytest.raises(ValueError, match="16 bytes"):
        capi.gated_gradient(_gated(capi), A, A, A, A, A + 8, need)


@pytest.mark.parametrize("kw,match", [
    (dict(dtype=3), "float32, float16 or bfloat16"),
    (dict(dim=0), "must be positive"),
    (dict(out_dim=-2), "must be positive"),
    (dict(dim=2**24 + 1), "at most 2\\^24"),
    (dict(rows=2**29 + 1), "rows must lie"),
    (dict(x_stride=7), "smaller than dim"),
    (dict(weight_stride=1), "smaller than dim"),
    (dict(weight=None), "null device pointer"),
    (dict(adapter_count=-1), "adapter_count"),
    (dict(max_rank=0), "max_rank must lie"),
    (dict(max_rank=129), "max_rank must lie"),
    (dict(down=None), "null adapter pointer"),
    (dict(up=None), "null adapter pointer"),
])
def test_adapted_descriptor(capi, kw, match):
    with pytest.raises(ValueError, match=match):
        capi.adapted_projection_workspace_bytes(_adapted(capi, **kw))
    with pytest.raises(ValueError, match=match):
        capi.adapted_projection(_adapted(capi, **kw), A, capi.F32, A, 1 << 30)


def test_adapted_operands(capi):
    assert capi.library().zcgvs_adapted_max_rank() == 128
    with pytest.raises(ValueError, match="the operands' or float32"):
        capi.adapted_projection(_adapted(capi), A, capi.F16, A, 1 << 30)
    with pytest.raises(ValueError, match="smaller than out_dim"):
        capi.adapted_projection(_adapted(capi), A, capi.F32, A, 1 << 30, out_stride=5)
    with pytest.raises(ValueError, match="null device pointer"):
        capi.adapted_projection(_adapted(capi), None, capi.F32, A, 1 << 30)
    need = capi.adapted_projection_workspace_bytes(_adapted(capi))
    with pytest.raises(ValueError, match="too small"):
        capi.adapted_projection(_adapted(capi), A, capi.F32, A, need - 1)
    with pytest.raises(ValueError, match="16 bytes"):
        capi.adapted_projection(_adapted(capi), A, capi.F32, A + 1, need)


def test_null_descriptors(capi):
    lib = capi.library()
    assert lib.zcgvs_embedding_lookup(None, A, 0, capi.F32, None) == capi.ERR_INVALID_ARGUMENT
    assert lib.zcgvs_gated_projection(None, A, 0, None) == capi.ERR_INVALID_ARGUMENT
    assert lib.zcgvs_adapted_projection(None, A, 0, capi.F32, A, 0, None) == capi.ERR_INVALID_ARGUMENT
    assert lib.zcgvs_gated_gradient_workspace_bytes(None) == 0 and "null descriptor" in capi.last_error()


def test_empty_work_returns_ok(capi):
    capi.embedding_lookup(_embedding(capi, token_count=0, ids=None), None, capi.F32)
    capi.embedding_gradient(_embedding(capi, token_count=0), None, capi.F32, None, capi.F32, None, 0, accumulate=True)
    capi.gated_projection(_gated(capi, rows=0, x=None), None)
    capi.gated_gradient(_gated(capi), None, None, None, None, None, 0)  # no gradient is wanted
    capi.adapted_projection(_adapted(capi, rows=0, x=None), None, capi.F32, None, 0)


def test_stores_do_not_take_bfloat16(capi):
    with pytest.raises(ValueError, match="unknown corpus dtype"):
        capi.search_workspace_bytes(capi.search_desc(capi.store_desc(A, 100, 64, capi.BF16), A, 1, 10))
    with pytest.raises(ValueError, match="unknown storage dtype"):
        capi.launch_similarity(A, capi.BF16, 1.0, 10, 32, A, 1, None, 0, A)
    with pytest.raises(ValueError, match="unknown dtype"):
        capi.launch_gather_rescore(A, capi.BF16, 1.0, 10, 32, A, 1, A, 1, 0, A)
