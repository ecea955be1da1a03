"""Sizes beyond what the embedding-model operators' launches can index are refused, without a GPU."""

import pytest

A = 1 << 20  # an address that nothing reads here


@pytest.mark.parametrize("dim", [2 ** 23 + 1, 2 ** 24, 2 ** 31 - 1])
def test_embedding_dim(capi, dim):
    desc = capi.embedding_desc(A, 10, dim, capi.F32, A, 5)
    with pytest.raises(ValueError, match="dim must be at most 2\\^23"):
        capi.embedding_lookup(desc, A, capi.F32)
    with pytest.raises(ValueError, match="dim must be at most 2\\^23"):
        capi.embedding_gradient_workspace_bytes(desc)
    with pytest.raises(ValueError, match="dim must be at most 2\\^23"):
        capi.embedding_gradient(desc, A, capi.F32, A, capi.F32, A, 1 << 60)


def test_largest_embedding_dim(capi):
    assert capi.embedding_gradient_workspace_bytes(capi.embedding_desc(A, 10, 2 ** 23, capi.F32, A, 5)) > 2 * 2 ** 23 * 4


@pytest.mark.parametrize("dtype", ["F32", "F16", "BF16"])
@pytest.mark.parametrize("rows,dim,hidden", [(64, 768, 2048), (500, 384, 1024), (16_384, 768, 2048), (3000, 1024, 4096)])
def test_gradient_workspace_goes_by_the_sizes(capi, dtype, rows, dim, hidden):
    """Not by the alignment of the operands, on which the tiles depend: a workspace serves all calls of its sizes."""
    size = {capi.gated_gradient_workspace_bytes(capi.gated_desc(A + x, rows, dim, A + w, A + w, hidden, getattr(capi, dtype),
                                                                capi.ACT_SILU, x_stride=dim + pad, weight_stride=dim + pad))
            for x in (0, 4) for w in (0, 4) for pad in (0, 1)}
    assert len(size) == 1
