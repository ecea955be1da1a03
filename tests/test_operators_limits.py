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
