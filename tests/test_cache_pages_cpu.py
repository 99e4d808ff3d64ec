"""Refusals of the page operators, before any CUDA call: sizes that no memory has, and a tensor in place of the list."""
import ctypes

import pytest
import torch

ONE = ctypes.c_void_p(256)  # never dereferenced
NULL = ctypes.c_void_p(None)


@pytest.mark.parametrize("pages,size", [(1 << 24, 1 << 40), (2**31 - 1, 1 << 40), (1 << 30, 1 << 34), (1 << 19, 1 << 30)])
def test_sizes_past_the_address_space(cabi, pages, size):
    """Their product may wrap, and with it the test that the tensors do not overlap."""
    lib = cabi.load()
    table = (ctypes.c_void_p * 2)(4096, 4096)
    assert lib.b200ops_copy_pages(table, 2, pages, size, ONE, ONE, 0, NULL) == cabi.EINVAL
    assert lib.b200ops_copy_pages(table, 1, pages, size, ONE, ONE, 0, NULL) == cabi.EINVAL
    assert "bad cache shape" in cabi.last_error()
    need = lib.b200ops_compact_pages_workspace_size(pages)
    assert lib.b200ops_compact_pages(table, 2, pages, size, ONE, ONE, 2, 3, ctypes.c_void_p(8192), ONE, ONE,
                                     ONE, need, NULL) == cabi.EINVAL


def test_one_tensor_in_place_of_the_list(ops):
    """A tensor is a sequence too, of its pages: taken for the list, each page's tokens would be moved as pages."""
    cache = torch.zeros(8, 8, 2, 16)
    ids = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="copy_pages: caches must be a list"):
        ops.copy_pages(cache, ids, ids)
    with pytest.raises(RuntimeError, match="compact_pages: caches must be a list"):
        ops.compact_pages(cache, ids[None], ids[:1])
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.copy_pages((cache,), ids, ids)
