"""Sizes the page entries cannot plan, refused before the device is touched."""
import ctypes

import pytest

from npu_sparse_attn_sharedkv_int8 import runtime
from tests.test_tree_pages_boundary import ERANGE, page_args


@pytest.mark.parametrize("op", [0, 1])
@pytest.mark.parametrize("batch, width, rows", [(8192, 1 << 19, 32), (8192, (1 << 19) + 1, 32), (4, 1 << 30, 1), (8193, 1, 1)])
def test_tables_beyond_32_bits(op, batch, width, rows):
    """A resize of the whole table would need 2^32 fresh pages or more, whose number wraps."""
    args = page_args(batch=batch, width=width, pageRows=rows)
    assert runtime._library().sharedkv_page(ctypes.addressof(args), op, 1 << 20, 0, 0, -1, None) == ERANGE


def test_workspace_of_a_large_table():
    assert runtime._library().sharedkv_page_workspace_bytes(8192, (1 << 19) - 1) > 4 * 8192 * ((1 << 19) - 1)
