"""Refusals of the drafted-tree and page-pool entry points that need no GPU: the C entries check their
arguments before they touch the device."""
import ctypes

import pytest
import torch

from npu_sparse_attn_sharedkv_int8 import PagePool, PreparedTreeAttention
from npu_sparse_attn_sharedkv_int8 import pages, runtime, tree_attention
from npu_sparse_attn_sharedkv_int8.reference import make_case

EINVAL, ERANGE, EVARIANT = -22, -34, -2


def lib():
    return runtime._library()


def test_struct_sizes():
    assert lib().sharedkv_tree_args_size() == ctypes.sizeof(tree_attention._Args) == 192
    assert lib().sharedkv_page_args_size() == ctypes.sizeof(pages._Args) == 64


def tree_args(**changes):
    args = tree_attention._Args()
    for name in tree_attention._POINTERS:
        setattr(args, name, 1 << 20)
    args.cmpPaths = args.lse = 0
    args.oriStride = args.cmpStride = 16384
    args.tokens, args.heads, args.batch, args.oriTableWidth, args.cmpTableWidth, args.oriPages, args.cmpPages = 4, 8, 1, 2, 2, 2, 2
    args.ratio, args.window, args.topk, args.softmaxScale = 4, 128, 16, 1.0
    for name, value in changes.items():
        setattr(args, name, value)
    return args


@pytest.mark.parametrize("changes", [
    dict(ratio=2), dict(heads=0), dict(heads=12), dict(heads=136), dict(window=0), dict(window=65537), dict(topk=0), dict(topk=1025),
    dict(indices=0), dict(indices=2), dict(q=0), dict(q=8), dict(ori=8), dict(cmp=0), dict(paths=0), dict(paths=4), dict(out=2), dict(sinks=0),
    dict(workspace=0), dict(workspace=128), dict(oriStride=16392), dict(oriStride=16368), dict(cmpStride=512), dict(oriTableWidth=0),
    dict(cmpPages=0), dict(oriPages=1 << 26), dict(cuQ=0), dict(seqLens=2), dict(lse=2), dict(ratio=128, cmpPaths=4), dict(cmpScale=0)])
def test_tree_entry_refuses(changes):
    args = tree_args(**changes)
    assert lib().sharedkv_tree_attention(ctypes.addressof(args), -1, None) == EINVAL


def test_tree_entry_with_nothing_to_do():
    assert lib().sharedkv_tree_attention(0, -1, None) == EINVAL
    args = tree_args(tokens=0)
    assert lib().sharedkv_tree_attention(ctypes.addressof(args), -1, None) == 0


def page_args(**changes):
    args = pages._Args()
    for name in pages._POINTERS:
        setattr(args, name, 1 << 20)
    args.layers, args.pages, args.pageRows, args.batch, args.width = 1, 8, 32, 2, 3
    for name, value in changes.items():
        setattr(args, name, value)
    return args


PAGE_REFUSALS = [(op, changes, status) for ops, changes, status in (
    (range(4), dict(caches=0), EINVAL), (range(4), dict(caches=4), EINVAL), (range(4), dict(layers=0), EINVAL), (range(4), dict(pages=0), EINVAL),
    (range(4), dict(pageRows=0), EINVAL), ((0, 1, 3), dict(table=0), EINVAL), ((0, 1, 3), dict(width=0), EINVAL),
    ((0, 1, 3), dict(width=1 << 27), EINVAL), ((0, 1), dict(lens=0), EINVAL), ((0, 1), dict(refs=2), EINVAL),
    ((0, 1), dict(workspace=64), EINVAL), ((0, 1), dict(batch=8193), ERANGE)) for op in ops]


@pytest.mark.parametrize("op, changes, status", PAGE_REFUSALS)
def test_page_entries_refuse(op, changes, status):
    args = page_args(**changes)
    assert lib().sharedkv_page(ctypes.addressof(args), op, 1 << 20, 1 << 20, 4, -1, None) == status


def test_page_entry_arrays():
    args = page_args()
    call = lambda op, a, b, n: lib().sharedkv_page(ctypes.addressof(args), op, a, b, n, -1, None)  # noqa: E731
    for op in range(4):
        assert call(op, 0, 1 << 20, 4) == EINVAL
        assert call(op, (1 << 20) + 2, 1 << 20, 4) == EINVAL
    assert call(2, (1 << 20) + 4, 0, 1) == EINVAL
    assert call(3, 1 << 20, 0, 1) == EINVAL
    assert call(3, 1 << 20, 1 << 20, 65) == EINVAL
    assert call(4, 1 << 20, 0, 1) == EVARIANT
    assert call(2, 1 << 20, 0, 0) == 0 and call(3, 1 << 20, 1 << 20, 0) == 0
    assert lib().sharedkv_page(0, 0, 1 << 20, 0, 0, -1, None) == EINVAL


def test_host_tensors_are_refused():
    case = make_case()
    with pytest.raises(ValueError, match="CUDA"):
        PreparedTreeAttention(case, torch.zeros(1, dtype=torch.int64), torch.ones(512))
    with pytest.raises(ValueError, match="CUDA"):
        PagePool([torch.zeros(4, 32, 1, 512, dtype=torch.int8)])


def test_path_masks():
    assert tree_attention.path_masks([-1, 0, 0, 1, -1]).tolist() == [1, 3, 5, 11, 16]
    assert tree_attention.path_masks(range(-1, 63))[63] == -1
    assert tree_attention.path_masks([]).tolist() == []
    for parents in ([0], [-1, 1], [-2], list(range(-1, 64))):
        with pytest.raises(ValueError):
            tree_attention.path_masks(parents)


def test_reference_counts():
    table = torch.tensor([[3, 1, 9], [3, 7, 7], [0, 0, 0]], dtype=torch.int32)
    assert pages.count_references(table, torch.tensor([33, 64, 0], dtype=torch.int32), 32, 8).tolist() == [0, 1, 0, 2, 0, 0, 0, 1]
