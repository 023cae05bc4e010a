"""Attention of a tree of drafted tokens over the INT8 shared-KV cache.

The speculative-decoding counterpart of `PreparedAttention`: the query tokens of a request are the
nodes of a draft tree whose rows the cache writer has put behind the committed rows, and every token
attends the committed rows and its own path only.  The reference has no such operator; inputs, pages
and padding follow `SharedKVCase` and `PreparedAttention`.
"""
import ctypes

import torch

from .attention import DIM, _address, _check_case, _require
from .runtime import Kernels, check, current_stream

DRAFT_ROWS = 64                  # drafted rows of a request a path mask can name
_POINTERS = ("q", "ori", "cmp", "oriScale", "cmpScale", "oriTable", "cmpTable", "indices", "paths", "cmpPaths", "cuQ",
             "seqLens", "sinks", "out", "lse", "workspace", "oriStride", "cmpStride")
_COUNTS = ("tokens", "heads", "batch", "oriTableWidth", "cmpTableWidth", "oriPages", "cmpPages", "ratio", "window", "topk")
_CASE_POINTERS = (("q", "q"), ("ori", "ori"), ("cmp", "cmp"), ("oriTable", "ori_block_table"), ("cmpTable", "cmp_block_table"),
                  ("indices", "cmp_indices"), ("cuQ", "cu_q"), ("seqLens", "seq_lens"), ("sinks", "sink"))


class _Args(ctypes.Structure):
    """TreeAttentionArgs of the C ABI, 192 bytes."""
    _fields_ = ([(n, ctypes.c_uint64) for n in _POINTERS] + [(n, ctypes.c_uint32) for n in _COUNTS]
                + [("softmaxScale", ctypes.c_float), ("reserved", ctypes.c_uint32)])


def path_masks(parents):
    """Path masks of one draft tree: `parents[i]` is the index of token i's parent among the drafted
    tokens (below i), -1 for a child of the last committed token.  Returns INT64[n] on the host."""
    masks = []
    for token, parent in enumerate(parents):
        if not -1 <= parent < token:
            raise ValueError("A drafted token's parent comes before it")
        if token >= DRAFT_ROWS:
            raise ValueError(f"A path mask names at most {DRAFT_ROWS} drafted tokens")
        masks.append((masks[parent] if parent >= 0 else 0) | 1 << token)
    return torch.tensor([m - (1 << 64) if m >> 63 else m for m in masks], dtype=torch.int64)


def _check_masks(masks, tokens, device, name):
    _require(masks.dtype == torch.int64 and tuple(masks.shape) == (tokens,) and masks.device == device and masks.is_contiguous(),
             f"Expected contiguous INT64 {name}[T] on the query device")


class PreparedTreeAttention:
    """Holds every input and output tensor of one call; `run()` allocates nothing, reads nothing back
    and launches on the current stream of the inputs' device.

    `case` is a `SharedKVCase` whose query tokens are drafted tokens: request b has
    n = cu_q[b+1] - cu_q[b] of them and seq_lens[b] - n committed rows, and its token j owns the
    original cache's row seq_lens[b] - n + j.  `paths` INT64[T]: bit j of a token's mask is drafted row
    j of its request; a path holds the token itself and its ancestors (`path_masks`).  The committed
    rows of the window are those that the path leaves room for.  Ratio 4: the token's own top-k list,
    entries up to 64 rows behind the committed groups.  Ratio 128: every committed group and, with
    `cmp_paths` INT64[T], drafted compressed rows behind them.  BF16 Q[T,H,512] with H a multiple of 8
    up to 128, window 1..65536, INT8 pages of 32 rows at strides and addresses that are multiples of 16.

    The workspace belongs to the operator: two of its launches must not overlap in time.
    """

    def __init__(self, case, paths, ori_scale, cmp_scale=None, *, cmp_paths=None, output=None, return_lse=False, lse_output=None,
                 scratch_allocator=None):
        tokens, heads, device = _check_case(case, ori_scale, cmp_scale)
        _require(heads % 8 == 0, "Tree attention needs a multiple of eight heads")
        _require(case.window <= 65536, "Tree attention needs a window of at most 65536 rows")
        _require(case.ori_indices is None, "Tree attention takes the window from the path, not explicit original slots")
        caches = (case.ori,) if case.ratio == 1 else (case.ori, case.cmp)
        _require(all(c.shape[1] == 32 and c.stride(0) % 16 == 0 and c.data_ptr() % 16 == 0 for c in caches),
                 "Tree attention needs 32-row pages at 16-byte aligned addresses and strides")
        _require(case.ratio != 4 or case.cmp_indices.shape[-1] <= 1024, "Tree attention needs top-k <= 1024")
        _check_masks(paths, tokens, device, "paths")
        _require(cmp_paths is None or case.ratio == 128, "Compressed path masks belong to ratio-128 layers")
        if cmp_paths is not None:
            _check_masks(cmp_paths, tokens, device, "cmp_paths")
        self.device, self.device_index = device, device.index
        self.scales = (ori_scale, cmp_scale)
        self.kernels = Kernels()
        if self.kernels.lib.sharedkv_tree_args_size() != ctypes.sizeof(_Args):
            raise RuntimeError("Native library ABI changed; rebuild libsharedkv_cuda.so")
        self.args = args = _Args()
        args.oriScale, args.cmpScale = _address(ori_scale), _address(cmp_scale if case.ratio > 1 else None)
        args.oriStride, args.oriPages, args.oriTableWidth = case.ori.stride(0), case.ori.shape[0], case.ori_block_table.shape[1]
        if case.ratio > 1:
            args.cmpStride, args.cmpPages, args.cmpTableWidth = case.cmp.stride(0), case.cmp.shape[0], case.cmp_block_table.shape[1]
        args.tokens, args.heads, args.batch = tokens, heads, case.seq_lens.numel()
        args.ratio, args.window, args.softmaxScale = case.ratio, case.window, case.softmax_scale
        args.topk = case.cmp_indices.shape[-1] if case.ratio == 4 else 0
        out = torch.empty_like(case.q) if output is None else output
        lse = lse_output
        if lse is None and return_lse:
            lse = torch.empty((tokens, heads), dtype=torch.float32, device=device)
        need = self.kernels.lib.sharedkv_tree_workspace_bytes(tokens, heads, args.batch, case.ratio, args.topk)
        allocate = scratch_allocator or (lambda name, shape, dtype, where: torch.empty(shape, dtype=dtype, device=where))
        self.workspace = allocate("tree_workspace", (max(need, 1024),), torch.uint8, device)
        _require(self.workspace.data_ptr() % 256 == 0, "Attention workspace must be 256-byte aligned")
        args.workspace = self.workspace.data_ptr()
        # Launches need no prepared workspace, so it does not matter which stream this runs on and when, or that a graph
        # captures it: it only clears the status word, which recycled memory may hold.
        self.workspace[:4].zero_()
        self.argument_address = ctypes.addressof(args)
        self._rebind_same_geometry(case, paths, cmp_paths=cmp_paths, output=out, lse_output=lse)

    def _rebind_same_geometry(self, case, paths, *, cmp_paths=None, output=None, lse_output=None):
        """Serving fast path: other pointers, the same shapes, strides and types; inputs are not validated
        again."""
        self.case, self.paths, self.cmp_paths = case, paths, cmp_paths
        self.out = torch.empty_like(case.q) if output is None else output
        self.lse = lse_output
        tokens, heads, _ = case.q.shape
        _require(self.out.shape == case.q.shape and self.out.dtype == torch.bfloat16 and self.out.device == case.q.device
                 and self.out.is_contiguous(), "Invalid output buffer")
        _require(lse_output is None or (tuple(lse_output.shape) == (tokens, heads) and lse_output.dtype == torch.float32
                                        and lse_output.device == case.q.device and lse_output.is_contiguous()),
                 "Invalid FP32 LSE[T,H] output buffer")
        for field, attribute in _CASE_POINTERS:
            setattr(self.args, field, _address(getattr(case, attribute)))
        self.args.paths, self.args.cmpPaths = paths.data_ptr(), _address(cmp_paths)
        self.args.out, self.args.lse = self.out.data_ptr(), _address(lse_output)

    def run(self):
        if self.args.tokens:
            check(self.kernels.lib.sharedkv_tree_attention(self.argument_address, self.device_index, current_stream(self.device_index)),
                  "tree attention launch")
        return self.out

    def status(self):
        """Synchronises the current stream; raises RuntimeError if a wait inside a launch of this operator ran
        out (its results are then invalid).  Diagnostic only."""
        with torch.cuda.device(self.device):
            check(self.kernels.lib.sharedkv_tree_status(self.args.workspace, current_stream(self.device_index)), "tree attention kernel")


__all__ = ["DIM", "DRAFT_ROWS", "PreparedTreeAttention", "path_masks"]
