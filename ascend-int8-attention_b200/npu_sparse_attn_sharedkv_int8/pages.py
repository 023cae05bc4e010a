"""Page bookkeeping of INT8 shared-KV caches on the device.

`cache_layout` plans where pages live; a `PagePool` says which sequence holds which page.  Block table,
lengths and reference counts are device tensors that the pool changes in place, so a captured decode
loop (drafted trees, beams) grows, forks, trims and frees sequences without a host round trip.  The
reference leaves this to the host's block manager.
"""
import ctypes

import torch

from .runtime import Kernels, NativeError, check, current_stream

ROW = 512                        # bytes of a cache row
MAX_KEPT = 64                    # rows of a drafted tree that `keep` can move per sequence
MAX_SEQUENCES = 8192
_POINTERS = ("caches", "table", "lens", "refs", "workspace")
_COUNTS = ("layers", "pages", "pageRows", "batch", "width", "reserved")
_RESIZE, _FORK, _COPY, _KEEP = range(4)
_REFUSED = -34                   # SHAREDKV_ERANGE


class _Args(ctypes.Structure):
    """PagePoolArgs of the C ABI, 64 bytes."""
    _fields_ = [(n, ctypes.c_uint64) for n in _POINTERS] + [(n, ctypes.c_uint32) for n in _COUNTS]


def _require(ok, message):
    if not ok:
        raise ValueError(message)


def count_references(table, lens, page_rows, pages):
    """INT32[pages]: how many sequences hold each page (sequence b holds the first
    ceil(lens[b] / page_rows) entries of its table row)."""
    live = torch.arange(table.shape[1], device=table.device) < ((lens.long() + page_rows - 1) // page_rows)[:, None]
    return torch.bincount(table[live].long(), minlength=pages).to(torch.int32)


class PagePool:
    """The pages of `caches` (INT8 [pages, rows, 1, 512] views of equal shape, one per layer, any page
    stride that is a multiple of 16 bytes) and the sequences that hold them.

    `table` INT32[B, W], `lens` INT32[B] (rows) and `refs` INT32[pages] (counted from the first two when
    not given) are changed in place.  A page is free when its count is zero; a count the caller raises
    pins the page.  Fresh pages are the lowest-numbered free ones.  Operations launch on the current
    stream of the caches' device, allocate and read back nothing, and must be ordered among themselves
    and with the readers of the table.  `copy` and `keep` need no lengths and counts.
    """

    def __init__(self, caches, table=None, lens=None, refs=None):
        caches = list(caches)
        _require(len(caches) > 0, "A page pool needs at least one cache")
        device, shape = caches[0].device, tuple(caches[0].shape)
        for cache in caches:
            _require(cache.device.type == "cuda" and cache.dtype == torch.int8 and cache.ndim == 4 and tuple(cache.shape[-2:]) == (1, ROW),
                     "Expected INT8 CUDA cache[pages,page_size,1,512]")
            _require(tuple(cache.shape) == shape and cache.device == device, "The caches of a pool have one shape and one device")
            _require(shape[0] > 0 and shape[1] > 0 and cache.stride(1) == ROW and cache.stride(-1) == 1
                     and (shape[0] == 1 or cache.stride(0) >= shape[1] * ROW) and shape[1] <= 1 << 20, "Invalid cache strides or empty page storage")
            _require(cache.data_ptr() % 16 == 0 and cache.stride(0) % 16 == 0, "Pages must be 16-byte aligned")
        _require(len({cache.data_ptr() for cache in caches}) == len(caches), "A cache is in the pool twice")
        _require(lens is None or table is not None, "Lengths need a block table")
        if table is not None:
            _require(table.dtype == torch.int32 and table.ndim == 2 and table.is_contiguous() and table.device == device
                     and table.shape[1] > 0, "Expected contiguous INT32 table[B,W] on the caches' device")
            _require(table.shape[1] * shape[1] < 2 ** 31, "The block table addresses too many rows")
        if lens is not None:
            _require(table.shape[0] <= MAX_SEQUENCES, f"A pool holds at most {MAX_SEQUENCES} sequences")
            _require(table.numel() < 2 ** 32, "The block table has too many entries")
            self._check_sequences(lens, table, "lens")
            if refs is None:
                refs = count_references(table, lens, shape[1], shape[0])
            _require(refs.dtype == torch.int32 and tuple(refs.shape) == (shape[0],) and refs.is_contiguous() and refs.device == device,
                     "Expected contiguous INT32 refs[pages] on the caches' device")
        self.caches, self.table, self.lens, self.refs = caches, table, lens, refs
        self.device, self.pages, self.page_rows = device, shape[0], shape[1]
        self.kernels = Kernels()
        if self.kernels.lib.sharedkv_page_args_size() != ctypes.sizeof(_Args):
            raise RuntimeError("Native library ABI changed; rebuild libsharedkv_cuda.so")
        batch, width = (0, 0) if table is None else table.shape
        # One buffer: the caches' addresses and page strides, padded to 256 bytes, then the workspace, whose head
        # holds the sticky status (operations write the rest before they read it).  The copy has arrived when it
        # returns, so that the pool may be used on any stream.
        words = [word for c in caches for word in (c.data_ptr(), c.stride(0))]
        lead = -(-len(words) // 32) * 32
        start = torch.tensor(words + [0] * (lead - len(words) + 32), dtype=torch.int64)
        self._buffer = torch.empty(lead + -(-self.kernels.lib.sharedkv_page_workspace_bytes(batch, width) // 8), dtype=torch.int64, device=device)
        self._buffer[:lead + 32].copy_(start)
        self.workspace = self._buffer[lead:]
        _require(self.workspace.data_ptr() % 256 == 0, "The pool's workspace must be 256-byte aligned")
        self.args = _Args()
        for name, tensor in (("caches", self._buffer), ("table", table), ("lens", lens), ("refs", refs), ("workspace", self.workspace)):
            setattr(self.args, name, 0 if tensor is None else tensor.data_ptr())
        self.args.layers, self.args.pages, self.args.pageRows = len(caches), self.pages, self.page_rows
        self.args.batch, self.args.width = batch, width
        self.argument_address = ctypes.addressof(self.args)
        self._page, self._index = self.kernels.lib.sharedkv_page, device.index

    @staticmethod
    def _check_sequences(tensor, table, name):
        if (tensor.dtype != torch.int32 or tensor.ndim != 1 or len(tensor) != len(table) or not tensor.is_contiguous()
                or tensor.get_device() != table.get_device()):
            raise ValueError(f"Expected contiguous INT32 {name}[B] on the caches' device")

    def _launch(self, op, first, second=0, count=0):
        index = self._index
        status = self._page(self.argument_address, op, first, second, count, index, current_stream(index))
        if status:
            check(status, "page pool launch")

    def resize(self, lens):
        """Sequence b gets lens[b] rows (INT32[B]): more take fresh pages, fewer give pages back, 0 frees
        the sequence.  A growing sequence whose last page is partly filled and shared gets its own copy of
        it.  With too few free pages, or a length the table cannot hold, nothing changes (`status`)."""
        if self.lens is None:
            raise ValueError("resize needs lengths and reference counts")
        self._check_sequences(lens, self.table, "lens")
        address = lens.data_ptr()
        if address == self.args.lens and address:
            raise ValueError("The new lens are a tensor of their own: the pool's still say what it holds")
        self._launch(_RESIZE, address)

    def fork(self, parents):
        """Sequence b continues sequence parents[b] (INT32[B]; negative: it ends).  The children of a
        sequence share its full pages; the first keeps the partly filled last page, the others get copies.
        With too few free pages or a parent outside the batch nothing changes (`status`)."""
        if self.lens is None:
            raise ValueError("fork needs lengths and reference counts")
        self._check_sequences(parents, self.table, "parents")
        self._launch(_FORK, parents.data_ptr())

    def copy(self, pairs):
        """Pages pairs[i, 0] -> pairs[i, 1] (INT32[N, 2]) in every cache; pairs outside the pool are
        skipped.  No page may be a destination twice, or a destination and a source."""
        address = pairs.data_ptr()
        if (pairs.dtype != torch.int32 or pairs.ndim != 2 or pairs.shape[1] != 2 or not pairs.is_contiguous()
                or pairs.get_device() != self._index or address % 8):
            raise ValueError("Expected contiguous INT32 pairs[N,2] on the caches' device")
        count = len(pairs)
        if count:
            self._launch(_COPY, address, 0, count)

    def keep(self, base, kept):
        """Rows base[b] + kept[b, i] -> base[b] + i in every cache (INT32[B], INT32[B, K], K <= 64): packs the
        accepted rows of drafted trees behind the committed ones.  Negative entries and rows without a page
        are skipped; all rows of a sequence are read before one is written.  The pages that hold drafted
        rows belong to one sequence.  `base` is a tensor of its own: the pool's lens include the draft since the
        resize that made room for it."""
        if self.table is None:
            raise ValueError("keep needs a block table")
        self._check_sequences(base, self.table, "base")
        if (kept.dtype != torch.int32 or kept.ndim != 2 or len(kept) != len(self.table) or kept.shape[1] > MAX_KEPT
                or not kept.is_contiguous() or kept.get_device() != self._index):
            raise ValueError(f"Expected contiguous INT32 kept[B,K <= {MAX_KEPT}] on the caches' device")
        width, address = kept.shape[1], base.data_ptr()
        if address == self.args.lens and address:
            raise ValueError("base is a tensor of its own, the committed lengths: the pool's lens include the draft")
        if width and len(kept):
            self._launch(_KEEP, address, kept.data_ptr(), width)

    def status(self):
        """Synchronises the current stream; raises RuntimeError if a resize or fork of this pool was
        refused on the device (its tables were then left as they were), ever or since `clear_status`.
        Diagnostic only."""
        with torch.cuda.device(self.device):
            status = self.kernels.lib.sharedkv_page_status(self.workspace.data_ptr(), current_stream(self.device.index))
        if status == _REFUSED:
            raise NativeError("A page pool operation was refused: too few free pages, a length beyond the block table or an unknown parent")
        check(status, "page pool status")

    def clear_status(self):
        """Forgets a refusal, in stream order: a server that has freed pages and tries again asks `status`
        about the second attempt."""
        self.workspace[:1].zero_()


__all__ = ["MAX_KEPT", "MAX_SEQUENCES", "PagePool", "count_references"]
