"""Upkeep of the pages of a paged cache on the device: copying, forking, growing, releasing and compacting.

``PagePool`` is a handle on tensors that the program owns: the K and V pools of every layer (``[pages, page_size, ...]``,
the layout ``attn_decode`` and ``attn_paged`` read; state pools of other kinds with pages of one "token" work too), the
page table ``[rows, cols]`` and lengths ``[rows]`` that the attention calls take, and ``refs [pages]``, the number of
page-table entries that hold each page (0 = free). A row holds ``ceil(len / page_size)`` entries; -1 stands for a released
page, which the attention with first tokens (``attn_paged``) never reads. New pages are the lowest free ones, in the
order of the call's entries, so the outcome is the same on every run.

Every method is asynchronous on the current stream, synchronises nothing, and can be captured into a CUDA graph; calls on
one pool have to be ordered on one stream. Indices are int32 or int64 device tensors. Nothing outside the pool is touched
whatever they say; what a call could not do is left out and leaves a sticky status word (``STATUS_NAMES``,
``check_status``).
"""

from __future__ import annotations

import ctypes
import logging
from typing import Sequence

import torch

from greenattention_b200 import _C, dispatch

CHUNK = 16384  # bytes of a copy item of the kernels
MAX_ROWS = 32768
MAX_PAGES = (1 << 31) - 1 - 32768
STATUS_NAMES = {
    1: "a bounded wait for a copy ran out", 3: "a page id was out of range", 5: "a length exceeded the row's entries",
    7: "a row or page index was out of range", 8: "no free page was left", 9: "the page counts did not match the page table",
    10: "entries of one call contradict one another, or a forked row was not empty",
}
_NO_SCRATCH = ("ga_pages_free", "ga_pages_evict")
logger = logging.getLogger(__name__)


def _no(why: str):
    raise dispatch.Declined(f"kv_pages: {why}")


class PagePool:
    def __init__(self, caches: Sequence[torch.Tensor], page_table: torch.Tensor, seqlens: torch.Tensor, refs: torch.Tensor):
        caches = list(caches)
        if not caches:
            _no("no tensors")
        for t in (*caches, page_table, seqlens, refs):
            if not isinstance(t, torch.Tensor):
                _no("not a tensor")
        dev = refs.device
        if any(t.device != dev for t in (*caches, page_table, seqlens)):
            _no("the tensors are on different devices")
        if any(t.dtype != torch.int32 for t in (page_table, seqlens, refs)) or page_table.dim() != 2 or seqlens.dim() != 1 or refs.dim() != 1:
            _no("page_table [rows, cols], seqlens [rows] and refs [pages] are int32")
        rows, cols = page_table.shape
        pages = refs.shape[0]
        if seqlens.shape[0] != rows or (rows > 1 and not seqlens.is_contiguous()) or (pages > 1 and not refs.is_contiguous()):
            _no("seqlens and refs are dense, seqlens as long as the page table")
        if (rows > 1 and page_table.stride(0) < cols * max(1, page_table.stride(1))) or (cols > 1 and page_table.stride(1) < 1):
            _no("page_table rows overlap")
        if pages > MAX_PAGES:
            _no(f"{pages} pages, at most {MAX_PAGES}")
        page_size = caches[0].shape[1] if caches[0].dim() >= 2 else 0
        if page_size < 1 or page_size & (page_size - 1):
            _no(f"page_size {page_size} is not a power of two")
        seen, stride, tok, chunk_tensor, chunk_first = [], [], [], [], []
        for i, t in enumerate(caches):
            if t.dim() < 2 or t.shape[0] != pages or t.shape[1] != page_size:
                _no(f"tensor {i} is not [{pages}, {page_size}, ...]")
            el = t.element_size()
            if pages and not t[0].is_contiguous():
                _no(f"tensor {i}: the tokens of a page are not dense")
            tb, ps = t[0, 0].numel() * el if pages else 0, t.stride(0) * el
            if not pages or tb == 0 or tb % 16 or ps % 16 or t.data_ptr() % 16 or (pages > 1 and ps < tb * page_size):
                _no(f"tensor {i}: tokens, pages and the base are multiples of 16 bytes and pages do not overlap")
            if tb * page_size >= 1 << 30:
                _no(f"tensor {i}: a page of {tb * page_size} bytes")
            seen.append((t.data_ptr(), t.data_ptr() + (pages - 1) * ps + tb * page_size, ps, tb * page_size))
            stride.append(ps)
            tok.append(tb)
            chunk_first.append(len(chunk_tensor))
            chunk_tensor += [i] * -(-tb * page_size // CHUNK)
        if len({s[0] for s in seen}) != len(seen):
            _no("one tensor is listed twice")
        if not refs.is_cuda:
            raise _C.GreenAttentionError(f"tensors are on {dev}: the green kernels have no CPU path")
        if torch.cuda.is_current_stream_capturing():
            _no("a pool is set up before a CUDA graph is captured")
        _C.init(dev.index)
        self.caches, self.page_table, self.seqlens, self.refs = caches, page_table, seqlens, refs
        self.device, self.page_size, self.num_pages = dev, page_size, pages
        self._scratch_bytes: dict = {}  # entries of a call -> bytes
        self.status = torch.zeros(1, dtype=torch.int32, device=dev)
        # what the kernels read about the tensors
        self._base = torch.tensor([s[0] for s in seen], dtype=torch.int64, device=dev)
        self._stride = torch.tensor(stride, dtype=torch.int64, device=dev)
        self._tok = torch.tensor(tok, dtype=torch.int32, device=dev)
        self._chunk_tensor = torch.tensor(chunk_tensor, dtype=torch.int32, device=dev)
        self._chunk_first = torch.tensor(chunk_first, dtype=torch.int32, device=dev)
        torch.cuda.synchronize(dev)  # they are there before a kernel on any stream reads them
        self._p = _C.GaPagePool(
            self._base.data_ptr(), self._stride.data_ptr(), self._tok.data_ptr(), self._chunk_tensor.data_ptr(),
            self._chunk_first.data_ptr(), len(caches), len(chunk_tensor), pages, page_size, page_table.data_ptr(),
            page_table.stride(0), page_table.stride(1), rows, cols, seqlens.data_ptr(), refs.data_ptr(), self.status.data_ptr(),
            None, 0,
        )

    # ------------------------------------------------------------------------------------------------- plumbing

    def _index(self, name: str, t) -> int:
        if not isinstance(t, torch.Tensor) or t.dtype not in (torch.int32, torch.int64) or t.dim() != 1:
            _no(f"{name} must be a 1-D int32 or int64 tensor")
        if t.device != self.device:
            _no(f"{name} is on {t.device}, the pool on {self.device}")
        if t.shape[0] > 1 and t.stride(0) != 1:
            _no(f"{name} is not dense")
        return int(t.dtype == torch.int64)

    def _entries(self, rows) -> int:
        n = rows.shape[0]
        if n > MAX_ROWS:
            _no(f"{n} entries in one call, at most {MAX_ROWS}")
        return n

    def _pair(self, a_name: str, a, b_name: str, b) -> int:
        is64 = self._index(a_name, a)
        if self._index(b_name, b) != is64 or a.shape != b.shape:
            _no(f"{a_name} and {b_name} differ in type or length")
        return is64

    def _call(self, name: str, n: int, *args) -> None:
        lib = _C.lib()
        # A copy of the handle's struct: calls of several host threads do not share one.
        p = _C.GaPagePool.from_buffer_copy(self._p)
        if name not in _NO_SCRATCH:
            nbytes = self._scratch_bytes.get(n)
            if nbytes is None:
                nbytes = self._scratch_bytes[n] = lib.ga_pages_scratch_bytes(ctypes.byref(p), n)
            scratch = self.refs.new_empty(nbytes, dtype=torch.uint8)
            p.scratch, p.scratch_bytes = scratch.data_ptr(), nbytes
        fn = getattr(lib, name)
        index = self.device.index
        if torch.cuda.current_device() == index:
            rc = fn(ctypes.byref(p), *args, _C.raw_stream(index))
        else:
            with torch.cuda.device(self.device):  # the library launches on the current device
                rc = fn(ctypes.byref(p), *args, _C.raw_stream(index))
        if rc:
            _C.check(rc, name)

    def check_status(self, reset: bool = True) -> int:
        """The status word (0 = fine; ``STATUS_NAMES``), logged when it is not 0 and put back. Synchronises."""
        val = int(self.status.item())
        if val:
            logger.error("green_attention: page pool status %d on %s: %s", val, self.device, STATUS_NAMES.get(val, "unknown"))
            if reset:
                self.status.zero_()
        return val

    # ------------------------------------------------------------------------------------------------ operators

    def copy(self, src: torch.Tensor, dst: torch.Tensor) -> None:
        """Page ``dst[i]`` becomes a copy of page ``src[i]`` in every tensor; counts and table stay. Of entries with one
        destination the last counts; one that copies a page onto itself says nothing. An entry whose source another entry writes is left out (status 10): what it would
        copy depends on the order. Entries that name no page are left out (status 7)."""
        is64 = self._pair("src", src, "dst", dst)
        n = src.shape[0]
        if n:
            self._call("ga_pages_copy", n, src.data_ptr(), dst.data_ptr(), is64, n)

    def fork(self, parents: torch.Tensor, children: torch.Tensor) -> None:
        """Row ``children[i]``, which is empty, becomes a copy of row ``parents[i]``: the full pages are shared, the tokens
        of a partial last page are copied to the lowest free page (copy on write ahead of the write). A child that is not
        empty or is named before is left alone (status 10), one that finds no free page too (status 8)."""
        is64 = self._pair("parents", parents, "children", children)
        n = self._entries(parents)
        if n:
            self._call("ga_pages_fork", n, parents.data_ptr(), children.data_ptr(), is64, n)

    def grow(self, rows: torch.Tensor, lens: torch.Tensor) -> None:
        """Row ``rows[i]`` grows to ``lens[i]`` tokens, with the lowest free pages for what does not fit the row's last page;
        a smaller length leaves it alone. From the first row on whose pages are not there, rows that need some are left
        as they were (status 8)."""
        is64, lens64 = self._index("rows", rows), self._index("lens", lens)
        n = self._entries(rows)
        if lens.shape[0] != n:
            _no("rows and lens differ in length")
        if n:
            self._call("ga_pages_grow", n, rows.data_ptr(), lens.data_ptr(), is64, lens64, n)

    def free(self, rows: torch.Tensor) -> None:
        """Releases the rows' pages; their lengths become 0."""
        is64 = self._index("rows", rows)
        n = self._entries(rows)
        if n:
            self._call("ga_pages_free", n, rows.data_ptr(), is64, n)

    def evict(self, rows: torch.Tensor, window_left: int, sink_tokens: int = 0) -> None:
        """Releases the pages of the rows that no query from position ``len`` on sees with ``window_size=(window_left, 0)``
        and ``sink_tokens``; their entries become -1, the lengths stay."""
        is64 = self._index("rows", rows)
        for name, v in (("window_left", window_left), ("sink_tokens", sink_tokens)):
            if not isinstance(v, int) or isinstance(v, bool) or not 0 <= v < 1 << 31:
                _no(f"{name} {v} is not a count")
        n = self._entries(rows)
        if n:
            self._call("ga_pages_evict", n, rows.data_ptr(), is64, n, window_left, sink_tokens)

    def compact(self) -> tuple:
        """Moves the held pages with the highest ids into the gaps, so that the held pages are those below their number;
        the table, the counts and every tensor follow. Returns ``(map, live)``: ``map[page]`` is the page's new id or -1
        for a free one, ``live`` the number of held pages, both int32 on the device."""
        out = torch.empty(self.num_pages, dtype=torch.int32, device=self.device)
        live = torch.empty(1, dtype=torch.int32, device=self.device)
        self._call("ga_pages_compact", 0, out.data_ptr(), live.data_ptr())
        return out, live
