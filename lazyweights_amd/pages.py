"""Page tables of a paged key-value cache (KvCache, KvCache8) and the pool of its free pages, kept on the GPU (lw_pages_advance
of include/lazyweights_amd.h): a serving loop says how many tokens every sequence gets, and keeps, and one launch gives the
lengths, tables and row starts that a Batch reads, without the host knowing which pages there are.

    pages = Pages.empty(cache_pages, page_size, seqs, table_pages)
    q_start, position, slot = pages.advance(new, rows=n)       # new int32 [seqs] on the GPU, their sum at most n
    batch = Batch(cache, heads, q_start, pages.kv_len, pages.table, max_new, max_kv)   # kept; later steps pass q_start=q_start
    pages.advance(new, keep=keep, q_start=q_start, position=position, slot=slot)     # keep[s] = 0: a request that ended

Calls go to torch's current stream unless `stream` (a hipStream_t as an integer) is given, then as with KvCache's. A call can be
captured; calls on one Pages must not overlap. Bad arguments raise ValueError, a refused call RuntimeError.
"""
import ctypes

import torch

from ._lib import last_error, load_library
from .attention import _current_device, _current_stream


class _Pages(ctypes.Structure):
    _fields_ = [("table", ctypes.c_void_p), ("table_stride", ctypes.c_int64), ("table_pages", ctypes.c_int32),
                ("seqs", ctypes.c_int32), ("page_size", ctypes.c_int32), ("pages", ctypes.c_int32), ("free", ctypes.c_void_p),
                ("kv_len", ctypes.c_void_p), ("left", ctypes.c_void_p), ("workspace", ctypes.c_void_p)]


class Pages:
    """Sequences' tables int32 [seqs, table_pages] and lengths kv_len int32 [seqs], and the free pages: free int32 [pages], a stack of
    which the first left[0] are free (left int32 [2]; left[1] says what the last step lacked: 0 nothing, else the sum of 1: pages, 2:
    room in the table, 4: rows; then it has changed nothing). All on one GPU, contiguous (the table's rows may lie apart). A page belongs to
    one sequence: what is given back is taken again, whoever else's table names it."""

    def __init__(self, page_size, kv_len, table, free, left):
        seqs = kv_len.shape[0] if kv_len.dim() == 1 else -1
        if table.dim() != 2 or table.shape[0] != seqs or free.dim() != 1 or left.shape != (2,):
            raise ValueError("kv_len [seqs], table [seqs, pages], free [pages] and left [2] are wanted, not %s, %s, %s, %s"
                             % tuple(tuple(t.shape) for t in (kv_len, table, free, left)))
        if not kv_len.is_cuda or any(t.dtype != torch.int32 or t.device != kv_len.device for t in (kv_len, table, free, left)):
            raise ValueError("kv_len, table, free and left must be int32 tensors on one GPU")
        if any(t.numel() > 1 and t.stride(-1) != 1 for t in (kv_len, table, free, left)):
            raise ValueError("kv_len, the table's rows, free and left must be contiguous")
        if not 0 < page_size <= 65536 or page_size & (page_size - 1):
            raise ValueError("page_size must be a power of two up to 65536")
        if seqs > 8192:
            raise ValueError("up to 8192 sequences")
        self.lib, self.index, self.seqs = load_library(), kv_len.get_device(), seqs
        self.page_size, self.kv_len, self.table, self.free, self.left = page_size, kv_len, table, free, left
        self.workspace = torch.zeros(272, dtype=torch.int32, device=kv_len.device)
        self._current, self._device = _current_stream(), _current_device()
        self.c = _Pages(table.data_ptr(), table.stride(0) if seqs > 1 else table.shape[1], table.shape[1], seqs, page_size,
                        free.shape[0], free.data_ptr(), kv_len.data_ptr(), left.data_ptr(), self.workspace.data_ptr())
        self.ptr = ctypes.addressof(self.c)

    @classmethod
    def empty(cls, pages, page_size, seqs, table_pages, device="cuda"):
        """Sequences of no tokens, and all pages free (page 0 is the first to be taken)."""
        def whole(x):
            return torch.tensor(x, dtype=torch.int32, device=device)

        return cls(page_size, torch.zeros(seqs, dtype=torch.int32, device=device),
                   torch.full((seqs, table_pages), -1, dtype=torch.int32, device=device),
                   torch.arange(pages - 1, -1, -1, dtype=torch.int32, device=device), whole([pages, 0]))

    def _whole(self, what, t, size, dtype=torch.int32):
        """Address of a contiguous tensor [size] of whole numbers on the pages' device."""
        if t.dtype != dtype or t.shape != (size,) or t.get_device() != self.index or not t.is_contiguous():
            raise ValueError("%s: %s [%d], contiguous, on the pages' device is wanted" % (what, dtype, size))
        return t.data_ptr()

    def advance(self, new, keep=None, rows=None, kv_len_out=None, left_out=None, q_start=None, position=None, slot=None,
                places=True, stream=None):
        """Every sequence is cut to keep[s] tokens (not at all without keep) and grown by new[s] (int32 [seqs]): lengths, table, pool
        and left are brought up to date, or with kv_len_out and left_out written there, the pages' own left as they were.
        Returns (q_start int32 [seqs + 1], position int32 [rows], slot int64 [rows]): the rows' starts, every new row's position,
        and page * page_size + its row there (-1 for no page). What is not given is allocated; `rows` is the most that new may add
        up to (else that of position or slot); with places=False positions and slots that are not given are not made."""
        if self._device() != self.index:  # launches go to the current device
            with torch.cuda.device(self.index):
                return self.advance(new, keep, rows, kv_len_out, left_out, q_start, position, slot, places, stream)
        if rows is None:
            if position is None and slot is None:
                raise ValueError("rows, position or slot must be given")
            rows = (slot if position is None else position).shape[0]
        if not 0 <= rows < 1 << 30:
            raise ValueError("rows must be less than 2^30")
        other = None
        if stream is not None and stream != self._current(self.index):
            other = torch.cuda.ExternalStream(stream, self.index) if stream else torch.cuda.default_stream(self.index)
        if q_start is None or (places and (position is None or slot is None)):
            with torch.cuda.stream(other):  # (None: the current one)
                if q_start is None:
                    q_start = torch.empty(self.seqs + 1, dtype=torch.int32, device=self.kv_len.device)
                if places and position is None:
                    position = torch.empty(rows, dtype=torch.int32, device=self.kv_len.device)
                if places and slot is None:
                    slot = torch.empty(rows, dtype=torch.int64, device=self.kv_len.device)
        n, c = self.seqs, self.c
        if self.lib.lw_pages_advance(
                self.ptr, self._whole("new", new, n), None if keep is None else self._whole("keep", keep, n), rows,
                c.kv_len if kv_len_out is None else self._whole("kv_len_out", kv_len_out, n),
                c.left if left_out is None else self._whole("left_out", left_out, 2), self._whole("q_start", q_start, n + 1),
                None if position is None else self._whole("position", position, rows),
                None if slot is None else self._whole("slot", slot, rows, torch.int64),
                self._current(self.index) if stream is None else stream) != 0:
            raise RuntimeError(last_error())
        if other is not None:
            for t in (self.kv_len, self.table, self.free, self.left, self.workspace, new, keep, kv_len_out, left_out, q_start,
                      position, slot):
                if t is not None:
                    t.record_stream(other)
        return q_start, position, slot
