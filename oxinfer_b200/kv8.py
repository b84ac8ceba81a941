"""The 8-bit cache and the attention over it (``b2_kv8_*`` and ``b2_attend_kv8_dev`` of ``include/b200qmm.h``): keys and values as integers
of -127 .. 127 with a power of two as the scale of every block of 32 tokens, KV head and kind. No counterpart in the reference, whose
caches are f32. Everything is on the device, launched on the backend's stream, and not synchronized.
"""
from __future__ import annotations

import ctypes as C
from dataclasses import dataclass

from . import _lib

BLOCK = 32  # tokens of a block


@dataclass
class Kv8Seqs:
    """The sequences of a call. ``start``: int32 [n], the position of each one's first row. ``rows``: int32 [n + 1], sequence ``s`` has rows
    ``rows[s] .. rows[s + 1] - 1`` of the call's tensors, or None: ``max_rows`` each. ``table``: int32 [n, max_blocks], the pool's number of
    each one's blocks, or None: sequence ``s`` has blocks ``s * max_blocks ..``. All int32 tensors on the device. ``n_rows``: rows in all (None: ``n *
    max_rows``); ``max_rows``: the most rows of a sequence."""
    start: object
    max_blocks: int
    max_rows: int = 1
    rows: object = None
    n_rows: int | None = None
    table: object = None

    def c(self, device) -> _lib.Kv8Seqs:
        import torch

        n = self.start.numel()
        assert self.rows is None or self.rows.numel() == n + 1
        assert self.table is None or tuple(self.table.shape) == (n, self.max_blocks)
        for x in (self.start, self.rows, self.table):
            assert x is None or (x.dtype == torch.int32 and x.device == device and x.is_contiguous())
        ptr = lambda x: x.data_ptr() if x is not None else None
        assert self.rows is None or self.n_rows is not None
        return _lib.Kv8Seqs(n, n * self.max_rows if self.n_rows is None else self.n_rows, self.max_rows, self.max_blocks, ptr(self.table), ptr(self.start),
                            ptr(self.rows))


class Kv8Cache:
    """A pool of ``n_blocks`` blocks of 32 tokens for ``nkv`` KV heads of ``hd`` (``Backend.kv8``). The calls return False where the backend declines."""

    def __init__(self, backend, handle: int, nkv: int, hd: int, n_blocks: int):
        import torch

        self.backend, self.handle, self.nkv, self.hd, self.n_blocks = backend, handle, nkv, hd, n_blocks
        self.device = torch.device("cuda", backend.ordinal)
        self._work_bytes = _lib.lib().b2_attend_kv8_work_bytes(backend._ctx, handle)

    def bytes(self) -> int:
        return _lib.lib().b2_kv8_bytes(self.backend._ctx, self.handle)

    def free(self) -> None:
        if self.handle and self.backend._ctx:
            _lib.lib().b2_kv8_free(self.backend._ctx, self.handle)
        self.handle = 0

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass

    def append(self, seqs: Kv8Seqs, k, v) -> bool:
        """Keys and values ``[n_rows][nkv][hd]`` (f32, bf16 or f16; any strides of rows and heads, the same for both)."""
        from .backend import _dtype_code

        s = seqs.c(self.device)
        for x in (k, v):
            assert tuple(x.shape) == (s.n_rows, self.nkv, self.hd) and x.device == self.device and x.stride(2) == 1
        assert k.dtype == v.dtype and (s.n_rows == 0 or k.stride() == v.stride())
        return self.backend._check(self.backend._L.b2_kv8_append_dev(self.backend._ctx, self.handle, C.byref(s), k.data_ptr(), v.data_ptr(), _dtype_code(k),
                                                                     k.stride(0), k.stride(1)))

    def read(self, seqs: Kv8Seqs, k, v) -> bool:
        """The values that the rows stand for into f32 ``[n_rows][nkv][hd]``."""
        import torch

        s = seqs.c(self.device)
        for x in (k, v):
            assert tuple(x.shape) == (s.n_rows, self.nkv, self.hd) and x.device == self.device and x.dtype == torch.float32 and x.is_contiguous()
        return self.backend._check(self.backend._L.b2_kv8_read_dev(self.backend._ctx, self.handle, C.byref(s), k.data_ptr(), v.data_ptr()))

    def attend(self, seqs: Kv8Seqs, q, out, scale: float, cap: float = 0.0, window: int | None = None, slopes=None, prefix=None) -> bool:
        """Row ``i`` of a sequence attends from position ``start + i``; ``q`` and ``out`` are ``[n_rows][nh][hd]`` of one type (rows of any
        stride). Scores are ``cap * tanh(scale * q.k / cap)`` (``cap`` 0: ``scale * q.k``) ``+ slopes[h] * (key - position)``; a key is seen up to the row's own
        position or below ``prefix`` (int32 [n]), and with a ``window`` only if it is less than that far behind."""
        import torch

        from .backend import _dtype_code

        s = seqs.c(self.device)
        nh = q.shape[1]
        for x in (q, out):
            assert tuple(x.shape) == (s.n_rows, nh, self.hd) and x.device == self.device and x.dtype == q.dtype
            assert x.stride(2) == 1 and x.stride(1) == self.hd
        assert slopes is None or (slopes.dtype == torch.float32 and slopes.numel() == nh and slopes.is_contiguous() and slopes.device == self.device)
        assert prefix is None or (prefix.dtype == torch.int32 and prefix.numel() == s.n_seqs and prefix.is_contiguous() and prefix.device == self.device)
        # (memory of the call's own, from torch's allocator: calls on other streams and captured ones have theirs)
        work = torch.empty(self._work_bytes, dtype=torch.uint8, device=self.device) if q.dtype == torch.float32 or s.max_rows * (nh // self.nkv) <= 8 else None
        a = _lib.Kv8Attention(nh, scale, cap, window or 0, slopes.data_ptr() if slopes is not None else None, prefix.data_ptr() if prefix is not None else None,
                              work.data_ptr() if work is not None else None)
        return self.backend._check(self.backend._L.b2_attend_kv8_dev(self.backend._ctx, self.handle, C.byref(s), C.byref(a), q.data_ptr(), q.stride(0),
                                                                     out.data_ptr(), out.stride(0), _dtype_code(q)))
