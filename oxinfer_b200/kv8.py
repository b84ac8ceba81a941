"""The 8-bit cache and the attention over it (``b2_kv8_*`` and ``b2_attend_kv8_dev`` of ``include/b200qmm.h``): keys and values as integers
of -127 .. 127 with a power of two as the scale of every block of 32 tokens, KV head and kind. No counterpart in the reference, whose
caches are f32. Everything is on the device, launched on the backend's stream, and not synchronized.
"""
from __future__ import annotations

import ctypes as C
from dataclasses import dataclass

from . import _lib

BLOCK = 32  # tokens of a block
DEALT_FROM = 768  # positions of a sequence: below, its keys are never shared out over all of the GPU


@dataclass(frozen=True)
class Kv8Seqs:
    """The sequences of a call. ``start``: int32 [n], the position of each one's first row. ``rows``: int32 [n + 1], sequence ``s`` has rows
    ``rows[s] .. rows[s + 1] - 1`` of the call's tensors, or None: ``max_rows`` each. ``table``: int32 [n, max_blocks], the pool's number of
    each one's blocks, or None: sequence ``s`` has blocks ``s * max_blocks ..``. All int32 tensors on the device; what they hold may change from call to call.
    ``n_rows``: rows in all (None: ``n * max_rows``); ``max_rows``: the most rows of a sequence."""
    start: object
    max_blocks: int
    max_rows: int = 1
    rows: object = None
    n_rows: int | None = None
    table: object = None

    def __post_init__(self):
        import torch

        n, device = self.start.numel(), self.start.device
        assert self.rows is None or (self.rows.numel() == n + 1 and self.n_rows is not None)
        assert self.table is None or tuple(self.table.shape) == (n, self.max_blocks)
        for x in (self.start, self.rows, self.table):
            assert x is None or (x.dtype == torch.int32 and x.device == device and x.is_contiguous())
        ptr = lambda x: x.data_ptr() if x is not None else None
        if self.n_rows is None:
            object.__setattr__(self, "n_rows", n * self.max_rows)
        object.__setattr__(self, "device", device)
        object.__setattr__(self, "n_seqs", n)
        # (the tensors are held by this object, so their addresses stay)
        object.__setattr__(self, "_c", _lib.Kv8Seqs(n, self.n_rows, self.max_rows, self.max_blocks, ptr(self.table), ptr(self.start), ptr(self.rows)))
        object.__setattr__(self, "_ref", C.byref(self._c))

    def c(self, device=None) -> _lib.Kv8Seqs:
        return self._c


class Kv8Cache:
    """A pool of ``n_blocks`` blocks of 32 tokens for ``nkv`` KV heads of ``hd`` (``Backend.kv8``). The calls return False where the backend declines."""

    def __init__(self, backend, handle: int, nkv: int, hd: int, n_blocks: int):
        import torch

        self._torch, self._f32 = torch, torch.float32
        self._codes = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}
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

    def _work(self):
        """Memory of the call's own, from torch's allocator, for the backend's stream: calls on other streams and captured ones have theirs."""
        torch, stream = self._torch, self.backend.stream
        if torch._C._cuda_getCurrentRawStream(self.device.index) == stream:
            return torch.empty(self._work_bytes, dtype=torch.uint8, device=self.device)
        with torch.cuda.stream(torch.cuda.ExternalStream(stream, device=self.device) if stream else torch.cuda.default_stream(self.device)):
            return torch.empty(self._work_bytes, dtype=torch.uint8, device=self.device)

    @staticmethod
    def _strides(x):
        """Of ``[rows][heads][hd]``; a dimension of one has whatever stride torch gave it, and counts as if it lay side by side."""
        rows, heads, hd = x.shape
        a, b, c = x.stride()
        if heads == 1:
            b = hd
        return (heads * hd if rows == 1 else a), b, c

    def append(self, seqs: Kv8Seqs, k, v) -> bool:
        """Keys and values ``[n_rows][nkv][hd]`` (f32, bf16 or f16; any strides of rows and heads, the same for both)."""
        shape, stride = (seqs.n_rows, self.nkv, self.hd), k.stride()
        assert k.shape == shape and v.shape == shape and k.dtype == v.dtype and k.device == self.device == v.device == seqs.device
        if v.stride() != stride:
            stride = self._strides(k)
            assert self._strides(v) == stride
        assert stride[2] == 1
        be = self.backend
        return be._check(be._L.b2_kv8_append_dev(be._ctx, self.handle, seqs._ref, k.data_ptr(), v.data_ptr(), self._codes[k.dtype], stride[0], stride[1]))

    def read(self, seqs: Kv8Seqs, k, v) -> bool:
        """The values that the rows stand for into f32 ``[n_rows][nkv][hd]``."""
        shape = (seqs.n_rows, self.nkv, self.hd)
        assert k.shape == shape and v.shape == shape and k.dtype == v.dtype == self._f32 and k.is_contiguous() and v.is_contiguous()
        assert k.device == self.device == v.device == seqs.device
        be = self.backend
        return be._check(be._L.b2_kv8_read_dev(be._ctx, self.handle, seqs._ref, k.data_ptr(), v.data_ptr()))

    def attend(self, seqs: Kv8Seqs, q, out, scale: float, cap: float = 0.0, window: int | None = None, slopes=None, prefix=None) -> bool:
        """Row ``i`` of a sequence attends from position ``start + i``; ``q`` and ``out`` are ``[n_rows][nh][hd]`` of one type (rows of any
        stride). Scores are ``cap * tanh(scale * q.k / cap)`` (``cap`` 0: ``scale * q.k``) ``+ slopes[h] * (key - position)``; a key is seen up to the row's own
        position or below ``prefix`` (int32 [n]), and with a ``window`` only if it is less than that far behind."""
        n, nh, hd = q.shape
        dtype, qs, os = q.dtype, q.stride(), out.stride()
        if nh == 1:
            qs, os = self._strides(q), self._strides(out)
        assert out.shape == q.shape and n == seqs.n_rows and hd == self.hd and out.dtype == dtype and q.device == self.device == out.device == seqs.device
        assert qs[2] == os[2] == 1 and qs[1] == os[1] == hd
        assert slopes is None or (slopes.dtype == self._f32 and slopes.numel() == nh and slopes.is_contiguous() and slopes.device == self.device)
        assert prefix is None or (prefix.dtype == self._torch.int32 and prefix.numel() == seqs.n_seqs and prefix.is_contiguous() and prefix.device == self.device)
        assert window is None or window >= 0
        few = dtype == self._f32 or seqs.max_rows * nh <= 8 * self.nkv
        work = self._work() if few and seqs.max_blocks * BLOCK >= DEALT_FROM else None
        a = _lib.Kv8Attention(nh, scale, cap, min(window or 0, 0xFFFFFFFF), None if slopes is None else slopes.data_ptr(), None if prefix is None else prefix.data_ptr(),
                              None if work is None else work.data_ptr())
        be = self.backend
        return be._check(be._L.b2_attend_kv8_dev(be._ctx, self.handle, seqs._ref, C.byref(a), q.data_ptr(), qs[0], out.data_ptr(), os[0], self._codes[dtype]))
