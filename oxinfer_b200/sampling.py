"""Rules on logits before a token is chosen (``b2_logits_dev``): penalties for the tokens of a history, biases, a grammar's mask. The reference
does this on the host (``src/sampler.rs``).
"""
from __future__ import annotations

from dataclasses import dataclass

import numpy as np

from . import _lib


@dataclass
class GenerateRules:
    """Rules for every step of ``DecodePlan.generate`` (``b2_generate_rules``), host arrays: the history is ``prompt`` and what the call has chosen so far."""
    repeat: float = 1.0
    frequency: float = 0.0
    presence: float = 0.0
    prompt: np.ndarray | None = None     # int32
    bias_ids: np.ndarray | None = None   # int32
    bias: np.ndarray | None = None       # float32
    mask: np.ndarray | None = None       # uint32 words, bit i % 32 of word i / 32: token i is allowed

    def c(self, n: int):
        """The struct, and the arrays that it points into."""
        prompt, ids = (None if x is None else np.ascontiguousarray(x, dtype=np.int32) for x in (self.prompt, self.bias_ids))
        bias = None if self.bias is None else np.ascontiguousarray(self.bias, dtype=np.float32)
        mask = None if self.mask is None else np.ascontiguousarray(self.mask).view(np.uint32)
        assert (ids is None) == (bias is None) and (ids is None or ids.size == bias.size)
        assert mask is None or mask.size == (n + 31) // 32
        ptr = lambda x: x.ctypes.data if x is not None and x.size else None
        size = lambda x: x.size if x is not None else 0
        return _lib.GenerateRules(self.repeat, self.frequency, self.presence, size(prompt), size(ids), ptr(prompt), ptr(ids), ptr(bias), ptr(mask)), (prompt, ids, bias, mask)


@dataclass
class LogitRules:
    """What changes rows of logits, in this order: ``l / repeat`` (``l * repeat`` where ``l <= 0``) and ``- (frequency * count + presence)`` for tokens of the
    history; ``+ bias``; ``-inf`` where ``mask`` has no bit. ``history`` and ``bias_ids`` are int32 lists on the device, ``bias`` f32; row ``r`` has the part
    ``ptr[r] .. ptr[r + 1] - 1`` of a list, or all of it where the ``ptr`` is None. ``mask``: int32 words, ``[words]`` or ``[1, words]`` for all rows, or
    ``[t, words]``, with ``words`` at least ``(n + 31) // 32`` (exactly that many in the first form)."""
    repeat: float = 1.0
    frequency: float = 0.0
    presence: float = 0.0
    history: object = None
    history_ptr: object = None
    bias_ids: object = None
    bias: object = None
    bias_ptr: object = None
    mask: object = None

    def c(self, t: int, n: int, device) -> _lib.LogitRules:
        import torch

        r = _lib.LogitRules(self.repeat, self.frequency, self.presence)
        int32 = torch.int32
        ok = lambda x, dtype: x.dtype == dtype and x.device == device and x.is_contiguous()
        h, b, m = self.history, self.bias_ids, self.mask
        if h is not None:
            assert ok(h, int32)
            r.n_history, r.history = h.numel(), h.data_ptr()
            if self.history_ptr is not None:
                assert ok(self.history_ptr, int32) and self.history_ptr.numel() == t + 1
                r.history_ptr = self.history_ptr.data_ptr()
        if b is not None:
            assert ok(b, int32) and ok(self.bias, torch.float32) and self.bias.numel() == b.numel()
            r.n_bias, r.bias_ids, r.bias = b.numel(), b.data_ptr(), self.bias.data_ptr()
            if self.bias_ptr is not None:
                assert ok(self.bias_ptr, int32) and self.bias_ptr.numel() == t + 1
                r.bias_ptr = self.bias_ptr.data_ptr()
        if m is not None:
            assert m.dim() > 0 and ok(m, int32)
            width, words = m.shape[-1], (n + 31) // 32
            # (a list of words is one row: the rows of several would all get the first one's bits)
            assert width >= words and m.numel() in (width, t * width) and (m.dim() > 1 or t == 1 or width == words)
            r.mask, r.mask_stride = m.data_ptr(), width if m.numel() == t * width else 0
        return r
