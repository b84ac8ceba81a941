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
    ``ptr[r] .. ptr[r + 1] - 1`` of a list, or all of it where the ``ptr`` is None. ``mask``: int32 words, one row for all or a row each."""
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

        for x in (self.history, self.history_ptr, self.bias_ids, self.bias_ptr, self.mask):
            assert x is None or (x.dtype == torch.int32 and x.device == device and x.is_contiguous())
        for x in (self.history_ptr, self.bias_ptr):
            assert x is None or x.numel() == t + 1
        assert (self.bias_ids is None) == (self.bias is None)
        assert self.bias is None or (self.bias.dtype == torch.float32 and self.bias.device == device and self.bias.numel() == self.bias_ids.numel() and self.bias.is_contiguous())
        words = (n + 31) // 32
        assert self.mask is None or (self.mask.shape[-1] >= words and self.mask.numel() in (self.mask.shape[-1], t * self.mask.shape[-1]))
        ptr = lambda x: x.data_ptr() if x is not None and x.numel() else None
        size = lambda x: x.numel() if x is not None else 0
        stride = 0 if self.mask is None or (self.mask.numel() == self.mask.shape[-1] and t != 1) else self.mask.shape[-1]
        return _lib.LogitRules(self.repeat, self.frequency, self.presence, size(self.history), size(self.bias_ids), ptr(self.history), ptr(self.history_ptr),
                               ptr(self.bias_ids), ptr(self.bias), ptr(self.bias_ptr), ptr(self.mask), stride)
