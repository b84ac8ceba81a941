"""Rules on logits before a token is chosen (``b2_logits_dev``): penalties for the tokens of a history, biases, a grammar's mask. The reference
does this on the host (``src/sampler.rs``).
"""
from __future__ import annotations

from dataclasses import dataclass

from . import _lib


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
