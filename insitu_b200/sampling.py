"""Sampling tokens from logits on the GPU (``ins_sample``).

    from insitu_b200.sampling import Sampler
    sampler = Sampler(temperature=0.8, top_k=50, top_p=0.95)
    tokens, logprobs = sampler(logits, torch.rand_like(logits, dtype=torch.float32))

The random numbers are the caller's, one per logit, so a run repeats from its
generator's seed and no state lives here. A ``Sampler`` holds the settings,
one value for all rows or one a row, on the device.
"""

from __future__ import annotations

import torch

from . import _lib
from .engine import _raise_mapped

MAX_VOCAB = 1 << 18

# name: (type, value that cuts nothing, what a value must satisfy, in words)
_SETTINGS = {
    "temperature": (torch.float32, 1.0, lambda v: (v == 0) | ((v >= 1e-5) & (v <= 1e5)),
                    "0 (the largest logit) or in [1e-5, 1e5]"),
    "top_k": (torch.int32, 0, lambda v: v >= 0, "at least 0 (0: no cut)"),
    "top_p": (torch.float32, 1.0, lambda v: (v > 0) & (v <= 1), "in (0, 1]"),
    "min_p": (torch.float32, 0.0, lambda v: (v >= 0) & (v <= 1), "in [0, 1]"),
}


class Sampler:
    """Settings of a batch of rows; calling it draws one token a row.

    ``temperature`` (0 takes the largest logit), ``top_k`` (0: off), ``top_p``
    and ``min_p`` are numbers, or 1-D tensors or sequences of one value a row.
    They are checked here, so a call reads nothing back from the device. One
    ``Sampler`` may be used on several streams."""

    def __init__(self, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
        self._rows = None
        self._per_row, self._scalar, self._filled = {}, {}, {}
        for name, value in (("temperature", temperature), ("top_k", top_k), ("top_p", top_p), ("min_p", min_p)):
            dtype, neutral, valid, words = _SETTINGS[name]
            t = torch.as_tensor(value)
            if t.dim() > 1:
                raise ValueError(f"{name} must be a number or one value a row")
            if dtype == torch.int32 and (t.is_floating_point() or t.dtype == torch.bool):
                raise TypeError(f"{name} must be an integer")
            held = (t.clamp(max=MAX_VOCAB) if dtype == torch.int32 else t).to(dtype).contiguous()
            # (reading the check's answer also waits for `held`, where t is on the device)
            if not bool(valid(t if dtype == torch.int32 else held).all()):
                raise ValueError(f"{name} must be {words}")
            if t.dim() == 0:
                if held.item() != neutral:
                    self._scalar[name] = held.item()
                continue
            if self._rows not in (None, t.numel()):
                raise ValueError(f"{name} holds {t.numel()} values; other settings hold {self._rows}")
            self._rows = t.numel()
            self._per_row[name] = held

    def _values(self, n: int, device) -> list:
        """The settings' device tensors for n rows. Calls on any stream share
        them, so they come by copies from the host that the host waits for
        (the first call, and one with more rows than any before), and the
        operator tells the allocator which streams read them."""
        if self._rows not in (None, n):
            raise ValueError(f"the settings are for {self._rows} rows; logits hold {n}")
        out = []
        for name in _SETTINGS:
            t = self._per_row.get(name)
            if t is not None:
                if t.device != device:
                    t = self._per_row[name] = t.cpu().to(device)
            elif name in self._scalar:
                t = self._filled.get(name)
                if t is None or t.device != device or t.numel() < n:
                    rows = max(256, 1 << (n - 1).bit_length())
                    t = torch.full((rows,), self._scalar[name], dtype=_SETTINGS[name][0]).to(device)
                    self._filled[name] = t
                t = t[:n]
            out.append(t)
        return out

    def __call__(self, logits: torch.Tensor, uniform: torch.Tensor):
        """``logits`` (rows, vocab) float32, float16 or bfloat16 on the GPU,
        rows at any stride; ``uniform`` float32 of the same shape, in [0, 1).
        Returns tokens (rows,) int64 and their log-probabilities among the
        tokens kept (rows,) float32. A row of nothing but -inf and NaN gives
        -1 and -inf."""
        if logits.dim() != 2 or logits.device.type != "cuda":
            raise ValueError("logits must be a (rows, vocab) tensor on the GPU")
        try:
            return _lib.ops().sample(logits, uniform, *self._values(logits.shape[0], logits.device))
        except (RuntimeError, ValueError) as e:
            _raise_mapped(e)
