"""Penalties of the tokens so far, biases and masks on logits (``ins_penalize``).

    from insitu_b200.penalties import Penalties
    penalties = Penalties(repetition=1.1, frequency=0.2)
    logits = penalties(logits, tokens, lengths, prompts=prompts, mask=allowed)
    token, logprob = sampler(logits, uniform)

The tokens are the caller's, as it has them: a row of token ids for each
sequence, prompt first. Nothing is counted from one call to the next.
"""

from __future__ import annotations

import torch

from . import _lib
from .engine import _raise_mapped
from .sampling import RowSettings


def _finite(v):
    return (v >= -1e5) & (v <= 1e5)


class Penalties(RowSettings):
    """Settings of a batch of rows; calling it changes rows of logits.

    ``repetition`` divides a positive logit of a token seen so far (in the
    prompt or since), and multiplies a negative one; ``presence`` is taken from
    the logit of a token said since the prompt, ``frequency`` as often as it has
    been said. Numbers, or 1-D tensors or sequences of one value a row. One
    ``Penalties`` may be used on several streams."""

    SETTINGS = {
        "repetition": (torch.float32, 1.0, lambda v: (v >= 1e-5) & (v <= 1e5), "in [1e-5, 1e5]"),
        "presence": (torch.float32, 0.0, _finite, "in [-1e5, 1e5]"),
        "frequency": (torch.float32, 0.0, _finite, "in [-1e5, 1e5]"),
    }

    def __init__(self, repetition=1.0, presence=0.0, frequency=0.0):
        super().__init__(repetition=repetition, presence=presence, frequency=frequency)

    def __call__(self, logits: torch.Tensor, tokens: torch.Tensor | None = None,
                 lengths: torch.Tensor | None = None, *, prompts: torch.Tensor | None = None,
                 of: torch.Tensor | None = None, drafted: torch.Tensor | None = None,
                 bias: torch.Tensor | None = None, mask: torch.Tensor | None = None,
                 out: torch.Tensor | None = None) -> torch.Tensor:
        """``logits`` (rows, vocab) float32, float16 or bfloat16 on the GPU, rows
        at any stride. Returns them changed, in a new tensor or ``out`` (which
        may be ``logits``, and shares memory with no other argument). All other tensors are on the same device:

        ``tokens`` (sequences, n) int64, a sequence a row of logits, or row i's
        sequence ``of[i]`` (int32); ``lengths`` (sequences,) int32, how many of
        its columns hold tokens (all); ``prompts`` (sequences,) int32, how many
        of those are its prompt (none); ``drafted`` (rows, m) int64, tokens that
        a row adds to its sequence's, e.g. ``DraftTree.paths``. Ids outside the
        vocabulary (-1) are no tokens.
        ``bias`` float32, (vocab,) for all rows or (rows, vocab), is added.
        ``mask`` int32, (words,) or (rows, words): a token is allowed where bit
        t % 32 of word t // 32 is set, and becomes -inf where it is not."""
        if logits.dim() != 2 or logits.device.type != "cuda":
            raise ValueError("logits must be a (rows, vocab) tensor on the GPU")
        bias, mask = (t[None] if t is not None and t.dim() == 1 else t for t in (bias, mask))
        if out is None:
            out = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
        try:
            _lib.ops().penalize(logits, tokens, lengths, prompts, of, drafted,
                                *self._values(logits.shape[0], logits.device), bias, mask, out)
        except (RuntimeError, ValueError) as e:
            _raise_mapped(e)
        return out
