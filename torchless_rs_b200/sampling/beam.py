"""The selection step of a beam search on the device (kernels in csrc/beam_select.cu).

The reference keeps one continuation of a prompt (src/sampler/mod.rs:269-305); a beam search keeps several and
goes on with the likeliest of all their next tokens."""
from __future__ import annotations

from typing import Tuple

import torch

from ..csrc import ops


class BeamSelector:
    MAX_N = ops.BeamOps.MAX_N

    def __init__(self, device: torch.device):
        self.device = torch.device(device)
        self.ops = ops.beam_ops()

    def select(self, logits: torch.Tensor, scores: torch.Tensor,
               n: int) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        """The `n` continuations of each sequence with the highest log-probability.

        `logits` [sequences * beams, vocabulary]: the step's logits, a sequence's beams in consecutive rows;
        `scores` [sequences, beams]: each beam's log-probability so far, -inf for a place without a beam (its row of
        logits does not matter).  Returns (values, beams, tokens), each [sequences, n] on the device, in falling order of
        scores[s, b] + log softmax(logits[s, b])[t]; of equal ones the lower beam comes first, then its larger logit, then the lower token.
        Sums are compared in 64 bits; the values are rounded to 32.  Continuations of one beam come in the order of its logits, and
        beams with the same logits and score tie to the last bit.  Each row's logarithm is off by less than 2^-19 (up to 2^18
        entries: most of its exponentials run in 32 bits), so continuations of different beams that are closer than twice that may come in
        either order.  A logit that is NaN or -inf is no continuation, +inf counts as the largest finite number;
        where fewer than `n` continuations exist, the last places hold -inf, -1, -1.

        The result is in buffers of its own; nothing is kept between calls."""
        out = self.ops.select(logits, scores, n)
        return out[0].view(torch.float32), out[1], out[2]
