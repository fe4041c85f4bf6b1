"""Log probabilities of tokens, as the engine gives them out."""
from __future__ import annotations

from typing import List, NamedTuple, Sequence, Tuple

import numpy as np
import torch

from .. import ops


class TokenScore(NamedTuple):
    """A token under the distribution it was drawn from or scored by: its log probability (natural), its rank (0: the most probable), the
    distribution's entropy, and the most probable tokens with their log probabilities, best first."""

    id: int
    logprob: float
    rank: int
    entropy: float
    top: Tuple[Tuple[int, float], ...]


class PendingScores:
    """The scores of some rows of logits, on their way to the host."""

    def __init__(self, logits: torch.Tensor, ids: torch.Tensor, top: int, status: torch.Tensor):
        got = ops.token_logprobs(logits, ids, top, status)
        self.host = [torch.empty(t.shape, dtype=t.dtype).pin_memory() for t in got]
        for h, t in zip(self.host, got):
            h.copy_(t, non_blocking=True)
        self.event = ops.record_event(None)

    def scores(self, ids: Sequence[int]) -> List[TokenScore]:
        """Waits for them; ``ids``: the rows' tokens."""
        self.event.synchronize()
        lp, rank, entropy, top_ids, top_lp = [h.numpy() for h in self.host]
        return [TokenScore(int(t), float(lp[r]), int(rank[r]), float(entropy[r]), tuple(zip(top_ids[r].tolist(), np.asarray(top_lp[r]).tolist())))
                for r, t in enumerate(ids)]
