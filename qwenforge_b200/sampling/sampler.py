"""Next-token choice. The reference chooses greedily only (student_engine.py:1320, :982, :1158:
argmax of the last position's logits) and accepts a seed that no stochastic operation reads
(:316, :425-427). This library adds temperature sampling: temperature 0 is the reference's greedy
choice (lowest id on ties), temperature > 0 draws from softmax(logits / temperature) with the
Gumbel-max kernel, keyed by (seed, sequence id, number of tokens the sequence has generated), so a
sequence's tokens do not depend on which batch it runs in."""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional

import torch

from .. import ops


# `verify` draws behind a refused draft under another seed than `__call__`, which may have drawn the draft: its own with these bits changed.
REDRAW_BITS = 0x9E3779B97F4A7C15


@dataclass(frozen=True)
class SamplingParams:
    temperature: float = 0.0
    seed: int = 0

    def __post_init__(self):
        if self.temperature < 0:
            raise ValueError(f"temperature must be >= 0, got {self.temperature}")


class Sampler:
    def __init__(self, params: SamplingParams = SamplingParams()):
        self.params = params

    @property
    def greedy(self) -> bool:
        return self.params.temperature <= 0.0

    def __call__(self, logits: torch.Tensor, seq_ids: Optional[torch.Tensor] = None,
                 steps: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None, scratch=None) -> torch.Tensor:
        """logits float32 [rows, vocab] -> int32 [rows]; seq_ids int64 [rows] and steps int32 [rows] when sampling."""
        if out is None:
            out = torch.empty(logits.shape[0], dtype=torch.int32, device=logits.device)
        ops.sample(logits, self.params.temperature, self.params.seed, seq_ids, steps, out, scratch)
        return out

    def verify(self, logits: torch.Tensor, drafted: torch.Tensor, first: torch.Tensor, most: int, uniforms: Optional[torch.Tensor] = None,
               draft_logits: Optional[torch.Tensor] = None, seq_ids: Optional[torch.Tensor] = None,
               steps: Optional[torch.Tensor] = None, scratch=None) -> tuple[torch.Tensor, torch.Tensor]:
        """Which drafted tokens stay, and the token behind them (`ops.verify_drafts`). logits float32 [rows, vocab]: a row per drafted
        token and one more per entry, entry s's from first[s] on; drafted int32, uniforms float32 and draft_logits float32 [.., vocab] one
        after another; seq_ids and steps as when sampling. Returns accepted int32 [entries] and tokens int32 [entries, most + 1].

        Drafts that come with draft_logits may be this sampler's own draws from them, for the same seq_ids and steps, or any other's; without, they
        must not be draws at random. The uniforms are independent of either, and new ones every time."""
        n = first.numel() - 1
        accepted = torch.empty(n, dtype=torch.int32, device=logits.device)
        tokens = torch.empty((n, most + 1), dtype=torch.int32, device=logits.device)
        if uniforms is None:
            if not self.greedy:
                raise ValueError("verify: sampling needs uniforms")
            uniforms = torch.empty(0, dtype=torch.float32, device=logits.device)
        ops.verify_drafts(logits, draft_logits, drafted, first, uniforms, self.params.temperature, self.params.seed, seq_ids, steps,
                          accepted, tokens, scratch, redraw_seed=self.params.seed ^ REDRAW_BITS)
        return accepted, tokens
