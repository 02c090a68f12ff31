"""What a model thinks of tokens: log-probabilities of given ones, the entropy of their distribution and the most likely alternatives.

The reference reports one log-probability a token (generate.py:101-117,134-135); here the same pass over a row of logits gives the row's entropy and its best tokens as well,
in one kernel that reads the logits once (csrc/paged/token_scores.cuh)."""
from dataclasses import dataclass
from typing import Optional

import torch

from . import _abi_paged

MAX_ALTERNATIVES = _abi_paged.MAX_TOP


@dataclass
class TokenScores:
    logprob: Optional[torch.Tensor]   # [T] fp32: log-probability of each row's target, 0 where it has none (None without targets)
    entropy: torch.Tensor             # [T] fp32, in nats
    top_ids: torch.Tensor             # [T, top] int64, most likely first; of equal ones the lowest index
    top_logprobs: torch.Tensor        # [T, top] fp32


    def rows(self, r0: int, r1: int) -> "TokenScores":
        """Rows r0 .. r1 - 1, sharing memory."""
        return TokenScores(None if self.logprob is None else self.logprob[r0:r1], self.entropy[r0:r1], self.top_ids[r0:r1], self.top_logprobs[r0:r1])


def empty_scores(T: int, top: int, scored: bool, device: torch.device) -> TokenScores:
    return TokenScores(torch.empty(T, dtype=torch.float32, device=device) if scored else None, torch.empty(T, dtype=torch.float32, device=device),
                       torch.empty(T, top, dtype=torch.long, device=device), torch.empty(T, top, dtype=torch.float32, device=device))


def token_scores(logits: torch.Tensor, targets: Optional[torch.Tensor] = None, top: int = 0, out: Optional[TokenScores] = None) -> TokenScores:
    """Scores of the rows of `logits` [T, V] (fp32 or bf16; rows may be part of wider ones).  targets [T] int64: a token of each row, or -1 (score 0); a target past the
    vocabulary scores NaN, as does a row that holds NaN or +infinity, or nothing but -infinity.  Other entries of -infinity (masked tokens) weigh nothing.  `out`: results
    of the caller's, contiguous."""
    assert logits.dim() == 2 and logits.dtype in (torch.float32, torch.bfloat16) and logits.shape[1] >= 1, f"logits [T, V], fp32 or bf16, got {tuple(logits.shape)} {logits.dtype}"
    T, V = logits.shape
    assert logits.stride(1) == 1 and (T <= 1 or logits.stride(0) >= V), "rows of logits are contiguous and do not overlap"
    assert targets is None or (targets.dtype == torch.long and targets.shape == (T,)), "targets: one int64 a row"
    assert 0 <= top <= min(MAX_ALTERNATIVES, V), f"{top} alternatives (at most {MAX_ALTERNATIVES}, and no more than tokens)"
    if out is None:
        out = empty_scores(T, top, targets is not None, logits.device)
    else:
        f32 = torch.float32
        assert (out.logprob is None) == (targets is None) and (out.logprob is None or (out.logprob.shape == (T,) and out.logprob.dtype == f32)), "out.logprob [T] fp32, with targets"
        assert out.entropy.shape == (T,) and out.top_ids.shape == out.top_logprobs.shape == (T, top) and out.entropy.dtype == out.top_logprobs.dtype == f32 and out.top_ids.dtype == torch.long, "out"
    if 0 < T <= _abi_paged.MAX_SCORE_ROWS:
        _abi_paged.token_scores(logits, targets, out.logprob, out.entropy, out.top_ids, out.top_logprobs, top)
    else:
        for r in range(0, T, _abi_paged.MAX_SCORE_ROWS):
            n = min(T, r + _abi_paged.MAX_SCORE_ROWS)
            part = out.rows(r, n)
            _abi_paged.token_scores(logits[r:n], None if targets is None else targets[r:n], part.logprob, part.entropy, part.top_ids, part.top_logprobs, top)
    return out
