"""Beam search's selection over beams and vocabulary (MI355X).

``l20_beam_search_step`` takes a step's logits and the beams' scores and gives each request's next beams: tokens,
the beams that they continue, and their scores; candidates that end there are given apart.  The parents go to
``l20_reorder_block_tables`` (``l20_block_tables``), which lets the cache's block tables follow them, and
``l20_copy_pages`` copies what must not be shared.  The reference decodes greedily or by verification: no
counterpart there.
"""

from __future__ import annotations

from functools import lru_cache
from typing import NamedTuple, Optional, Sequence

import torch

import l20_paged_decode  # noqa: F401  (loads the ops library)
from l20_paged_split_kv import _gpu_facts

MAX_BEAMS = 32
MAX_END_TOKENS = 8


class BeamSearchStep(NamedTuple):
    """The next beams of ``l20_beam_search_step`` and the candidates that ended, all [requests, beams]."""

    tokens: torch.Tensor  # int64, -1: no such beam
    parents: torch.Tensor  # int32, the beam that it continues, -1: none
    scores: torch.Tensor  # fp32, -inf: none
    ended_tokens: torch.Tensor  # int64, the end token, -1: none
    ended_parents: torch.Tensor  # int32
    ended_scores: torch.Tensor  # fp32

    @staticmethod
    def empty(requests: int, beams: int, device) -> "BeamSearchStep":
        def one(dtype):
            return torch.empty(requests, beams, dtype=dtype, device=device)

        return BeamSearchStep(one(torch.int64), one(torch.int32), one(torch.float32),
                              one(torch.int64), one(torch.int32), one(torch.float32))


@lru_cache(maxsize=4096)
def _bytes(requests: int, beams: int, vocab: int, ends: int) -> int:
    import l20_pd_cabi

    a = l20_pd_cabi.L20PdBeamStepArgs()
    a.requests, a.beams, a.vocab, a.num_end_tokens = requests, beams, vocab, ends
    return int(l20_pd_cabi.load().l20_pd_beam_step_workspace(l20_pd_cabi.ctypes.byref(a)))


def allocate_l20_beam_search_workspace(logits: torch.Tensor, scores: torch.Tensor, *,
                                       end_tokens: Sequence[int] = ()) -> torch.Tensor:
    """The workspace of ``l20_beam_search_step`` for up to these requests, beams, vocabulary and number of end tokens
    (uint8).  Calls that may overlap each need their own; its contents do not matter."""
    size = _bytes(scores.shape[0], scores.shape[1], logits.shape[-1], len(end_tokens))
    return torch.empty(size, dtype=torch.uint8, device=logits.device)


def l20_beam_search_step(
    logits: torch.Tensor,
    scores: torch.Tensor,
    *,
    end_tokens: Sequence[int] = (),
    out: Optional[BeamSearchStep] = None,
    workspace: Optional[torch.Tensor] = None,
) -> BeamSearchStep:
    """One step of beam search for every request.

    ``logits`` [requests * beams, vocab] or [requests, beams, vocab] (bf16, fp16 or fp32; rows of any stride) and
    ``scores`` fp32 [requests, beams], the beams' summed log-probabilities.  A candidate is a beam and a token; its
    score is the beam's plus the token's log-probability.  The next beams are the best candidates whose token is not
    in ``end_tokens`` (at most 8); candidates with an end token are given apart where they are among the first
    ``beams`` of all.  Candidates are ordered by score (in 64 bits), then lower beam, higher logit, lower token.

    A beam whose score is not finite is dead and its logits do not matter: a first step has scores 0 and, for all but
    one beam, -inf; a finished request has -inf alone, and gets parents of -1.  Masked tokens (-inf) are never taken,
    and a row with a NaN or +inf, or masked throughout, gives no candidates.  Where there are fewer candidates than
    beams the rest are tokens and parents of -1 with a score of -inf.

    ``out.scores`` may be ``scores`` itself; other outputs must share no bytes with the inputs.  With ``out`` and
    ``workspace`` given nothing is allocated and the call can be captured in a graph."""
    if not (logits.is_cuda and _gpu_facts(logits.device)[0]):
        raise RuntimeError("l20_beam_search_step requires an MI355X (gfx950) GPU")
    if scores.ndim != 2 or not 1 <= scores.shape[1] <= MAX_BEAMS:
        raise RuntimeError(f"scores must be [requests, beams] with 1 to {MAX_BEAMS} beams")
    if out is None:
        out = BeamSearchStep.empty(scores.shape[0], scores.shape[1], scores.device)
    if workspace is None:
        workspace = allocate_l20_beam_search_workspace(logits, scores, end_tokens=end_tokens)
    torch.ops.l20_stack.beam_search_step(logits, scores, end_tokens, *out, workspace)
    return out


def _register_fake() -> None:
    @torch.library.register_fake("l20_stack::beam_search_step")
    def _beam_search_step_fake(logits, scores, end_tokens, tokens, parents, scores_out, ended_tokens, ended_parents,
                               ended_scores, workspace):
        return None


_register_fake()
