"""Beam search over the paged cache: ``chill_beam_select`` chooses the candidates, ``chill_pages_fork`` (cache.py) gives every beam the pages of the one that it
continues.

    scores = torch.full((groups, beams), -inf); scores[:, 0] = 0            # float32: the beams of a request are one to begin with
    while ...:
        ...                                                                 # a step of the model: logits [groups * beams, vocab]
        scores, parents, tokens = chill_beam_select(logits, scores)
        lens, copies = chill_pages_fork(pages, shared, lens, parents.view(-1), page_size)
        chill_cache_copy(k_cache, v_cache, copies)                          # for every layer's caches, or for all in one call

Nothing here synchronises, and every call can be captured into a CUDA graph.  The reference has no counterpart.
"""
from __future__ import annotations

import typing

import torch

from . import _decode_abi, _eager, cache, rotary


class ChillBeams(typing.NamedTuple):
    """Chosen candidates of every group, best first: scores float32, parents (row of the logits, group * beams + beam) and tokens int32, [groups, count]."""

    scores: torch.Tensor
    parents: torch.Tensor
    tokens: torch.Tensor


def _check_select(logits, scores, count, finished, end_token):
    assert logits.is_cuda, "the selection runs on CUDA tensors only"
    cache._check_sizes(logits=logits)
    assert logits.ndim == 2 and logits.numel() > 0 and logits.dtype in cache._DTYPES, "logits must be [groups * beams, vocab], fp16 / bf16 / fp32"
    V = logits.shape[1]
    assert logits.stride(1) == 1 or V == 1, "the elements of a row of logits must lie beside each other"
    assert V <= 2 ** 26 and logits.shape[0] <= 65535
    assert scores.ndim == 2 and scores.dtype == torch.float32 and scores.is_contiguous() and scores.device == logits.device and \
        scores.numel() == logits.shape[0], "scores must be a contiguous float32 tensor [groups, beams] with a row of logits for each"
    K = scores.shape[1]
    assert K <= _decode_abi.SELECT_MAX and 1 <= count <= _decode_abi.SELECT_MAX, f"at most {_decode_abi.SELECT_MAX} beams and candidates"
    assert count <= K * V, "a group has fewer candidates than are asked for"
    if finished is not None:
        assert finished.dtype == torch.bool and finished.shape == scores.shape and finished.is_contiguous() and finished.device == logits.device, \
            "finished must be a contiguous bool tensor [groups, beams]"
        assert 0 <= end_token < V, "end_token must be in the vocabulary"
    assert not (torch.is_grad_enabled() and (logits.requires_grad or scores.requires_grad)), \
        "the selection has no gradients: call it under torch.no_grad() or with detached tensors"
    cache._check_grad(logits, scores)


@torch.library.custom_op("chill_attention::beam_select", mutates_args=(), device_types=("cuda",))
def _select_op(logits: torch.Tensor, scores: torch.Tensor, count: int, finished: typing.Optional[torch.Tensor],
               end_token: int) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    _check_select(logits, scores, count, finished, end_token)
    return _eager.extension().beam_select(rotary._native(), logits, scores, count, finished, end_token)


@_select_op.register_fake
def _(logits, scores, count, finished, end_token):
    G = scores.shape[0]
    ints = lambda: scores.new_empty(G, count, dtype=torch.int32)  # noqa: E731
    return scores.new_empty(G, count), ints(), ints()


def chill_beam_select(logits: torch.Tensor, scores: torch.Tensor, count: int | None = None, finished: torch.Tensor | None = None,
                      end_token: int = 0) -> ChillBeams:
    """The ``count`` best continuations of every group of beams.

    Candidate (beam, token) of a group has ``scores[group, beam] + log_softmax(logits[row])[token]``, row = group * beams + beam; -inf where the logit or the beam's score
    is -inf (a row of nothing but -inf has no candidates).  They are ranked by that value in 64 bits, and it is rounded to fp32 at the end; of equal ones the lowest
    beam, then the largest logit, then the lowest token comes first.  The exponentials of the row's sum are fp32, so its logarithm is good to 1e-7 (1e-5 where the
    maximum rises again and again along the row): a beam's candidates are in the exact order of their logits, those of different beams may change places where they are
    nearer than that.  Equal rows have equal sums, bit for bit.  A NaN or +inf among a row's logits, or a NaN as score, makes its candidates NaN, which rank first: they
    show.  They are all alike, and so are those of a score of +inf: the lowest token first.

    Args:
        logits: [groups * beams, vocab], fp16 / bf16 / fp32; rows any stride apart.
        scores: float32 [groups, beams], sums of log-probabilities; -inf: no such beam (in the first step all but one of a request's beams).
        count: candidates to keep, default the number of beams; up to 64, as are the beams.  (Twice the beams leave enough where tokens end some of them.)
        finished: bool [groups, beams]: beams at their end; they have one candidate, ``end_token`` at their score, and their logits are not read.

    Returns: ChillBeams.  With fewer candidates than ``count`` the last ones have score -inf (parents and tokens: the first ones that are left over).
    ``parents.view(-1)`` is what ``chill_pages_fork`` takes where count is the number of beams.
    """
    if count is None:
        count = scores.shape[-1]
    if cache._direct():
        out = _eager.extension().beam_select(rotary._NATIVE or rotary._native(), logits, scores, count, finished, end_token)
        if out is not None:
            return ChillBeams(*out)
    _check_select(logits, scores, count, finished, end_token)
    return ChillBeams(*_select_op(logits, scores, count, finished, end_token))
