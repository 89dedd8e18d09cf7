"""Beam search: choosing the next beams and reordering their paged cache.

CUDA tensors run the kernels of ``csrc/beam.cu``, CPU tensors the formulas
below (also the numerics oracle of the kernel tests).  Neither has a backward
pass; on CUDA results are detached.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from ._ext import native
from .paged import check_range


def beam_select(logits: torch.Tensor, scores: torch.Tensor, finished: Optional[torch.Tensor] = None,
                eos_token_id: int = -1) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """The ``K`` best continuations of each batch entry's ``K`` beams.

    ``logits [B, K, V]`` (bf16 or fp32), ``scores [B, K]`` fp32 (log-probability
    of each beam so far; ``-inf`` for a beam that holds nothing yet).  Candidate
    ``(k, v)`` scores ``scores[k] + log_softmax(logits[k])[v]``; a beam with
    ``finished[b, k]`` offers only ``eos_token_id``, at its unchanged score.
    Candidates are ordered by their fp32 score, ties by ``(k, v)``.

    Returns ``(scores [B, K] fp32, parents [B, K] int32, tokens [B, K] int32,
    finished [B, K] bool)``, best first.  A NaN logit or score counts as ``-inf`` and
    an infinite one as the largest finite float; a row of ``-inf`` offers nothing
    (score ``-inf``).  Up to 32 beams on CUDA.
    """
    if logits.is_cuda:
        return native().beam_select(logits, scores, finished, eos_token_id)
    bsz, beams, vocab = logits.shape
    if vocab < beams:
        raise ValueError(f"beam_select needs at least as many tokens ({vocab}) as beams ({beams})")
    if finished is not None and not 0 <= eos_token_id < vocab:
        raise ValueError("finished beams need an end token inside the vocabulary")
    big = torch.finfo(torch.float32).max
    ninf = torch.tensor(float("-inf"))
    x = torch.where(torch.isnan(logits), ninf.to(logits.dtype), logits).float().clamp(max=big)
    top = x.amax(-1, keepdim=True).clamp(min=-big)
    scores = torch.where(torch.isnan(scores), ninf, scores).clamp(max=big)
    total = torch.exp(x - top).sum(-1, keepdim=True)
    logp = torch.where(total > 0, (x - top) - torch.log(total), ninf)
    if finished is not None:
        frozen = torch.full((vocab,), float("-inf"))
        frozen[eos_token_id] = 0.0
        logp = torch.where(finished[..., None], frozen, logp)
    cand = (scores[..., None] + logp).flatten(1)
    value, at = torch.sort(cand, dim=1, descending=True, stable=True)
    value, at = value[:, :beams].contiguous(), at[:, :beams]
    parent, token = at // vocab, at % vocab
    done = token == eos_token_id
    if finished is not None:
        done = done | finished.gather(1, parent)
    return value, parent.int(), token.int(), done


def beam_reorder(pages: torch.Tensor, block_table: torch.Tensor, parents: torch.Tensor,
                 seq_lens: torch.Tensor) -> torch.Tensor:
    """Let beam ``i`` of every batch entry continue beam ``parents[b, i]``.

    ``pages [layers, pool, page, width]``, ``block_table [B * K, columns]``,
    ``parents [B, K]``, ``seq_lens [B]`` (the cached length, common to the beams
    of an entry).  Returns the new block table.  Full pages are shared: the new
    row lists the parent's.  The page that is being filled must stay private: a
    beam's first child keeps it, and each further child takes that of a beam
    without children (there are as many) and gets its rows copied in, in every
    layer (in place).  Later columns, and the current one when it is empty,
    stay each beam's own, so the pages being written are always distinct
    within an entry if they were to begin with.

    On CUDA a parent, page or length out of range is skipped and reported by
    ``ops._ext.check_status`` (a negative length counts as zero); on the CPU it
    raises ``IndexError``.
    """
    if pages.is_cuda:
        return native().beam_reorder(pages, block_table, parents, seq_lens)
    bsz, beams = parents.shape
    page = pages.shape[2]
    check_range("parent", parents, beams)
    check_range("length", seq_lens, block_table.shape[1] * page + 1)
    for b in range(bsz):                     # all checks before the first page is written
        col, rem = divmod(int(seq_lens[b]), page)
        if rem:
            check_range("page", block_table[b * beams:(b + 1) * beams, col], pages.shape[1])
    out = block_table.clone()
    for b in range(bsz):
        col, rem = divmod(int(seq_lens[b]), page)
        old = block_table[b * beams:(b + 1) * beams]
        new = out[b * beams:(b + 1) * beams]
        par = parents[b].long()
        new[:, :col] = old[par, :col]
        if rem == 0:
            continue
        spare = [int(old[i, col]) for i in range(beams) if i not in par.tolist()]
        kept = set()
        for i, p in enumerate(par.tolist()):
            src = int(old[p, col])
            dst = spare.pop(0) if p in kept else src
            kept.add(p)
            if dst != src:
                pages[:, dst, :rem] = pages[:, src, :rem]
            new[i, col] = dst
    return out
