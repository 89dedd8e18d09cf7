"""Paged latent cache: writing new rows and attending over them.

The dense cache of ``models.mla`` holds ``max_seq_len`` rows per batch row and
one position per call.  Here the cache is a pool of pages shared by all
sequences, and a call takes a *ragged* batch: any number of sequences, each
with any number of new tokens (a decode step, a speculative check, a chunk of
a prompt, an idle slot) on top of any cached length.

Metadata (int32 tensors on the pages' device, read there only, so nothing
synchronises and a CUDA graph stays valid while they change):

* ``block_table [B, columns]``: page of positions ``[j * page, (j + 1) * page)``;
* ``cu_seqlens [B + 1]``: the new tokens of sequence ``b`` are rows
  ``cu[b]:cu[b + 1]`` of the token-major inputs;
* ``seq_lens [B]``: cached length *including* the new tokens, so token ``i`` of
  ``n`` sits at position ``seq_lens[b] - n + i``.

``pages [pool, page, R + dr]`` bf16 holds the RMS-normalised latent followed by
the rotated shared key, one layer per tensor (a layer of a stacked
``[layers, pool, page, R + dr]`` buffer will do).  The page size is a power of
two from 8 to 256; R is a multiple of 8 up to 512 and dr one up to 64.

CUDA tensors run the kernels of ``csrc/paged.cu``, CPU tensors the formulas
below.  On CUDA a page or position out of range is skipped and reported by
``ops._ext.check_status``; on the CPU it raises ``IndexError``.
"""
from __future__ import annotations

import torch

from ._ext import native


def token_positions(cu_seqlens: torch.Tensor, seq_lens: torch.Tensor, total: int):
    """``(sequence, position)`` of each of ``total`` new tokens (int64)."""
    t = torch.arange(total, device=cu_seqlens.device)
    seq = torch.searchsorted(cu_seqlens[1:].long().contiguous(), t, right=True)
    if total and int(seq[-1]) >= seq_lens.numel():
        raise IndexError(f"cu_seqlens covers {int(cu_seqlens[-1])} of {total} tokens")
    return seq, seq_lens.long()[seq] - cu_seqlens.long()[seq + 1] + t


def latent_cache_append(pages: torch.Tensor, kv_a: torch.Tensor, weight: torch.Tensor, cos: torch.Tensor,
                        sin: torch.Tensor, block_table: torch.Tensor, cu_seqlens: torch.Tensor,
                        seq_lens: torch.Tensor, eps: float = 1e-6) -> torch.Tensor:
    """Write the cache rows of new tokens into their pages (in place); returns ``pages``.

    ``kv_a [T, R + dr]`` (bf16 or fp32) is the output of the ``wkv_a``
    projection: its first R columns are RMS-normalised with ``weight [R]``
    (fp32), the others are rotated as interleaved pairs by the tables
    ``cos``/``sin [positions, dr / 2]`` (fp32) at the token's position.
    """
    if pages.is_cuda:
        native().latent_cache_append(pages, kv_a, weight, cos, sin, block_table, cu_seqlens, seq_lens, eps)
        return pages
    rank, page = weight.numel(), pages.shape[1]
    seq, pos = token_positions(cu_seqlens, seq_lens, kv_a.shape[0])
    x = kv_a.float()
    lat, pe = x[:, :rank], x[:, rank:]
    lat = lat * torch.rsqrt(lat.square().mean(-1, keepdim=True) + eps) * weight
    c, s = cos[pos], sin[pos]
    a, b = pe[:, 0::2], pe[:, 1::2]
    pe = torch.stack([a * c - b * s, a * s + b * c], dim=-1).flatten(1)
    pages[block_table.long()[seq, pos // page], pos % page] = torch.cat([lat, pe], 1).to(pages.dtype)
    return pages


def paged_latent_attention(q: torch.Tensor, pages: torch.Tensor, block_table: torch.Tensor,
                           cu_seqlens: torch.Tensor, seq_lens: torch.Tensor, kv_rank: int,
                           scale: float) -> torch.Tensor:
    """Absorbed causal attention of new tokens over their cached rows.

    ``q [T, H, R + dr]`` holds each head's query multiplied by ``W_k`` (R)
    followed by its rotated part (dr).  Row ``t`` sees the cached rows up to its
    own position; the result ``[T, H, R]`` is the weighted sum of their latents.
    A token that sees no row (its position is negative) gets zeros.
    """
    if q.is_cuda:
        return native().paged_latent_attention(q.contiguous(), pages, block_table, cu_seqlens, seq_lens, kv_rank,
                                               scale)
    out = torch.zeros(*q.shape[:2], kv_rank, dtype=q.dtype)
    page = pages.shape[1]
    for b in range(seq_lens.numel()):
        lo, hi, n = int(cu_seqlens[b]), int(cu_seqlens[b + 1]), int(seq_lens[b])
        if hi <= lo or n <= 0:
            continue
        key = torch.arange(n)
        kv = pages[block_table[b].long()[key // page], key % page].float()
        pos = torch.arange(n - (hi - lo), n)
        s = torch.einsum("thd,jd->thj", q[lo:hi].float(), kv) * scale
        s = s.masked_fill((key[None, :] > pos[:, None])[:, None, :], float("-inf"))
        p = torch.where((pos >= 0)[:, None, None], s.softmax(dim=-1), torch.zeros_like(s))
        out[lo:hi] = torch.einsum("thj,jr->thr", p, kv[:, :kv_rank]).to(q.dtype)
    return out
