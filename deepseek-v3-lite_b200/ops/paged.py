"""Paged latent cache: writing new rows and attending over them.

The dense cache of ``models.mla`` holds ``max_seq_len`` rows per batch row and
one position per call.  Here the cache is a pool of pages shared by all
sequences, and a call takes a *ragged* batch: any number of sequences, each
with any number of new tokens (a decode step, drafted tokens, a chunk of a
prompt, an idle slot) on top of any cached length.

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
below.  On CUDA a page or position out of range, or a token that the offsets
leave out, is skipped and reported by ``ops._ext.check_status``; on the CPU it
raises ``IndexError`` (the attention alone gives a token left out zeros).

These operators serve: they have no backward pass.  On CUDA their results are
detached, whether gradients are enabled or not (``models.mla`` trains).
"""
from __future__ import annotations

from typing import List

import torch

from . import norm as norm_ops
from ._ext import native


def check_range(what: str, values: torch.Tensor, end: int) -> torch.Tensor:
    """``values`` of a CPU form, all in ``[0, end)``; else ``IndexError`` (a negative one would count from the end)."""
    if values.numel() and (int(values.min()) < 0 or int(values.max()) >= end):
        raise IndexError(f"{what} {int(values.min())} to {int(values.max())}, not in 0 to {end - 1}")
    return values


def ragged_positions(cu_seqlens: torch.Tensor, seq_lens: torch.Tensor, total: int):
    """``(sequence, position)`` of each of ``total`` new tokens (int64), without a look at the values on the host.

    A token that no sequence holds gets a sequence in range and position -1,
    which the kernels skip and report.
    """
    if total and not seq_lens.numel():
        raise IndexError(f"{total} tokens without a sequence")
    t = torch.arange(total, device=cu_seqlens.device)
    cu, lens = cu_seqlens.long(), seq_lens.long()
    seq = torch.searchsorted(cu[1:].contiguous(), t, right=True)
    held = seq < lens.numel()
    seq = seq.clamp(max=max(lens.numel() - 1, 0))
    held &= t >= cu[seq]
    return seq, torch.where(held, lens[seq] - cu[seq + 1] + t, -1)


def token_positions(cu_seqlens: torch.Tensor, seq_lens: torch.Tensor, total: int):
    """``ragged_positions``; on the CPU a token that no sequence holds raises ``IndexError``."""
    seq, pos = ragged_positions(cu_seqlens, seq_lens, total)
    if total and not pos.is_cuda and (int(cu_seqlens[0]) > 0 or int(cu_seqlens[-1]) < total):
        raise IndexError(f"cu_seqlens covers {int(cu_seqlens[0])} to {int(cu_seqlens[-1])} of {total} tokens")
    return seq, pos


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
    check_range("position", pos, min(cos.shape[0], block_table.shape[1] * page))
    x = kv_a.float()
    lat, pe = x[:, :rank], x[:, rank:]
    lat = lat * torch.rsqrt(lat.square().mean(-1, keepdim=True) + eps) * weight
    c, s = cos[pos], sin[pos]
    a, b = pe[:, 0::2], pe[:, 1::2]
    pe = torch.stack([a * c - b * s, a * s + b * c], dim=-1).flatten(1)
    ids = check_range("page", block_table.long()[seq, pos // page], pages.shape[0])
    pages[ids, pos % page] = torch.cat([lat, pe], 1).to(pages.dtype)
    return pages


def paged_latent_attention(q: torch.Tensor, pages: torch.Tensor, block_table: torch.Tensor,
                           cu_seqlens: torch.Tensor, seq_lens: torch.Tensor, kv_rank: int,
                           scale: float) -> torch.Tensor:
    """Absorbed causal attention of new tokens over their cached rows.

    ``q [T, H, R + dr]`` holds each head's query multiplied by ``W_k`` (R)
    followed by its rotated part (dr).  Row ``t`` sees the cached rows up to its
    own position; the result ``[T, H, R]`` is the weighted sum of their latents.
    A token that sees no row (its position is negative) or that no sequence holds
    (reported on CUDA) gets zeros.  Rows at and
    past ``seq_lens`` may hold anything; those before it have to be finite, also
    for earlier tokens that do not see them (their weight there is zero, and zero
    times infinity is not).  ``scale`` is positive; ``q`` is copied if it is not
    contiguous.  On CUDA scores, sums and partial results are fp32 and the
    weights are rounded to bf16 for the second product: against 64 bits the
    result is off by 2.1e-3 (relative, root mean square), of which its own
    rounding to bf16 is 1.7e-3.
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
        kv = pages[check_range("page", block_table[b].long()[key // page], pages.shape[0]), key % page].float()
        pos = torch.arange(n - (hi - lo), n)
        s = torch.einsum("thd,jd->thj", q[lo:hi].float(), kv) * scale
        s = s.masked_fill((key[None, :] > pos[:, None])[:, None, :], float("-inf"))
        p = torch.where((pos >= 0)[:, None, None], s.softmax(dim=-1), torch.zeros_like(s))
        out[lo:hi] = torch.einsum("thj,jr->thr", p, kv[:, :kv_rank]).to(q.dtype)
    return out


class PagedLatentCache:
    """Pages of the latent cache of every layer, and a host-side list of free ones.

    ``pages [layers, pool, page, R + dr]``; ``take`` and ``give`` hand page ids
    out and back (the caller writes them into its block tables).  One id stands
    for the same page in every layer.
    """

    def __init__(self, config: dict, pool: int, page_size: int = 64, device=None, dtype=torch.bfloat16):
        if page_size < 8 or page_size > 256 or page_size & (page_size - 1):
            raise ValueError(f"page_size must be a power of two from 8 to 256, got {page_size}")
        self.page_size = page_size
        width = config["kv_lora_rank"] + config["qk_rope_head_dim"]
        self.pages = torch.empty(config["n_layers"], pool, page_size, width, device=device, dtype=dtype)
        self._free: List[int] = list(range(pool - 1, -1, -1))

    @property
    def free(self) -> int:
        """Number of pages that are not handed out."""
        return len(self._free)

    def take(self, n: int) -> List[int]:
        """``n`` page ids; raises ``RuntimeError`` if fewer are free."""
        if n > len(self._free):
            raise RuntimeError(f"paged cache: {n} pages wanted, {len(self._free)} of {self.pages.shape[1]} free")
        return [self._free.pop() for _ in range(n)]

    def give(self, ids: List[int]) -> None:
        """Return pages that ``take`` handed out."""
        self._free.extend(ids)


@torch.no_grad()
def paged_step(model, tokens: torch.Tensor, cache: PagedLatentCache, block_table: torch.Tensor,
               cu_seqlens: torch.Tensor, seq_lens: torch.Tensor) -> torch.Tensor:
    """Run the new ``tokens [T]`` of a ragged batch through the model.

    Writes their cache rows and returns the logits after the last new token of
    each sequence, ``[B, vocab]`` (a sequence without new tokens gets an
    unspecified row).  Only those: a check of drafted tokens, which wants the
    logits after each of them, calls the operators above layer by layer.
    Metadata as above.
    """
    if not tokens.numel():                   # every slot idle
        return model.head.weight.new_zeros(seq_lens.numel(), model.config["vocab_size"],
                                           dtype=torch.bfloat16 if tokens.is_cuda else None)
    if tokens.is_cuda:
        return model.native_inference().forward_paged(tokens, cache, block_table, cu_seqlens, seq_lens)
    from .decode import _row_rope
    from .rope import rope_cos_sin
    cfg = model.config
    cos, sin = rope_cos_sin(cfg["max_seq_len"], cfg["qk_rope_head_dim"], float(cfg["rope_theta"]))
    _, pos = token_positions(cu_seqlens, seq_lens, tokens.numel())
    h = model.embed(tokens.long()).unsqueeze(1)                                    # [T, 1, dim]
    for i, layer in enumerate(model.layers):
        attn = layer.attn
        x = norm_ops.rms_norm(h, layer.attn_norm.weight, layer.attn_norm.eps)
        attn._extend_rope(attn.max_seq_len, x.device)
        latent_cache_append(cache.pages[i], attn.wkv_a(x)[:, 0], attn.kv_norm.weight, cos, sin, block_table, cu_seqlens,
                            seq_lens)
        q_nope, q_pe = attn._queries(x)
        q_pe = _row_rope(q_pe, attn.freqs_cis[pos])
        w_k, w_v = attn._wkv_b_split()
        q = torch.cat([torch.einsum("thd,hdr->thr", q_nope[:, 0], w_k), q_pe[:, 0]], dim=-1)
        o = paged_latent_attention(q, cache.pages[i], block_table, cu_seqlens, seq_lens, attn.kv_lora_rank,
                                   attn.softmax_scale)
        h = h + attn.wo(torch.einsum("thr,hdr->thd", o, w_v).reshape(tokens.numel(), 1, -1))
        h = h + layer.ffn(norm_ops.rms_norm(h, layer.ffn_norm.weight, layer.ffn_norm.eps))
    last = (cu_seqlens[1:].long() - 1).clamp(min=0)
    return model.head(model.final_hidden(h[last, 0]))
