"""Beam search over the paged latent cache.

``BeamSearchDecoder`` prefills prompts of any lengths in chunks (one ragged call
per chunk), then advances ``num_beams`` beams per prompt: a model step over all
beams, ``ops.beam.beam_select`` over (beam, token) candidates, and
``ops.beam.beam_reorder``, which shares the full pages of a parent between its
children and copies only the page being filled.  Nothing in a step waits for
the device except the end-of-sequence test when ``eos_token_id`` is given.

``python inference/beam_search.py [--batch 8] [--beams 4] [--prompt 512] [--new 64]``
times it on the 412M dims with random weights.
"""
from __future__ import annotations

import argparse
import json
import sys
import time
from pathlib import Path
from typing import List, Optional, Sequence, Tuple, Union

import torch
import yaml

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

from models.transformer import Transformer  # noqa: E402
from ops.beam import beam_reorder, beam_select  # noqa: E402
from ops.paged import PagedLatentCache, paged_step  # noqa: E402


class BeamSearchDecoder:
    """Beam search for a batch of prompts of different lengths."""

    def __init__(self, model: Transformer, num_beams: int = 4, page_size: int = 64, prefill_chunk: int = 512):
        if not 1 <= num_beams <= 32:
            raise ValueError(f"num_beams must be 1 to 32, got {num_beams}")
        if prefill_chunk < 1:
            raise ValueError(f"prefill_chunk must be positive, got {prefill_chunk}")
        self.model = model
        self.beams = num_beams
        self.page_size = page_size
        self.chunk = prefill_chunk

    def _tables(self, lens: Sequence[int], new: int) -> Tuple[PagedLatentCache, torch.Tensor]:
        """A cache of the size needed and its tables ``[B * K, columns]``: the beams of a prompt share its
        full pages and own every later one."""
        page, beams, m = self.page_size, self.beams, self.model
        weight = m.embed.weight
        need = [(n // page, (n + new + page - 1) // page) for n in lens]          # shared columns, all columns
        cols = max(c for _, c in need)
        dtype = torch.bfloat16 if weight.is_cuda else weight.dtype
        cache = PagedLatentCache(m.config, sum(s + beams * (c - s) for s, c in need), page, weight.device, dtype)
        table = torch.zeros(len(lens) * beams, cols, dtype=torch.int32)
        for b, (s, c) in enumerate(need):
            shared = torch.tensor(cache.take(s), dtype=torch.int32)
            for k in range(beams):
                row = table[b * beams + k]
                row[:s] = shared
                row[s:c] = torch.tensor(cache.take(c - s), dtype=torch.int32)
        return cache, table.to(weight.device)

    def _prefill(self, prompts: List[torch.Tensor], cache: PagedLatentCache, table: torch.Tensor) -> torch.Tensor:
        """Logits ``[B, V]`` after each prompt; the rows go to its first beam's pages."""
        dev = table.device
        lens = [p.numel() for p in prompts]
        done, logits = 0, None
        while done < max(lens):
            part = [p[done:done + self.chunk] for p in prompts]
            new = torch.tensor([0] + [p.numel() for p in part])
            upto = torch.tensor([min(n, done + self.chunk) for n in lens], dtype=torch.int32)
            out = paged_step(self.model, torch.cat(part), cache, table[::self.beams], new.cumsum(0).int().to(dev),
                             upto.to(dev))
            # a prompt that ended in an earlier chunk keeps its logits
            live = (new[1:] > 0).to(dev)[:, None]
            logits = out.float() if logits is None else torch.where(live, out.float(), logits)
            done += self.chunk
        return logits

    @torch.no_grad()
    def generate(self, prompts: Union[torch.Tensor, Sequence[torch.Tensor]], max_new_tokens: int = 64,
                 eos_token_id: Optional[int] = None, length_penalty: float = 0.0
                 ) -> Tuple[torch.Tensor, torch.Tensor]:
        """``(tokens [B, K, max_new_tokens], scores [B, K])`` of the new tokens, best beam first.

        ``scores`` are sums of log-probabilities, divided by ``length **
        length_penalty`` (tokens up to and with the end token) where that is not
        zero.  A beam that produced ``eos_token_id`` repeats it from there on.
        """
        prompts = [p.reshape(-1) for p in prompts]
        if not prompts or min(p.numel() for p in prompts) == 0:
            raise ValueError("beam search needs at least one prompt, and none of them empty")
        if max_new_tokens < 1:
            raise ValueError(f"max_new_tokens must be positive, got {max_new_tokens}")
        lens = [p.numel() for p in prompts]
        if max(lens) + max_new_tokens > self.model.max_seq_len:
            raise ValueError(f"prompt + new tokens ({max(lens) + max_new_tokens}) exceeds max_seq_len "
                             f"{self.model.max_seq_len}")
        was_training = self.model.training
        self.model.eval()
        try:
            return self._search(prompts, lens, max_new_tokens, eos_token_id, length_penalty)
        finally:
            self.model.train(was_training)

    def _search(self, prompts, lens, new, eos, alpha):
        bsz, beams, dev = len(prompts), self.beams, prompts[0].device
        cache, table = self._tables(lens, new)
        length = torch.tensor(lens, dtype=torch.int32, device=dev)
        cu = torch.arange(bsz * beams + 1, dtype=torch.int32, device=dev)
        scores = torch.full((bsz, beams), float("-inf"), device=dev)
        scores[:, 0] = 0.0                                   # one beam holds the prompt
        finished = None if eos is None else torch.zeros(bsz, beams, dtype=torch.bool, device=dev)
        end = -1 if eos is None else eos
        tokens = torch.zeros(bsz, beams, new, dtype=torch.long, device=dev)
        logits = self._prefill(prompts, cache, table)[:, None].expand(bsz, beams, -1)
        for i in range(new):
            scores, parents, chosen, done = beam_select(logits, scores, finished, end)
            tokens = tokens.gather(1, parents.long()[..., None].expand(-1, -1, new))
            tokens[:, :, i] = chosen
            if eos is not None:
                finished = done
                if bool(done.all()):
                    tokens[:, :, i + 1:] = eos
                    break
            if i + 1 < new:
                table = beam_reorder(cache.pages, table, parents, length)
                length = length + 1
                logits = paged_step(self.model, chosen.reshape(-1), cache, table, cu,
                                    length.repeat_interleave(beams)).view(bsz, beams, -1)
        if alpha != 0.0:
            size = torch.full((bsz, beams), float(new), device=dev)
            if eos is not None:
                hit = tokens == eos
                size = torch.where(hit.any(-1), hit.float().argmax(-1) + 1.0, size)
            scores = scores / size ** alpha
            scores, order = scores.sort(dim=1, descending=True, stable=True)
            tokens = tokens.gather(1, order[..., None].expand(-1, -1, new))
        return tokens, scores


def main() -> None:
    ap = argparse.ArgumentParser(description="Beam search throughput on the 412M dims, random weights")
    ap.add_argument("--batch", type=int, default=8)
    ap.add_argument("--beams", type=int, default=4)
    ap.add_argument("--prompt", type=int, default=512)
    ap.add_argument("--new", type=int, default=64)
    a = ap.parse_args()
    cfg = yaml.safe_load(open(Path(__file__).resolve().parent.parent / "configs" / "pretrain_412m.yaml"))["model"]
    torch.manual_seed(0)
    model = Transformer(cfg).cuda().eval()
    decoder = BeamSearchDecoder(model, num_beams=a.beams)
    prompts = [torch.randint(0, cfg["vocab_size"], (max(1, a.prompt - 7 * b),), device="cuda") for b in range(a.batch)]
    decoder.generate(prompts, max_new_tokens=4)              # weight copies, allocations
    torch.cuda.synchronize()
    t0 = time.perf_counter()
    decoder.generate(prompts, max_new_tokens=a.new)
    torch.cuda.synchronize()
    s = time.perf_counter() - t0
    print(json.dumps({"batch": a.batch, "beams": a.beams, "prompt": a.prompt, "new_tokens": a.new,
                      "seconds": round(s, 4), "beam_tokens_per_s": round(a.batch * a.beams * a.new / s, 1)}))


if __name__ == "__main__":
    main()
