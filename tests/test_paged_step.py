"""The paged model step against the full causal forward, token by token: chunks, single tokens and idle slots in one call.

Bound of the native path.  A layer rounds to bf16 (2^-9 relative) the normalised input, queries, latent, attention
weights, attention output and the FFN's input, hidden values and weights: 8 roundings per layer, each of a quantity no
larger than the residual stream, and two more in front of the logits.  They are independent, so that the error of the
26 roundings of three layers is about sqrt(26) 2^-9 of the largest logit of a row; the test allows 2.5 times that.
The CPU path is fp32 throughout.
"""
import math

import pytest
import torch

CFG = {
    "vocab_size": 1000, "dim": 256, "n_layers": 3, "n_heads": 4, "n_dense_layers": 3,
    "n_routed_experts": 8, "n_shared_experts": 1, "n_activated_experts": 2, "inter_dim": 512,
    "moe_inter_dim": 128, "kv_lora_rank": 64, "q_lora_rank": 0, "qk_nope_head_dim": 48,
    "qk_rope_head_dim": 16, "v_head_dim": 64, "max_seq_len": 128, "rope_theta": 10000,
    "rope_factor": 1.0, "mscale": 1.0, "mtp_depth": 1, "mtp_loss_weight": 0.3,
    "attn_impl": "sdpa", "weight_tying": False,
}
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
BOUND = {"cpu": 1e-4, "cuda": 2.5 * math.sqrt(26) * 2.0 ** -9}
# new tokens of each of five sequences, step by step: whole prompts, chunks over page edges, single tokens, idle slots
STEPS = [(16, 0, 70, 1, 5), (1, 12, 0, 1, 11), (1, 12, 1, 0, 16), (0, 12, 1, 1, 1), (1, 1, 1, 29, 0), (14, 0, 1, 1, 17),
         (1, 1, 1, 1, 1)]


def _model(device, cfg):
    from models.transformer import Transformer
    torch.manual_seed(0)
    model = Transformer(cfg).to(device).eval()
    with torch.no_grad():
        for layer in model.layers:           # let attention weigh as much as the rest, and depend on position
            layer.attn.wo.weight.mul_(4.0)
            layer.attn.wkv_a.weight.mul_(4.0)
    return model


def _full(model, tokens):
    with torch.enable_grad():                # the module path
        return model(tokens[None], use_cache=False).detach()[0].float()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("q_lora", [0, 64], ids=["direct_q", "lora_q"])
@pytest.mark.parametrize("page", [8, 32])
def test_logits_of_every_step(device, q_lora, page):
    from ops.paged import PagedLatentCache, paged_step
    cfg = dict(CFG, q_lora_rank=q_lora)
    model = _model(device, cfg)
    g = torch.Generator().manual_seed(1)
    total = [sum(s[b] for s in STEPS) for b in range(5)]
    seqs = [torch.randint(0, 1000, (n,), generator=g).to(device) for n in total]
    want = [_full(model, s) for s in seqs]
    cols = -(-max(total) // page)
    cache = PagedLatentCache(cfg, 5 * cols, page, device, torch.bfloat16 if device == "cuda" else torch.float32)
    cache.pages.fill_(float("nan"))
    table = torch.randperm(5 * cols, generator=g).int().view(5, cols).to(device)
    done = [0] * 5
    for step in STEPS:
        cu = torch.tensor([0, *torch.tensor(step).cumsum(0).tolist()], dtype=torch.int32, device=device)
        new = torch.cat([s[d:d + n] for s, d, n in zip(seqs, done, step)])
        done = [d + n for d, n in zip(done, step)]
        lens = torch.tensor(done, dtype=torch.int32, device=device)
        got = paged_step(model, new, cache, table, cu, lens).float()
        for b, n in enumerate(step):
            if n:
                ref = want[b][done[b] - 1]
                assert (got[b] - ref).abs().max() <= BOUND[device] * ref.abs().max(), (step, b)
    assert done == total
    # the bound is narrow enough to tell a position from the next one
    for s, w in zip(seqs, want):
        if s.numel() > 8:
            off = _full(model, s[1:])[-1]
            assert (off - w[-1]).abs().max() > 3 * BOUND[device] * w[-1].abs().max()


@pytest.mark.parametrize("device", DEVICES)
def test_beam_scores_are_the_log_probabilities_of_their_tokens(device):
    """A beam's score sums ``new`` log-probabilities, each off by no more than twice the bound of the logits."""
    from inference.beam_search import BeamSearchDecoder
    model = _model(device, CFG)
    g = torch.Generator().manual_seed(3)
    prompts = [torch.randint(0, 1000, (n,), generator=g).to(device) for n in (37, 16, 5)]
    new = 20
    tokens, scores = BeamSearchDecoder(model, num_beams=4, page_size=16, prefill_chunk=12).generate(prompts,
                                                                                                    max_new_tokens=new)
    assert (scores[:, :-1] >= scores[:, 1:]).all()
    for b, p in enumerate(prompts):
        for k in range(4):
            logits = _full(model, torch.cat([p, tokens[b, k]]))[p.numel() - 1:-1]
            want = torch.log_softmax(logits, -1).gather(1, tokens[b, k][:, None]).sum().item()
            bound = 2 * BOUND[device] * logits.abs().amax(-1).sum().item()
            assert abs(float(scores[b, k]) - want) <= bound
