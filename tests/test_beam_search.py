"""BeamSearchDecoder: against exhaustive bookkeeping on the CPU, and the kernels' path on a B200."""
import math

import pytest
import torch


def _log_probs(model, seq):
    with torch.enable_grad():
        out = model(seq[None], use_cache=False).detach()
    return torch.log_softmax(out[0, -1].double(), -1)


def _reference(model, prompt, beams, new, eos):
    """Beam search with a full forward per beam and step."""
    live = [(0.0, [], False)]
    for _ in range(new):
        cand = []
        for k, (score, toks, stop) in enumerate(live):
            if stop:
                cand.append((-score, k, eos, True))
                continue
            lp = _log_probs(model, torch.cat([prompt, torch.tensor(toks, dtype=torch.long)]))
            cand += [(-(score + float(p)), k, v, v == eos) for v, p in enumerate(lp)]
        cand.sort()
        live = [(-s, live[k][1] + [v], stop) for s, k, v, stop in cand[:beams]]
    return live


@pytest.fixture(scope="module")
def cpu_model(small_cfg):
    from models.transformer import Transformer
    torch.manual_seed(3)
    model = Transformer(dict(small_cfg, vocab_size=61)).eval()
    with torch.no_grad():
        model.head.weight.mul_(8.0)       # spread the logits
    return model


@pytest.mark.parametrize("eos", [None, 7])
def test_matches_full_recomputation(cpu_model, eos):
    from inference.beam_search import BeamSearchDecoder
    g = torch.Generator().manual_seed(0)
    prompts = [torch.randint(0, 61, (n,), generator=g) for n in (13, 8, 1)]
    tokens, scores = BeamSearchDecoder(cpu_model, num_beams=3, page_size=8, prefill_chunk=5).generate(
        prompts, max_new_tokens=11, eos_token_id=eos)
    for b, p in enumerate(prompts):
        want = _reference(cpu_model, p, 3, 11, eos)
        for k in range(3):
            assert abs(float(scores[b, k]) - want[k][0]) < 1e-3
            got = tokens[b, k].tolist()
            assert got == want[k][1] + [eos] * (11 - len(want[k][1]))


def test_length_penalty_orders_by_mean(cpu_model):
    from inference.beam_search import BeamSearchDecoder
    p = torch.arange(6)[None]
    d = BeamSearchDecoder(cpu_model, num_beams=4, page_size=8)
    _, plain = d.generate(p, max_new_tokens=5)
    _, mean = d.generate(p, max_new_tokens=5, length_penalty=1.0)
    torch.testing.assert_close(mean, plain / 5)


def test_refusals(cpu_model):
    from inference.beam_search import BeamSearchDecoder
    from ops.paged import PagedLatentCache
    for bad in (0, 33):
        with pytest.raises(ValueError, match="num_beams"):
            BeamSearchDecoder(cpu_model, num_beams=bad)
    d = BeamSearchDecoder(cpu_model, num_beams=2, page_size=8)
    with pytest.raises(ValueError, match="max_seq_len"):
        d.generate([torch.zeros(60, dtype=torch.long)], max_new_tokens=5)
    with pytest.raises(ValueError, match="empty"):
        d.generate([torch.zeros(0, dtype=torch.long)], max_new_tokens=5)
    with pytest.raises(ValueError, match="max_new_tokens"):
        d.generate([torch.zeros(3, dtype=torch.long)], max_new_tokens=0)
    with pytest.raises(ValueError, match="page_size"):
        PagedLatentCache(cpu_model.config, 4, page_size=12)
    cache = PagedLatentCache(cpu_model.config, 4, page_size=8)
    ids = cache.take(3)
    with pytest.raises(RuntimeError, match="1 of 4 free"):
        cache.take(2)
    cache.give(ids)
    assert cache.free == 4


@pytest.mark.gpu
@pytest.mark.parametrize("q_lora", [0, 64], ids=["direct_q", "lora_q"])
def test_native_path(q_lora):
    """One beam is greedy decoding; more beams score what the eager model says of their tokens."""
    from inference.beam_search import BeamSearchDecoder
    from models.transformer import Transformer
    from ops._ext import check_status
    from test_infer_gpu import CFG
    torch.manual_seed(0)
    m = Transformer(dict(CFG, q_lora_rank=q_lora)).cuda().eval()
    for moe in m.moe_layers():
        moe.gate.weight.data.mul_(10.0)
    with torch.no_grad():
        m.head.weight.mul_(6.0)           # greedy choices well apart
    g = torch.Generator(device="cuda").manual_seed(1)
    prompts = torch.randint(0, CFG["vocab_size"], (3, 37), device="cuda", generator=g)
    greedy = m.generate(prompts, max_new_tokens=24, temperature=0.0)[:, 37:]
    one, _ = BeamSearchDecoder(m, num_beams=1, page_size=16, prefill_chunk=16).generate(prompts, max_new_tokens=24)
    assert (one[:, 0] == greedy).float().mean() > 0.8      # bf16 near-ties may part the two
    assert (one[:, 0, :4] == greedy[:, :4]).all()
    ragged = [p[:n] for p, n in zip(prompts, (37, 16, 5))]
    tokens, scores = BeamSearchDecoder(m, num_beams=4, page_size=16, prefill_chunk=12).generate(ragged, max_new_tokens=20)
    check_status()
    assert (scores[:, :-1] >= scores[:, 1:]).all()
    for b, p in enumerate(ragged):
        assert len({tuple(t.tolist()) for t in tokens[b]}) == 4
        for k in range(4):
            seq = torch.cat([p, tokens[b, k]])[None]
            with torch.enable_grad():
                lp = torch.log_softmax(m(seq, use_cache=False).detach()[0].float(), -1)
            at = torch.arange(p.numel() - 1, seq.shape[1] - 1, device="cuda")
            want = lp[at, seq[0, p.numel():]].sum().item()
            assert math.isclose(float(scores[b, k]), want, rel_tol=0.1, abs_tol=0.5)
