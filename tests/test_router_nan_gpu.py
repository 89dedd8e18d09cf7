"""The router on scores that are not numbers: expert ids stay in range and distinct."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("experts,k", [(8, 2), (20, 4), (64, 8), (256, 8), (4, 4)])
def test_experts_are_in_range_when_scores_are_nan(experts, k):
    from ops._ext import native
    g = torch.Generator(device="cuda").manual_seed(experts)
    logits = torch.randn(300, experts, device="cuda", generator=g)
    bias = torch.randn(experts, device="cuda", generator=g) * 0.01

    def route(x, b):
        t = x.shape[0]
        idx = torch.empty(t, k, device="cuda", dtype=torch.int32)
        w, s = torch.empty(t, k, device="cuda"), torch.empty(t, k, device="cuda")
        counts = torch.zeros(experts, device="cuda", dtype=torch.int32)
        native().router_topk(x, b, experts, k, 1.0, idx, w, s, counts)
        return idx, w, counts

    want_idx, want_w, _ = route(logits, bias)
    x = logits.clone()
    x[::3] = float("nan")                                     # every score of a token
    x[1::3, 1:] = float("nan")                                # all but one
    idx, w, counts = route(x, bias)
    assert idx.min() >= 0 and idx.max() < experts
    assert (idx.sort(1).values.diff(dim=1) > 0).all()
    assert torch.equal(counts.long(), torch.bincount(idx.flatten().long(), minlength=experts))
    assert torch.equal(idx[::3], torch.arange(k, device="cuda", dtype=torch.int32).expand(100, k))
    assert (idx[1::3, 0] == 0).all()                          # a number goes before a NaN
    assert w[::3].isnan().all()
    assert torch.equal(idx[2::3], want_idx[2::3]) and torch.equal(w[2::3], want_w[2::3])
    off = torch.where(torch.arange(experts, device="cuda") < 1, 0.0, float("-inf"))
    idx, _, _ = route(logits, off)                            # experts switched off by their bias
    assert torch.equal(idx, torch.arange(k, device="cuda", dtype=torch.int32).expand(300, k))
