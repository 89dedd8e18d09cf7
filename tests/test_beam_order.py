"""Order and special values of the beam selection, the same on the CPU and on a B200."""
import pytest
import torch

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
NINF = float("-inf")


@pytest.mark.parametrize("device", DEVICES)
def test_end_token_outside_the_vocabulary_ends_nothing(device):
    from ops.beam import beam_select
    logits = torch.zeros(1, 2, 10, device=device)
    logits[0, :, 5] = 3.0
    for eos in (-1, 10, (1 << 32) + 5, -(1 << 32) + 5):
        _, _, token, done = beam_select(logits, torch.zeros(1, 2, device=device), None, eos)
        assert (token == 5).any() and not done.any()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("vocab", [40, 5000, 100018])
def test_zeros_of_either_sign_tie(device, dtype, vocab):
    """-0.0 and 0.0 are equal logits, and equal scores of finished beams: the lowest index goes first."""
    from ops.beam import beam_select
    logits = torch.full((1, 2, vocab), -5.0, device=device, dtype=dtype)
    at = [3, 7, vocab // 2, vocab - 2]
    logits[0, 0, at] = torch.tensor([-0.0, 0.0, -0.0, 0.0], device=device, dtype=dtype)
    scores = torch.tensor([[0.0, NINF]], device=device)
    _, parent, token, _ = beam_select(logits, scores)
    assert parent.tolist() == [[0, 0]] and token.tolist() == [[3, 7]]
    finished = torch.tensor([[True, True]], device=device)
    _, parent, token, _ = beam_select(logits, torch.tensor([[-0.0, 0.0]], device=device), finished, 1)
    assert parent.tolist() == [[0, 1]] and token.tolist() == [[1, 1]]


@pytest.mark.parametrize("device", DEVICES)
def test_scores_that_are_no_numbers(device):
    """A NaN score counts as -inf, an infinite one as the largest finite float, for live and finished beams."""
    from ops.beam import beam_select
    g = torch.Generator().manual_seed(0)
    logits = torch.randn(1, 3, 3000, generator=g).to(device)
    for bad in (float("nan"), NINF):
        for fin in (None, torch.tensor([[True, False, False]], device=device)):
            value, parent, token, _ = beam_select(logits, torch.tensor([[bad, -1.0, -2.0]], device=device), fin, 4)
            want = beam_select(logits[:, 1:], torch.tensor([[-1.0, -2.0]], device=device), None, 4)
            assert torch.isfinite(value).all() and (parent > 0).all()
            assert torch.equal(parent[:, :2], want[1] + 1) and torch.equal(token[:, :2], want[2])
            assert torch.equal(value[:, :2], want[0])
    big = torch.finfo(torch.float32).max
    value, parent, token, _ = beam_select(logits, torch.tensor([[-1.0, float("inf"), -2.0]], device=device))
    assert (value == big).all() and (parent == 1).all()
    fin = torch.tensor([[False, True, False]], device=device)
    value, parent, token, done = beam_select(logits, torch.tensor([[-1.0, float("inf"), -2.0]], device=device), fin, 4)
    assert value[0, 0] == big and parent[0, 0] == 1 and token[0, 0] == 4 and done[0, 0]
    assert torch.isfinite(value).all() and (parent[0, 1:] != 1).all()
