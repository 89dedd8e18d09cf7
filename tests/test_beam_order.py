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
