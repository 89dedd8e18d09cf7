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
