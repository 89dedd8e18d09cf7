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


def _check_order(device, logits, scores, finished=None, eos=-1, ties=True):
    """Against candidates in 64 bits, rounded once to fp32 and ordered by (score, index).

    ``ties`` says what the inputs are made for: candidates near the cut that lie so far from a rounding boundary that
    fp32 arithmetic (a few roundings of numbers up to 16) has to give the same scores; else, all of them clearly apart.
    Either is asserted."""
    from ops.beam import beam_select
    beams, vocab = logits.shape[1:]
    cand = scores.double()[..., None] + torch.log_softmax(logits.double(), -1)
    if finished is not None:
        frozen = torch.full((vocab,), NINF, dtype=torch.float64)
        frozen[eos] = 0.0
        cand = torch.where(finished[..., None], scores.double()[..., None] + frozen, cand)
    cand = cand.flatten(1)
    value, at = torch.sort(cand.float(), dim=1, descending=True, stable=True)
    if ties:
        near = cand >= value[:, beams - 1:beams].double() - 1e-3
        assert torch.equal((cand + 4e-6).float()[near], (cand - 4e-6).float()[near])
    else:
        assert (cand.sort(1, descending=True).values[:, :beams + 1].diff(dim=1) < -1e-3).all()
    got = beam_select(logits.to(device), scores.to(device), None if finished is None else finished.to(device), eos)
    assert got[1].cpu().tolist() == (at[:, :beams] // vocab).tolist()
    assert got[2].cpu().tolist() == (at[:, :beams] % vocab).tolist()
    torch.testing.assert_close(got[0].cpu(), value[:, :beams], rtol=0, atol=0 if ties else 1e-4)


@pytest.mark.parametrize("device", DEVICES)
def test_equal_scores_of_unequal_logits_go_by_index(device):
    """A large score rounds neighbouring logits to one candidate score: the lowest tokens win, also over larger
    logits, and also where more candidates tie than there are beams."""
    e = 2.0 ** -23
    for vocab in (64, 5000, 100018):
        logits = torch.full((1, 2, vocab), -50.0)
        logits[0, 0, [9, 7, 3]] = torch.tensor([1 + 2 * e, 1 + e, 1.0])
        logits[0, 1] = logits[0, 0]
        _check_order(device, logits, torch.tensor([[-1000.0, NINF]]))          # 3 before 7, 9 left out
        _check_order(device, logits, torch.tensor([[NINF, -1000.0]]))
        logits[0, 0, [9, 7, 3]] = torch.tensor([1 + e, 1.0, 1.0])
        _check_order(device, logits, torch.tensor([[-1000.0, NINF]]))          # a larger logit behind two equal ones
        logits[0, 0, [9, 7, 3]] = torch.tensor([1.0, 1.0, 1 + e])
        _check_order(device, logits, torch.tensor([[-1000.0, NINF]]))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("beams", [1, 4, 8, 11, 32])
def test_many_candidates_tie_at_the_cut(device, beams):
    """60 tokens per row, close together, whose logits differ in the last bits; rows and beams tie as well."""
    g = torch.Generator().manual_seed(beams)
    vocab, n = 50257, 60
    logits = torch.full((3, beams, vocab), -60.0)
    for b in range(3):
        for k in range(beams):
            at = torch.randperm(1500, generator=g)[:n] + 12000 * b + 300
            logits[b, k, at] = 1.0 + torch.randperm(n, generator=g) * 2.0 ** -23
    scores = torch.full((3, beams), -1000.0)
    scores[1, 0] = -998.0                                      # one beam above the others
    scores[2, : beams // 2] = -1003.0                          # the first half below
    _check_order(device, logits, scores)
    finished = torch.zeros(3, beams, dtype=torch.bool)
    finished[:, beams // 2] = True
    scores[0, beams // 2] = (-1000.0 - torch.log(torch.tensor(float(n)))).item()     # ties with the live beams
    _check_order(device, logits, scores, finished, 17)


@pytest.mark.parametrize("device", DEVICES)
def test_equal_scores_of_bf16_logits(device):
    logits = torch.full((1, 2, 9000), -50.0)
    logits[0, 0, [900, 700, 300]] = torch.tensor([1 + 2.0 ** -6, 1 + 2.0 ** -7, 1.0])
    logits[0, 0, 8000:8100] = 0.75
    _check_order(device, logits.bfloat16(), torch.tensor([[-2.0 ** 20, NINF]]))
    _check_order(device, logits.bfloat16(), torch.tensor([[-1.0, NINF]]), ties=False)


@pytest.mark.parametrize("device", DEVICES)
def test_ties_below_the_cut_change_nothing(device):
    g = torch.Generator().manual_seed(3)
    logits = torch.randn(2, 4, 30000, generator=g)
    logits[:, :, 100::1000] = 12.0 + torch.arange(30) / 16.0   # the best candidates well apart
    _check_order(device, logits, torch.tensor([[0.0, -0.3, -0.61, -0.92], [-100.0, NINF, NINF, NINF]]),
                 ties=False)


@pytest.mark.parametrize("device", DEVICES)
def test_an_infinite_score_swallows_every_logit(device):
    """All candidates of the beam tie at the largest finite float."""
    from ops.beam import beam_select
    g = torch.Generator().manual_seed(0)
    logits = torch.randn(1, 3, 30000, generator=g).to(device)
    _, parent, token, _ = beam_select(logits, torch.tensor([[-1.0, float("inf"), -2.0]], device=device))
    assert parent.tolist() == [[1, 1, 1]] and token.tolist() == [[0, 1, 2]]
