"""Beam selection and reordering on a B200 against plain 64-bit / exact implementations.

Scores: the kernel and the oracle agree to a few fp32 roundings of numbers of
the size of score + |logit| + log-sum-exp; the tests allow 8 * 2^-24 of that
plus 2^-20 for the log-sum-exp of a row.  Where two candidates are closer than
that their order is not defined by the data, so the integer results are
compared where candidates are exactly equal or clearly apart, and otherwise
through the scores that they select.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def status():
    from ops._ext import check_status, native
    native().status_reset()
    yield
    check_status()


def oracle(logits, scores, finished, eos):
    """(candidates [B, K * V] in 64 bits)."""
    x = torch.where(torch.isnan(logits), float("-inf"), logits.double()).clamp(max=torch.finfo(torch.float32).max)
    dead = (x == float("-inf")).all(-1, keepdim=True)
    lp = torch.where(dead, float("-inf"), torch.log_softmax(torch.where(dead, 0.0, x), -1))
    if finished is not None:
        frozen = torch.full((x.shape[-1],), float("-inf"), device=x.device, dtype=torch.float64)
        frozen[eos] = 0.0
        lp = torch.where(finished[..., None], frozen, lp)
    return (scores.double()[..., None] + lp).flatten(1)


def check(logits, scores, finished, eos, order=True):
    from ops.beam import beam_select
    got, parent, token, done = beam_select(logits, scores, finished, eos)
    bsz, beams, vocab = logits.shape
    cand = oracle(logits, scores, finished, eos)
    want, at = torch.sort(cand, dim=1, descending=True, stable=True)
    want, at = want[:, :beams], at[:, :beams]
    size = scores.abs().nan_to_num(posinf=0).max() + torch.nan_to_num(logits.float(), 0, 0, 0).abs().max() + 12
    tol = 8 * 2.0 ** -24 * size.item() + 2.0 ** -20
    fine = torch.isfinite(want)
    assert torch.equal(fine, torch.isfinite(got)) and (got[~fine] == float("-inf")).all()
    assert ((got.double() - want)[fine].abs() <= tol).all()
    flat = parent.long() * vocab + token.long()
    assert flat.sort(1).values.diff(dim=1).ne(0).all(), "a candidate was chosen twice"
    picked = cand.gather(1, flat)
    assert torch.equal(torch.isfinite(picked), fine) and ((picked - want)[fine].abs() <= 2 * tol).all()
    if order:
        assert torch.equal(flat, at)
    stop = token == eos
    if finished is not None:
        stop = stop | finished.gather(1, parent.long())
    assert torch.equal(done, stop)
    assert parent.dtype == torch.int32 and token.dtype == torch.int32


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("bsz,beams,vocab", [(1, 1, 1), (1, 4, 100018), (3, 5, 50257), (2, 32, 4096), (40, 2, 1000),
                                             (2, 8, 8193), (1, 3, 3), (5, 16, 2048), (1, 32, 33)])
def test_select_matches_64_bits(bsz, beams, vocab, dtype):
    g = torch.Generator(device="cuda").manual_seed(beams + vocab)
    logits = (torch.randn(bsz, beams, vocab, device="cuda", generator=g) * 3).to(dtype)
    scores = -10 * torch.rand(bsz, beams, device="cuda", generator=g)
    check(logits, scores, None, -1, order=False)
    fin = torch.rand(bsz, beams, device="cuda", generator=g) < 0.4
    check(logits, scores, fin, vocab // 2, order=False)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
def test_select_ties_go_to_the_lowest_index(dtype):
    """Equal rows with whole logits: equal candidates within a beam and across beams are equal in any arithmetic."""
    g = torch.Generator(device="cuda").manual_seed(0)
    for vocab in (100, 9000, 30000):
        base = torch.randint(-3, 4, (vocab,), device="cuda", generator=g).float()
        rows = base.expand(2, 4, vocab).contiguous()
        scores = torch.tensor([[0.0, 0.0, -1.0, 0.0], [-2.0, -1.0, -1.0, -1.0]], device="cuda")
        check(rows.to(dtype), scores, None, -1, order=True)
    check(torch.zeros(1, 6, 20000, device="cuda", dtype=dtype), torch.zeros(1, 6, device="cuda"), None, 5)


def test_select_masks_and_special_values():
    g = torch.Generator(device="cuda").manual_seed(2)
    ninf = float("-inf")
    logits = torch.randn(6, 3, 10000, device="cuda", generator=g)
    scores = torch.tensor([[0.0, ninf, ninf]] * 6, device="cuda")     # first step: one beam holds the prompt
    check(logits, scores, None, -1)
    one = torch.full((1, 3, 10000), ninf, device="cuda")              # every token banned
    check(one, torch.zeros(1, 3, device="cuda"), None, -1)
    one[0, 1, 77] = -4.0                                              # a single token left
    check(one, torch.zeros(1, 3, device="cuda"), None, -1)
    one[0, 2, 9999] = torch.finfo(torch.float32).min                  # masked by the type's lowest value
    check(one, torch.zeros(1, 3, device="cuda"), None, -1)
    bad = logits[:1].clone()
    bad[0, 0, 5], bad[0, 1, 8], bad[0, 2, 11] = float("nan"), ninf, 1e30
    check(bad, torch.zeros(1, 3, device="cuda"), None, -1)
    huge = logits[:1].clone()
    huge[0, 1, 3] = float("inf")
    check(huge, torch.zeros(1, 3, device="cuda"), None, -1)
    fin = torch.ones(1, 3, dtype=torch.bool, device="cuda")
    check(logits[:1], torch.tensor([[-1.0, -2.0, -3.0]], device="cuda"), fin, 4)
    check(torch.full_like(logits[:1], float("nan")), torch.tensor([[-1.0, -2.0, -3.0]], device="cuda"), fin, 0)
    check(logits[:1], torch.full((1, 3), ninf, device="cuda"), None, -1)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
def test_select_strided_and_unaligned_rows(dtype):
    from ops.beam import beam_select
    g = torch.Generator(device="cuda").manual_seed(3)
    buf = torch.randn(3, 4, 2, 5011, device="cuda", generator=g).to(dtype)
    view = buf[:, :, 1, 3:5006]
    scores = -torch.rand(3, 4, device="cuda", generator=g)
    got = beam_select(view, scores)
    want = beam_select(view.contiguous(), scores)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    check(view, scores, None, -1, order=False)


def test_select_refusals():
    from ops.beam import beam_select
    x, s = torch.zeros(2, 3, 10, device="cuda"), torch.zeros(2, 3, device="cuda")

    def refused(match, *a):
        with pytest.raises(RuntimeError, match=match):
            beam_select(*a)
    refused("logits", x.half(), s)
    refused("logits", x[..., ::2], s)
    refused("scores", x, s[:, :2])
    refused("scores", x, s.double())
    refused("beams", x[..., :2].contiguous(), s)
    refused("beams", torch.zeros(1, 33, 64, device="cuda"), torch.zeros(1, 33, device="cuda"))
    refused("finished", x, s, torch.zeros(2, 3, device="cuda"), 1)
    refused("end token", x, s, torch.zeros(2, 3, dtype=torch.bool, device="cuda"), -1)
    assert all(t.shape == (0, 3) for t in beam_select(x[:0], s[:0]))


@pytest.mark.parametrize("layers,beams,page,width,lens", [(1, 1, 8, 32, [5]), (3, 4, 16, 216, [37, 16, 0]),
                                                        (2, 32, 64, 576, [130]), (5, 8, 128, 80, [127, 128, 129]),
                                                        (2, 7, 32, 216, [64, 65])])
def test_reorder_equals_the_plain_copy(layers, beams, page, width, lens):
    from ops.beam import beam_reorder
    bsz, cols = len(lens), max(lens) // page + 2
    g = torch.Generator().manual_seed(beams)
    pool = bsz * beams * cols
    table = torch.randperm(pool, generator=g).view(bsz * beams, cols).int()
    pages = torch.randn(layers, pool, page, width, generator=g).to(torch.bfloat16)
    n = torch.tensor(lens, dtype=torch.int32)
    cases = [torch.randint(0, beams, (bsz, beams), generator=g), torch.zeros(bsz, beams, dtype=torch.long),
             torch.arange(beams).expand(bsz, beams), torch.arange(beams).flip(0).expand(bsz, beams)]
    for par in cases:
        par = par.int().contiguous()
        want_pages = pages.clone()
        want = beam_reorder(want_pages, table, par, n)
        # what the plain form promises: each new beam reads its parent's rows
        for b, length in enumerate(lens):
            for i in range(beams):
                for pos in {0, length // 2, length - 1} if length else ():
                    old = pages[:, table[b * beams + par[b, i], pos // page], pos % page]
                    assert torch.equal(want_pages[:, want[b * beams + i, pos // page], pos % page], old)
        gp = pages.cuda()
        got = beam_reorder(gp, table.cuda(), par.cuda(), n.cuda())
        assert torch.equal(got.cpu(), want) and torch.equal(gp.cpu(), want_pages)
        here = [got.view(bsz, beams, cols)[b, :, lens[b] // page].tolist() for b in range(bsz)]
        assert all(len(set(h)) == beams for h in here)


def test_reorder_strided_layers_and_bad_input():
    from ops._ext import check_status
    from ops.beam import beam_reorder
    g = torch.Generator(device="cuda").manual_seed(5)
    buf = torch.randn(8, 3, 16, 64, device="cuda", generator=g).to(torch.bfloat16)    # [pool, layers, page, width]
    pages = buf.transpose(0, 1)
    table = torch.arange(8, dtype=torch.int32, device="cuda").view(4, 2)
    par, n = torch.tensor([[1, 1, 2, 1]], dtype=torch.int32, device="cuda"), torch.tensor([21], dtype=torch.int32, device="cuda")
    plain = pages.cpu().clone()
    want = beam_reorder(plain, table.cpu(), par.cpu(), n.cpu())
    assert torch.equal(beam_reorder(pages, table, par, n).cpu(), want)
    assert torch.equal(pages.cpu(), plain)
    before = pages.clone()
    beam_reorder(pages, table + 100, par, n)
    with pytest.raises(RuntimeError, match="index bounds check"):
        check_status()
    beam_reorder(pages, table, par + 50, n)
    with pytest.raises(RuntimeError, match="index bounds check"):
        check_status()
    assert torch.equal(pages, before)
    for match, a in [("int32", (pages, table, par.long(), n)), ("B \\* K", (pages, table[:3], par, n)),
                     ("seq_lens", (pages, table, par, n.long())), ("contiguous pages", (pages[..., :32], table, par, n))]:
        with pytest.raises(RuntimeError, match=match):
            beam_reorder(*a)
