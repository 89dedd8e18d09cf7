"""Metadata of the paged path that is out of range: skipped and reported, never read or written."""
import pytest
import torch


def _i32(x, device="cpu"):
    return torch.tensor(x, dtype=torch.int32, device=device)


@pytest.fixture()
def reported():
    """``reported()`` checks that a bounds error was recorded, and clears it."""
    from ops._ext import check_status, native
    native().status_reset()

    def seen():
        with pytest.raises(RuntimeError, match="index bounds check"):
            check_status()
    yield seen
    check_status()


@pytest.mark.gpu
def test_rotation_skips_positions_outside_its_tables(reported):
    from ops._ext import native
    from ops.rope import rope_cos_sin
    C = native()
    cos, sin = rope_cos_sin(20, 16, 10000.0, "cuda")
    x = torch.randn(7, 3, 40, device="cuda").bfloat16()
    pos = _i32([0, 19, 20, -1, 5, 1 << 30, -(1 << 31)], "cuda")
    y = x.clone()
    C.rope_inplace(y, 24, 8, cos, sin, pos, 1, 0, False)
    reported()
    good = [0, 1, 4]
    want = x[good].clone()
    C.rope_inplace(want, 24, 8, cos, sin, pos[good].contiguous(), 1, 0, False)
    assert torch.equal(y[good], want) and not torch.equal(want, x[good])
    bad = [2, 3, 5, 6]
    assert torch.equal(y[bad], x[bad])
    for match, a in [("tables", (x, 24, 8, cos[:, :4], sin[:, :4], pos, 1, 0, False)),
                     ("one position per token", (x, 24, 8, cos, sin, pos[:3], 1, 0, False)),
                     ("one position per token", (x, 24, 8, cos, sin, pos.long(), 1, 0, False))]:
        with pytest.raises(RuntimeError, match=match):
            C.rope_inplace(*a)


@pytest.mark.gpu
@pytest.mark.parametrize("heads,rank", [(4, 64), (16, 512), (12, 192)])
@pytest.mark.parametrize("cu", [[2, 5, 8], [0, 3, 7], [3, 6, 10], [0, 12, 10], [4, 2, 10]], ids=str)
def test_attention_gives_zeros_to_tokens_of_no_sequence(cu, heads, rank, reported):
    """Offsets that leave tokens out: those rows are zeros, the tokens of intact sequences get their result."""
    from ops.paged import paged_latent_attention
    g = torch.Generator(device="cuda").manual_seed(rank)
    width, total = rank + 16, 10
    pages = torch.randn(6, 64, width, device="cuda", generator=g).bfloat16()
    table = _i32([[0, 1, 2], [3, 4, 5]], "cuda")
    q = torch.randn(total, heads, width, device="cuda", generator=g).bfloat16()
    lens = _i32([150, 90], "cuda")
    del_me = torch.full((total, heads, rank), float("nan"), device="cuda", dtype=torch.bfloat16)
    del del_me                                               # the result is likely to get this memory
    out = paged_latent_attention(q, pages, table, _i32(cu, "cuda"), lens, rank, 0.1)
    reported()
    held = torch.zeros(total, dtype=torch.bool)
    for b in range(2):
        lo, hi = cu[b], cu[b + 1]
        if lo < hi <= total:
            held[lo:hi] = True
            want = paged_latent_attention(q[lo:hi].contiguous(), pages, table[b:b + 1], _i32([0, hi - lo], "cuda"),
                                          lens[b:b + 1], rank, 0.1)
            torch.testing.assert_close(out[lo:hi].float(), want.float(), rtol=2.0 ** -6, atol=1e-3)
    assert (out[~held.cuda()] == 0).all()
