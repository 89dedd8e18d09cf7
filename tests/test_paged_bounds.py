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
