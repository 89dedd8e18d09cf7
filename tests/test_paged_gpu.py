"""Paged latent cache on a B200: append and attention against a plain 64-bit implementation.

Error bound of the attention: its weights are rounded to bf16 (relative 2^-9
each), so a result moves by at most 2^-9 * sum_j p_j |v_j|, and its own
rounding to bf16 adds 2^-9 |out|.  The scores are fp32 sums of exact products
of bf16 values; their error moves the weights by far less than that.  The
tests allow twice the sum of the two.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

F64 = torch.float64
BF16 = torch.bfloat16


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def make(seqs, heads, rank, rope, page, seed=0, spare=3, hole=float("nan"), q_gain=1.0):
    """Queries, pool, table, offsets and lengths for ``seqs`` = [(new, cached length)]; rows that no
    sequence holds are filled with ``hole``."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    width = rank + rope
    cols = max(1, max(-(-max(c, 0) // page) for _, c in seqs)) + 1
    need = [-(-max(c, 0) // page) for _, c in seqs]
    pool = sum(need) + spare
    order = torch.randperm(pool, generator=torch.Generator().manual_seed(seed)).tolist()
    pages = torch.full((pool, page, width), hole, device="cuda", dtype=BF16)
    table = torch.zeros(len(seqs), cols, dtype=torch.int32)
    at = 0
    for b, (_, c) in enumerate(seqs):
        for j in range(need[b]):
            pg = order[at]
            at += 1
            table[b, j] = pg
            rows = min(page, c - j * page)
            pages[pg, :rows] = torch.randn(rows, width, device="cuda", generator=g).to(BF16)
    total = sum(n for n, _ in seqs)
    q = (torch.randn(total, heads, width, device="cuda", generator=g) * q_gain).to(BF16)
    cu = [0]
    for n, _ in seqs:
        cu.append(cu[-1] + n)
    return q, pages, table.cuda(), _i32(cu), _i32([c for _, c in seqs])


def oracle(q, pages, table, cu, lens, rank, scale):
    """(out, sum_j p_j |v_j|) in 64 bits."""
    out = torch.zeros(q.shape[0], q.shape[1], rank, dtype=F64, device=q.device)
    size = torch.zeros_like(out)
    page = pages.shape[1]
    cu, lens = cu.tolist(), lens.tolist()
    for b, n in enumerate(lens):
        for t in range(cu[b], cu[b + 1]):
            pos = n - cu[b + 1] + t
            if pos < 0:
                continue
            key = torch.arange(pos + 1, device=q.device)
            kv = pages[table[b].long()[key // page], key % page].to(F64)
            p = torch.softmax(q[t].to(F64) @ kv.t() * scale, dim=-1)
            out[t] = p @ kv[:, :rank]
            size[t] = p @ kv[:, :rank].abs()
    return out, size


def check(got, want, size):
    err = (got.to(F64) - want).abs()
    bound = 2.0 ** -8 * (want.abs() + size) + 1e-6
    worst = ((err - bound).max().item() if err.numel() else -1.0)
    assert worst <= 0, f"exceeds the bound by {worst:.3g} (largest error {err.max().item():.3g})"


@pytest.fixture(autouse=True)
def status():
    from ops._ext import check_status, native
    native().status_reset()
    yield
    check_status()


SEQS = {
    "one": [(1, 1)],
    "tile_edges": [(1, 127), (1, 128), (1, 129), (1, 255), (1, 256), (1, 257)],
    "prompt": [(300, 300)],
    "chunk_on_cache": [(130, 391), (17, 1000)],
    "mixed": [(1, 77), (0, 50), (9, 9), (0, 0), (64, 640), (1, 1), (2, 513)],
    "row_sees_nothing": [(5, 2), (3, 3), (4, 0)],
}
SHAPES = [(12, 192, 24), (16, 512, 64), (4, 64, 16), (4, 16, 16), (5, 136, 8), (1, 320, 40), (128, 512, 64)]


@pytest.mark.parametrize("seqs", list(SEQS), ids=list(SEQS))
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "h%d_r%d_d%d" % s)
def test_attention_matches_64_bits(shape, seqs):
    from ops.paged import paged_latent_attention
    heads, rank, rope = shape
    page = [8, 16, 32, 64, 128, 256][(heads + len(seqs)) % 6]
    args = make(SEQS[seqs], heads, rank, rope, page, seed=heads + rank)
    scale = (rank + rope) ** -0.5
    got = paged_latent_attention(*args, rank, scale)
    assert got.shape == (args[0].shape[0], heads, rank) and got.dtype == BF16
    check(got, *oracle(*args, rank, scale))


@pytest.mark.parametrize("page", [8, 16, 32, 64, 128, 256])
def test_attention_page_sizes(page):
    from ops.paged import paged_latent_attention
    args = make([(3, 700), (70, 333), (1, 2049)], 12, 192, 24, page, seed=page)
    check(paged_latent_attention(*args, 192, 0.11), *oracle(*args, 192, 0.11))


@pytest.mark.parametrize("gain", [0.0, 1.0, 30.0])
def test_attention_flat_and_peaked_scores(gain):
    """Equal scores (q = 0), ordinary ones, and scores whose maximum moves by hundreds between tiles."""
    from ops.paged import paged_latent_attention
    args = make([(1, 3000), (20, 1500)], 16, 512, 64, 64, seed=7, q_gain=gain)
    check(paged_latent_attention(*args, 512, 0.07), *oracle(*args, 512, 0.07))


@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_attention_growing_scores(sign):
    """The running maximum moves at every tile (or never after the first): keys scaled along the sequence."""
    from ops.paged import paged_latent_attention
    q, pages, table, cu, lens = make([(1, 2000), (33, 1300)], 12, 192, 24, 64, seed=8)
    q = q.abs() * sign
    page = pages.shape[1]
    for b, n in enumerate(lens.tolist()):
        key = torch.arange(n, device="cuda")
        at = (table[b].long()[key // page], key % page)
        pages[at] = (pages[at].float().abs() * (0.2 + key[:, None] / 300.0)).to(BF16)
    check(paged_latent_attention(q, pages, table, cu, lens, 192, 0.05),
          *oracle(q, pages, table, cu, lens, 192, 0.05))


def test_attention_strided_pool_and_table():
    from ops.paged import paged_latent_attention
    q, pages, table, cu, lens = make([(7, 300), (1, 90)], 16, 512, 64, 32, seed=9)
    pool, page, width = pages.shape
    layered = torch.full((pool, 2, page, width + 24), float("nan"), device="cuda", dtype=BF16)
    view = layered[:, 1, :, 8:8 + width]
    view.copy_(pages)
    wide = torch.zeros(table.shape[0], table.shape[1] + 5, dtype=torch.int32, device="cuda")
    wide[:, 2:2 + table.shape[1]] = table
    want = paged_latent_attention(q, pages, table, cu, lens, 512, 0.07)
    got = paged_latent_attention(q, view, wide[:, 2:2 + table.shape[1]], cu, lens, 512, 0.07)
    assert torch.equal(got, want)
    qt = q.transpose(0, 1).contiguous().transpose(0, 1)     # heads outermost in memory
    assert torch.equal(paged_latent_attention(qt, pages, table, cu, lens, 512, 0.07), want)


@pytest.mark.parametrize("heads,new", [(4, 1), (40, 1), (12, 12)])
def test_attention_of_more_sequences_than_threads(heads, new):
    """1,300 sequences of 0 to ``new`` tokens over 0 to 200 rows: the search for a share takes several rounds."""
    from ops.paged import paged_latent_attention
    g = torch.Generator().manual_seed(heads)
    n = torch.randint(0 if new > 1 else 1, new + 1, (1300,), generator=g).tolist()
    c = torch.randint(0, 200, (1300,), generator=g).tolist()
    args = make([(a, max(a, b)) for a, b in zip(n, c)], heads, 64, 16, 32, seed=heads)
    check(paged_latent_attention(*args, 64, 0.11), *oracle(*args, 64, 0.11))


def test_attention_is_repeatable_on_any_stream():
    from ops.paged import paged_latent_attention
    args = make([(1, 5000), (200, 900), (3, 30)], 16, 512, 64, 64, seed=10)
    first = paged_latent_attention(*args, 512, 0.07)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        others = [paged_latent_attention(*args, 512, 0.07) for _ in range(3)]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(first, o) for o in others)


def test_attention_in_a_graph_follows_lengths():
    """A captured call reads lengths and table at replay."""
    from ops.paged import paged_latent_attention
    q, pages, table, cu, lens = make([(1, 600), (1, 450)], 12, 192, 24, 64, seed=11, hole=0.0)
    n = lens.clone()
    paged_latent_attention(q, pages, table, cu, n, 192, 0.1)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = paged_latent_attention(q, pages, table, cu, n, 192, 0.1)
    for cut in (0, 200, 449):
        n.copy_(lens - cut)
        graph.replay()
        check(out, *oracle(q, pages, table, cu, n, 192, 0.1))


def test_attention_pool_past_32_bit_offsets():
    """The used pages lie past 2^32 bytes and 2^31 elements of the pool."""
    from ops.paged import latent_cache_append, paged_latent_attention
    rank, rope, page, width = 512, 64, 64, 576
    pool = (1 << 31) // (page * width) + 40
    small = make([(5, 700)], 16, rank, rope, page, seed=12)
    q, pages, table, cu, lens = small
    big = torch.empty(pool, page, width, dtype=BF16, device="cuda")
    shift = pool - pages.shape[0]
    big[shift:] = pages
    got = paged_latent_attention(q, big, table + shift, cu, lens, rank, 0.07)
    assert torch.equal(got, paged_latent_attention(q, pages, table, cu, lens, rank, 0.07))
    x = torch.randn(5, width, device="cuda").to(BF16)
    w, cos, sin = torch.rand(rank, device="cuda") + 0.5, torch.rand(700, 32, device="cuda"), torch.rand(700, 32, device="cuda")
    latent_cache_append(big, x, w, cos, sin, table + shift, cu, lens)
    latent_cache_append(pages, x, w, cos, sin, table, cu, lens)
    assert torch.equal(big[shift:].nan_to_num(), pages.nan_to_num())


def test_bad_pages_are_skipped_and_reported():
    from ops._ext import check_status
    from ops.paged import latent_cache_append, paged_latent_attention
    q, pages, table, cu, lens = make([(1, 200), (2, 100)], 12, 192, 24, 64, seed=13, hole=0.0)
    want = paged_latent_attention(q, pages, table, cu, lens, 192, 0.1)
    bad = table.clone()
    bad[0, 1] = pages.shape[0] + 5
    bad[0, 2] = -3
    got = paged_latent_attention(q, pages, bad, cu, lens, 192, 0.1)
    assert torch.equal(got[1:], want[1:]) and torch.isfinite(got).all()
    with pytest.raises(RuntimeError, match="index bounds check"):
        check_status()
    long = lens.clone()
    long[1] = 100000                                           # more rows than the table has columns for
    paged_latent_attention(q, pages, table, cu, long, 192, 0.1)
    with pytest.raises(RuntimeError, match="index bounds check"):
        check_status()
    before = pages.clone()
    x = torch.randn(3, 216, device="cuda").to(BF16)
    w, cos = torch.ones(192, device="cuda"), torch.ones(50, 12, device="cuda")   # table of 50 positions
    latent_cache_append(pages, x, w, cos, cos, table, cu, lens)
    with pytest.raises(RuntimeError, match="index bounds check"):
        check_status()
    assert torch.equal(pages, before)


@pytest.mark.parametrize("dtype", [BF16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("shape", [(192, 24), (512, 64), (16, 16), (136, 8)], ids=lambda s: "r%d_d%d" % s)
def test_append_matches_64_bits(shape, dtype):
    """bf16 results: within one rounding (2^-8 relative, two roundings' worth of slack) of the 64-bit values."""
    from ops.paged import latent_cache_append
    rank, rope = shape
    seqs = [(1, 1), (0, 40), (33, 70), (128, 128), (1, 65), (5, 300)]
    _, pages, table, cu, lens = make(seqs, 1, rank, rope, 32, seed=rank, hole=0.0)
    before = pages.clone()
    g = torch.Generator(device="cuda").manual_seed(1)
    total = int(cu[-1])
    buf = torch.randn(total, rank + rope + 16, device="cuda", generator=g).to(dtype)
    x = buf[:, 8:8 + rank + rope] * 3 if rank == 16 else buf[:, 8:8 + rank + rope]
    w = torch.rand(rank, device="cuda", generator=g) + 0.5
    ang = torch.rand(300, rope // 2, device="cuda", generator=g) * 6
    cos, sin = ang.cos(), ang.sin()
    out = latent_cache_append(pages, x, w, cos, sin, table, cu, lens)
    assert out is pages
    want = before.to(F64)
    size = want.abs()
    for b, (n, c) in enumerate(seqs):
        for i in range(n):
            pos, t = c - n + i, int(cu[b]) + i
            r = x[t].to(F64)
            lat = r[:rank] * torch.rsqrt(r[:rank].square().mean() + 1e-6) * w.to(F64)
            a, d = r[rank::2], r[rank + 1::2]
            cc, ss = cos[pos].to(F64), sin[pos].to(F64)
            row = torch.cat([lat, torch.stack([a * cc - d * ss, a * ss + d * cc], -1).flatten()])
            at = (int(table[b, pos // 32]), pos % 32)
            want[at] = row
            size[at] = torch.cat([lat.abs(), torch.stack([(a * cc).abs() + (d * ss).abs()] * 2, -1).flatten()])
    err = (pages.to(F64) - want).abs()
    assert (err <= 2.0 ** -8 * want.abs() + 2.0 ** -20 * size + 1e-30).all()


def test_append_of_a_zero_row():
    from ops.paged import latent_cache_append
    _, pages, table, cu, lens = make([(2, 5)], 1, 64, 16, 16, seed=3, hole=0.0)
    latent_cache_append(pages, torch.zeros(2, 80, device="cuda"), torch.ones(64, device="cuda"),
                        torch.ones(5, 8, device="cuda"), torch.zeros(5, 8, device="cuda"), table, cu, lens)
    assert (pages[int(table[0, 0]), 3:5] == 0).all()


def test_refusals():
    from ops.paged import latent_cache_append, paged_latent_attention
    q, pages, table, cu, lens = make([(2, 20)], 4, 64, 16, 16, seed=4)

    def refused(match, *a):
        with pytest.raises(RuntimeError, match=match):
            paged_latent_attention(*a)
    refused("bf16", q.float(), pages, table, cu, lens, 64, 0.1)
    refused("bf16", q, pages.float(), table, cu, lens, 64, 0.1)
    refused("int32", q, pages, table.long(), cu, lens, 64, 0.1)
    refused("B \\+ 1", q, pages, table, cu[:-1], lens, 64, 0.1)
    refused("seq_lens", q, pages, table, cu, lens.long(), 64, 0.1)
    refused("same width", q[..., :72].contiguous(), pages, table, cu, lens, 64, 0.1)
    refused("latent rank", q, pages, table, cu, lens, 60, 0.1)
    refused("latent rank", q, pages, table, cu, lens, 80, 0.1)
    refused("power of two", q, pages[:, :12], table, cu, lens, 64, 0.1)
    refused("16-byte", q[..., 4:76].contiguous(), pages[..., 4:76], table, cu, lens, 64, 0.1)
    refused("device", q, pages, table.cpu(), cu, lens, 64, 0.1)
    x, w, c = torch.zeros(2, 80, device="cuda"), torch.ones(64, device="cuda"), torch.ones(20, 8, device="cuda")
    with pytest.raises(RuntimeError, match="wide"):
        latent_cache_append(pages, x[:, :72], w, c, c, table, cu, lens)
    with pytest.raises(RuntimeError, match="fp32 tensor"):
        latent_cache_append(pages, x, w.to(BF16), c, c, table, cu, lens)
    with pytest.raises(RuntimeError, match="tables"):
        latent_cache_append(pages, x, w, c, c[:10], table, cu, lens)
    assert paged_latent_attention(q[:0], pages, table, cu, lens, 64, 0.1).shape == (0, 4, 64)
