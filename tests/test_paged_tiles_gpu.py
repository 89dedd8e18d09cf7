"""Every row tile of the paged attention, with row tiles that are cut and joined in either way, against 64 bits.

The bound is that of the other attention tests: weights rounded to bf16 (2^-9 each) and the result once more, allowed
twice.  A one-token batch of 17 to 32 heads takes the 32-row tile, which the other tests do not reach.
"""
import pytest
import torch

from test_paged_gpu import check, make, oracle, status  # noqa: F401

pytestmark = pytest.mark.gpu

# few long sequences: one or two row tiles, cut over most CTAs (joined a row per CTA);
# many of mixed length: as many row tiles as CTAs or more (joined a row per warp)
FEW = [(1, 9000)]
MANY = [(1, 1 + 97 * (b % 23)) for b in range(200)]
EDGES = [(1, c) for c in (1, 2, 63, 64, 65, 127, 128, 129, 191, 192, 193, 700)]
SPARSE = [(1, 300), (1, 0), (1, 1), (1, 640), (1, 64)]       # a row that sees nothing between others


@pytest.mark.parametrize("seqs", [FEW, MANY, EDGES, SPARSE], ids=["few", "many", "edges", "sparse"])
@pytest.mark.parametrize("heads,rank,rope", [(17, 64, 16), (24, 64, 16), (32, 64, 16), (24, 192, 24), (24, 512, 64),
                                             (32, 512, 64), (31, 136, 8), (32, 8, 8)])
def test_one_token_batches_of_17_to_32_heads(heads, rank, rope, seqs):
    from ops.paged import paged_latent_attention
    args = make(seqs, heads, rank, rope, [16, 64, 128][heads % 3], seed=heads + rank)
    scale = (rank + rope) ** -0.5
    check(paged_latent_attention(*args, rank, scale), *oracle(*args, rank, scale))


@pytest.mark.parametrize("gain", [0.0, 30.0])
@pytest.mark.parametrize("heads,rank", [(24, 192), (32, 512)])
def test_flat_and_peaked_scores_of_the_32_row_tile(heads, rank, gain):
    from ops.paged import paged_latent_attention
    args = make([(1, 3000), (1, 1500), (1, 64)], heads, rank, 24, 64, seed=7, q_gain=gain)
    check(paged_latent_attention(*args, rank, 0.1), *oracle(*args, rank, 0.1))


@pytest.mark.parametrize("seqs", [[(2, 9000)], [(1 + b % 3, 3 + 61 * (b % 19)) for b in range(160)]], ids=["few", "many"])
@pytest.mark.parametrize("heads,rank,rope", [(4, 64, 16), (16, 64, 16), (12, 192, 24), (16, 512, 64), (40, 192, 24),
                                             (128, 192, 24)])
def test_cut_row_tiles_of_every_width(heads, rank, rope, seqs):
    from ops.paged import paged_latent_attention
    args = make(seqs, heads, rank, rope, 32, seed=heads)
    scale = (rank + rope) ** -0.5
    check(paged_latent_attention(*args, rank, scale), *oracle(*args, rank, scale))
