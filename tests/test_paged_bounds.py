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


def test_positions_of_tokens_that_no_sequence_holds():
    """Before the first offset, past the last one, and without any sequence: no index leaves its range."""
    from ops.paged import ragged_positions, token_positions
    lens = _i32([10, 4])
    for cu, want in [([0, 3, 5], [7, 8, 9, 2, 3]), ([1, 3, 5], [-1, 8, 9, 2, 3]), ([0, 3, 4], [7, 8, 9, 3, -1]),
                     ([0, 0, 2], [2, 3, -1, -1, -1]), ([0, 9, 9], [1, 2, 3, 4, 5])]:
        seq, pos = ragged_positions(_i32(cu), lens, 5)
        assert pos.tolist() == want
        assert seq.min() >= 0 and seq.max() < 2
        if -1 in want:
            with pytest.raises(IndexError, match="tokens"):
                token_positions(_i32(cu), lens, 5)
        else:
            assert token_positions(_i32(cu), lens, 5)[1].tolist() == want
    with pytest.raises(IndexError, match="without a sequence"):
        ragged_positions(_i32([0]), _i32([]), 2)
    assert ragged_positions(_i32([0]), _i32([]), 0)[1].numel() == 0


STEP_CFG = {
    "vocab_size": 1000, "dim": 256, "n_layers": 2, "n_heads": 4, "n_dense_layers": 1,
    "n_routed_experts": 8, "n_shared_experts": 1, "n_activated_experts": 2, "inter_dim": 512,
    "moe_inter_dim": 128, "kv_lora_rank": 64, "q_lora_rank": 0, "qk_nope_head_dim": 48,
    "qk_rope_head_dim": 16, "v_head_dim": 64, "max_seq_len": 96, "rope_theta": 10000,
    "rope_factor": 1.0, "mscale": 1.0, "mtp_depth": 1, "mtp_loss_weight": 0.3,
    "attn_impl": "sdpa", "weight_tying": True,
}


@pytest.mark.gpu
def test_model_step_survives_bad_metadata(reported):
    """Offsets that leave tokens out or pass them, positions past the model's length, unknown token ids: reported,
    and the sequences that are in order get their logits."""
    from models.transformer import Transformer
    from ops.paged import PagedLatentCache, paged_step
    torch.manual_seed(0)
    model = Transformer(STEP_CFG).cuda().eval()
    g = torch.Generator(device="cuda").manual_seed(2)
    tokens = torch.randint(0, 1000, (12,), device="cuda", generator=g)
    table = torch.arange(24, dtype=torch.int32, device="cuda").view(2, 12)

    def step(cu, lens, toks=tokens):
        cache = PagedLatentCache(STEP_CFG, 24, 16, "cuda")
        cache.pages.zero_()
        return paged_step(model, toks, cache, table, _i32(cu, "cuda"), _i32(lens, "cuda")).float()

    want = step([0, 5, 12], [5, 7])
    for cu, lens in [([0, 5, 9], [5, 4]), ([0, 5, 20], [5, 15]), ([0, 5, 12], [5, 120]), ([0, 5, 12], [5, 3]),
                     ([0, 5, 12], [5, -9]), ([0, 5, 12], [5, 1 << 30])]:
        got = step(cu, lens)
        reported()
        torch.testing.assert_close(got[0], want[0], rtol=2e-2, atol=2e-2)
    got = step([3, 5, 12], [2, 7])
    reported()
    torch.testing.assert_close(got[1], want[1], rtol=2e-2, atol=2e-2)
    wrong = tokens.clone()
    wrong[6], wrong[7] = 1000, -1
    got = step([0, 5, 12], [5, 7], wrong)
    reported()
    torch.testing.assert_close(got[0], want[0], rtol=2e-2, atol=2e-2)


@pytest.mark.gpu
@pytest.mark.parametrize("length", [-1, -16, -17, -100000, -(1 << 31), 49, 64, 100000, (1 << 31) - 1])
def test_reorder_reports_lengths_outside_the_table(length, reported):
    from ops.beam import beam_reorder
    pages = torch.randn(2, 12, 16, 32, device="cuda").bfloat16()
    before = pages.clone()
    table = torch.arange(12, dtype=torch.int32, device="cuda").view(4, 3)
    out = beam_reorder(pages, table, _i32([[1, 1, 2, 1]], "cuda"), _i32([length], "cuda"))
    reported()
    assert torch.equal(pages, before)
    assert torch.equal(out, table if length < 0 else table[[1, 1, 2, 1]])


@pytest.mark.gpu
def test_select_refuses_vocabularies_whose_segments_pass_32_bits():
    from ops.beam import beam_select
    scores = torch.zeros(0, 1, device="cuda")
    for vocab in ((1 << 31) - 100, (1 << 31) - 4096):
        with pytest.raises(RuntimeError, match="2\\^31"):
            beam_select(torch.empty(0, 1, vocab, device="cuda"), scores)
    assert beam_select(torch.empty(0, 1, (1 << 31) - 4097, device="cuda"), scores)[0].shape == (0, 1)


def _empty_step(cfg, device):
    from models.transformer import Transformer
    from ops.paged import PagedLatentCache, paged_step
    torch.manual_seed(0)
    model = Transformer(cfg).to(device).eval()
    dtype = torch.bfloat16 if device == "cuda" else torch.float32
    cache = PagedLatentCache(cfg, 6, 8, device, dtype)
    cache.pages.normal_()
    before = cache.pages.clone()
    for batch in (3, 0):
        out = paged_step(model, torch.zeros(0, dtype=torch.long, device=device), cache,
                         torch.zeros(batch, 2, dtype=torch.int32, device=device), _i32([0] * (batch + 1), device),
                         _i32([4] * batch, device))
        assert out.shape == (batch, cfg["vocab_size"])
    assert torch.equal(cache.pages, before)


def test_step_without_new_tokens(small_cfg):
    """Every slot of the batch idle: one row of logits per sequence, and the cache as it was."""
    _empty_step(small_cfg, "cpu")


@pytest.mark.gpu
def test_step_without_new_tokens_on_the_kernels():
    from ops._ext import check_status
    _empty_step(STEP_CFG, "cuda")
    check_status()


def test_cpu_forms_refuse_indices_below_zero():
    """Python would count them from the end of the tensor: rows of other sequences."""
    from ops.beam import beam_reorder
    from ops.paged import latent_cache_append, paged_latent_attention
    pages = torch.randn(4, 8, 24)
    before = pages.clone()
    table = _i32([[1, 0], [2, 3]])
    w, cos = torch.ones(16), torch.ones(16, 4)

    def append(rows, tab, cu, lens, **kw):
        latent_cache_append(pages, torch.randn(rows, 24), w, kw.get("cos", cos), kw.get("cos", cos), tab, _i32(cu),
                            _i32(lens))

    with pytest.raises(IndexError, match="position"):
        append(3, table, [0, 3, 3], [1, 5])                   # positions -2, -1, 0
    with pytest.raises(IndexError, match="position"):
        append(1, table, [0, 1, 1], [12, 5], cos=torch.ones(8, 4))
    with pytest.raises(IndexError, match="page"):
        append(1, _i32([[-1, 0], [2, 3]]), [0, 1, 1], [3, 5])
    with pytest.raises(IndexError, match="page"):
        append(1, _i32([[4, 0], [2, 3]]), [0, 1, 1], [3, 5])
    with pytest.raises(IndexError):
        append(1, table, [0, 1, 1], [17, 5], cos=torch.ones(32, 4))
    with pytest.raises(IndexError, match="page"):
        paged_latent_attention(torch.randn(1, 2, 24), pages, _i32([[-3, 0], [2, 3]]), _i32([0, 1, 1]), _i32([9, 5]), 16,
                               0.2)
    stack = pages[None].clone()
    for match, par, tab, length in [("parent", [[0, -1]], table, 5), ("parent", [[0, 2]], table, 5),
                                    ("length", [[0, 0]], table, -3), ("length", [[0, 0]], table, 17),
                                    ("page", [[0, 0]], _i32([[-1, 0], [2, 3]]), 5),
                                    ("page", [[0, 0]], _i32([[1, 0], [4, 3]]), 5)]:
        with pytest.raises(IndexError, match=match):
            beam_reorder(stack, tab, _i32(par), _i32([length]))
    assert torch.equal(pages, before) and torch.equal(stack[0], before)
    assert beam_reorder(stack, table, _i32([[0, 0]]), _i32([16])).tolist() == [[1, 0], [1, 0]]


@pytest.mark.gpu
@pytest.mark.parametrize("rank,rope", [(64, 16), (16, 12)], ids=["by_16_bytes", "by_elements"])
def test_append_skips_tokens_of_no_sequence(rank, rope, reported):
    """In front of the first offset and past the last one: nothing is written, the others are."""
    from ops.paged import latent_cache_append
    width = rank + rope
    pages = torch.zeros(6, 16, 96, device="cuda", dtype=torch.bfloat16)[..., :width]
    table = _i32([[0, 1, 2], [3, 4, 5]], "cuda")
    x = torch.randn(9, width, device="cuda")
    w, cos = torch.ones(rank, device="cuda"), torch.ones(48, rope // 2, device="cuda")
    latent_cache_append(pages, x, w, cos, torch.zeros_like(cos), table, _i32([3, 5, 7], "cuda"), _i32([20, 33], "cuda"))
    reported()
    written = (pages != 0).any(-1).nonzero().tolist()
    assert written == [[1, 2], [1, 3], [4, 15], [5, 0]]        # positions 18 and 19, 31 and 32


@pytest.mark.gpu
def test_attention_reports_more_key_tiles_than_it_counts(reported):
    """2^20 rows over 2^24 cached ones (of one page): not computed, zeros and a report."""
    from ops.paged import paged_latent_attention
    q = torch.ones(256, 4096, 24, device="cuda", dtype=torch.bfloat16)
    pages = torch.ones(1, 256, 24, device="cuda", dtype=torch.bfloat16)
    table = torch.zeros(1, 1 << 16, dtype=torch.int32, device="cuda")
    out = paged_latent_attention(q, pages, table, _i32([0, 256], "cuda"), _i32([1 << 24], "cuda"), 16, 0.1)
    reported()
    assert (out == 0).all()
    out = paged_latent_attention(q[:2], pages, table, _i32([0, 2], "cuda"), _i32([1 << 16], "cuda"), 16, 0.1)
    assert (out == 1).all()


@pytest.mark.gpu
@pytest.mark.parametrize("heads,rank,new", [(12, 192, 1), (5, 64, 1), (20, 512, 1), (12, 192, 7), (16, 512, 5)])
def test_attention_of_a_sequence_ignores_its_neighbours(heads, rank, new):
    """A row tile's spare rows hold the next sequence's queries; peaked ones there change no bit of the result."""
    from ops._ext import check_status
    from ops.paged import paged_latent_attention
    g = torch.Generator(device="cuda").manual_seed(heads)
    batch, cols, page = 30, 40, 32
    width = rank + 24
    pages = torch.randn(batch * cols, page, width, device="cuda", generator=g).bfloat16()
    table = torch.randperm(batch * cols, device="cuda", generator=g).int().view(batch, cols)
    lens = torch.randint(new, cols * page, (batch,), device="cuda", generator=g).int()
    cu = _i32([new * b for b in range(batch + 1)], "cuda")
    q = torch.randn(batch, new, heads, width, device="cuda", generator=g)
    peaked = q.clone()
    peaked[1::2] *= 30.0
    want, got = [paged_latent_attention(x.bfloat16().flatten(0, 1), pages, table, cu, lens, rank, width ** -0.5)
                 for x in (q, peaked)]
    check_status()
    assert torch.equal(got.view(batch, new, heads, rank)[::2], want.view(batch, new, heads, rank)[::2])


@pytest.mark.gpu
def test_a_layout_that_tma_refuses_raises():
    """A page stride of 2^40 bytes (of a pool of one page): an exception with the driver's code, not a crash."""
    from ops.paged import paged_latent_attention
    pages = torch.zeros(64 * 80, device="cuda", dtype=torch.bfloat16).as_strided((1, 64, 80), (1 << 39, 80, 1))
    q = torch.zeros(1, 4, 80, device="cuda", dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="cuTensorMapEncodeTiled failed with code [0-9]+"):
        paged_latent_attention(q, pages, _i32([[0]], "cuda"), _i32([0, 1], "cuda"), _i32([5], "cuda"), 64, 0.1)


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_reorder_of_a_table_alone(device):
    """Pages without a layer, or without a column: the new table, and no copy."""
    from ops.beam import beam_reorder
    table = torch.arange(12, dtype=torch.int32, device=device).view(4, 3)
    for shape in ((0, 12, 16, 32), (2, 12, 16, 0)):
        pages = torch.zeros(shape, device=device, dtype=torch.bfloat16)
        out = beam_reorder(pages, table, _i32([[1, 1, 2, 1]], device), _i32([21], device))
        assert out.tolist() == [[3, 4, 2], [3, 1, 5], [6, 7, 8], [3, 10, 11]]
