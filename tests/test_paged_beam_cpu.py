"""Paged cache and beam operators on the CPU: the formulas against the dense cache path and brute force."""
import math

import pytest
import torch


def _paged_setup(small_cfg, seqs, page=8):
    from models.mla import MultiHeadLatentAttention
    torch.manual_seed(0)
    attn = MultiHeadLatentAttention(small_cfg)
    cols = max(-(-c // page) for _, c in seqs)
    table = torch.randperm(len(seqs) * cols).view(len(seqs), cols).int()
    pages = torch.zeros(len(seqs) * cols, page, attn.kv_lora_rank + attn.qk_rope_head_dim)
    return attn, pages, table


def test_paged_attention_equals_dense_cache(small_cfg):
    """Append + absorbed paged attention, chunk by chunk, equals the dense-cache layer."""
    from ops.attention import mla_absorbed
    from ops.paged import latent_cache_append, paged_latent_attention
    from ops.rope import apply_rope_complex, rope_cos_sin, rope_table
    attn, pages, table = _paged_setup(small_cfg, [(0, 30), (0, 21)])
    rank, dr, heads = attn.kv_lora_rank, attn.qk_rope_head_dim, attn.n_heads
    cos, sin = rope_cos_sin(64, dr, 10000.0)
    freqs = rope_table(64, dr, 10000.0)
    w_k, w_v = attn._wkv_b_split()
    x = [torch.randn(1, 30, attn.dim), torch.randn(1, 21, attn.dim)]
    done = [0, 0]
    for take in ([12, 1], [1, 20], [17, 0]):
        lens = torch.tensor([done[b] + take[b] for b in range(2)], dtype=torch.int32)
        cu = torch.tensor([0, take[0], take[0] + take[1]], dtype=torch.int32)
        xs = [x[b][:, done[b]:done[b] + take[b]] for b in range(2)]
        kv_a = torch.cat([attn.wkv_a(v)[0] for v in xs])
        latent_cache_append(pages, kv_a.detach(), attn.kv_norm.weight.detach(), cos, sin, table, cu, lens)
        q = []
        for b in range(2):
            if take[b] == 0:
                continue
            qn, qp = attn._queries(xs[b])
            qp = apply_rope_complex(qp, freqs[done[b]:done[b] + take[b]])
            q.append(torch.cat([torch.einsum("bshd,hdr->bshr", qn, w_k), qp], -1)[0])
        out = paged_latent_attention(torch.cat(q).detach(), pages, table, cu, lens, rank, attn.softmax_scale)
        for b in range(2):
            if take[b] == 0:
                continue
            got = torch.einsum("thr,hdr->thd", out[cu[b]:cu[b + 1]], w_v).reshape(take[b], -1)
            ref = _dense(attn, x[b][:, :done[b] + take[b]])[0, done[b]:]
            torch.testing.assert_close(attn.wo(got), ref, rtol=1e-4, atol=1e-5)
        done = [done[b] + take[b] for b in range(2)]


def _dense(attn, x):
    n = x.shape[1]
    mask = torch.full((n, n), float("-inf")).triu(1).view(1, 1, n, n)
    return attn(x, 0, mask, use_cache=False)


def test_attention_empty_rows():
    from ops.paged import paged_latent_attention
    pages = torch.randn(4, 8, 24)
    table = torch.arange(4, dtype=torch.int32).view(2, 2)
    q = torch.randn(5, 3, 24)
    out = paged_latent_attention(q, pages, table, torch.tensor([0, 5, 5], dtype=torch.int32),
                                 torch.tensor([2, 0], dtype=torch.int32), 16, 0.2)
    assert (out[:3] == 0).all() and torch.isfinite(out).all() and (out[3:] != 0).any()
    with pytest.raises(IndexError):
        from ops.paged import latent_cache_append
        latent_cache_append(pages, torch.randn(5, 24), torch.ones(16), torch.ones(9, 4), torch.ones(9, 4), table,
                            torch.tensor([0, 1, 2], dtype=torch.int32), torch.tensor([1, 1], dtype=torch.int32))


def test_select_against_enumeration():
    from ops.beam import beam_select
    torch.manual_seed(0)
    logits, scores = torch.randn(2, 3, 7), -torch.rand(2, 3)
    fin = torch.tensor([[False, True, False], [False, False, False]])
    got, parent, token, done = beam_select(logits, scores, fin, 4)
    for b in range(2):
        cand = []
        for k in range(3):
            lp = torch.log_softmax(logits[b, k].double(), -1)
            for v in range(7):
                if fin[b, k]:
                    s = float(scores[b, k]) if v == 4 else -math.inf
                else:
                    s = float(scores[b, k]) + float(lp[v])
                cand.append((-s, k, v))
        cand.sort()
        for i in range(3):
            assert (int(parent[b, i]), int(token[b, i])) == cand[i][1:]
            assert abs(float(got[b, i]) + cand[i][0]) < 1e-5
            assert bool(done[b, i]) == (cand[i][2] == 4 or bool(fin[b, cand[i][1]]))


def test_reorder_shares_full_pages_and_copies_the_open_one():
    from ops.beam import beam_reorder
    pages = torch.arange(12.0).view(1, 12, 1, 1).expand(2, 12, 4, 8).clone()
    table = torch.arange(12, dtype=torch.int32).view(3, 4)
    out = beam_reorder(pages, table, torch.tensor([[2, 2, 1]], dtype=torch.int32), torch.tensor([6], dtype=torch.int32))
    assert out.tolist() == [[8, 9, 2, 3], [8, 1, 6, 7], [4, 5, 10, 11]]
    assert (pages[:, 1, :2] == 9).all() and (pages[:, 1, 2:] == 1).all()
    again = beam_reorder(pages, table, torch.tensor([[0, 0, 0]], dtype=torch.int32), torch.tensor([8], dtype=torch.int32))
    assert again.tolist() == [[0, 1, 2, 3], [0, 1, 6, 7], [0, 1, 10, 11]]
