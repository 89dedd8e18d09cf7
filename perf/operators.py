"""Workloads of the serving operators: paged latent cache, its attention, and beam search.

Four operators that a batch of requests goes through at every model step:

* ``append``: RMS-norm of the compressed latent, rotation of the shared key and the
  write of both into the pages of a latent cache;
* ``attend``: absorbed attention of a ragged batch of new tokens over that paged cache;
* ``select``: the choice of the next beams over (beam, token) pairs;
* ``reorder``: the new beams' block tables, and the copy of the page that is being filled.

With ``own`` false ``run`` is their plain form in elementary fp32 torch operations.
Model sizes ("412m", "14b", tiny) are those of the YAML configs of this repository.
"""
import math
import os
import random
import sys

import torch

own = False

# heads, latent rank, rotary width, query/key head width, layers, vocabulary
MODELS = {
    "tiny": dict(heads=4, rank=16, rope=16, qk=32, layers=4, vocab=50257),
    "small": dict(heads=4, rank=64, rope=16, qk=64, layers=3, vocab=4096),
    "412m": dict(heads=12, rank=192, rope=24, qk=72, layers=18, vocab=100018),
    "wide": dict(heads=8, rank=256, rope=32, qk=96, layers=12, vocab=32000),
    "14b": dict(heads=16, rank=512, rope=64, qk=192, layers=24, vocab=102400),
}


# ------------------------------------------------------------------- cases
def _attend(name, model, batch, new, ctx, page, lens_seed=1, group=1, idle=0.0):
    return {"name": name, "op": "attend", "model": model, "batch": batch, "new_lo": new[0], "new_hi": new[1],
            "ctx_lo": ctx[0], "ctx_hi": ctx[1], "page": page, "lens_seed": lens_seed, "group": group, "idle": idle}


def listed():
    return [
        # one interactive request, one token: the smallest attention call of a decode step
        _attend("attend_412m_one", "412m", 1, (1, 1), (700, 700), 64),
        # continuous batching: 64 requests, one token each, contexts spread up to the model's 4096
        _attend("attend_14b_decode", "14b", 64, (1, 1), (512, 4096), 64, lens_seed=2),
        # 8 beams of each of 6 prompts: the beams' tables share the prompt's pages
        _attend("attend_412m_beams", "412m", 48, (1, 1), (900, 2048), 16, lens_seed=3, group=8),
        # chunked prefill mixed with decodes and idle slots in one ragged batch
        _attend("attend_412m_mixed", "412m", 16, (1, 509), (509, 2048), 32, lens_seed=4, idle=0.1),
        # the largest prefill chunk: 4 prompts, 512 new tokens each on top of their cache
        _attend("attend_14b_chunk", "14b", 4, (512, 512), (3001, 4096), 64, lens_seed=5),
        # long documents: two requests, a few speculative tokens, far past the training length
        _attend("attend_14b_long", "14b", 2, (1, 3), (98304, 131071), 128, lens_seed=6),
        # a decode step's 64 new cache rows
        {"name": "append_14b_decode", "op": "append", "model": "14b", "batch": 64, "new_lo": 1, "new_hi": 1,
         "ctx_lo": 1, "ctx_hi": 512, "page": 64, "lens_seed": 7, "fp32": False},
        # prefill of ragged prompts, about 8 thousand rows
        {"name": "append_14b_prefill", "op": "append", "model": "14b", "batch": 8, "new_lo": 700, "new_hi": 1400,
         "ctx_lo": 1400, "ctx_hi": 2048, "page": 64, "lens_seed": 8, "fp32": False},
        # one prompt, four beams
        {"name": "select_one", "op": "select", "batch": 1, "beams": 4, "vocab": 100018, "fp32": False, "done": 0.0},
        # a batch of prompts with fp32 logits, some beams already finished
        {"name": "select_batch", "op": "select", "batch": 32, "beams": 8, "vocab": 102400, "fp32": True, "done": 0.1},
        # one prompt, four beams, all layers of the small model
        {"name": "reorder_one", "op": "reorder", "model": "412m", "batch": 1, "beams": 4, "page": 64, "prompt": 200,
         "step": 37},
        # a batch of prompts, all layers of the large model
        {"name": "reorder_batch", "op": "reorder", "model": "14b", "batch": 8, "beams": 8, "page": 64, "prompt": 90,
         "step": 100},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "append", "select", "reorder"])
    model = rng.choice(list(MODELS))
    if op == "attend":
        while True:
            kind = rng.choice(["decode", "verify", "chunk", "beams"])
            new = {"decode": (1, 1), "verify": (1, rng.randint(2, 9)), "beams": (1, 1)}.get(kind)
            if new is None:
                new = (1, _log_int(rng, 10, 700))
            hi = _log_int(rng, 60, 20000)
            c = _attend("", model, _log_int(rng, 1, 128), new, (max(1, hi // rng.randint(1, 9)), hi),
                        rng.choice([16, 32, 64, 128]), rng.randrange(1 << 20),
                        rng.randint(2, 8) if kind == "beams" else 1, rng.choice([0.0, 0.0, 0.2]))
            del c["name"]
            c["batch"] = max(c["batch"], c["group"])
            c["batch"] -= c["batch"] % c["group"]
            m = MODELS[model]
            rows = c["batch"] * c["new_hi"] * m["heads"]
            if rows * c["ctx_hi"] <= 1.2e8 and work(c)["flops"] <= 2.0e11 and c["batch"] * c["ctx_hi"] <= 260000:
                return c
    if op == "append":
        hi = _log_int(rng, 1, 1500)
        batch = max(1, min(_log_int(rng, 1, 256), 9000 // hi))
        return {"op": "append", "model": model, "batch": batch, "new_lo": rng.randint(1, hi), "new_hi": hi,
                "ctx_lo": hi, "ctx_hi": hi + rng.randint(0, 400), "page": rng.choice([16, 32, 64, 128]),
                "lens_seed": rng.randrange(1 << 20), "fp32": rng.random() < 0.3}
    if op == "select":
        beams = rng.randint(1, 16)
        vocab = _log_int(rng, 2000, 150000)
        return {"op": "select", "batch": max(1, min(_log_int(rng, 1, 64), int(2.6e7 / (beams * vocab)))),
                "beams": beams, "vocab": vocab, "fp32": rng.random() < 0.4, "done": rng.choice([0.0, 0.1, 0.5])}
    page = rng.choice([16, 32, 64, 128])
    beams, m = rng.randint(2, 8), MODELS[model]
    prompt, step = rng.randint(1, 300), rng.randint(1, 200)
    per = (prompt // page + 1 + beams * (step // page + 2)) * page * (m["rank"] + m["rope"]) * 2 * m["layers"]
    return {"op": "reorder", "model": model, "batch": max(1, min(_log_int(rng, 1, 32), int(2.5e8 / per))),
            "beams": beams, "page": page, "prompt": prompt, "step": step}


def _lens(case):
    """(new tokens, cached length after them) of every sequence."""
    rng = random.Random(case["lens_seed"])
    new, ctx = [], []
    for b in range(case["batch"]):
        if case.get("group", 1) > 1 and b % case["group"]:
            new.append(new[-1])             # the beams of one prompt advance together
            ctx.append(ctx[-1])
            continue
        n = rng.randint(case["new_lo"], case["new_hi"])
        if b and rng.random() < case.get("idle", 0.0):
            n = 0                           # an idle slot of the batch
        new.append(n)
        ctx.append(max(n, rng.randint(case["ctx_lo"], case["ctx_hi"])))
    return new, ctx


# ----------------------------------------------------------------- prepare
def _own_package():
    src = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "deepseek-v3-lite_b200")
    if src not in sys.path:
        sys.path.insert(0, src)


def _tables(case, dev):
    """Block tables over a shuffled pool, offsets and lengths; beams of a group share their prefix's full pages."""
    new, ctx = _lens(case)
    page, group, batch = case["page"], case.get("group", 1), case["batch"]
    cols = max(1, -(-max(ctx) // page))
    table = torch.zeros(batch, cols, dtype=torch.int64)
    used = 0
    for b in range(batch):
        n = -(-ctx[b] // page)
        lead = b - b % group
        shared = max(0, (ctx[b] * 3 // 4) // page) if group > 1 and b != lead else 0
        table[b, :shared] = table[lead, :shared]
        table[b, shared:n] = torch.arange(used, used + n - shared)
        used += n - shared
    pool = used + 2
    perm = torch.randperm(pool, generator=torch.Generator().manual_seed(case["lens_seed"]))
    cu = torch.zeros(batch + 1, dtype=torch.int32)
    cu[1:] = torch.tensor(new).cumsum(0)
    return (perm[table].to(torch.int32).to(dev), cu.to(dev), torch.tensor(ctx, dtype=torch.int32).to(dev), pool,
            new, ctx)


def _rope_tables(n, dim, dev):
    inv = 1.0 / (10000.0 ** (torch.arange(0, dim, 2, dtype=torch.float32, device=dev) / dim))
    ang = torch.outer(torch.arange(n, dtype=torch.float32, device=dev), inv)
    return torch.cos(ang).contiguous(), torch.sin(ang).contiguous()


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    randn = lambda *s: torch.randn(*s, device=dev, generator=g)  # noqa: E731
    st = {"case": case}
    op = case["op"]
    if op in ("attend", "append"):
        m = MODELS[case["model"]]
        width = m["rank"] + m["rope"]
        table, cu, lens, pool, new, ctx = _tables(case, dev)
        st.update(table=table, cu=cu, lens=lens, new_max=max(new), ctx_max=max(ctx), rank=m["rank"],
                  pages=randn(pool, case["page"], width).to(torch.bfloat16))
        if op == "attend":
            st.update(q=randn(sum(new), m["heads"], width).to(torch.bfloat16), scale=m["qk"] ** -0.5)
        else:
            kv_a = randn(sum(new), width) * 0.7
            cos, sin = _rope_tables(max(ctx), m["rope"], dev)
            st.update(kv_a=kv_a if case["fp32"] else kv_a.to(torch.bfloat16), weight=1.0 + 0.1 * randn(m["rank"]),
                      cos=cos, sin=sin)
    elif op == "select":
        b, k, v = case["batch"], case["beams"], case["vocab"]
        # a language model's logits: a broad bulk and a few likely tokens per row
        logits = 1.5 * randn(b, k, v)
        hot = torch.randint(0, v, (b, k, 24), device=dev, generator=g)
        bump = torch.rand(b, k, 24, device=dev, generator=g) * 9.0 + 4.0
        logits.scatter_(2, hot, bump)
        st.update(logits=logits if case["fp32"] else logits.to(torch.bfloat16), eos=2,
                  scores=-6.0 * torch.rand(b, k, device=dev, generator=g),
                  finished=torch.rand(b, k, device=dev, generator=g) < case["done"])
    else:
        m = MODELS[case["model"]]
        page, b, k = case["page"], case["batch"], case["beams"]
        length = case["prompt"] + case["step"]
        shared, cols = case["prompt"] // page, length // page + 2
        per_group = shared + k * (cols - shared)
        table = torch.empty(b, k, cols, dtype=torch.int64)
        base = (torch.arange(b) * per_group).view(b, 1, 1)
        table[:, :, :shared] = base + torch.arange(shared)
        table[:, :, shared:] = base + shared + torch.arange(k * (cols - shared)).view(1, k, cols - shared)
        perm = torch.randperm(b * per_group, generator=torch.Generator().manual_seed(seed))
        st.update(table=perm[table].view(b * k, cols).to(torch.int32).to(dev),
                  pages=randn(m["layers"], b * per_group, page, m["rank"] + m["rope"]).to(torch.bfloat16),
                  parents=torch.randint(0, k, (b, k), device=dev, generator=g).to(torch.int32),
                  lens=torch.full((b,), length, dtype=torch.int32, device=dev))
    return st


# --------------------------------------------------------------------- run
def run(st):
    return {"attend": _run_attend, "append": _run_append, "select": _run_select,
            "reorder": _run_reorder}[st["case"]["op"]](st)


def _positions(cu, lens, total):
    """Sequence and absolute position of every new token."""
    t = torch.arange(total, device=cu.device)
    seq = torch.searchsorted(cu[1:].long(), t, right=True)
    return seq, (lens[seq].long() - cu[seq + 1].long()) + t


def _run_attend(st):
    q, pages, table, cu, lens, rank = st["q"], st["pages"], st["table"], st["cu"], st["lens"], st["rank"]
    if own:
        _own_package()
        from ops.paged import paged_latent_attention
        return paged_latent_attention(q, pages, table, cu, lens, rank, st["scale"])
    total, heads, width = q.shape
    batch, page = table.shape[0], pages.shape[1]
    key = torch.arange(st["ctx_max"], device=q.device)
    kv = pages[table.long()[:, key // page], key % page].float()                     # [B, L, D]
    kv = torch.where((key[None, :] < lens[:, None])[..., None], kv, torch.zeros_like(kv))
    i = torch.arange(max(st["new_max"], 1), device=q.device)
    count = (cu[1:] - cu[:-1]).long()
    token = (cu[:-1].long()[:, None] + i[None, :]).clamp(max=max(total - 1, 0))      # [B, n]
    qb = q.float()[token].reshape(batch, -1, width)                                  # [B, n * H, D]
    s = torch.matmul(qb, kv.transpose(1, 2)) * st["scale"]
    pos = (lens.long() - count)[:, None] + i[None, :]
    seen = (key[None, None, :] <= pos[:, :, None]) & (key[None, None, :] < lens[:, None, None])
    s = s.view(batch, -1, heads, key.numel())
    seen = seen[:, :, None, :]
    s = torch.where(seen, s, torch.full_like(s, float("-inf")))
    top = s.amax(-1, keepdim=True)
    top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
    p = torch.exp(s - top)
    total_p = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(batch, -1, key.numel()), kv[..., :rank]).view(batch, -1, heads, rank)
    o = torch.where(total_p > 0, o / total_p, torch.zeros_like(o))
    seq, where = _positions(cu, lens, total)
    return o[seq, where - (lens.long() - count)[seq]].to(q.dtype)


def _run_append(st):
    pages, kv_a, weight, rank = st["pages"], st["kv_a"], st["weight"], st["rank"]
    if own:
        _own_package()
        from ops.paged import latent_cache_append
        return latent_cache_append(pages, kv_a, weight, st["cos"], st["sin"], st["table"], st["cu"], st["lens"])
    page = pages.shape[1]
    seq, pos = _positions(st["cu"], st["lens"], kv_a.shape[0])
    x = kv_a.float()
    lat, pe = x[:, :rank], x[:, rank:]
    lat = lat * torch.rsqrt((lat * lat).mean(-1, keepdim=True) + 1e-6) * weight
    c, s = st["cos"][pos], st["sin"][pos]
    a, b = pe[:, 0::2], pe[:, 1::2]
    pe = torch.stack([a * c - b * s, a * s + b * c], -1).flatten(1)
    pages[st["table"].long()[seq, pos // page], pos % page] = torch.cat([lat, pe], 1).to(pages.dtype)
    return pages


def _run_select(st):
    logits, scores, finished, eos = st["logits"], st["scores"], st["finished"], st["eos"]
    if own:
        _own_package()
        from ops.beam import beam_select
        return beam_select(logits, scores, finished, eos)
    batch, beams, vocab = logits.shape
    x = logits.float()
    top = x.amax(-1, keepdim=True)
    z = x - top
    logp = z - torch.log(torch.exp(z).sum(-1, keepdim=True))
    frozen = torch.full((vocab,), float("-inf"), device=x.device)
    frozen[eos] = 0.0
    logp = torch.where(finished[..., None], frozen, logp)
    cand = (scores[..., None] + logp).view(batch, -1)
    # the `beams` largest, ties to the lowest index
    least = torch.topk(cand, beams).values[:, -1:]
    above, tie = cand > least, cand == least
    take = above | (tie & (tie.cumsum(1) <= beams - above.sum(1, keepdim=True)))
    n = cand.shape[1]
    at = n - torch.topk(torch.where(take, n - torch.arange(n, device=x.device), 0), beams).values
    value, order = torch.sort(cand.gather(1, at), dim=1, descending=True, stable=True)
    at = at.gather(1, order)
    parent, token = at // vocab, at % vocab
    return value, parent.to(torch.int32), token.to(torch.int32), finished.gather(1, parent) | (token == eos)


def _run_reorder(st):
    pages, table, parents, lens = st["pages"], st["table"], st["parents"], st["lens"]
    if own:
        _own_package()
        from ops.beam import beam_reorder
        return beam_reorder(pages, table, parents, lens), pages
    batch, beams = parents.shape
    page, cols = pages.shape[2], table.shape[1]
    old = table.view(batch, beams, cols).long()
    par = parents.long()
    col, rem = (lens // page).long(), (lens % page).long()
    full = torch.arange(cols, device=table.device)[None, None, :] < col[:, None, None]
    taken = old.gather(1, par[..., None].expand(-1, -1, cols))
    out = torch.where(full, taken, old)
    # the page being filled: the first child of a beam keeps it, each further child copies it into a childless beam's
    cur = old.gather(2, col[:, None, None].expand(-1, beams, 1))[..., 0]
    same = par[:, :, None] == par[:, None, :]
    again = torch.tril(same, -1).any(2)
    dead = ~(par[:, None, :] == torch.arange(beams, device=table.device)[None, :, None]).any(2)
    spare = cur.gather(1, torch.argsort((~dead).to(torch.int32), dim=1, stable=True))
    source = cur.gather(1, par)
    target = torch.where(again, spare.gather(1, (again.cumsum(1) - 1).clamp(min=0)), source)
    part = (rem > 0)[:, None]
    target, source = torch.where(part, target, cur), torch.where(part, source, cur)
    out.scatter_(2, col[:, None, None].expand(-1, beams, 1), target[..., None])
    rows = torch.arange(page, device=table.device)[None, None, :] < rem[:, None, None]
    moved = torch.where(rows[None, ..., None], pages[:, source], pages[:, target])
    pages[:, target] = moved
    return out.view(batch * beams, cols).to(torch.int32), pages


# -------------------------------------------------------------------- work
def work(case):
    op = case["op"]
    if op == "select":
        rows = case["batch"] * case["beams"]
        return {"bytes": rows * case["vocab"] * (4 if case["fp32"] else 2) + rows * 18,
                "flops": rows * case["vocab"] * 4}
    m = MODELS[case["model"]]
    width = m["rank"] + m["rope"]
    if op == "reorder":
        k, length = case["beams"], case["prompt"] + case["step"]
        copies = case["batch"] * k * (1.0 - 1.0 / k) ** k       # expected number of childless beams
        return {"bytes": int(copies * (length % case["page"]) * width * 2 * 2 * m["layers"]
                             + case["batch"] * k * (length // case["page"] + 2) * 8), "flops": 0}
    new, ctx = _lens(case)
    total = sum(new)
    if op == "append":
        return {"bytes": total * width * ((4 if case["fp32"] else 2) + 2) + m["rank"] * 4 + total * m["rope"] * 4,
                "flops": total * (4 * m["rank"] + 3 * m["rope"])}
    group, page, keys = case["group"], case["page"], 0
    for b in range(case["batch"]):
        if new[b]:
            keys += ctx[b] - ((ctx[b] * 3 // 4) // page * page if group > 1 and b % group else 0)
    pairs = sum(n * (c - n) + n * (n + 1) // 2 for n, c in zip(new, ctx))
    return {"bytes": keys * width * 2 + total * m["heads"] * (width + m["rank"]) * 2,
            "flops": pairs * m["heads"] * 2 * (width + m["rank"])}


# ------------------------------------------------------------------- exact
def exact(case, seed):
    """The operators from their definitions, in 64 bits, sequence by sequence."""
    st = prepare(case, seed)
    op = case["op"]
    if op == "attend":
        q, pages, table, rank = st["q"].double(), st["pages"], st["table"].tolist(), st["rank"]
        new, ctx = _lens(case)
        out, t0 = torch.zeros(q.shape[0], q.shape[1], rank, dtype=torch.float64, device=q.device), 0
        for b, (n, c) in enumerate(zip(new, ctx)):
            if n == 0:
                continue
            cols = -(-c // case["page"])
            keys = pages[torch.tensor(table[b][:cols], device=q.device)].flatten(0, 1)[:c].double()
            hidden = torch.ones(n, c, dtype=torch.bool, device=q.device).triu(c - n + 1)
            for h in range(q.shape[1]):
                logit = torch.addmm(torch.zeros((), dtype=torch.float64, device=q.device),
                                    q[t0:t0 + n, h], keys.t(), alpha=st["scale"]).masked_fill_(hidden, -math.inf)
                out[t0:t0 + n, h] = torch.exp(logit - torch.logsumexp(logit, 1, keepdim=True)) @ keys[:, :rank]
            t0 += n
        return out
    if op == "append":
        pages, x = st["pages"].double(), st["kv_a"].double()
        new, ctx = _lens(case)
        rank, rope, page, t0 = st["rank"], st["cos"].shape[1] * 2, case["page"], 0
        inv = 10000.0 ** (-torch.arange(0, rope, 2, dtype=torch.float64, device=x.device) / rope)
        for b, (n, c) in enumerate(zip(new, ctx)):
            rows = x[t0:t0 + n]
            t0 += n
            pos = torch.arange(c - n, c, device=x.device)
            lat = rows[:, :rank]
            lat = lat / torch.sqrt(lat.square().mean(1, keepdim=True) + 1e-6) * st["weight"].double()
            turn = torch.polar(torch.ones(n, rope // 2, dtype=torch.float64, device=x.device), pos[:, None] * inv)
            pe = torch.view_as_real(torch.view_as_complex(rows[:, rank:].reshape(n, -1, 2).contiguous()) * turn)
            pages[st["table"][b].long()[pos // page], pos % page] = torch.cat([lat, pe.flatten(1)], 1)
        return pages
    if op == "select":
        b, k, v = st["logits"].shape
        cand = st["scores"].double()[..., None] + torch.log_softmax(st["logits"].double(), -1)
        stopped = torch.full((b, k, v), -math.inf, dtype=torch.float64, device=cand.device)
        stopped[..., st["eos"]] = st["scores"].double()
        cand = torch.where(st["finished"][..., None], stopped, cand)
        value = torch.topk(cand.view(b, -1), k).values
        return value, None, None, None
    # copies: the plain integers decide, and the pages hold bf16 values as they are
    pages, table = st["pages"], st["table"].tolist()
    parents, length, page, k = st["parents"].tolist(), case["prompt"] + case["step"], case["page"], case["beams"]
    col, rem = length // page, length % page
    for b in range(case["batch"]):
        cur = [table[b * k + i][col] for i in range(k)]
        free = [cur[i] for i in range(k) if i not in parents[b]]
        kept = set()
        for i, p in enumerate(parents[b]):
            if p in kept and rem:
                pages[:, free.pop(0), :rem] = pages[:, cur[p], :rem]
            kept.add(p)
    return None, pages.double()
