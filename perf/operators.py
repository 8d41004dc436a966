"""The operators that serve a prompt and its answers on the paged KV cache, at the sizes their users run.

Three groups of calls:

  chunk      decode.ChunkAttention.run: attention of a chunk of new tokens of each of several sequences over the paged
             bf16 cache, with the q/k head norms, RoPE and the cache append folded in: a prompt, a further piece of one,
             a few drafted tokens to verify, a ragged batch of them
  logprobs   decode.log_probs: log probability and rank of a given token, entropy and top alternatives of every row of
             logits: one decode step, a batch of them, all rows of a prompt
  pool       cache.PagePool: pages given to new sequences and freed again ("admit"), sequences forked ("fork"), pages
             moved together ("compact") and copied ("copy"), over the caches of all layers

The plain forms below are elementary torch operations in 32 bits with the bf16 rounding points that the operators define
(q and k after their norm and after RoPE, the results); exact() restates them in 64 bits."""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

HEAD_DIM, PAGE, EPS, THETA = 128, 16, 1e-6, 1e6
Q_HEADS, KV_HEADS, VOCAB, LAYERS = 16, 8, 151936, 28     # the decoder of the repository's decode step
MOST_SCORES = Q_HEADS * 8192 * 8192                       # scores of the largest chunk case


def listed():
    return [
        # four drafted tokens of one sequence to verify: the smallest chunk, latency counts
        dict(name="chunk verify b1", kind="chunk", batch=1, tokens=4, start=1000, ragged=False, q_heads=16, kv_heads=8, page=16, pad=0, shape=1),
        # the same for a decode batch of ragged sequences, in a buffer with room for more rows
        dict(name="chunk verify b24", kind="chunk", batch=24, tokens=5, start=3500, ragged=True, q_heads=16, kv_heads=8, page=16, pad=16, shape=2),
        # a prompt from its beginning
        dict(name="chunk prompt 2048", kind="chunk", batch=1, tokens=2048, start=0, ragged=False, q_heads=16, kv_heads=8, page=16, pad=0, shape=3),
        # a ragged batch of prompts behind shared openings, three q heads to a kv head, larger pages
        dict(name="chunk ragged b8", kind="chunk", batch=8, tokens=1501, start=777, ragged=True, q_heads=12, kv_heads=4, page=32, pad=3, shape=4),
        # a further piece of a long document
        dict(name="chunk 512 at 30000", kind="chunk", batch=1, tokens=512, start=30000, ragged=False, q_heads=16, kv_heads=8, page=16, pad=0, shape=5),
        # a long prompt at once: the largest call
        dict(name="chunk prompt 8192", kind="chunk", batch=1, tokens=8192, start=0, ragged=False, q_heads=16, kv_heads=8, page=16, pad=0, shape=6),
        # one decode step of one sequence: the sampled token and the alternatives that an API shows
        dict(name="logprobs r1", kind="logprobs", rows=1, vocab=VOCAB, stride=VOCAB, dtype="bf16", top_k=20, temperature=1.0),
        # a decode batch of a smaller, oddly sized vocabulary in fp32
        dict(name="logprobs r64 fp32", kind="logprobs", rows=64, vocab=32003, stride=32003, dtype="fp32", top_k=5, temperature=0.7),
        # every row of a prompt
        dict(name="logprobs r2048", kind="logprobs", rows=2048, vocab=VOCAB, stride=VOCAB, dtype="bf16", top_k=8, temperature=1.0),
        # 32 prompts get their pages, and give them back when they are answered: no page moves, latency counts
        dict(name="pool admit 32", kind="admit", layers=1, pages=20000, page=16, kv_heads=8, sequences=128, tokens=1500, count=32, live=0.5),
        # eight answers to one prompt: the full pages shared, the last one copied in every layer
        dict(name="pool fork 8", kind="fork", layers=LAYERS, pages=1400, page=16, kv_heads=8, sequences=24, tokens=1100, count=8, live=0.6),
        # a pool whose live pages lie all over it is moved together
        dict(name="pool compact", kind="compact", layers=LAYERS, pages=1400, page=16, kv_heads=8, sequences=64, tokens=400, count=0, live=0.5),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["chunk", "chunk", "chunk", "logprobs", "logprobs", "admit", "fork", "compact", "copy"])
    if kind == "chunk":
        q_heads, kv_heads = rng.choice([(16, 8), (16, 8), (32, 8), (12, 4), (8, 8), (24, 3), (16, 1)])
        tokens, batch = _log_int(rng, 1, 8192), _log_int(rng, 1, 32)
        start = rng.choice([0, _log_int(rng, 1, 32000)])
        while batch > 1 and (batch * q_heads * tokens * (start + tokens) > MOST_SCORES // 4 or batch * (start + tokens) > 150000):
            batch -= 1
        while q_heads * tokens * (start + tokens) > MOST_SCORES // 2:
            tokens = max(1, tokens * 3 // 4)
        return dict(kind=kind, batch=batch, tokens=tokens, start=start, ragged=rng.random() < 0.6, q_heads=q_heads, kv_heads=kv_heads,
                    page=rng.choice([16, 16, 16, 32, 64, 8, 20]), pad=rng.choice([0, 0, 1, 13]), shape=rng.randrange(1 << 16))
    if kind == "logprobs":
        vocab = rng.choice([VOCAB, VOCAB, _log_int(rng, 1000, 200000)])
        rows = _log_int(rng, 1, min(2048, 2048 * VOCAB // (2 * vocab)))
        return dict(kind=kind, rows=rows, vocab=vocab, stride=vocab + rng.choice([0, 0, 0, 8, 37]), dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                    top_k=rng.choice([0, 1, 5, 20, 32]), temperature=rng.choice([1.0, 1.0, 0.6, 1.3]))
    page, kv_heads = rng.choice([16, 16, 32, 5]), rng.choice([8, 8, 4, 1])
    layers, live = rng.randint(2, LAYERS), rng.uniform(0.2, 0.8)
    if kind == "admit":
        return dict(kind=kind, layers=1, pages=_log_int(rng, 2000, 60000), page=page, kv_heads=1, sequences=rng.randint(40, 256),
                    tokens=_log_int(rng, 100, 4000), count=rng.randint(1, 32), live=live)
    pages = _log_int(rng, 200, 1400 * 16 * 8 * LAYERS // (page * max(kv_heads, 4) * LAYERS))
    return dict(kind=kind, layers=layers, pages=pages, page=page, kv_heads=kv_heads, sequences=rng.randint(24, 96), tokens=_log_int(rng, 64, 1500),
                count=rng.randint(1, 16) if kind == "fork" else rng.randint(1, pages // 3) if kind == "copy" else 0, live=live)


# ------------------------------------------------------------------ the shapes that a case stands for


def _lens(case):
    """New tokens and first positions of each sequence of a chunk case: the first sequence has the most of both."""
    r, b = np.random.RandomState(case["shape"]), case["batch"]
    if not case["ragged"]:
        return np.full(b, case["tokens"]), np.full(b, case["start"])
    tokens, starts = r.randint(0, case["tokens"] + 1, b), r.randint(0, case["start"] + 1, b)
    tokens[0], starts[0] = case["tokens"], case["start"]
    return tokens, starts


def _pool(case, r):
    """A page pool in use: page table, lengths and reference counts.  Every second sequence shares the full pages of the first
    half of the one before it; the pages lie in no order; the last `count` rows of an "admit" or "fork" case are empty."""
    pages, page, rows = case["pages"], case["page"], case["sequences"]
    used = rows - (case["count"] if case["kind"] in ("admit", "fork") else 0)
    width = 2 * (-(-case["tokens"] // page)) + 2
    table, lengths, refs = np.full((rows, width), -1, np.int32), np.zeros(rows, np.int32), np.zeros(pages, np.int32)
    order, at, most = r.permutation(pages).astype(np.int32), 0, int(case["live"] * pages)
    for s in range(used):
        n = int(r.randint(max(1, case["tokens"] // 2), case["tokens"] + 1))
        shared = min(n, int(lengths[s - 1]) // 2) // page if s & 1 else 0
        need = -(-n // page) - shared
        if at + need > most:
            break
        table[s, :shared] = table[s - 1, :shared]
        table[s, shared:shared + need] = order[at:at + need]
        lengths[s], at = n, at + need
    held = table[table >= 0]
    np.add.at(refs, held, 1)
    return table, lengths, refs


# ------------------------------------------------------------------ inputs


def _gen(seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    return gen


def _normal(gen, *shape):
    return torch.randn(*shape, device="cuda", generator=gen, dtype=torch.bfloat16)


def _ints(a):
    return torch.from_numpy(np.ascontiguousarray(a, np.int32)).cuda()


def _prepare_chunk(case, gen, r):
    tokens, starts = _lens(case)
    h, kv, page, batch = case["q_heads"], case["kv_heads"], case["page"], case["batch"]
    rows, context = int(tokens.sum()), int((tokens + starts).max())
    logical = -(-context // page)
    physical = batch * logical + 3
    bounds = np.concatenate([[0], np.cumsum(tokens)])
    angles = np.arange(logical * page)[:, None] * THETA ** (-np.arange(0, HEAD_DIM, 2) / HEAD_DIM)[None, :]
    near_one = lambda: (1 + 0.1 * torch.randn(HEAD_DIM, device="cuda", generator=gen)).to(torch.bfloat16)   # noqa: E731
    state = dict(case=case, rows=rows, context=context, longest=int(tokens.max()),
                 qkv=_normal(gen, rows + case["pad"], (h + 2 * kv) * HEAD_DIM), q_norm=near_one(), k_norm=near_one(),
                 cos=torch.from_numpy(np.cos(angles).astype(np.float32)).cuda(), sin=torch.from_numpy(np.sin(angles).astype(np.float32)).cuda(),
                 # pages in the order a running server would have handed them out: no order
                 table=_ints(r.permutation(physical)[:batch * logical].reshape(batch, logical)), positions=_ints(starts), row_starts=_ints(bounds),
                 keys=_normal(gen, physical, page, kv, HEAD_DIM), values=_normal(gen, physical, page, kv, HEAD_DIM),
                 out=torch.zeros(rows + case["pad"], h * HEAD_DIM, dtype=torch.bfloat16, device="cuda"))
    if own:
        from garnet_b200 import decode
        cfg = decode.DecoderConfig(q_heads=h, kv_heads=kv, page_size=page, eps=EPS)
        state["attention"] = decode.ChunkAttention(cfg, max_tokens=rows + case["pad"], max_context=logical * page, max_logical_pages=logical,
                                                   rope_positions=logical * page)
    return state


def _prepare_logprobs(case, gen):
    rows, vocab, stride = case["rows"], case["vocab"], case["stride"]
    dtype = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}[case["dtype"]]
    # a model's logits: a broad bulk, and a few tokens that stand out, more of them in some rows than in others
    x = torch.randn(rows, stride, device="cuda", generator=gen).mul_(2.0)
    few = torch.randint(0, vocab, (rows, 12), device="cuda", generator=gen)
    x.scatter_add_(1, few, torch.rand(rows, 12, device="cuda", generator=gen) * 18 * torch.rand(rows, 1, device="cuda", generator=gen))
    logits = x.to(dtype)[:, :vocab]
    # tokens drawn from the rows' own distribution
    noise = torch.rand(rows, vocab, device="cuda", generator=gen).clamp_(min=1e-30).log_().neg_().log_().neg_()
    targets = noise.add_(logits.float() / case["temperature"]).argmax(1).to(torch.int32)
    return dict(case=case, logits=logits, targets=targets)


def _prepare_pool(case, gen, r):
    table, lengths, refs = _pool(case, r)
    rows, count, kind = case["sequences"], case["count"], case["kind"]
    shape = (case["layers"], case["pages"], case["page"], case["kv_heads"], HEAD_DIM)
    state = dict(case=case, table=_ints(table), lengths=_ints(lengths), refs=_ints(refs))
    if kind == "admit":
        shape = (1, case["pages"], case["page"], 1, 8)      # no page is read or written: what a position holds does not matter
        state["which"] = _ints(r.permutation(np.arange(rows - count, rows)))
        state["tokens"] = _ints(r.randint(max(1, case["tokens"] // 3), case["tokens"] + 1, count))
    elif kind == "fork":
        held = np.flatnonzero(lengths)
        state["which"] = _ints(r.permutation(np.arange(rows - count, rows)))
        state["parents"] = _ints(np.full(count, held[r.randint(len(held))]) if count > 1 and r.rand() < 0.5 else held[r.randint(0, len(held), count)])
    elif kind == "copy":
        pair = r.permutation(case["pages"])[:2 * count]
        state["src"], state["dst"] = _ints(pair[:count]), _ints(pair[count:])
    state["keys"], state["values"] = _normal(gen, *shape), _normal(gen, *shape)
    if own:
        from garnet_b200 import cache
        pool = cache.PagePool(state["keys"], state["values"], sequences=rows, max_logical_pages=table.shape[1])
        state["pool"] = pool
        pool.page_tables.copy_(state["table"])
        pool.lengths.copy_(state["lengths"])
        pool.refcounts.copy_(state["refs"])
        state["now"] = (pool.page_tables, pool.lengths, pool.refcounts)
    else:
        state["now"] = (state["table"].clone(), state["lengths"].clone(), state["refs"].clone())
    return state


def prepare(case, seed):
    gen, r = _gen(seed), np.random.RandomState(seed % (1 << 31))
    if case["kind"] == "chunk":
        return _prepare_chunk(case, gen, r)
    if case["kind"] == "logprobs":
        return _prepare_logprobs(case, gen)
    return _prepare_pool(case, gen, r)


# ------------------------------------------------------------------ plain forms: attention of a chunk


def _bf(x):
    return x.to(torch.bfloat16).float()


def _head(x, w, cos, sin):
    """RMS norm of a head and rotate-half RoPE, each rounded to bf16."""
    x = x.float()
    x = _bf(x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * w.float())
    a, b = x[..., :HEAD_DIM // 2], x[..., HEAD_DIM // 2:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1).to(torch.bfloat16)


def _plain_chunk(s):
    case, rows = s["case"], s["rows"]
    h, kv, page, batch = case["q_heads"], case["kv_heads"], case["page"], case["batch"]
    t_max, c_max = s["longest"], s["context"]
    bounds = s["row_starts"].long()
    row = torch.arange(rows, device="cuda")
    seq = torch.searchsorted(bounds, row, right=True) - 1
    t = row - bounds[seq]
    slot = s["positions"].long()[seq] + t
    cos, sin = s["cos"][slot][:, None, :], s["sin"][slot][:, None, :]
    x = s["qkv"][:rows].view(rows, h + 2 * kv, HEAD_DIM)
    q = _head(x[:, :h], s["q_norm"], cos, sin)
    where = s["table"].long()[seq, slot // page]
    s["keys"][where, slot % page] = _head(x[:, h:h + kv], s["k_norm"], cos, sin)
    s["values"][where, slot % page] = x[:, h + kv:]
    # every sequence padded to the longest: queries [batch, kv, group * t_max, 128], keys and values [batch, kv, c_max, 128]
    group = h // kv
    to = (bounds[:-1, None] + torch.arange(t_max, device="cuda")).clamp(max=max(rows - 1, 0))
    q = q[to].float().view(batch, t_max, kv, group, HEAD_DIM).permute(0, 2, 3, 1, 4).reshape(batch, kv, group * t_max, HEAD_DIM)
    at = torch.arange(c_max, device="cuda")
    ids = s["table"].long()[:, at // page]
    k = s["keys"][ids, at % page].float().permute(0, 2, 3, 1)
    v = s["values"][ids, at % page].float().permute(0, 2, 1, 3)
    score = torch.matmul(q, k).view(batch, kv, group, t_max, c_max).mul_(1 / math.sqrt(HEAD_DIM))
    last = s["positions"].long()[:, None] + torch.arange(t_max, device="cuda")
    score.masked_fill_((at > last[:, :, None])[:, None, None], -math.inf)
    p = score.sub_(score.amax(-1, keepdim=True)).exp_()
    # positions behind a sequence's last row hold whatever the cache held: their weight is zero, and so is what they add
    o = torch.matmul(p.view(batch, kv, group * t_max, c_max), v).view(batch, kv, group, t_max, HEAD_DIM) / p.sum(-1, keepdim=True)
    s["out"][:rows] = o.permute(0, 3, 1, 2, 4).reshape(batch, t_max, h * HEAD_DIM)[seq, t].to(torch.bfloat16)
    return s["out"], s["keys"], s["values"]


# ------------------------------------------------------------------ plain forms: log probabilities


def _plain_logprobs(s):
    case, k = s["case"], s["case"]["top_k"]
    raw = s["logits"].float()
    x = raw / case["temperature"]
    x = x.sub_(x.amax(1, keepdim=True))
    p = x.exp()
    total = p.sum(1, dtype=torch.float64)
    log_total = total.log()
    entropy = log_total - (p * x).sum(1, dtype=torch.float64) / total
    del p
    to = s["targets"].long()[:, None]
    log_prob = x.gather(1, to)[:, 0].double() - log_total
    rank = (raw > raw.gather(1, to)).sum(1) + 1
    result = [log_prob.float(), rank.to(torch.int32), entropy.float()]
    if k:
        ids = torch.sort(raw, dim=1, descending=True, stable=True)[1][:, :k]     # equal logits: the lowest index first
        result += [(x.gather(1, ids).double() - log_total[:, None]).float(), ids.to(torch.int32)]
    return result


# ------------------------------------------------------------------ plain forms: pages


def _free_ids(refs):
    """The free pages in ascending order, then the others, and how many are free."""
    held = (refs > 0).to(torch.int32)
    return torch.sort(held, stable=True)[1].to(torch.int32), refs.numel() - held.sum()


def _given(need, refs):
    """First page of each entry's share in the order of free pages, and which entries get theirs: the free pages are given out in the
    order of the list until one does not get what it needs; entries that need none always do."""
    ids, free = _free_ids(refs)
    upto = need.cumsum(0)
    fine = (need == 0) | (upto <= free)
    return ids, upto - need, fine


def _plain_extend(now, which, tokens, page):
    table, lengths, refs = now
    have = (lengths[which].long() + page - 1) // page
    size = lengths[which].long() + tokens.long()
    need = (size + page - 1) // page - have
    ids, first, fine = _given(need, refs)
    col = torch.arange(table.shape[1], device="cuda")
    new = fine[:, None] & (col >= have[:, None]) & (col < (have + need)[:, None])
    page_of = ids[(first[:, None] + col - have[:, None]).clamp(0, ids.numel() - 1)]
    table[which] = torch.where(new, page_of, table[which])
    refs.index_add_(0, page_of.reshape(-1).long(), new.reshape(-1).to(torch.int32))
    lengths[which] = torch.where(fine, size, lengths[which].long()).to(torch.int32)
    return torch.where(fine, 0, 5).to(torch.int32)


def _plain_free(now, which, page):
    table, lengths, refs = now
    rows = table[which].long()
    held = torch.arange(table.shape[1], device="cuda") < ((lengths[which].long() + page - 1) // page)[:, None]
    refs.index_add_(0, rows.clamp(min=0).reshape(-1), -held.reshape(-1).to(torch.int32))
    table[which] = -1
    lengths[which] = 0


def _plain_fork(now, keys, values, parents, children, page):
    table, lengths, refs = now
    size, rows = lengths[parents].long(), table[parents]
    full, part = size // page, size % page
    ids, first, fine = _given((part > 0).long(), refs)
    col = torch.arange(table.shape[1], device="cuda")
    shared, last = fine[:, None] & (col < full[:, None]), fine[:, None] & (part > 0)[:, None] & (col == full[:, None])
    new = ids[first.clamp(max=ids.numel() - 1)]
    # the positions of the last pages; an entry that has none copies a page of its parent's over itself
    copies = fine & (part > 0)
    src = rows.gather(1, full.clamp(max=table.shape[1] - 1)[:, None])[:, 0].clamp(min=0).long()
    src = torch.where(copies, src, rows[:, 0].clamp(min=0).long())
    dst = torch.where(copies, new.long(), src)
    kept = (torch.arange(page, device="cuda") < part[:, None])[None, :, :, None, None]
    keys[:, dst] = torch.where(kept, keys[:, src], keys[:, dst])
    values[:, dst] = torch.where(kept, values[:, src], values[:, dst])
    rows = torch.where(last, new[:, None], torch.where(shared, rows, -1))
    refs.index_add_(0, rows.clamp(min=0).reshape(-1).long(), (rows >= 0).reshape(-1).to(torch.int32))
    table[children] = torch.where(fine[:, None], rows, table[children])
    lengths[children] = torch.where(fine, size, lengths[children].long()).to(torch.int32)
    return torch.where(fine, 0, 5).to(torch.int32)


def _plain_compact(now, keys, values):
    table, lengths, refs = now
    held, at = refs > 0, torch.arange(refs.numel(), device="cuda")
    live = held.sum()
    src, dst = torch.nonzero(held & (at >= live))[:, 0], torch.nonzero(~held & (at < live))[:, 0]
    keys[:, dst] = keys[:, src]
    values[:, dst] = values[:, src]
    to = at.to(torch.int32)
    to[src] = dst.to(torch.int32)
    refs[dst] = refs[src]
    refs[src] = 0
    table.copy_(torch.where(table >= 0, to[table.clamp(min=0).long()], table))
    return live.to(torch.int32).reshape(1)


# ------------------------------------------------------------------ one pass


def _snapshot(now):
    """Page tables, lengths and reference counts as a scheduler takes them."""
    return [t.clone() for t in now]


def run(state):
    s, case = state, state["case"]
    kind, page = case["kind"], case.get("page")
    if kind == "chunk":
        if not own:
            return _plain_chunk(s)
        out = s["attention"].run(s["qkv"], s["q_norm"], s["k_norm"], s["cos"], s["sin"], s["keys"], s["values"], s["table"], s["positions"],
                                 s["row_starts"], s["out"])
        return out, s["keys"], s["values"]
    if kind == "logprobs":
        if not own:
            return _plain_logprobs(s)
        from garnet_b200 import decode
        r = decode.log_probs(s["logits"], s["targets"], top_k=case["top_k"], temperature=case["temperature"])
        return [r.log_probs, r.ranks, r.entropy] + ([r.top_log_probs, r.top_ids] if case["top_k"] else [])
    now, pool = s["now"], s.get("pool")
    if kind == "admit":          # new sequences come, are seen in the tables, and go
        status = pool.extend(s["which"], s["tokens"]) if own else _plain_extend(now, s["which"], s["tokens"], page)
        seen = _snapshot(now)
        pool.free(s["which"]) if own else _plain_free(now, s["which"], page)
        return status, seen
    if kind == "fork":           # the same for the children of a fork
        status = pool.fork(s["parents"], s["which"]) if own else _plain_fork(now, s["keys"], s["values"], s["parents"], s["which"], page)
        seen = _snapshot(now)
        pool.free(s["which"]) if own else _plain_free(now, s["which"], page)
        return status, seen, s["keys"], s["values"]
    if kind == "copy":
        if own:
            pool.copy_pages(s["src"], s["dst"])
        else:
            s["keys"][:, s["dst"].long()] = s["keys"][:, s["src"].long()]
            s["values"][:, s["dst"].long()] = s["values"][:, s["src"].long()]
        return s["keys"], s["values"]
    # a pass finds the pool scattered as it was
    now[0].copy_(s["table"]), now[1].copy_(s["lengths"]), now[2].copy_(s["refs"])
    live = pool.compact() if own else _plain_compact(now, s["keys"], s["values"])
    return live, now, s["keys"], s["values"]


# ------------------------------------------------------------------ what a pass cannot do without


def work(case):
    kind = case["kind"]
    if kind == "chunk":
        tokens, starts = _lens(case)
        h, kv, rows = case["q_heads"], case["kv_heads"], int(tokens.sum())
        pairs = int((tokens * starts + tokens * (tokens + 1) // 2).sum())
        row = 2 * kv * HEAD_DIM * 2                                # K and V of a position
        read = int(starts[tokens > 0].sum()) * row + rows * (h + 2 * kv) * HEAD_DIM * 2
        return {"bytes": read + rows * (row + h * HEAD_DIM * 2), "flops": 4 * h * HEAD_DIM * pairs}
    if kind == "logprobs":
        values = case["rows"] * case["vocab"]
        return {"bytes": values * (4 if case["dtype"] == "fp32" else 2) + case["rows"] * (16 + 8 * case["top_k"]), "flops": 5 * values}
    table, lengths, refs = _pool(case, np.random.RandomState(1))
    page_bytes = 2 * case["layers"] * case["page"] * case["kv_heads"] * HEAD_DIM * 2
    meta = 2 * 4 * (table.size + lengths.size + refs.size)
    if kind == "admit":
        return {"bytes": meta, "flops": 0}
    if kind == "fork":                                             # the last page of a parent is half full on average
        return {"bytes": meta + case["count"] * page_bytes, "flops": 0}
    if kind == "copy":
        return {"bytes": 2 * case["count"] * page_bytes, "flops": 0}
    live = int((refs > 0).sum())
    return {"bytes": meta + 2 * int((refs[live:] > 0).sum()) * page_bytes, "flops": 0}


# ------------------------------------------------------------------ the operators' definitions in 64 bits


def _exact_head(x, w, cos, sin):
    x = x.double()
    x = (x * (x.pow(2).sum(-1, keepdim=True) / HEAD_DIM + EPS).rsqrt() * w.double()).to(torch.bfloat16).double()
    turned = torch.cat([-x[..., HEAD_DIM // 2:], x[..., :HEAD_DIM // 2]], -1)
    return x * torch.cat([cos, cos], -1) + turned * torch.cat([sin, sin], -1)


def _exact_chunk(case, seed):
    s = prepare(case, seed)
    h, kv, page = case["q_heads"], case["kv_heads"], case["page"]
    tokens, starts = _lens(case)
    result = torch.zeros(s["out"].shape, dtype=torch.float64, device="cuda")
    keys, values = s["keys"].double(), s["values"].double()
    row0 = 0
    for b in range(case["batch"]):
        n, first = int(tokens[b]), int(starts[b])
        if not n:
            continue
        x = s["qkv"][row0:row0 + n].view(n, h + 2 * kv, HEAD_DIM)
        cos, sin = (s[c][first:first + n, None, :].double() for c in ("cos", "sin"))
        q = _exact_head(x[:, :h], s["q_norm"], cos, sin).to(torch.bfloat16).double()
        slots = torch.arange(first, first + n, device="cuda")
        pages = s["table"][b].long()
        keys[pages[slots // page], slots % page] = _exact_head(x[:, h:h + kv], s["k_norm"], cos, sin).to(torch.bfloat16).double()
        values[pages[slots // page], slots % page] = x[:, h + kv:].double()
        seen = torch.arange(first + n, device="cuda")
        K, V = keys[pages[seen // page], seen % page], values[pages[seen // page], seen % page]
        for head in range(h):
            kh, vh = K[:, head // (h // kv)], V[:, head // (h // kv)]
            for t0 in range(0, n, 2048):
                part = slice(t0, min(n, t0 + 2048))
                score = q[part, head] @ kh.T / math.sqrt(float(HEAD_DIM))
                p = torch.softmax(score.masked_fill(seen[None, :] > slots[part, None], -math.inf), -1)
                result[row0 + t0:row0 + t0 + p.shape[0], head * HEAD_DIM:(head + 1) * HEAD_DIM] = p @ vh
        row0 += n
    return result, keys, values


def _exact_logprobs(case, seed):
    s = prepare(case, seed)
    log_probs, entropies, tops = [], [], []
    for r0 in range(0, case["rows"], 256):
        x = torch.log_softmax(s["logits"][r0:r0 + 256].double() / case["temperature"], 1)
        log_probs.append(x.gather(1, s["targets"][r0:r0 + 256].long()[:, None])[:, 0])
        entropies.append(-(x.exp() * x).sum(1))
        if case["top_k"]:
            tops.append(torch.topk(x, case["top_k"], dim=1)[0])
    return [torch.cat(log_probs), None, torch.cat(entropies)] + ([torch.cat(tops), None] if case["top_k"] else [])


def exact(case, seed):
    if case["kind"] == "chunk":
        return _exact_chunk(case, seed)
    if case["kind"] == "logprobs":
        return _exact_logprobs(case, seed)
    return None      # whole numbers, and pages that are copied as they are
