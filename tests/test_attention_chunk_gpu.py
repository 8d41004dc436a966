"""garnet_b200_attention_chunk against a plain implementation: float64 attention over the cache, head norms and RoPE in the kernel's own
fp32 steps.

The rows hold whole numbers times a power of two, so that a head's sum of squares is exact in any order and the fp32 restatement of norm
and RoPE gives the kernel's q and k bit for bit: the appended k and v are compared exactly.  A result is off by its own rounding
(2^-8 of itself) and by the rounding of the weights p to bf16 before they multiply v (2^-8 of sum p |v|); the scores' fp32 sums of 128
products, the exponentials and the fp32 (or tensor-core) sums of the weights' products add less than 2^-11 of sum p |v| at these
lengths (scores below 2^7: 2^-24 2^7 8 for the weights; 2^-24 per position for the sums, of at most 5000 positions)."""
import numpy as np
import pytest
import torch

import garnet_b200
from garnet_b200 import cache, decode as dec

pytestmark = pytest.mark.gpu
f32 = np.float32


def bf(a):
    """fp32 rounded to bf16 (nearest even), as fp32."""
    return torch.from_numpy(np.ascontiguousarray(a, f32)).to(torch.bfloat16).float().numpy()


def fma(a, b, c):
    """fp32 a b + c rounded once (the float64 sum of the exact product is rounded to fp32; that this rounds twice matters once in 2^29)."""
    a, b, c = (np.asarray(v, np.float64) for v in (a, b, c))
    return (a * b + c).astype(f32)


def head(x, w, cos, sin, eps):
    """x [..., 128] fp32: the kernel's fp32 steps."""
    mean = (x.astype(np.float64) ** 2).sum(-1, keepdims=True) / 128 + np.float64(f32(eps))
    r = f32(1) / np.sqrt(mean.astype(f32))
    c = f32(0.5) * r * (1 - mean * (r.astype(np.float64) * r)).astype(f32)
    v = x * w
    x = bf(fma(v, r, v * c))
    a, b = x[..., :64], x[..., 64:]

    def turned(a, b):
        p = b * sin
        return fma(a, cos, p) + fma(b, sin, -p)

    return bf(np.concatenate([turned(a, -b), turned(b, a)], -1))


class Case:
    def __init__(self, lens, starts, q_heads=4, kv_heads=2, page_size=16, pad=0, seed=0, max_context=None, spare=3, scale=0.25):
        gen = torch.Generator().manual_seed(seed)
        self.cfg = dec.DecoderConfig(q_heads=q_heads, kv_heads=kv_heads, page_size=page_size)
        self.lens, self.starts = list(lens), list(starts)
        rows, batch = sum(lens), len(lens)
        context = max(max(n + max(s, 0) for n, s in zip(lens, starts)), 1)
        self.width = -(-context // page_size) + 1
        self.positions_room = self.width * page_size
        self.max_context = max_context or self.positions_room
        pages = batch * self.width + spare
        ints = lambda *shape: torch.randint(-8, 9, shape, generator=gen).float() * scale   # noqa: E731
        self.qkv = ints(rows + pad, (q_heads + 2 * kv_heads) * 128).to(torch.bfloat16)
        self.q_norm, self.k_norm = ((1 + 0.2 * torch.randn(128, generator=gen)).to(torch.bfloat16) for _ in range(2))
        self.keys, self.values = (torch.randn(pages, page_size, kv_heads, 128, generator=gen).to(torch.bfloat16) for _ in range(2))
        self.table = torch.randperm(pages, generator=gen)[:batch * self.width].reshape(batch, self.width).to(torch.int32)
        cos, sin = dec.rope_tables(self.positions_room, 128, self.cfg.rope_theta)
        self.cos, self.sin = torch.from_numpy(cos), torch.from_numpy(sin)
        self.row_starts = torch.from_numpy(np.concatenate([[0], np.cumsum(lens)]).astype(np.int32))
        self.rows, self.pad, self.batch, self.pages = rows, pad, batch, pages

    def device(self):
        d = lambda t: t.cuda()   # noqa: E731
        return dict(qkv=d(self.qkv), q_norm_w=d(self.q_norm), k_norm_w=d(self.k_norm), cos=d(self.cos), sin=d(self.sin), key_pages=d(self.keys),
                    value_pages=d(self.values), page_tables=d(self.table), positions=torch.tensor(self.starts, dtype=torch.int32, device="cuda"),
                    row_starts=d(self.row_starts), out=torch.full((self.rows + self.pad, self.cfg.q_heads * 128), 7.0, dtype=torch.bfloat16, device="cuda"))

    def op(self):
        return dec.ChunkAttention(self.cfg, self.rows + self.pad, self.max_context, self.width, self.positions_room)

    def expect(self):
        """(results, tolerances, keys, values), float64 / bf16."""
        cfg, ps = self.cfg, self.cfg.page_size
        h, kv = cfg.q_heads, cfg.kv_heads
        keys, values = self.keys.float().numpy().copy(), self.values.float().numpy().copy()
        x = self.qkv.float().numpy().reshape(self.rows + self.pad, h + 2 * kv, 128)
        wq, wk = self.q_norm.float().numpy(), self.k_norm.float().numpy()
        cos, sin, table = self.cos.numpy(), self.sin.numpy(), self.table.numpy()
        out = np.full((self.rows + self.pad, h, 128), 7.0)
        tol = np.zeros_like(out)
        page_ok = (table >= 0) & (table < self.pages)
        queries = {}
        for b in range(self.batch):
            for t in range(self.lens[b]):
                r, slot = int(self.row_starts[b]) + t, self.starts[b] + t
                out[r] = 0
                if self.starts[b] < 0 or slot >= self.max_context:
                    continue
                c, s = cos[slot], sin[slot]
                queries[r] = (b, slot, head(x[r, :h], wq, c, s, cfg.eps))
                if page_ok[b, slot // ps]:
                    at = table[b, slot // ps], slot % ps
                    keys[at] = head(x[r, h:h + kv], wk, c, s, cfg.eps)
                    values[at] = x[r, h + kv:]
        for r, (b, slot, q) in queries.items():
            n = slot + 1
            seen = np.flatnonzero(page_ok[b, np.arange(n) // ps])
            if not len(seen):
                continue
            pg, of = table[b, seen // ps], seen % ps
            K, V = keys[pg, of].astype(np.float64), values[pg, of].astype(np.float64)
            for i in range(h):
                g = i // (h // kv)
                with np.errstate(invalid="ignore", over="ignore"):
                    s = K[:, g] @ q[i].astype(np.float64) / np.sqrt(128.0)
                    p = np.exp(s - s.max())
                    p /= p.sum()
                    out[r, i] = (p[:, None] * V[:, g])[p != 0].sum(0) if not np.isnan(p).any() else np.nan
                    mass = (p[:, None] * np.abs(V[:, g]))[p != 0].sum(0)
                tol[r, i] = 2.0 ** -8 * np.abs(out[r, i]) + (2.0 ** -8 + 2.0 ** -11) * mass
        return out.reshape(self.rows + self.pad, -1), tol.reshape(self.rows + self.pad, -1), keys, values

    def run(self):
        d = self.device()
        self.op().run(**d)
        torch.cuda.synchronize()
        return d

    def check(self, tight=True):
        d = self.run()
        want, tol, keys, values = self.expect()
        got = d["out"].double().cpu().numpy()
        both = np.isnan(got) & np.isnan(want)
        with np.errstate(invalid="ignore"):
            bad = ~both & (got != want) & ~(np.abs(got - want) <= tol)
        assert not bad.any(), f"{bad.sum()} of {bad.size}, first at {np.argwhere(bad)[0]}: {got[bad][:4]} for {want[bad][:4]}"
        if tight and np.isfinite(want).all() and self.rows:
            off = got[:self.rows] - want[:self.rows]
            assert np.linalg.norm(off) <= 2.0 ** -8 * np.linalg.norm(want[:self.rows])
        for t, a in ((d["key_pages"], keys), (d["value_pages"], values)):
            assert np.array_equal(t.float().cpu().numpy(), a, equal_nan=True)
        return d


@pytest.mark.parametrize("q_heads,kv_heads", [(4, 2), (16, 8), (3, 3), (6, 2), (8, 1), (40, 1)])
@pytest.mark.parametrize("lens,starts", [([1], [0]), ([1], [200]), ([5, 0, 17, 1], [0, 3, 130, 64]), ([70, 33], [0, 45])])
def test_heads_and_lengths(q_heads, kv_heads, lens, starts):
    Case(lens, starts, q_heads, kv_heads, pad=3, seed=q_heads).check()


def test_a_group_as_large_as_a_tile():
    Case([5, 2], [0, 40], 128, 1).check()


@pytest.mark.parametrize("page_size", [1, 5, 8, 16, 24, 64, 128, 200])
def test_page_sizes(page_size):
    Case([150, 9], [31, 250], page_size=page_size, seed=page_size).check()


@pytest.mark.parametrize("tokens", [63, 64, 65, 127, 128, 129, 255, 256, 257])
@pytest.mark.parametrize("start", [0, 1, 127, 128])
def test_edges_of_tiles(tokens, start):
    Case([tokens], [start], 2, 1, seed=tokens).check()


@pytest.mark.parametrize("q_heads,kv_heads,tokens,start", [(2, 2, 3, 4900), (4, 1, 40, 3000), (16, 8, 1, 2047), (2, 1, 300, 1500)])
def test_few_rows_after_a_long_context(q_heads, kv_heads, tokens, start):
    Case([tokens], [start], q_heads, kv_heads, seed=tokens).check()


def test_many_sequences():
    r = np.random.RandomState(0)
    lens = [int(n) for n in r.randint(0, 9, 70)]
    Case(lens, [int(n) for n in r.randint(0, 150, 70)], 4, 2).check()


def test_more_sequences_than_threads_order_them():
    """Blocks of rows are ordered by what they see: 600 sequences, many without rows, two of many blocks, in a buffer with room to spare."""
    r = np.random.RandomState(1)
    lens = [int(n) for n in r.randint(0, 4, 600)]
    lens[17], lens[598], lens[599] = 700, 90, 1
    Case(lens, [int(n) for n in r.randint(0, 60, 600)], 8, 1, pad=5).check()


@pytest.mark.parametrize("q_heads,kv_heads,lens,starts,page_size", [
    (16, 8, [130, 90, 1, 127, 128, 129, 64, 65, 260, 0, 33, 100, 77, 128], [0, 5, 300, 128, 127, 1, 64, 63, 0, 9, 500, 250, 1, 0], 16),
    (18, 6, [90, 43, 85, 130, 84, 42, 41, 100, 100, 86, 129, 60, 70, 127, 3, 1, 88, 99, 47, 90], [20 * i for i in range(20)], 20),
    (30, 30, [129, 257, 200, 255], [0, 100, 37, 1], 64)])
def test_batches_that_fill_the_gpu(q_heads, kv_heads, lens, starts, page_size):
    """Two tiles of query rows to a CTA."""
    Case(lens, starts, q_heads, kv_heads, page_size=page_size, pad=2, seed=q_heads).check()


@pytest.mark.parametrize("batch,q_heads,kv_heads,tokens,start", [
    (1, 2, 1, 1, 0), (16, 8, 8, 1, 1500), (6, 8, 8, 1, 500), (1, 2, 1, 1, 500),
    (16, 8, 8, 1, 300), (3, 8, 8, 300, 500), (16, 6, 2, 1, 3000), (1, 2, 1, 1, 4500),
    (16, 8, 8, 130, 500), (6, 8, 8, 130, 1500), (3, 8, 8, 130, 3000), (6, 6, 2, 64, 4500)])
def test_every_kind_of_cta_and_share_of_keys(batch, q_heads, kv_heads, tokens, start):
    """One tile with a short or a long ring, two tiles; keys in 1, 2, 4 or 8 shares; contexts with pages missing here and there, the first
    third of one missing altogether, so that shares of it hold nothing."""
    c = Case([tokens] * batch, [start] * batch, q_heads, kv_heads, seed=batch + tokens)
    c.table[:, 3::7] = -1
    c.table[0, :start // 48] = -1
    c.check()


def test_sharp_scores():
    """Scores of some hundreds: all weight on single positions, maxima that grow from tile to tile, rows whose largest score comes last."""
    c = Case([140], [400], 2, 1, seed=5)
    c.k_norm = (c.k_norm.float() * 16).to(torch.bfloat16)
    c.keys = (c.keys.float() * torch.linspace(0.1, 30, c.pages)[:, None, None, None]).to(torch.bfloat16)
    d = c.run()
    want, _, keys, values = c.expect()
    got = d["out"].double().cpu().numpy()
    # scores up to 2^12: their fp32 rounding, 2^-24 2^12 8, moves a weight by up to 2^-9 of itself, beside the two roundings to bf16
    mass = np.abs(values).max()
    assert np.isfinite(got).all() and (np.abs(got - want) <= 2.0 ** -8 * np.abs(want) + (2.0 ** -8 + 2.0 ** -8) * mass).all()


def test_what_lies_behind_a_sequence_does_not_matter():
    """NaN and infinities in the rest of the last page, in pages behind it and in pages of nobody."""
    for ps in (16, 5, 64):
        c = Case([37, 1, 20], [50, 33, 0], page_size=ps, seed=1)
        used = torch.zeros(c.pages, ps, dtype=torch.bool)
        for b in range(c.batch):
            for s in range(c.starts[b] + c.lens[b]):
                used[c.table[b, s // ps], s % ps] = True
        junk = torch.tensor([float("nan"), float("inf"), -float("inf")])[torch.randint(0, 3, c.keys.shape)].to(torch.bfloat16)
        for t in (c.keys, c.values):
            t[~used] = junk[~used]
        c.check()


def test_infinities_and_nan_in_later_tokens_and_in_the_context():
    """v of a later token of the chunk is inf or NaN: earlier rows do not see it, later ones do.  k that is inf or NaN likewise."""
    c = Case([150], [10], 2, 1, seed=2)
    x = c.qkv.view(-1, 4, 128)
    x[60, 3, 5], x[100, 3, 7], x[101, 3, 9] = float("inf"), float("nan"), -float("inf")
    c.check()
    c = Case([40], [100], 2, 1, seed=3)
    x = c.qkv.view(-1, 4, 128)
    x[20, 2, 5] = float("nan")          # k: rows from 20 on are NaN
    c.check()
    c = Case([40], [100], 2, 1, seed=3)
    page, off = c.table[0, 70 // 16], 70 % 16
    c.values[page, off, 0, 3] = float("inf")
    c.check()


def test_pages_that_do_not_exist():
    """Slots without a page are neither written nor seen; a row that sees none is zeros."""
    c = Case([30, 4, 3], [64, 40, 0], seed=4)
    c.table[0, 1], c.table[0, 5] = -1, c.pages          # one in the context, one that new rows fall into
    c.table[1, :] = -7
    c.table[2, 0] = 2 ** 31 - 1
    c.check()


def test_slots_outside():
    """A negative first slot; rows that run over max_context."""
    c = Case([6, 20, 3], [-1, 90, 2], seed=6, max_context=100)
    d = c.check()
    assert (d["out"][:6] == 0).all() and (d["out"][6 + 10:26] == 0).all()


def test_shared_pages():
    """Two sequences share the pages of their opening."""
    c = Case([10, 10], [64, 64], seed=7)
    c.table[1, :4] = c.table[0, :4]
    c.check()


def test_general_values_against_the_decode_kernel():
    """Rows of one token each: the same as garnet_b200_attention_decode, but for the rounding of the weights."""
    batch, starts = 6, [0, 15, 16, 300, 511, 127]
    c = Case([1] * batch, starts, 16, 8, seed=8)
    gen = torch.Generator().manual_seed(0)
    c.qkv = torch.randn(c.qkv.shape, generator=gen).to(torch.bfloat16)
    d = c.run()
    e = c.device()
    attn = dec.PagedAttention(c.cfg, batch, c.max_context, c.width, c.positions_room)
    attn.run(e["qkv"], e["q_norm_w"], e["k_norm_w"], e["cos"], e["sin"], e["key_pages"], e["value_pages"], e["page_tables"], e["positions"], e["out"])
    assert torch.equal(d["value_pages"], e["value_pages"])
    dk = (d["key_pages"].float() - e["key_pages"].float()).abs()
    assert (dk <= e["key_pages"].float().abs() * 2.0 ** -7).all() and (dk > 0).float().mean() < 1e-3     # sums of squares in another order
    a, b = d["out"].float(), e["out"].float()
    # two roundings of results and one of weights, each 2^-8 of values whose rms is the row's
    assert ((a - b).norm(dim=1) <= 3 * 2.0 ** -8 * b.norm(dim=1)).all()


def test_same_bits_every_time_captured_and_on_another_stream():
    c = Case([33, 150, 1], [100, 0, 700], 16, 8, seed=9)
    first = c.run()
    d, op = c.device(), c.op()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        op.run(**d, pdl=True)
    side.synchronize()
    assert torch.equal(d["out"], first["out"]) and torch.equal(d["key_pages"], first["key_pages"])
    # captured with other row boundaries and positions in place, replayed with these; two graphs that share the workspace
    e = c.device()
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    for g in graphs:
        with torch.cuda.graph(g):
            op.run(**e)
    e["row_starts"].zero_()
    graphs[0].replay()
    torch.cuda.synchronize()
    assert (e["out"] == 7).all()                       # rows of no sequence are left as they are
    e["row_starts"].copy_(c.row_starts)
    for g in graphs:
        e["out"].zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(e["out"], first["out"])


def test_calls_one_after_the_other_share_a_workspace():
    """Launched without a wait between them, each starting while the one before ends, as the layers of a step are."""
    cases = [Case([5, 9], [700, 30], 4, 2, seed=1), Case([150, 1], [0, 400], 4, 2, seed=2), Case([1, 1], [63, 64], 4, 2, seed=3)]
    alone = [c.run()["out"] for c in cases]
    shared = max(cases, key=lambda c: c.rows)
    op = dec.ChunkAttention(shared.cfg, 160, 4096, 256, 4096)
    cos, sin = (torch.from_numpy(t).cuda() for t in dec.rope_tables(4096, 128, shared.cfg.rope_theta))
    given = []
    for c in cases:
        d = c.device()
        table = torch.full((c.batch, 256), -1, dtype=torch.int32, device="cuda")
        table[:, :c.width] = d["page_tables"]
        given.append(dict(d, cos=cos, sin=sin, page_tables=table))
    torch.cuda.synchronize()
    for _ in range(20):
        for d in given:
            op.run(**d, pdl=True)
    torch.cuda.synchronize()
    for d, want in zip(given, alone):
        off = (d["out"].double() - want.double()).norm()
        assert off <= 2.0 ** -8 * want.double().norm()     # the keys may be shared out otherwise: P's rounding, the result's own


def test_piece_after_piece_is_the_whole_prompt():
    """A prompt in one call, and in three pieces of odd lengths: the same keys and values, results within the two calls' roundings."""
    c = Case([300], [0], 4, 2, seed=10)
    whole = c.run()
    d, op = c.device(), c.op()
    at = 0
    for n in (1, 166, 133):
        part = dict(d, qkv=d["qkv"][at:at + n].contiguous(), positions=torch.tensor([at], dtype=torch.int32, device="cuda"),
                    row_starts=torch.tensor([0, n], dtype=torch.int32, device="cuda"), out=d["out"][at:at + n])
        op.run(**part)
        at += n
    assert torch.equal(d["key_pages"], whole["key_pages"]) and torch.equal(d["value_pages"], whole["value_pages"])
    a, b = d["out"].float(), whole["out"].float()
    assert ((a - b).norm(dim=1) <= 4 * 2.0 ** -8 * b.norm(dim=1)).all()


def test_refusals():
    c = Case([4], [0])
    d, op = c.device(), c.op()
    for name, bad in dict(qkv=d["qkv"].float(), q_norm_w=d["q_norm_w"][:64], cos=d["cos"][:3], key_pages=d["key_pages"].transpose(1, 2), value_pages=d["value_pages"][1:],
                          page_tables=d["page_tables"].long(), positions=d["positions"].cpu(), row_starts=d["row_starts"][:1], out=d["out"][:, :128]).items():
        with pytest.raises(ValueError):
            op.run(**dict(d, **{name: bad}))
    small = dec.ChunkAttention(c.cfg, 1, c.max_context, c.width, c.positions_room)
    with pytest.raises(garnet_b200.GarnetB200Error):
        small.run(**d)                                  # more rows than the workspace is for
    for cfg, kw in ((dec.DecoderConfig(q_heads=3, kv_heads=2), {}), (dec.DecoderConfig(head_dim=64), {}), (dec.DecoderConfig(q_heads=129, kv_heads=1), {}),
                    (c.cfg, dict(max_context=c.positions_room + 1)), (c.cfg, dict(max_tokens=0))):
        with pytest.raises(garnet_b200.GarnetB200Error):
            dec.ChunkAttention(**dict(dict(cfg=cfg, max_tokens=4, max_context=c.max_context, max_logical_pages=c.width, rope_positions=c.positions_room), **kw))
    op.run(**dict(d, qkv=d["qkv"][:0], out=d["out"][:0]))      # no rows: nothing to do


def test_prompt_fork_answers_and_log_probabilities_together():
    """As a server uses them: pages for a prompt, the prompt in two pieces, two forks, one decode step of each sequence, pages freed and moved
    together, another step, log probabilities of the greedy tokens."""
    cfg = dec.DecoderConfig(hidden=512, q_heads=4, kv_heads=2)
    gen = torch.Generator(device="cuda").manual_seed(0)
    keys, values = (torch.full((1, 40, 16, 2, 128), float("nan"), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    pool = cache.PagePool(keys, values, sequences=4, max_logical_pages=8)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")   # noqa: E731
    cos, sin = (torch.from_numpy(t).cuda() for t in dec.rope_tables(128, 128, cfg.rope_theta))
    qn, kn = ((1 + 0.1 * torch.randn(128, device="cuda", generator=gen)).to(torch.bfloat16) for _ in range(2))
    rows = torch.randn(100, cfg.qkv_width, device="cuda", generator=gen).to(torch.bfloat16)
    chunk = dec.ChunkAttention(cfg, 100, 128, 8, 128)
    decode = dec.PagedAttention(cfg, 4, 128, 8, 128)
    assert pool.extend(i32(3, 1), i32(33, 50)).tolist() == [0, 0]       # sequence 3 is in the way and goes later
    out = torch.zeros(100, 512, dtype=torch.bfloat16, device="cuda")
    for at, n in ((0, 30), (30, 20)):
        chunk.run(rows[at:at + n], qn, kn, cos, sin, keys[0], values[0], pool.page_tables[1:2], i32(at), i32(0, n), out[at:at + n])
    assert pool.fork(i32(1, 1), i32(0, 2)).tolist() == [0, 0]
    pool.free(i32(3))
    head_w = garnet_b200.W4A16Linear().prepare(*garnet_b200.quantize_int4(torch.randn(640, 512, device="cuda", generator=gen)), 640, 512)

    def step(slot):
        """The three sequences get the same token: their results have the same bits as long as their pages hold the same."""
        assert pool.extend(i32(0, 1, 2), i32(1, 1, 1)).tolist() == [0, 0, 0]
        y = torch.zeros(4, 512, dtype=torch.bfloat16, device="cuda")
        decode.run(rows[slot:slot + 1].repeat(4, 1), qn, kn, cos, sin, keys[0], values[0], pool.page_tables, i32(slot, slot, slot, -1), y)
        assert y.isfinite().all() and torch.equal(y[0], y[1]) and torch.equal(y[1], y[2]) and (y[3] == 0).all()
        return y

    for slot in range(50, 64):
        step(slot)
    tables = pool.page_tables.clone()
    assert int((tables[:3, :3] != tables[1, :3]).sum()) == 0 and len(set(tables[:3, 3].tolist())) == 3      # shared, and their own
    again = decode_only(decode, rows, qn, kn, cos, sin, keys, values, pool, i32)
    live = int(pool.compact())
    assert live == 3 + 3 and int(pool.page_tables.max()) == live - 1 and int(pool.refcounts.sum()) == 12
    assert torch.equal(again, decode_only(decode, rows, qn, kn, cos, sin, keys, values, pool, i32))
    y = step(64)
    logits = head_w.forward(y[:3])
    token = torch.zeros(3, dtype=torch.int32, device="cuda")
    dec.argmax_bf16(logits, token)
    r = dec.log_probs(logits, token, top_k=3)
    want = torch.log_softmax(logits.double(), 1)
    assert (r.ranks == 1).all() and torch.equal(r.top_ids[:, 0], token)
    # logits below 2^6, sums of 640 terms: 2^-24 (4 2^6 + 3 2^7 + 30) < 2^-14
    assert (r.log_probs.double() - want.gather(1, token.long()[:, None])[:, 0]).abs().max() <= 2.0 ** -14
    # the same chunk rows of the three sequences at once, over the moved pages: drafted tokens behind slot 64
    assert pool.extend(i32(0, 1, 2), i32(4, 4, 4)).tolist() == [0, 0, 0]
    z = torch.zeros(12, 512, dtype=torch.bfloat16, device="cuda")
    chunk.run(rows[65:69].repeat(3, 1), qn, kn, cos, sin, keys[0], values[0], pool.page_tables[:3].contiguous(), i32(65, 65, 65), i32(0, 4, 8, 12), z)
    assert z.isfinite().all() and torch.equal(z[:4], z[4:8]) and torch.equal(z[:4], z[8:])


def decode_only(decode, rows, qn, kn, cos, sin, keys, values, pool, i32):
    """The step at slot 63 again (its k and v are written over themselves)."""
    y = torch.zeros(4, 512, dtype=torch.bfloat16, device="cuda")
    decode.run(rows[63:64].repeat(4, 1), qn, kn, cos, sin, keys[0], values[0], pool.page_tables, i32(63, 63, 63, -1), y)
    return y


def test_the_decode_kernel_and_pages_that_do_not_exist():
    """garnet_b200_attention_decode on tables as PagePool leaves them: a slot without a page (-1) is neither written nor seen, a row that sees none is
    zeros; nothing else in the cache changes."""
    starts = [40, 300, 16, 129, 0, 255]
    c = Case([1] * len(starts), starts, 4, 2, seed=21)
    c.table[0, 1] = -1                               # a page of the context
    c.table[1, 300 // 16] = -1                       # the page that the new token falls into: a pool that was full
    c.table[2, 16 // 16] = -1
    c.table[3, :8] = -1                              # a whole split of the context
    c.table[4, :] = -1                               # a sequence without pages
    c.table[5, :] = -7
    want, tol, keys, values = c.expect()
    d = c.device()
    guard = [torch.full((c.pages + 2, *c.keys.shape[1:]), 3.0, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    for g, name in zip(guard, ("key_pages", "value_pages")):
        g[1:-1] = d[name]
    attn = dec.PagedAttention(c.cfg, c.batch, c.max_context, c.width, c.positions_room)
    for _ in range(2):
        attn.run(d["qkv"], d["q_norm_w"], d["k_norm_w"], d["cos"], d["sin"], guard[0][1:-1], guard[1][1:-1], d["page_tables"], d["positions"], d["out"])
        got = d["out"].double().cpu().numpy()
        assert (np.abs(got - want) <= tol).all() and (got[4:] == 0).all()
    assert all((g[0] == 3).all() and (g[-1] == 3).all() for g in guard)
    assert np.array_equal(guard[1][1:-1].float().cpu().numpy(), values)
    assert (np.abs(guard[0][1:-1].float().cpu().numpy() - keys) <= 2.0 ** -7 * np.abs(keys)).all()      # k by plain fp32 steps: a neighbour at most


@pytest.mark.parametrize("what", ["a key of the context", "a key of the chunk", "a query", "a value of the context"])
@pytest.mark.parametrize("tokens", [512, 3])
def test_rows_that_are_nan_cost_no_more_than_others(what, tokens):
    """A NaN that most rows of one sequence see: those of its kv head are NaN, all others have the bits that they have without it, and the
    call takes no longer than a few others (walked through one slot after the other, 512 such rows at 30000 took 100 times as long)."""
    cfg, start = dec.DecoderConfig(q_heads=16, kv_heads=8), 30000
    gen = torch.Generator(device="cuda").manual_seed(0)
    pages = (start + tokens) // 16 + 1
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")   # noqa: E731
    keys, values = (torch.randn(2 * pages, 16, 8, 128, device="cuda", generator=gen).to(torch.bfloat16) for _ in range(2))
    qkv = torch.randn(2 * tokens, 32, 128, device="cuda", generator=gen).to(torch.bfloat16)
    one = torch.ones(128, dtype=torch.bfloat16, device="cuda")
    cos, sin = (torch.from_numpy(t).cuda() for t in dec.rope_tables(16 * pages, 128, cfg.rope_theta))
    op = dec.ChunkAttention(cfg, 2 * tokens, 16 * pages, pages, 16 * pages)
    table = torch.randperm(2 * pages, device="cuda", generator=gen).to(torch.int32).view(2, pages)

    def run():
        out = torch.zeros(2 * tokens, 16 * 128, dtype=torch.bfloat16, device="cuda")
        begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        begin.record()
        op.run(qkv.view(2 * tokens, -1), one, one, cos, sin, keys, values, table, ints(start, start), ints(0, tokens, 2 * tokens), out)
        end.record()
        torch.cuda.synchronize()
        return out.view(2, tokens, 16, 128), begin.elapsed_time(end)

    run()
    clean, _ = run()
    first = 0                                            # row of sequence 0 from which on results are NaN
    hit = torch.zeros(16, 128, dtype=torch.bool, device="cuda")
    hit[6:8] = True
    if what == "a key of the context":
        keys[table[0, 0], 5, 3, 17] = float("nan")
    elif what == "a key of the chunk":
        qkv[0, 16 + 3, 17] = float("nan")
    elif what == "a query":
        qkv[:tokens, 6:8, 17] = float("nan")
    else:
        values[table[0, 0], 5, 3, 17] = float("nan")
        hit[:] = False
        hit[6:8, 17] = True
    got, ms = run()
    assert got[0, first:, hit].isnan().all()
    assert torch.equal(got[0][:, ~hit], clean[0][:, ~hit]) and torch.equal(got[1], clean[1])
    assert ms < 5, f"{ms} ms"


def test_values_that_rows_do_not_see_and_values_that_they_see():
    """Infinities and NaN in both: rows before the last of them are what they are without it, dims with one that a row sees are NaN."""
    for lens, starts, heads in (([150], [700], (2, 1)), ([9], [3000], (4, 1)), ([150, 20], [40, 90], (16, 8))):
        c = Case(lens, starts, *heads, seed=31)
        h, kv = heads
        x = c.qkv.view(-1, h + 2 * kv, 128)
        for row, dim, value in ((lens[0] // 2, 3, float("inf")), (lens[0] - 1, 4, float("nan")), (lens[0] // 3, 5, -float("inf"))):
            x[row, h + kv, dim] = value
        c.values[c.table[0, 1], 2, 0, 6] = float("nan")
        c.check()


@pytest.mark.parametrize("lens,starts,heads", [([130], [0], (16, 8)), ([5, 2, 0], [700, 1000, 3], (4, 2))])
def test_a_call_that_says_how_far_its_rows_reach(lens, starts, heads):
    """An object for 40000 slots: told the call's context it gives the bits of an object for just that; rows behind what it is told are zeros and
    append nothing."""
    c = Case(lens, starts, *heads, seed=41)
    want = c.run()
    reach, width, room = max(n + s for n, s in zip(lens, starts)), 2500, 40000
    fitted = dec.ChunkAttention(c.cfg, c.rows, reach, c.width, c.positions_room)
    cos, sin = (torch.from_numpy(t).cuda() for t in dec.rope_tables(room, 128, c.cfg.rope_theta))
    large = dec.ChunkAttention(c.cfg, c.rows + 3, room, width, room)
    table = torch.full((c.batch, width), -1, dtype=torch.int32, device="cuda")
    table[:, :c.width] = c.table.cuda()
    results = []
    for op, more in ((fitted, {}), (large, dict(cos=cos, sin=sin, page_tables=table, context=reach)), (large, dict(cos=cos, sin=sin, page_tables=table)),
                     (large, dict(cos=cos, sin=sin, page_tables=table, context=reach - 1))):
        d = c.device()
        op.run(**dict(d, **more))
        results.append(d)
    a, b, far, less = results
    for name in ("out", "key_pages", "value_pages"):
        assert torch.equal(a[name], b[name])
    assert torch.equal(far["key_pages"], want["key_pages"]) and (far["out"].float() - want["out"].float()).norm() <= 2.0 ** -8 * want["out"].float().norm()
    last = int(np.argmax([n + s for n, s in zip(lens, starts)]))
    row = int(c.row_starts[last + 1]) - 1
    assert (less["out"][row] == 0).all() and torch.equal(less["out"][:row], b["out"][:row])
    slot = starts[last] + lens[last] - 1
    page, off = int(c.table[last, slot // 16]), slot % 16
    assert torch.equal(less["key_pages"][page, off].cpu(), c.keys[page, off])
    for context in (0, -1, room + 1):
        with pytest.raises(ValueError):
            large.run(**dict(c.device(), cos=cos, sin=sin, page_tables=table, context=context))


@pytest.mark.parametrize("rows,start", [(96, 40), (5, 900)])
def test_between_linears_that_use_tensor_memory_too(rows, start):
    """Linear, attention, linear without a wait on the host, as the layers of a prompt follow one another: all three take tensor memory and may come
    up before the kernels that they wait for are done."""
    c = Case([rows], [start], 16, 8, seed=51)
    gen = torch.Generator(device="cuda").manual_seed(1)
    mk = lambda n, k: garnet_b200.W4A16Linear().prepare(*garnet_b200.quantize_int4(torch.randn(n, k, device="cuda", generator=gen) / 32), n, k)   # noqa: E731
    qkv_lin, o_lin = mk(c.cfg.qkv_width, 1024), mk(1024, 2048)
    x = torch.randn(rows, 1024, device="cuda", generator=gen).to(torch.bfloat16)
    d, op = c.device(), c.op()
    steps = []
    for sync in (True, False):
        y = x
        for _ in range(12):
            qkv = qkv_lin.forward(y)
            if sync:
                torch.cuda.synchronize()
            out = torch.zeros(rows, 2048, dtype=torch.bfloat16, device="cuda")
            op.run(**dict(d, qkv=qkv, out=out), pdl=not sync)
            if sync:
                torch.cuda.synchronize()
            y = o_lin.forward(out)
            if sync:
                torch.cuda.synchronize()
        steps.append(y)
    torch.cuda.synchronize()
    assert steps[0].isfinite().all() and torch.equal(steps[0], steps[1])
