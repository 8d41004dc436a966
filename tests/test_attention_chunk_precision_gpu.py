"""How exact chunk attention is beside its results' own rounding: weights of 16 bits, sums that do not lose with the length of the context.

Tolerances, relative to the value or to mass = sum p |v|.  A result's rounding to bf16 is half a step, 2^-8 at most.  A weight enters its
product with v as two bf16 numbers, eight bits cut off and eight rounded: 2^-7 2^-8 = 2^-15 of it is left out at most.  The scores of
these cases stay below 2^4 in powers of two and their 128 products below 2^7: the tensor core cuts them eight times at 2^-17 each, 2^-14 in
the sum and 2^-17 in the exponent after the scale 1 / sqrt(128) log2 e = 2^-3; the exponent's own rounding and the exponential add 2^-19,
both in the result and in its denominator.  Sums of up to 600 positions lose 2^-23 of themselves per MMA of eight per 64 positions at most,
half of that on average over their growth: 2^-18.  In all 2^-15 (1 + 2 (1/4 + 1/16) + 1/8), less than 2^-14 of the mass."""
import numpy as np
import pytest
import torch

from garnet_b200 import decode as dec
from test_attention_chunk_gpu import Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lens,starts,heads", [([200, 33], [0, 350], (4, 2)), ([5, 9, 1], [500, 130, 63], (16, 8)), ([150] * 20, [37] * 20, (16, 8)), ([3], [590], (2, 1))])
def test_weights_keep_sixteen_bits(lens, starts, heads):
    c = Case(lens, starts, *heads, seed=11)
    d = c.run()
    want, tol, _, _ = c.expect()
    mass = (tol - 2.0 ** -8 * np.abs(want)) / (2.0 ** -8 + 2.0 ** -11)
    off = np.abs(d["out"].double().cpu().numpy() - want)
    bad = off > 2.0 ** -8 * np.abs(want) + 2.0 ** -14 * mass
    assert not bad.any(), f"{bad.sum()} of {bad.size}, the largest by {(off - 2.0 ** -8 * np.abs(want))[bad].max() / mass.max()}"


@pytest.mark.parametrize("tokens,context,heads", [(1, 131072, 8), (2048, 32768, 16), (2048, 65536, 16), (9000, 9000, 8)])
def test_long_sums_lose_no_more_than_short_ones(tokens, context, heads):
    """Equal weights (queries of zeros) and positive values of many magnitudes: a tensor core that adds them all loses 2^-28.5 per key, in one
    direction (12 of 1024 results were a step too low after 32768 keys).  Added in fp32 after every 64 steps of 64 keys, a sum loses 2^-23 of
    itself per MMA of 256 at most, half of that on average over its growth: 2^-16.  A quarter of that again for all that follows: sums of up
    to 32 parts and a division in fp32."""
    gen = torch.Generator(device="cuda").manual_seed(tokens)
    kv, pages = 8, context // 16 + 1
    cfg = dec.DecoderConfig(q_heads=heads, kv_heads=kv)
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")   # noqa: E731
    cos, sin = (torch.from_numpy(t).cuda() for t in dec.rope_tables(16 * pages, 128, cfg.rope_theta))
    one = torch.ones(128, dtype=torch.bfloat16, device="cuda")
    table = torch.randperm(pages, device="cuda", generator=gen).to(torch.int32)[None]
    op = dec.ChunkAttention(cfg, tokens, 16 * pages, pages, 16 * pages)
    for _ in range(3):
        values = torch.exp2(-12 * torch.rand(16 * pages, kv, 128, device="cuda", generator=gen)).to(torch.bfloat16)
        cache = torch.empty(pages, 16, kv, 128, dtype=torch.bfloat16, device="cuda")
        cache[table[0].long()] = values.view(pages, 16, kv, 128)
        qkv = torch.zeros(tokens, heads + 2 * kv, 128, dtype=torch.bfloat16, device="cuda")
        qkv[:, heads + kv:] = values[context - tokens:context]
        out = torch.zeros(tokens, heads * 128, dtype=torch.bfloat16, device="cuda")
        op.run(qkv.view(tokens, -1), one, one, cos, sin, torch.zeros_like(cache), cache, table, ints(context - tokens), ints(0, tokens), out)
        for row in {0, tokens // 2, tokens - 1}:
            want = values[:context - tokens + row + 1].double().mean(0).repeat_interleave(heads // kv, 0)
            got = out[row].view(heads, 128).double()
            half_step = torch.exp2(torch.floor(torch.log2(want)) - 8)
            over = ((got - want).abs() - half_step) / want
            assert float(over.max()) <= 1.25 * 2.0 ** -16, f"row {row}: {int((over > 1.25 * 2.0 ** -16).sum())} of {over.numel()}, {float(over.max())}"


def test_weights_and_sums_after_a_long_context():
    """General weights, up to 41000 positions, pages missing; two tiles, one tile in shares."""
    for lens, starts, heads in (([3], [41000], (2, 1)), ([1], [41000], (4, 4)), ([130], [7000], (4, 1))):
        c = Case(lens, starts, *heads, seed=12)
        c.table[0, 5::97] = -1
        d = c.run()
        want, tol, _, _ = c.expect()
        mass = (tol - 2.0 ** -8 * np.abs(want)) / (2.0 ** -8 + 2.0 ** -11)
        off = np.abs(d["out"].double().cpu().numpy() - want)
        bad = off > 2.0 ** -8 * np.abs(want) + 2.0 ** -14 * mass
        assert not bad.any(), f"{bad.sum()} of {bad.size}"


@pytest.mark.parametrize("lens,starts,heads", [([140], [9000], (2, 1)), ([1], [70000], (2, 1))])
def test_maxima_that_grow_along_a_long_context(lens, starts, heads):
    """Kept sums are scaled to larger and larger maxima.  Scores up to 2^6 in powers of two, products up to 2^9: cut eight times at 2^-15, 2^-15 in
    the exponent, twice (result and denominator), beside what the others have: less than 2^-13 of the mass."""
    c = Case(lens, starts, *heads, seed=13)
    at = torch.arange(starts[0])
    scale = 0.05 + 10 * at / starts[0]
    pages, offsets = c.table[0, (at // 16).long()].long(), at % 16
    c.keys[pages, offsets] = (c.keys[pages, offsets].float() * scale[:, None, None]).to(torch.bfloat16)
    d = c.run()
    want, tol, _, _ = c.expect()
    mass = (tol - 2.0 ** -8 * np.abs(want)) / (2.0 ** -8 + 2.0 ** -11)
    off = np.abs(d["out"].double().cpu().numpy() - want)
    bad = off > 2.0 ** -8 * np.abs(want) + 2.0 ** -13 * mass
    assert not bad.any(), f"{bad.sum()} of {bad.size}"


def test_keys_of_general_rows_are_the_rounded_float64_results():
    """Norm and RoPE of normal rows against float64, rounded to fp32 and then to bf16.  The kernel carries what its fp32 steps are short of: its
    fp32 number before the norm's rounding to bf16 is the rounded float64 one; before RoPE's it has been rounded twice, so that it is a
    neighbour in half of the cases at most, and one gap of fp32 numbers in 2^16 changes the bf16 number: 2^-17, 8 of 10^6 (plain fp32 steps
    have 25)."""
    cfg, tokens = dec.DecoderConfig(q_heads=8, kv_heads=8), 4096
    gen = torch.Generator(device="cuda").manual_seed(5)
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")   # noqa: E731
    cos, sin = (torch.from_numpy(t).cuda() for t in dec.rope_tables(tokens, 128, cfg.rope_theta))
    w = (1 + 0.2 * torch.randn(128, device="cuda", generator=gen)).to(torch.bfloat16)
    one = torch.ones(128, dtype=torch.bfloat16, device="cuda")
    op = dec.ChunkAttention(cfg, tokens, tokens, tokens // 16, tokens)
    off = plain = count = 0
    for _ in range(4):
        qkv = torch.randn(tokens, 24, 128, device="cuda", generator=gen).to(torch.bfloat16)
        keys, values = (torch.zeros(tokens // 16, 16, 8, 128, dtype=torch.bfloat16, device="cuda") for _ in range(2))
        out = torch.empty(tokens, 8 * 128, dtype=torch.bfloat16, device="cuda")
        op.run(qkv.view(tokens, -1), one, w, cos, sin, keys, values, torch.arange(tokens // 16, dtype=torch.int32, device="cuda")[None], ints(0), ints(0, tokens), out)
        x = qkv[:, 8:16].double()
        x = (x * (x.pow(2).mean(-1, keepdim=True) + float(np.float32(cfg.eps))).rsqrt() * w.double()).float().to(torch.bfloat16).double()
        a, b, c, s = x[..., :64], x[..., 64:], cos.double()[:, None], sin.double()[:, None]
        want = torch.cat([a * c - b * s, b * c + a * s], -1).float().to(torch.bfloat16)
        off += int((keys.view(tokens, 8, 128) != want).sum())
        y = qkv[:, 8:16].float()
        y = (y / torch.sqrt((y * y).mean(-1, keepdim=True) + cfg.eps) * w.float()).to(torch.bfloat16).float()
        a, b, c, s = y[..., :64], y[..., 64:], cos[:, None], sin[:, None]
        plain += int((torch.cat([a * c - b * s, b * c + a * s], -1).to(torch.bfloat16) != want).sum())
        count += want.numel()
    print(f"{off / count * 1e6:.1f} of 10^6, plain fp32 steps {plain / count * 1e6:.1f}")
    assert off <= 8e-6 * count, f"{off} of {count}"


def test_squares_beyond_fp32():
    """Heads whose squares overflow come out as zeros, as the one-token kernel has them; an infinity among them is NaN."""
    cfg = dec.DecoderConfig(q_heads=4, kv_heads=2)
    gen = torch.Generator(device="cuda").manual_seed(6)
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")   # noqa: E731
    cos, sin = (torch.from_numpy(t).cuda() for t in dec.rope_tables(64, 128, cfg.rope_theta))
    w = torch.full((128,), 3.0, dtype=torch.bfloat16, device="cuda")
    qkv = torch.randn(3, 8, 128, device="cuda", generator=gen)
    qkv[0, 4] *= 2.0 ** 66                       # a key
    qkv[1, 0] *= 2.0 ** 126                      # a query: its product with the weight overflows too
    qkv[1, 4, 7] = 2.0 ** 65                     # one value of a key
    qkv[2, 5, 9] = float("inf")
    qkv = qkv.to(torch.bfloat16)
    got, want = [], []
    for results, op, more in ((got, dec.ChunkAttention(cfg, 3, 64, 4, 64), (ints(0, 1, 2, 3),)), (want, dec.PagedAttention(cfg, 3, 64, 4, 64), ())):
        keys, values = (torch.zeros(12, 16, 2, 128, dtype=torch.bfloat16, device="cuda") for _ in range(2))
        out = torch.zeros(3, 4 * 128, dtype=torch.bfloat16, device="cuda")
        op.run(qkv.view(3, -1), w, w, cos, sin, keys, values, torch.arange(12, dtype=torch.int32, device="cuda").view(3, 4), ints(5, 0, 20), *more, out)
        results += [out.view(3, 4, 128), keys]
    assert (got[1][0, 5, 0] == 0).all() and (got[1][4, 0, 0] == 0).all() and got[1][9, 4, 1].isnan().any()
    assert torch.equal(got[1].isnan(), want[1].isnan()) and torch.equal(got[1][4, 0, 0], want[1][4, 0, 0])
    assert torch.equal(got[0][:2], want[0][:2])          # one slot each: the value itself
    # a score of NaN: softmax is NaN (the one-token kernel leaves out what has such a sum)
    assert got[0][2, 2:].isnan().all() and not got[0][2, :2].isnan().any()
