"""garnet_b200_log_probs against float64: log probability and rank of given tokens, entropy, top alternatives.

Tolerances.  With u = 2^-24, d = (x - max) / T and E the mean under softmax: an fp32 d is off by 3 u |d| at most (difference, product with
1 / T, product with log2 e), its exponential by 4 u more, and a sum of n terms in chains of n / 256 and a tree by (n / 256 + 16) u of
itself.  So log S is off by u (3 E|d| + n / 256 + 20), a log probability by u (4 |lp| + 3 |d_t|) more, and the entropy, whose second
sum has terms e^d d, by u (E|d| (n / 256 + 24) + 3 E d^2) more than log S."""
import numpy as np
import pytest
import torch

import garnet_b200
from garnet_b200 import decode as dec

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def oracle(x, targets, k, temperature):
    """Everything of the operator in float64, and the tolerances, for x [rows, vocab] without NaN and +inf."""
    x = x.astype(np.float64)
    z = x / temperature
    top = z.max(1, keepdims=True)
    empty = np.isneginf(top[:, 0])
    d = z - np.where(np.isneginf(top), 0.0, top)
    e = np.exp(d)
    s = e.sum(1)
    with np.errstate(divide="ignore", invalid="ignore"):
        log_s = np.log(s)
        p = e / s[:, None]
        lp = d - log_s[:, None]
        ad = np.where(e > 0, np.abs(d), 0.0)
        entropy = np.where(empty, 0.0, -(p * np.where(e > 0, lp, 0.0)).sum(1))
        mean_d, mean_d2 = (p * ad).sum(1), (p * ad * ad).sum(1)
    lp[empty] = -np.inf
    lp[lp < -np.finfo(np.float32).max] = -np.inf     # beyond fp32
    n = x.shape[1]
    tol_s = U * (3 * mean_d + n / 256 + 20)
    tol_h = tol_s + U * (mean_d * (n / 256 + 24) + 3 * mean_d2)
    with np.errstate(invalid="ignore"):
        tol_lp = tol_s[:, None] + U * (4 * np.abs(lp) + 3 * np.abs(d))
    tol_lp[~np.isfinite(lp)] = 0
    order = np.argsort(-x, axis=1, kind="stable")[:, :k]
    given = (targets >= 0) & (targets < n)
    t = np.where(given, targets, 0)
    rows = np.arange(x.shape[0])
    rank = np.where(given, (x > x[rows, t][:, None]).sum(1) + 1, 0)
    return dict(lp=np.where(given, lp[rows, t], 0.0), tol=np.where(given, tol_lp[rows, t], 0.0), rank=rank, entropy=entropy,
                tol_h=np.where(empty, 0.0, tol_h), ids=order, top=np.take_along_axis(lp, order, 1), tol_top=np.take_along_axis(tol_lp, order, 1))


def near(got, want, tol, what):
    got = got.double().cpu().numpy()
    same = got == want     # infinities
    with np.errstate(invalid="ignore"):
        assert (same | (np.abs(got - want) <= tol)).all(), f"{what}: {np.nanmax(np.abs(got - want) - tol)}"


def check(logits, targets, k, temperature=1.0):
    r = dec.log_probs(logits, targets, top_k=k, temperature=temperature)
    temperature = float(1 / np.float64(np.float32(1.0 / np.float32(temperature))))     # the kernel multiplies by fp32(1 / T)
    want = oracle(logits.float().cpu().numpy(), targets.cpu().numpy(), k, temperature)
    near(r.log_probs, want["lp"], want["tol"], "log probability")
    near(r.entropy, want["entropy"], want["tol_h"], "entropy")
    near(r.top_log_probs, want["top"], want["tol_top"], "alternatives")
    assert np.array_equal(r.ranks.cpu().numpy(), want["rank"])
    assert np.array_equal(r.top_ids.cpu().numpy(), want["ids"])
    return r


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,vocab,pad,k", [(1, 1, 0, 1), (1, 151936, 0, 20), (3, 32003, 5, 32), (5, 2, 1, 2), (37, 257, 0, 7), (300, 1000, 8, 5),
                                              (2, 8192, 0, 0), (20, 65537, 3, 1), (160, 4099, 0, 32), (1, 31, 0, 31)])
def test_values(dtype, rows, vocab, pad, k):
    gen = torch.Generator(device="cuda").manual_seed(rows * 1000 + vocab)
    x = (torch.randn(rows, vocab + pad, device="cuda", generator=gen) * 3).to(dtype)
    x[:, vocab:] = 1000.0          # what lies between the rows is not theirs
    targets = torch.randint(0, vocab, (rows,), dtype=torch.int32, device="cuda", generator=gen)
    check(x[:, :vocab], targets, k)
    check(x[:, :vocab], targets, k, 0.6)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows", [1, 200])
def test_orders_and_ties(dtype, rows):
    """Rows in ascending and descending order, constant rows, few distinct values, single peaks, large magnitudes."""
    n = 5003
    base = torch.linspace(-20, 20, n, device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(3)
    kinds = [base, base.flip(0), torch.zeros(n, device="cuda"), torch.full((n,), -7.5, device="cuda"),
             torch.randint(-2, 3, (n,), device="cuda", generator=gen).float(), torch.full((n,), -30.0, device="cuda").index_fill(0, torch.tensor([4321], device="cuda"), 40.0),
             base * 500, torch.where(torch.arange(n, device="cuda") % 2 == 0, 0.0, -0.0)]
    x = torch.stack([kinds[i % len(kinds)] for i in range(max(rows, len(kinds)))]).to(dtype)[:max(rows, len(kinds))]
    targets = torch.randint(0, n, (x.shape[0],), dtype=torch.int32, device="cuda", generator=gen)
    targets[5] = 4321
    if rows == 1:
        for i in range(x.shape[0]):
            check(x[i:i + 1], targets[i:i + 1], 32)
    else:
        check(x, targets, 32)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows_each,temperature", [(1, 1.0), (60, 1.0), (1, 60000.0), (1, 2e-6)])
def test_masked_rows(dtype, rows_each, temperature):
    """-inf and the type's lowest value as masks, masks that leave one value or none, rows without a target."""
    n, inf, lowest = 3001, float("inf"), torch.finfo(dtype).min
    gen = torch.Generator(device="cuda").manual_seed(9)
    x = torch.randn(9, n, device="cuda", generator=gen)
    x[0, ::2] = -inf
    x[1] = -inf
    x[2] = -inf
    x[2, 1777] = -3.0
    x[3, 5:] = lowest
    x[4] = lowest
    x[5, :2990] = -inf
    x[6] = lowest                       # one mask over the other
    x[6, 100:2900] = -inf
    x[7] = -lowest
    x[8, :2000], x[8, 2000:] = lowest, -lowest
    x = x.to(dtype).repeat(rows_each, 1)
    targets = torch.tensor([0, 3, 1777, 7, -1, n, 5, 6, 2999], dtype=torch.int32, device="cuda").repeat(rows_each)
    r = check(x, targets, 32, temperature)
    assert r.entropy[1] == 0 and r.log_probs[1] == -inf and r.log_probs[2] == 0 and r.log_probs[4] == 0 and r.ranks[4] == 0 and r.ranks[5] == 0


@pytest.mark.parametrize("rows_each", [1, 60])
def test_nan_and_infinity(rows_each):
    n, inf, nan = 999, float("inf"), float("nan")
    x = torch.linspace(-3, 3, n, device="cuda").repeat(4, 1)
    x[0, 500] = nan
    x[1, 7] = inf
    x[2] = nan
    x[3] = nan
    x[3, [4, 900]] = torch.tensor([1.0, -inf], device="cuda")
    x = x.repeat(rows_each, 1)
    r = dec.log_probs(x, torch.zeros(4 * rows_each, dtype=torch.int32, device="cuda"), top_k=4)
    assert r.log_probs.isnan().all() and r.entropy.isnan().all() and r.top_log_probs.isnan().all()
    ids = r.top_ids.view(rows_each, 4, 4)
    for i in range(rows_each):
        assert ids[i, 0].tolist() == [998, 997, 996, 995]
        assert ids[i, 1].tolist() == [7, 998, 997, 996]
        assert ids[i, 2].tolist() == [-1] * 4
        assert ids[i, 3].tolist() == [4, 900, -1, -1]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,offset", [(1, 0), (3, 5), (700, 3)])
def test_ranks_beside_nan(dtype, rows, offset):
    """The rank counts the larger logits of the whole row, wherever a NaN lies and however the row is cut into blocks and parts; nothing
    is larger than a NaN."""
    n = 20011
    gen = torch.Generator(device="cuda").manual_seed(rows)
    flat = torch.randn(rows * n + offset, device="cuda", generator=gen).to(dtype)
    x = flat[offset:].view(rows, n)
    nans = torch.randint(0, n, (rows, 3), device="cuda", generator=gen)
    x.scatter_(1, nans, float("nan"))
    targets = torch.randint(0, n, (rows,), dtype=torch.int32, device="cuda", generator=gen)
    targets[rows // 2] = nans[rows // 2, 0]
    r = dec.log_probs(x, targets, top_k=2)
    want = (x > x.gather(1, targets.long()[:, None])).sum(1) + 1
    assert torch.equal(r.ranks.long(), want) and int(r.ranks[rows // 2]) == 1
    assert r.log_probs.isnan().all() and r.entropy.isnan().all()


def test_without_targets_unaligned_and_many_rows():
    gen = torch.Generator(device="cuda").manual_seed(2)
    flat = torch.randn(70000 * 17 + 3, device="cuda", generator=gen).to(torch.bfloat16)
    x = flat[3:].view(70000, 17)         # rows that start on any 2-byte boundary; more rows than a grid dimension of 65535
    targets = torch.randint(0, 17, (70000,), dtype=torch.int32, device="cuda", generator=gen)
    check(x, targets, 3)
    r = dec.log_probs(x)
    assert r.log_probs is None and r.ranks is None and r.top_ids.shape == (70000, 0)
    assert torch.equal(r.entropy, dec.log_probs(x, targets, top_k=5).entropy)
    empty = dec.log_probs(x[:0], targets[:0], top_k=2)
    assert empty.entropy.shape == (0,) and empty.top_ids.shape == (0, 2)


def test_same_bits_every_time_captured_and_on_another_stream():
    gen = torch.Generator(device="cuda").manual_seed(4)
    x = (torch.randn(5, 151936, device="cuda", generator=gen) * 2).to(torch.bfloat16)
    targets = torch.randint(0, 151936, (5,), dtype=torch.int32, device="cuda", generator=gen)
    first = dec.log_probs(x, targets, top_k=9)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        other = dec.log_probs(x, targets, top_k=9, pdl=True)
    side.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        held = dec.log_probs(x, targets, top_k=9)
    y = x.clone()
    x.neg_()
    g.replay()
    torch.cuda.synchronize()
    assert not torch.equal(held.entropy, first.entropy)
    x.copy_(y)
    g.replay()
    torch.cuda.synchronize()
    for a, b, c in zip(first, other, held):
        assert torch.equal(a, b) and torch.equal(a, c)


def test_top_one_is_the_greedy_token():
    gen = torch.Generator(device="cuda").manual_seed(6)
    x = torch.randn(8, 151936, device="cuda", generator=gen).to(torch.bfloat16)
    token = torch.zeros(8, dtype=torch.int32, device="cuda")
    dec.argmax_bf16(x, token)
    r = dec.log_probs(x, token, top_k=1)
    assert torch.equal(r.top_ids[:, 0], token) and torch.equal(r.top_log_probs[:, 0], r.log_probs) and (r.ranks == 1).all()


def test_refusals():
    x = torch.zeros(2, 64, device="cuda")
    t = torch.zeros(2, dtype=torch.int32, device="cuda")
    for bad in (lambda: dec.log_probs(x, t.long()), lambda: dec.log_probs(x, t[:1]), lambda: dec.log_probs(x.double(), t), lambda: dec.log_probs(x.T, t),
                lambda: dec.log_probs(x.cpu(), t), lambda: dec.log_probs(x[0], t), lambda: dec.log_probs(x, t.cpu())):
        with pytest.raises(ValueError):
            bad()
    for kw in (dict(top_k=33), dict(top_k=-1), dict(temperature=0.0), dict(temperature=float("nan")), dict(temperature=float("inf"))):
        with pytest.raises(garnet_b200.GarnetB200Error):
            dec.log_probs(x, t, **kw)
    with pytest.raises(garnet_b200.GarnetB200Error):
        dec.log_probs(x[:, :5], t, top_k=6)
