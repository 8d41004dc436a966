"""The page pool (garnet_b200_cache_*) against a plain model of it: whole numbers and copied bytes, compared exactly."""
import numpy as np
import pytest
import torch

import garnet_b200
from garnet_b200 import cache

pytestmark = pytest.mark.gpu
OK, REFUSED, FULL = 0, 1, 5


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


class Model:
    """The operators' definitions on host arrays, entry after entry."""

    def __init__(self, pool, keys, values):
        self.ps, self.width = pool.opt.page_size, pool.opt.max_logical_pages
        self.table, self.lengths, self.refs = (t.cpu().numpy().copy() for t in (pool.page_tables, pool.lengths, pool.refcounts))
        self.data = [t.cpu().clone() for t in (*keys, *values)]

    def grant(self, needs):
        """First fit in list order: (status, pages) per entry, None for a refused one."""
        free, at, result = [int(p) for p in np.flatnonzero(self.refs <= 0)], 0, []
        for need in needs:
            if need is None:
                result.append((REFUSED, []))
                continue
            got = need == 0 or at + need <= len(free)
            result.append((OK, free[at:at + need]) if got else (FULL, []))
            at += need
        return result

    def extend(self, seqs, tokens):
        needs, named = [], set()
        for s, n in zip(seqs, tokens):
            bad = not 0 <= s < len(self.lengths) or s in named or n < 0 or self.lengths[s] + n > self.width * self.ps
            needs.append(None if bad else -(-int(self.lengths[s] + n) // self.ps) - -(-int(self.lengths[s]) // self.ps))
            named.add(s)
        status = []
        for (st, pages), s, n in zip(self.grant(needs), seqs, tokens):
            status.append(st)
            if st == OK:
                have = -(-int(self.lengths[s]) // self.ps)
                self.table[s, have:have + len(pages)] = pages
                self.refs[pages] = 1
                self.lengths[s] += n
        return status

    def fork(self, parents, children):
        needs, named = [], set()
        for p, c in zip(parents, children):
            inside = 0 <= p < len(self.lengths) and 0 <= c < len(self.lengths)
            bad = not inside or c in named or p in children or self.lengths[c] != 0
            needs.append(None if bad else int(self.lengths[p] % self.ps > 0))
            named.add(c)
        status = []
        for (st, pages), p, c in zip(self.grant(needs), parents, children):
            status.append(st)
            if st != OK:
                continue
            full, part = divmod(int(self.lengths[p]), self.ps)
            self.table[c, :full] = self.table[p, :full]
            np.add.at(self.refs, self.table[p, :full], 1)
            if part:
                src = int(self.table[p, full])
                self.table[c, full], self.refs[pages[0]] = pages[0], 1
                for d in self.data:
                    d[pages[0], :part] = d[src, :part]
            self.lengths[c] = self.lengths[p]
        return status

    def free(self, seqs):
        for s in seqs:
            if 0 <= s < len(self.lengths):
                held = -(-int(self.lengths[s]) // self.ps)
                np.subtract.at(self.refs, self.table[s, :held], 1)
                self.table[s, :held] = -1
                self.lengths[s] = 0

    def compact(self):
        live = int((self.refs > 0).sum())
        src, dst = [p for p in np.flatnonzero(self.refs > 0) if p >= live], [p for p in np.flatnonzero(self.refs <= 0) if p < live]
        to = np.arange(len(self.refs))
        for s, d in zip(src, dst):
            to[s] = d
            self.refs[d], self.refs[s] = self.refs[s], 0
            for t in self.data:
                t[d] = t[s]
        self.table = np.where(self.table >= 0, to[np.maximum(self.table, 0)], self.table)
        return live

    def copy(self, src, dst):
        pages = self.data[0].shape[0]
        for s, d in zip(src, dst):
            if 0 <= s < pages and 0 <= d < pages:
                for t in self.data:
                    t[d] = t[s]

    def same(self, pool, keys, values):
        assert np.array_equal(pool.page_tables.cpu().numpy(), self.table)
        assert np.array_equal(pool.lengths.cpu().numpy(), self.lengths)
        assert np.array_equal(pool.refcounts.cpu().numpy(), self.refs)
        for got, want in zip((*keys, *values), self.data):
            assert torch.equal(got.cpu().view(torch.int16), want.view(torch.int16))


def make(layers, pages, page_size, kv_heads, head_dim, sequences, width, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    shape = (pages, page_size, kv_heads, head_dim)
    keys, values = ([torch.randint(-30000, 30000, shape, device="cuda", generator=gen, dtype=torch.int16).view(torch.bfloat16) for _ in range(layers)]
                    for _ in range(2))
    pool = cache.PagePool(keys, values, sequences, width)
    return pool, keys, values, Model(pool, keys, values)


@pytest.mark.parametrize("layers,pages,page_size,kv_heads,head_dim", [(2, 60, 16, 2, 128), (1, 33, 1, 1, 8), (3, 200, 5, 1, 64), (1, 7, 64, 8, 128), (2, 1500, 3, 1, 24)])
def test_random_use(layers, pages, page_size, kv_heads, head_dim):
    """Two hundred random calls: lists with repeated, wrong and exhausted entries among them."""
    sequences, width = 24, max(2, pages // 4)
    pool, keys, values, model = make(layers, pages, page_size, kv_heads, head_dim, sequences, width)
    r = np.random.RandomState(pages)
    most = max(2, width * page_size // 3)
    for step in range(200):
        what = r.randint(5)
        n = r.randint(1, 9)
        seqs = [int(s) for s in r.randint(-1 if r.rand() < 0.2 else 0, sequences + (r.rand() < 0.2), n)]
        if what == 0:
            tokens = [int(t) for t in r.randint(-1 if r.rand() < 0.1 else 0, most, n)]
            assert pool.extend(ints(seqs), ints(tokens)).tolist() == model.extend(seqs, tokens)
        elif what == 1:
            empty = [s for s in range(sequences) if model.lengths[s] == 0]
            children = [int(r.choice(empty)) if empty and r.rand() < 0.9 else int(r.randint(sequences)) for _ in seqs]
            assert pool.fork(ints(seqs), ints(children)).tolist() == model.fork(seqs, children)
        elif what == 2:
            seqs = seqs[:1 + n // 3]
            pool.free(ints(seqs))
            model.free(seqs)
        elif what == 3:
            assert pool.compact().tolist() == [model.compact()]
        else:
            src, dst = ([int(p) for p in r.randint(-1, pages + 1, n)] for _ in range(2))
            pool.copy_pages(ints(src), ints(dst))
            model.copy(src, dst)
        if step % 10 == 9:
            model.same(pool, keys, values)
    model.same(pool, keys, values)


@pytest.mark.parametrize("count", [1, 40, 700])
@pytest.mark.parametrize("kind", ["apart", "chain", "same destination", "swap", "into itself"])
def test_copies_in_the_order_of_the_list(count, kind):
    pages = 1500
    pool, keys, values, model = make(3, pages, 4, 1, 64, 4, 4, seed=count)
    r = np.random.RandomState(count)
    perm = [int(p) for p in r.permutation(pages)]
    src, dst = perm[:count], perm[count:2 * count]
    if kind == "chain":
        src, dst = perm[:count], perm[1:count + 1]
    elif kind == "same destination":
        dst = [dst[0]] * count
    elif kind == "swap":
        src, dst = src + dst, dst + src
    elif kind == "into itself":
        dst = src
    pool.copy_pages(ints(src), ints(dst))
    model.copy(src, dst)
    model.same(pool, keys, values)


def test_a_large_pool_and_long_lists():
    """More entries than the planning CTA has threads, pages in every warp's share, 40000 pages."""
    sequences, width, pages = 3000, 24, 40000
    pool, keys, values, model = make(1, pages, 2, 1, 8, sequences, width)
    r = np.random.RandomState(1)
    tokens = [int(t) for t in r.randint(0, 30, sequences)]
    order = [int(s) for s in r.permutation(sequences)]
    assert pool.extend(ints(order), ints(tokens)).tolist() == model.extend(order, tokens)
    gone = order[::2]
    pool.free(ints(gone))
    model.free(gone)
    model.same(pool, keys, values)
    parents = [order[1 + 2 * int(i)] for i in r.randint(0, sequences // 2, len(gone))]
    assert pool.fork(ints(parents), ints(gone)).tolist() == model.fork(parents, gone)
    model.same(pool, keys, values)
    gone = order[1::3]
    pool.free(ints(gone))
    model.free(gone)
    assert pool.compact().tolist() == [model.compact()]
    model.same(pool, keys, values)
    rest = [s for s in range(sequences) if model.lengths[s]]
    grow = [int(t) for t in r.randint(0, 18, len(rest))]
    grow[len(rest) // 2] = 10 ** 6                       # does not fit the row: refused, the others are served
    assert pool.extend(ints(rest), ints(grow)).tolist() == model.extend(rest, grow)
    model.same(pool, keys, values)


def test_a_pool_that_runs_out():
    pool, keys, values, model = make(1, 10, 4, 1, 8, 8, 10)
    seqs, tokens = [0, 1, 2, 3, 4], [9, 16, 20, 0, 4]      # 3 + 4 pages, 5 do not fit, 0 pages, then none are given any more
    assert pool.extend(ints(seqs), ints(tokens)).tolist() == model.extend(seqs, tokens) == [OK, OK, FULL, OK, FULL]
    assert pool.extend(ints([5]), ints([12])).tolist() == model.extend([5], [12]) == [OK]     # the rest
    parents, children = [0, 1, 5], [6, 7, 2]               # a partial last page: none is left; full pages are shared all the same
    assert pool.fork(ints(parents), ints(children)).tolist() == model.fork(parents, children) == [FULL, OK, OK]
    model.same(pool, keys, values)
    assert pool.compact().tolist() == [model.compact()] == [10]
    model.same(pool, keys, values)


def test_one_tensor_for_all_layers_and_captured_calls():
    """The pages of all layers as one tensor, and a captured extend - fork - free that is replayed on other lists."""
    gen = torch.Generator(device="cuda").manual_seed(0)
    keys, values = (torch.randn(3, 50, 16, 2, 128, device="cuda", generator=gen).to(torch.bfloat16) for _ in range(2))
    pool = cache.PagePool(keys, values, 6, 8)
    model = Model(pool, keys, values)
    seqs, tokens, parents, children, gone = ints([0, 1]), ints([40, 23]), ints([0, 0]), ints([2, 3]), ints([1, 2])

    def calls():
        return pool.extend(seqs, tokens), pool.fork(parents, children), (pool.free(gone), pool.compact())[1]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = calls()
    torch.cuda.current_stream().wait_stream(side)
    assert [t.tolist() for t in first] == [model.extend([0, 1], [40, 23]), model.fork([0, 0], [2, 3]), (model.free([1, 2]), [model.compact()])[1]]
    model.same(pool, keys, values)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        held = calls()
    model.same(pool, keys, values)                         # capture runs nothing
    seqs.copy_(ints([1, 0])), tokens.copy_(ints([5, 100])), parents.copy_(ints([3, 0])), children.copy_(ints([2, 5])), gone.copy_(ints([0, 0]))
    g.replay()
    torch.cuda.synchronize()
    want = [model.extend([1, 0], [5, 100]), model.fork([3, 0], [2, 5]), (model.free([0, 0]), [model.compact()])[1]]
    assert [t.tolist() for t in held] == want
    model.same(pool, keys, values)


def test_pages_behind_two_gigabytes():
    """Byte offsets above 2^32: a cache of 4.5 GB, pages copied to and from its end."""
    pages, shape = 70000, (16, 16, 128)                    # 64 KB per page
    keys = torch.zeros(1, pages, *shape, dtype=torch.bfloat16, device="cuda")
    values = torch.zeros_like(keys)
    pool = cache.PagePool(keys, values, 4, 8)
    gen = torch.Generator(device="cuda").manual_seed(0)
    keys[0, 5] = torch.randn(*shape, device="cuda", generator=gen).to(torch.bfloat16)
    values[0, pages - 1] = torch.randn(*shape, device="cuda", generator=gen).to(torch.bfloat16)
    want_k, want_v = keys[0, 5].clone(), values[0, pages - 1].clone()
    pool.copy_pages(ints([5, pages - 1]), ints([pages - 2, 6]))
    torch.cuda.synchronize()
    assert torch.equal(keys[0, pages - 2], want_k) and torch.equal(values[0, 6], want_v)
    # a live page at the end comes to the front
    pool.refcounts[pages - 2] = 2
    pool.page_tables[:2, 0] = pages - 2
    pool.lengths[:2] = 16
    assert pool.compact().tolist() == [1]
    assert pool.page_tables[:2, 0].tolist() == [0, 0] and pool.refcounts[0] == 2 and pool.refcounts[pages - 2] == 0
    assert torch.equal(keys[0, 0], want_k)


def test_pages_that_the_host_holds_are_found_again():
    """Pages whose only reference is a count of the host's: moved together with the others, found by `moved`, not handed out, given back."""
    pool, keys, values, model = make(2, 40, 4, 1, 64, 6, 20)
    seqs = [0, 1, 2, 3]
    assert pool.extend(ints(seqs), ints([30, 25, 17, 40])).tolist() == model.extend(seqs, [30, 25, 17, 40])
    pinned = [int(model.table[1, 0]), int(model.table[2, 4]), int(model.table[3, 9])]
    for p in pinned:
        pool.refcounts[p] += 1
        model.refs[p] += 1
    held = [[t[p].clone() for t in (*keys, *values)] for p in pinned]
    pool.free(ints([0, 1, 2]))
    model.free([0, 1, 2])
    before = model.refs.copy()
    moved = torch.full((40,), -9, dtype=torch.int32, device="cuda")
    assert pool.compact(moved).tolist() == [model.compact()] == [12]
    model.same(pool, keys, values)
    to = moved.tolist()
    live = [p for p in range(40) if before[p] > 0]
    assert sorted(to[p] for p in live) == list(range(12)) and all(to[p] == p for p in range(40) if before[p] <= 0 or p < 12)
    assert [to[p] for p in live if p >= 12] == [p for p in range(12) if before[p] <= 0]
    assert pool.extend(ints([5]), ints([70])).tolist() == model.extend([5], [70]) == [OK]
    model.same(pool, keys, values)
    for p, want in zip(pinned, held):
        assert all(torch.equal(t[to[p]].view(torch.int16), w.view(torch.int16)) for t, w in zip((*keys, *values), want))
        assert to[p] not in pool.page_tables[5].tolist()
        pool.refcounts[to[p]] -= 1
        model.refs[to[p]] -= 1
    # nothing moves now that pages 0 .. live - 1 are live but for those that were given back; a pool without holes says so
    pool.free(ints([3]))
    model.free([3])
    assert pool.compact(moved).tolist() == [model.compact()]
    model.same(pool, keys, values)
    assert pool.compact(moved).tolist() == [model.compact()] and moved.tolist() == list(range(40))
    for bad in (moved[:39], moved.long(), moved.cpu()):
        with pytest.raises(ValueError):
            pool.compact(bad)


def test_refusals():
    pool, keys, values, _ = make(1, 8, 4, 1, 8, 4, 4)
    for bad in (lambda: pool.extend(ints([0, 1]), ints([1])), lambda: pool.extend(torch.zeros(1, dtype=torch.int64, device="cuda"), ints([1])),
                lambda: pool.fork(ints([0]), ints([[1]])), lambda: pool.free(torch.zeros(1, dtype=torch.int32)), lambda: pool.free(ints([0] * 5)),
                lambda: pool.copy_pages(ints([0, 1]), ints([1])), lambda: cache.PagePool(keys, values + values, 4, 4), lambda: cache.PagePool([], [], 4, 4),
                lambda: cache.PagePool([keys[0].cpu()], values, 4, 4), lambda: cache.PagePool([keys[0].transpose(0, 1)], values, 4, 4),
                lambda: cache.PagePool([keys[0][:4]], values, 4, 4), lambda: cache.PagePool([keys[0][:0]], [values[0][:0]], 4, 4)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(garnet_b200.GarnetB200Error):       # 8 bytes per position
        cache.PagePool([torch.zeros(4, 4, 1, 4, dtype=torch.bfloat16, device="cuda")], [torch.zeros(4, 4, 1, 4, dtype=torch.bfloat16, device="cuda")], 4, 4)
    with pytest.raises(garnet_b200.GarnetB200Error):
        cache.PagePool(keys, values, 0, 4)
    assert pool.extend(ints([]), ints([])).tolist() == []
    pool.free(ints([]))
    pool.copy_pages(ints([]), ints([]))
