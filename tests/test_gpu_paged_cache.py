"""Page operations of the key/value cache on the GPU against list bookkeeping (tests/drafting.py).

Every operation moves bits and counts integers, so all comparisons are exact."""
from __future__ import annotations

import random

import pytest
import torch

import drafting
import tsac_cuda

pytestmark = pytest.mark.gpu

ROW = 64  # values of a row in the small tests: kv_heads 1, head_dim 64


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


class Pair:
    """A cache on the GPU and its list bookkeeping, stepped together and compared."""

    def __init__(self, pages=24, page_size=8, sequences=6, max_pages=8, layers=2, dtype=torch.bfloat16, heads=1, dim=ROW):
        self.gpu = tsac_cuda.PagedCache.empty(layers, pages, page_size, heads, dim, sequences, max_pages, dtype=dtype)
        self.book = drafting.Book(pages, page_size, sequences)
        self.layers, self.heads, self.dim, self.dtype = layers, heads, dim, dtype
        self.serial = 0
        self.errors = torch.zeros(1, dtype=torch.int32, device="cuda")

    def word(self):
        value = int(self.errors.item())
        self.errors.zero_()
        return value

    def values(self, serial, layer, which):
        """The row that append number `serial` stored: distinct in every layer, for keys and for values."""
        generator = torch.Generator().manual_seed(serial * 64 + layer * 2 + which)
        return torch.randn((self.heads, self.dim), generator=generator).to(self.dtype)

    def reserve(self, entries, **more):
        self.gpu.reserve(ints([m for _, m in entries]), sequences=ints([s for s, _ in entries]), error_word=self.errors, **more)
        return self.book.reserve(entries)

    def append(self, entries):
        most = max(n for _, n in entries)
        serials = []
        for s, n in entries:
            serials.append([self.serial + k for k in range(n)])
            self.book.append(s, serials[-1])
            self.serial += n
        for layer in range(self.layers):
            rows = torch.full((2, len(entries), most, self.heads, self.dim), float("nan"), dtype=self.dtype)
            for i, line in enumerate(serials):
                for n, serial in enumerate(line):
                    for which in (0, 1):
                        rows[which, i, n] = self.values(serial, layer, which)
            rows = rows.cuda()
            self.gpu.append(layer, rows[0], rows[1], nodes=ints([n for _, n in entries]),
                            sequences=ints([s for s, _ in entries]), error_word=self.errors)

    def keep(self, entries, width=None):
        width = width or max(1, max(len(p) for _, p in entries))
        path = [list(p) + [-7] * (width - len(p)) for _, p in entries]
        self.gpu.keep(ints(path), ints([len(p) for _, p in entries]), sequences=ints([s for s, _ in entries]),
                      error_word=self.errors)
        for s, p in entries:
            self.book.keep(s, p)

    def fork(self, pairs):
        self.gpu.fork(ints([a for a, _ in pairs]), ints([b for _, b in pairs]), error_word=self.errors)
        for a, b in pairs:
            self.book.fork(a, b)

    def release(self, entries):
        self.gpu.release(sequences=ints([s for s, _ in entries]), positions=ints([p for _, p in entries]), error_word=self.errors)
        for s, p in entries:
            self.book.release(s, p)

    def compact(self):
        assert int(self.gpu.compact(error_word=self.errors).item()) == self.book.compact()

    def check(self, rows=True):
        assert self.word() == 0
        assert self.gpu.refs.tolist() == self.book.refs
        assert self.gpu.lengths.tolist() == self.book.lengths
        assert self.gpu.counts.tolist() == [len(h) for h in self.book.held]
        width = self.gpu.max_pages
        assert self.gpu.tables.tolist() == [h + [-1] * (width - len(h)) for h in self.book.held]
        if rows:
            pool = self.gpu.pool.cpu()
            for (page, slot), serial in self.book.rows.items():
                if self.book.refs[page] > 0:
                    for layer in range(self.layers):
                        for which in (0, 1):
                            assert torch.equal(pool[layer, which, page, slot], self.values(serial, layer, which)), (page, slot)

    def grow(self, entries):
        """reserve, append and keep everything."""
        assert self.reserve(entries)
        self.append(entries)
        self.keep([(s, list(range(n))) for s, n in entries])


@pytest.mark.parametrize("page_size", [1, 4, 16, 64])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_step_after_step(page_size, dtype):
    pair = Pair(pages=200 // page_size + 20, page_size=page_size, sequences=4, max_pages=64 // page_size + 3, dtype=dtype)
    rng = random.Random(page_size)
    for _ in range(8):
        entries = [(s, rng.randint(1, 7)) for s in rng.sample(range(4), rng.randint(1, 4))]
        assert pair.reserve(entries)
        pair.append(entries)
        pair.keep([(s, sorted(rng.sample(range(n), rng.randint(0, n)))) for s, n in entries])
        pair.check()


@pytest.mark.parametrize("heads,dim", [(3, 64), (8, 128), (1, 8)])
def test_row_shapes(heads, dim):
    pair = Pair(pages=12, page_size=4, sequences=3, max_pages=6, layers=3, heads=heads, dim=dim)
    pair.grow([(2, 5), (0, 1)])
    pair.grow([(0, 9)])
    entries = [(0, 6), (2, 4)]
    assert pair.reserve(entries)
    pair.append(entries)
    pair.keep([(0, [0, 3, 5]), (2, [0, 1, 3])])
    pair.check()


def test_continuations_share_and_part():
    pair = Pair(pages=40, page_size=8, sequences=6, max_pages=8)
    pair.grow([(0, 19)])
    pair.fork([(0, 3), (0, 5), (0, 1)])
    pair.check()
    pair.grow([(3, 2), (1, 1), (0, 3), (5, 20)])  # the fourth holder keeps the page
    pair.check()
    pair.fork([(5, 2)])
    pair.release([(0, 0), (5, 3)])
    pair.check()
    pair.grow([(5, 9), (2, 1)])
    pair.check()
    pair.release([(s, 0) for s in (5, 3, 2, 1)])
    pair.check()
    assert pair.gpu.refs.sum().item() == 0


def test_random_operations():
    """A thousand-page life of the cache: every operation mixed, exact bookkeeping throughout."""
    for seed in range(4):
        rng = random.Random(seed)
        pair = Pair(pages=48, page_size=4, sequences=7, max_pages=12, layers=1)
        for _ in range(40):
            what = rng.choice(("grow", "grow", "grow", "draft", "fork", "release", "compact"))
            lengths, held = pair.book.lengths, pair.book.held
            room = [s for s in range(7) if lengths[s] < 40]
            if what in ("grow", "draft") and room:
                entries = [(s, rng.randint(1, min(7, 48 - lengths[s]))) for s in rng.sample(room, rng.randint(1, min(4, len(room))))]
                if not pair.reserve(entries):
                    assert pair.word() == 8
                    pair.check()
                    continue
                pair.append(entries)
                pair.keep([(s, sorted(rng.sample(range(n), rng.randint(0, n)))) for s, n in entries])
            elif what == "fork":
                empty = [s for s in range(7) if not held[s]]
                full = [s for s in range(7) if held[s]]
                if empty and full:
                    children = rng.sample(empty, rng.randint(1, len(empty)))
                    pair.fork([(rng.choice(full), c) for c in children])
            elif what == "release":
                pair.release([(s, rng.choice((0, rng.randint(0, 50)))) for s in rng.sample(range(7), rng.randint(1, 5))])
            elif what == "compact":
                pair.compact()
            pair.check()


def test_pool_without_room_changes_nothing():
    pair = Pair(pages=4, page_size=8, sequences=3, max_pages=4)
    pair.grow([(0, 17)])
    pair.fork([(0, 1)])
    assert not pair.reserve([(2, 1), (1, 1), (0, 8)])  # one page, one copy, one page: three of one
    assert pair.word() == 8
    pair.check()
    assert pair.reserve([(1, 7)])  # one copy
    pair.check()


def test_reservations_of_nothing_and_of_everything():
    pair = Pair(pages=30, page_size=8, sequences=6, max_pages=4)
    assert pair.reserve([(1, 0), (0, 0)])
    pair.check()
    pair.grow([(0, 32), (3, 31), (4, 32)])
    pair.grow([(3, 1)])
    pair.check()
    pair.gpu.reserve(ints([0, 0, 0, 0, 0, 0]), error_word=pair.errors)
    pair.check()


@pytest.mark.parametrize("pages", [1500, 40000])
def test_large_pools(pages):
    """More pages than one pass of the allocator covers; the free ones at its ends."""
    cache = tsac_cuda.PagedCache.empty(1, pages, 1, 1, 8, 3, 1024)
    refs = torch.ones(pages, dtype=torch.int32)
    free = sorted(random.Random(1).sample(range(pages), 700) + [0, pages - 1])
    free = sorted(set(free))
    refs[free] = 0
    cache.refs.copy_(refs)
    cache.reserve(ints([300, len(free) - 301, 1]))
    tables = cache.tables.tolist()
    assert tables[0][:300] + tables[1][:len(free) - 301] + tables[2][:1] == free
    assert cache.refs.tolist() == [1] * pages


@pytest.mark.parametrize("pages,live", [(1500, 700), (40000, 33000), (64, 64), (64, 0)])
def test_compaction(pages, live):
    cache = tsac_cuda.PagedCache.empty(2, pages, 1, 1, 8, 40, 1024)
    order = random.Random(live).sample(range(pages), live)
    cache.pool.copy_(torch.randn(cache.pool.shape))
    pool = cache.pool.clone()
    refs = torch.zeros(pages, dtype=torch.int32)
    refs[order] = torch.arange(live, dtype=torch.int32) + 1
    tables = torch.full((40, 1024), -1, dtype=torch.int32)
    counts = [min(1024, max(0, live - 1024 * s)) for s in range(40)]
    for s, n in enumerate(counts):
        tables[s, :n] = torch.tensor(order[1024 * s:1024 * s + n], dtype=torch.int32)
    cache.refs.copy_(refs)
    cache.tables.copy_(tables)
    cache.counts.copy_(ints(counts))
    new_tables, new_refs = torch.empty_like(cache.tables), torch.empty_like(cache.refs)
    word = torch.zeros(1, dtype=torch.int32, device="cuda")
    assert int(cache.compact(tables_out=new_tables, refs_out=new_refs, error_word=word).item()) == live
    assert torch.equal(cache.refs.cpu(), refs) and torch.equal(cache.tables.cpu(), tables) and word.item() == 0
    holes = [p for p in range(live) if refs[p] == 0]
    to = {p: (p if p < live else None) for p in range(pages) if refs[p] > 0}
    for p in sorted(to):
        if to[p] is None:
            to[p] = holes.pop(0)
    want = torch.zeros(pages, dtype=torch.int32)
    expected = pool.cpu().clone()
    for p, place in to.items():
        want[place] = refs[p]
        expected[:, :, place] = pool[:, :, p].cpu() if live <= 700 else expected[:, :, place]
    assert torch.equal(new_refs.cpu(), want)
    mapped = torch.tensor([to.get(p, -1) for p in range(pages)] + [-1], dtype=torch.int32)
    assert torch.equal(new_tables.cpu(), mapped[tables.long()])
    moved = sorted(p for p in to if to[p] != p)
    places = [to[p] for p in moved]
    assert torch.equal(cache.pool[:, :, places], pool[:, :, moved])
    still = sorted(set(range(pages)) - set(places))
    assert torch.equal(cache.pool[:, :, still], pool[:, :, still])


def test_strided_rows_and_other_starts():
    cache = tsac_cuda.PagedCache.empty(1, 8, 4, 2, 64, 2, 4)
    cache.reserve(ints([9, 9]))
    big = torch.randn(2, 3, 4, 4, 64, device="cuda").to(torch.bfloat16)
    keys, values = big[:, ::2, :, 1:3].flatten(1, 2)[:, ::2], big.transpose(0, 1)[0].transpose(1, 2)[:, :, :2]
    keys, values = big[:, 0, ::2, 1:3], big[:, 1:3, 3, ::2]
    cache.append(0, keys, values, starts=ints([7, 2]))
    flat = cache.pool.view(2, 32, 2, 64)
    tables = cache.tables.tolist()
    for b, start in enumerate((7, 2)):
        for n in range(2):
            at = tables[b][(start + n) // 4] * 4 + (start + n) % 4
            assert torch.equal(flat[0, at], keys[b, n]) and torch.equal(flat[1, at], values[b, n])
    assert (flat != 0).any(-1).any(-1).sum().item() == 8


def test_keep_with_starts_and_new_lengths():
    """Evicting rows of a committed region: any ascending path, long ones too."""
    cache = tsac_cuda.PagedCache.empty(2, 70, 16, 1, 64, 3, 64)
    cache.reserve(ints([1000, 0, 16]))
    cache.pool.copy_(torch.randn(cache.pool.shape))
    before = cache.pool.clone()
    rng = random.Random(0)
    path = sorted(rng.sample(range(990), 600))
    out = ints([5, 6, 7])
    word = torch.zeros(1, dtype=torch.int32, device="cuda")
    cache.keep(ints([path, [0] * 600]), ints([600, 0]), starts=ints([10, 3]), lengths_out=out, sequences=ints([0, 2]), error_word=word)
    assert word.item() == 0 and out.tolist() == [610, 6, 3] and cache.lengths.tolist() == [0, 0, 0]
    flat, old = cache.pool.view(2, 2, -1, 64), before.view(2, 2, -1, 64)
    table = cache.tables[0].tolist()
    at = lambda p: table[p // 16] * 16 + p % 16  # noqa: E731
    want = old.clone()
    want[:, :, [at(10 + j) for j in range(600)]] = old[:, :, [at(10 + p) for p in path]]
    assert torch.equal(flat, want)


def _state(cache):
    return [t.clone() for t in (cache.tables, cache.counts, cache.lengths, cache.refs, cache.pool)]


def _same(cache, state):
    return all(torch.equal(a, b) for a, b in zip(_state(cache), state))


def test_invalid_entries_are_reported_and_skipped():
    pair = Pair(pages=24, page_size=8, sequences=6, max_pages=8)
    pair.grow([(0, 10), (1, 5)])
    cache, errors = pair.gpu, pair.errors
    state = _state(cache)

    def expect(fn, unchanged=True):
        errors.zero_()
        fn()
        assert errors.item() == 16
        assert not unchanged or _same(cache, state)

    expect(lambda: cache.reserve(ints([1, 1]), sequences=ints([2, 6]), error_word=errors))
    expect(lambda: cache.reserve(ints([1, 1]), sequences=ints([2, -1]), error_word=errors))
    expect(lambda: cache.reserve(ints([1, 1]), sequences=ints([2, 2]), error_word=errors))
    expect(lambda: cache.reserve(ints([1, -1]), sequences=ints([2, 3]), error_word=errors))
    expect(lambda: cache.reserve(ints([60]), sequences=ints([1]), error_word=errors))  # past the table
    expect(lambda: cache.reserve(ints([2147483647]), sequences=ints([1]), error_word=errors))
    expect(lambda: cache.reserve(ints([9]), sequences=ints([1]), slots=1, error_word=errors))  # two pages, one slot
    expect(lambda: cache.fork(ints([0]), ints([1]), error_word=errors))      # a child with pages
    expect(lambda: cache.fork(ints([7]), ints([2]), error_word=errors))
    expect(lambda: cache.fork(ints([0]), ints([9]), error_word=errors))
    expect(lambda: cache.fork(ints([2]), ints([2]), error_word=errors))
    expect(lambda: cache.release(sequences=ints([-3]), error_word=errors))
    expect(lambda: cache.release(sequences=ints([0]), positions=ints([-1]), error_word=errors))
    rows = torch.ones(1, 7, 1, ROW, dtype=torch.bfloat16, device="cuda")
    expect(lambda: cache.append(0, rows, rows, sequences=ints([2]), error_word=errors))        # nothing reserved
    expect(lambda: cache.append(0, rows, rows, sequences=ints([6]), error_word=errors))
    expect(lambda: cache.append(0, rows, rows, sequences=ints([1]), starts=ints([-9]), error_word=errors))
    expect(lambda: cache.append(0, rows, rows, sequences=ints([1]), starts=ints([2147483647]), error_word=errors))
    expect(lambda: cache.keep(ints([[1, 0]]), ints([2]), sequences=ints([1]), error_word=errors))   # not ascending
    expect(lambda: cache.keep(ints([[0, 0]]), ints([2]), sequences=ints([1]), error_word=errors))
    expect(lambda: cache.keep(ints([[-1, 0]]), ints([2]), sequences=ints([1]), error_word=errors))
    expect(lambda: cache.keep(ints([[0, 90]]), ints([2]), sequences=ints([1]), error_word=errors))
    expect(lambda: cache.keep(ints([[0, 1]]), ints([3]), sequences=ints([1]), error_word=errors))
    expect(lambda: cache.keep(ints([[0, 1]]), ints([-1]), sequences=ints([1]), error_word=errors))
    expect(lambda: cache.keep(ints([[0, 1]]), ints([2]), sequences=ints([6]), error_word=errors))

    # A valid entry beside an invalid one goes through.
    expect(lambda: cache.fork(ints([0, 0, 2]), ints([2, 2, 3]), error_word=errors), unchanged=False)
    assert cache.counts.tolist() == [2, 1, 2, 0, 0, 0] and cache.refs.tolist()[:3] == [2, 2, 1]
    expect(lambda: cache.release(sequences=ints([2, 2]), error_word=errors), unchanged=False)
    assert _same(cache, state)

    # Rows of shared pages are refused, not written.
    errors.zero_()
    cache.fork(ints([0]), ints([4]), error_word=errors)
    assert errors.item() == 0
    state = _state(cache)
    expect(lambda: cache.append(0, rows[:, :6], rows[:, :6], sequences=ints([4]), error_word=errors))
    expect(lambda: cache.keep(ints([[1]]), ints([1]), starts=ints([3]), sequences=ints([4]), error_word=errors))


def test_pages_that_are_none_are_reported():
    """A table that names no page of the pool: skipped, never followed."""
    pair = Pair(pages=24, page_size=8, sequences=4, max_pages=8)
    pair.grow([(0, 20)])
    cache, errors = pair.gpu, pair.errors
    cache.tables[0, 1] = 24
    cache.tables[0, 2] = -5
    refs, pool = cache.refs.clone(), cache.pool.clone()
    cache.fork(ints([0]), ints([1]), error_word=errors)
    assert errors.item() == 16 and torch.equal(cache.refs, refs) and cache.counts.tolist() == [3, 0, 0, 0]
    errors.zero_()
    cache.reserve(ints([1]), sequences=ints([0]), error_word=errors)
    assert errors.item() == 16 and torch.equal(cache.refs, refs)
    errors.zero_()
    cache.keep(ints([[0, 2]]), ints([2]), sequences=ints([0]), error_word=errors)
    assert errors.item() == 16 and torch.equal(cache.pool, pool) and cache.lengths.tolist()[0] == 20
    errors.zero_()
    out = cache.tables.clone()
    cache.compact(tables_out=out, refs_out=refs.clone(), error_word=errors)
    assert errors.item() == 16 and out[0].tolist() == [0, -1, -1, -1, -1, -1, -1, -1]
    errors.zero_()
    cache.release(sequences=ints([0]), error_word=errors)
    assert errors.item() == 16 and cache.refs.tolist()[:3] == [0, 1, 1] and cache.counts.tolist()[0] == 0


def test_many_sequences_in_one_call():
    """The longest list: 4,096 sequences that share one page, all but one parting from it."""
    count = 4096
    cache = tsac_cuda.PagedCache.empty(1, count + 4, 4, 1, 8, count, 2)
    cache.reserve(ints([3] + [0] * (count - 1)))
    cache.lengths[0] = 3
    cache.pool[:, :, 0] = 1.5
    children = torch.arange(1, count, dtype=torch.int32, device="cuda")
    cache.fork(torch.zeros_like(children), children)
    assert cache.refs[0].item() == count
    errors = torch.zeros(1, dtype=torch.int32, device="cuda")
    order = torch.randperm(count, generator=torch.Generator().manual_seed(0)).to(torch.int32).cuda()
    cache.reserve(torch.ones_like(order), sequences=order, slots=1, error_word=errors)
    assert errors.item() == 0
    want = torch.empty(count, dtype=torch.int32)
    want[order.cpu().long()] = torch.cat((torch.arange(1, count, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)))
    assert torch.equal(cache.tables[:, 0].cpu(), want)
    assert (cache.refs[:count] == 1).all() and (cache.pool[:, :, :count] == 1.5).all()


def test_captured_step_replays():
    """reserve, append, keep and release in one CUDA graph, replayed as lengths move on."""
    pair = Pair(pages=40, page_size=8, sequences=2, max_pages=12, layers=1)
    cache = pair.gpu
    rows = torch.zeros(2, 2, 3, 1, ROW, dtype=torch.bfloat16, device="cuda")
    nodes, path, accepted = ints([3, 2]), ints([[0, 2, -1], [0, 1, -1]]), ints([2, 2])

    def step():
        cache.reserve(nodes, error_word=pair.errors)
        cache.append(0, rows[0], rows[1], nodes=nodes, error_word=pair.errors)
        cache.keep(path, accepted, error_word=pair.errors)
        cache.release(positions=cache.lengths, error_word=pair.errors)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            step()
    for turn in range(6):
        serials = [[10 * turn + n for n in range(3)], [10 * turn + 5 + n for n in range(2)]]
        for b, line in enumerate(serials):
            for n, serial in enumerate(line):
                rows[0, b, n], rows[1, b, n] = pair.values(serial, 0, 0).cuda(), pair.values(serial, 0, 1).cuda()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graph.replay()
        torch.cuda.synchronize()
        assert pair.book.reserve([(0, 3), (1, 2)])
        for b, line in enumerate(serials):
            pair.book.append(b, line)
        pair.book.keep(0, [0, 2])
        pair.book.keep(1, [0, 1])
        for b in (0, 1):
            pair.book.release(b, pair.book.lengths[b])
        pair.check()


def test_captured_reservation_outlives_larger_ones():
    """A graph's temporary memory stays its own when later calls need more."""
    cache = tsac_cuda.PagedCache.empty(1, 600, 4, 1, 8, 300, 4)
    first = ints([0])
    positions = ints([3])
    cache.reserve(positions, sequences=first, slots=1)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.release(sequences=first)
        cache.reserve(positions, sequences=first, slots=1)
    cache.reserve(torch.ones(300, dtype=torch.int32, device="cuda"))
    guards = [torch.full((n,), 17, dtype=torch.uint8, device="cuda") for n in (16, 64, 512, 4096, 8192, 20000) for _ in range(8)]
    want = cache.refs.clone(), cache.tables.clone()
    for _ in range(3):
        graph.replay()
    assert all((guard == 17).all() for guard in guards)
    assert torch.equal(cache.refs, want[0]) and torch.equal(cache.tables, want[1])


def test_long_reservation_among_short_ones():
    """A prompt's pages in one call with entries of none, one and two pages, taken in list order."""
    pair = Pair(pages=6000, page_size=4, sequences=6, max_pages=5000, layers=1)
    pair.grow([(4, 3), (0, 8)])
    assert pair.reserve([(1, 1), (3, 0), (0, 19800), (4, 1), (2, 8), (5, 2900)])
    pair.check()
    assert not pair.reserve([(2, 4000)])
    assert pair.word() == 8
    pair.check()


@pytest.mark.parametrize("outside", [True, False])
def test_several_shared_pages_in_a_range(outside):
    """Lengths taken back into shared pages: each writer copies each of them, but the last where no other holds it."""
    pair = Pair(pages=60, page_size=8, sequences=6, max_pages=8)
    pair.grow([(0, 40)])
    pair.fork([(0, s) for s in (1, 2, 3, 4)])
    if not outside:
        pair.release([(0, 0)])
    for s, length in ((1, 3), (2, 17), (3, 9), (4, 0)):
        pair.gpu.lengths[s] = length
        pair.book.lengths[s] = length
    assert pair.reserve([(2, 10), (4, 30), (1, 20), (5, 9), (3, 20)])
    pair.check()
    assert pair.reserve([(4, 3), (2, 30)])
    pair.check()


def test_many_sequences_share_many_pages():
    """4,095 sequences that hold the same 24 pages part from all of them in one call, one keeping them."""
    count, shared = 4095, 24
    cache = tsac_cuda.PagedCache.empty(1, count * shared + 3, 1, 1, 8, count, shared)
    cache.reserve(ints([shared] + [0] * (count - 1)))
    cache.lengths[0] = shared
    cache.pool[:, :, :shared] = torch.arange(shared, device="cuda", dtype=torch.bfloat16)[:, None, None, None]
    children = torch.arange(1, count, dtype=torch.int32, device="cuda")
    cache.fork(torch.zeros_like(children), children)
    assert (cache.refs[:shared] == count).all()
    cache.lengths.zero_()
    errors = torch.zeros(1, dtype=torch.int32, device="cuda")
    cache.reserve(torch.full((count,), shared, dtype=torch.int32, device="cuda"), error_word=errors)
    assert errors.item() == 0
    want = torch.arange(shared, shared * count, dtype=torch.int32, device="cuda").view(count - 1, shared)
    assert torch.equal(cache.tables[:-1], want) and torch.equal(cache.tables[-1], torch.arange(shared, dtype=torch.int32, device="cuda"))
    assert (cache.refs[:shared * count] == 1).all() and (cache.refs[shared * count:] == 0).all()
    rows = cache.pool[0, :, :shared * count, 0, 0, 0].view(2, count, shared)
    assert (rows == torch.arange(shared, device="cuda", dtype=torch.bfloat16)).all()


def test_temporary_memory_used_on_another_stream_is_not_handed_out():
    """A cache given up while another stream still works for it leaves its temporary memory alone."""
    cache = tsac_cuda.PagedCache.empty(1, 600, 4, 1, 8, 300, 4)
    positions = torch.ones(300, dtype=torch.int32, device="cuda")
    cache.reserve(positions, slots=1)
    place, size = cache._scratches[-1][0].data_ptr(), cache._scratches[-1][0].numel()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(200_000_000)
        cache.release()
        cache.reserve(positions, slots=1)
    buffers = cache.pool, cache.tables, cache.counts, cache.lengths, cache.refs  # the caller's
    del cache
    again = [torch.empty(size, dtype=torch.uint8, device="cuda") for _ in range(16)]
    assert not side.query() and all(block.data_ptr() != place for block in again)
    torch.cuda.synchronize()
    assert buffers[4].sum().item() == 300


def test_binding_refuses_other_dimensions():
    pair = Pair()
    with pytest.raises(tsac_cuda.TsacError, match="keys must be"):
        pair.gpu.append(0, torch.zeros(2, 1, ROW, device="cuda", dtype=torch.bfloat16), torch.zeros(2, 1, ROW, device="cuda", dtype=torch.bfloat16))
    with pytest.raises(tsac_cuda.TsacError, match="path must be"):
        pair.gpu.keep(ints([0]), ints([1]))
    with pytest.raises(tsac_cuda.TsacError, match="positions must be"):
        pair.gpu.reserve(ints([[1]]))
    with pytest.raises(tsac_cuda.TsacError, match="parents must be"):
        pair.gpu.fork(ints([[0]]), ints([[1]]))
    with pytest.raises(tsac_cuda.TsacError, match="sequences must be"):
        pair.gpu.release(sequences=ints([[0]]))
    with pytest.raises(tsac_cuda.TsacError, match="32-bit word"):
        pair.gpu.release(error_word=torch.zeros(4, dtype=torch.uint8, device="cuda"))
    pair.check()


@pytest.mark.parametrize("pages,in_place", [(64, False), (64, True), (1500, True), (40000, False)])
def test_compaction_of_inconsistent_counts(pages, in_place):
    """Negative counts and entries of pages without a count: reported, and never more moves than holes."""
    rng = random.Random(pages)
    cache = tsac_cuda.PagedCache.empty(1, pages, 2, 1, 8, 3, pages // 4)
    refs = torch.tensor([rng.choice((-3, -1, 0, 0, 1, 2)) for _ in range(pages)], dtype=torch.int32)
    refs[-1], refs[0] = 5, -1
    live = [p for p in range(pages) if refs[p] > 0]
    count = len(live)
    cache.refs.copy_(refs)
    cache.pool.copy_(torch.randn(cache.pool.shape))
    pool = cache.pool.clone()
    named = live[:pages // 8] + live[-pages // 16:] + [p for p in range(pages) if refs[p] <= 0][:pages // 16]
    rng.shuffle(named)
    cache.tables[1, :len(named)] = ints(named)
    cache.counts[1] = len(named)
    tables_out, refs_out = (cache.tables, cache.refs) if in_place else (torch.empty_like(cache.tables), torch.empty_like(cache.refs))
    word = torch.zeros(1, dtype=torch.int32, device="cuda")
    assert cache.compact(tables_out=tables_out, refs_out=refs_out, error_word=word).item() == count
    assert word.item() == 16
    holes = [p for p in range(count) if refs[p] <= 0]
    moved = [p for p in live if p >= count]
    assert len(holes) == len(moved)
    to = {p: p for p in live} | dict(zip(moved, holes))
    want = torch.zeros(pages, dtype=torch.int32)
    want[[to[p] for p in live]] = refs[live]
    assert torch.equal(refs_out.cpu(), want)
    assert tables_out[1, :len(named)].tolist() == [to.get(p, -1) for p in named]
    assert (tables_out[[0, 2]] == -1).all() and (tables_out[1, len(named):] == -1).all()
    expected = pool.clone()
    expected[:, :, holes] = pool[:, :, moved]
    assert torch.equal(cache.pool, expected)


def test_counts_below_the_entries_that_name_a_page():
    """Tables and counts that a caller built wrongly: reported, and no count falls below zero."""
    pair = Pair(pages=12, page_size=8, sequences=5, max_pages=4)
    pair.grow([(0, 20), (1, 9)])
    cache, errors = pair.gpu, pair.errors

    def word():
        value = errors.item()
        errors.zero_()
        return value

    # Sequence 2 names the pages of sequence 0 (0, 1, 2) without being counted.
    cache.tables[2], cache.counts[2], cache.lengths[2] = cache.tables[0].clone(), 3, 20
    cache.release(sequences=ints([0]), error_word=errors)
    assert word() == 0 and cache.refs.tolist()[:5] == [0, 0, 0, 1, 1]
    state = _state(cache)
    cache.reserve(ints([1, 3]), sequences=ints([3, 2]), error_word=errors)
    assert word() == 16 and _same(cache, state)
    cache.fork(ints([2]), ints([4]), error_word=errors)
    assert word() == 16 and _same(cache, state)
    cache.release(sequences=ints([2, 1]), error_word=errors)
    assert word() == 16 and cache.refs.tolist() == [0] * 12 and cache.counts.tolist() == [0] * 5
    assert (cache.tables == -1).all() and cache.lengths.tolist() == [0] * 5
    # Many holders of one page with a count of two, and a count that is negative already.
    cache = tsac_cuda.PagedCache.empty(1, 3, 4, 1, 8, 4096, 2)
    cache.tables[:, 0], cache.tables[:, 1] = 1, 2
    cache.counts.fill_(2)
    cache.lengths.fill_(8)
    cache.refs.copy_(ints([0, 2, -7]))
    cache.release(error_word=errors)
    assert word() == 16 and cache.refs.tolist() == [0, 0, -7] and cache.counts.sum().item() == 0


@pytest.mark.parametrize("name", ["pool", "tables", "counts", "lengths", "refs"])
def test_the_bound_tensors_cannot_be_exchanged(name):
    """The calls go on with the addresses that the cache was made with."""
    pair = Pair()
    pair.grow([(0, 5)])
    before = getattr(pair.gpu, name)
    with pytest.raises(tsac_cuda.TsacError, match=f"{name} is bound"):
        setattr(pair.gpu, name, before.clone())
    assert getattr(pair.gpu, name) is before
    pair.gpu.lengths += 0  # in place
    pair.check()
