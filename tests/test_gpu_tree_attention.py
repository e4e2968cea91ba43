"""Attention of drafted trees over the paged cache on the GPU against the formula in 64 bits.

Tolerances, with h = finfo(type).eps / 2 (half a rounding step of the type)
and A = sum_k p_k |v_k| / sum_k p_k of the element: rounding each p for the
second product moves the output by at most h A; the output's own rounding by
h |out|; 32-bit arithmetic moves each score by at most (D + 2) 2^-23 scale
sum |q k| <= (D + 2) 2^-23 S, so each p by twice that relative, and sums of n
terms by n 2^-23: in all (2 (D + 2) S + 2 n) 2^-23 A with S the largest sum of
|q k| scale.  The type's subnormals add at most their spacing for fp16
(2^-24) per output and, for p below 2^-14, 2^-24 |v| per key."""
from __future__ import annotations

import math
import random

import pytest
import torch

import drafting
import tsac_cuda

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def random_tree(rng, nodes, holes=False):
    parents = [-1]
    for n in range(1, nodes):
        parents.append(rng.choice([-1, -2, n - 1]) if holes and rng.random() < 0.3 else rng.randint(max(0, n - 4), n - 1))
    return parents


class Setup:
    def __init__(self, kind, dim, kv_heads, group, page, lengths, nodes, seed=0, spread=1.0, holes=False, layers=1, most=None):
        g = torch.Generator().manual_seed(seed)
        rng = random.Random(seed)
        self.kind, self.dim, self.group, self.kv_heads = kind, dim, group, kv_heads
        self.lengths, self.nodes, self.layers = lengths, nodes, layers
        self.most = most or max(1, max(nodes))
        count = len(lengths)
        held = [-(-(a + max(0, n)) // page) for a, n in zip(lengths, nodes)]
        pages = sum(held) + 2
        order = list(range(pages))
        rng.shuffle(order)
        dtype = TYPES[kind]
        self.pool = (torch.randn((layers, 2, pages, page, kv_heads, dim), generator=g) * spread).to(dtype)
        tables = torch.full((count, max(held) + 1), -1, dtype=torch.int32)
        for b, n in enumerate(held):
            tables[b, :n] = torch.tensor([order.pop() for _ in range(n)], dtype=torch.int32)
            # What lies behind a sequence's last position is anything.
            if n and (lengths[b] + max(0, nodes[b])) % page:
                self.pool[:, :, tables[b, n - 1], (lengths[b] + max(0, nodes[b])) % page:] = float("nan")
        self.tables = tables
        self.parents = [random_tree(rng, self.most, holes) for _ in range(count)]
        self.query = (torch.randn((count, self.most, kv_heads * group, dim), generator=g) * spread).to(dtype)
        refs = torch.zeros(pages, dtype=torch.int32)
        refs[tables[tables >= 0].long()] = 1
        self.cache = tsac_cuda.PagedCache(self.pool.cuda(), tables.cuda(), ints(held), ints(lengths), refs.cuda())

    def rows(self, b, layer=0):
        flat = self.pool[layer][:, self.tables[b][self.tables[b] >= 0].long()].flatten(1, 2)
        n = self.lengths[b] + max(0, self.nodes[b])
        return flat[0][:n].double(), flat[1][:n].double()

    def run(self, layer=0, **more):
        errors = torch.zeros(1, dtype=torch.int32, device="cuda")
        shape = (len(self.lengths), self.most, self.kv_heads * self.group)
        out = torch.full((*shape, self.dim), 77.0, dtype=TYPES[self.kind], device="cuda")
        lse = torch.full(shape, 77.0, device="cuda")
        self.cache.attention(layer, self.query.cuda(), ints(self.parents), out, nodes=ints(self.nodes), lse=lse,
                             error_word=errors, **more)
        assert errors.item() == 0
        return out.cpu().double(), lse.cpu().double()

    def check(self, out, lse, layer=0, scale=None, entries=None):
        scale = self.dim ** -0.5 if scale is None else scale
        half = torch.finfo(TYPES[self.kind]).eps / 2
        for b in range(len(self.lengths)) if entries is None else entries:
            n = max(0, min(self.nodes[b], self.most))
            assert (out[b, n:] == 77.0).all() and (lse[b, n:] == 77.0).all()
            if n == 0:
                continue
            keys, values = self.rows(b, layer)
            query = self.query[b, :n].double()
            want, want_lse, size = drafting.attention(query, keys, values, self.lengths[b], self.parents[b], n, self.group, scale)
            reach = abs(scale) * (query.abs().amax((0, 1)) * keys.abs().amax((0, 1))).sum().item()
            total = self.lengths[b] + n
            fine = (2 * (self.dim + 2) * reach + 2 * total) * 2.0 ** -23
            tiny = 2.0 ** -24 * (1 + total * values.abs().max().item()) if self.kind == "fp16" else 0.0
            bound = half * (1 + fine) * size + half * want.abs() + fine * size + tiny
            assert ((out[b, :n] - want).abs() <= bound).all(), (b, ((out[b, :n] - want).abs() - bound).max())
            finite = torch.isfinite(want_lse)
            assert torch.equal(lse[b, :n][~finite], want_lse[~finite])
            # The maximum is kept in units of log2(e): one more rounding of each, and the sum's.
            lse_bound = fine + 4 * 2.0 ** -23 * (1 + want_lse[finite].abs())
            assert ((lse[b, :n][finite] - want_lse[finite]).abs() <= lse_bound).all()


@pytest.mark.parametrize("kind", ["bf16", "fp16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("page", [1, 16, 128])
def test_lengths(kind, dim, page):
    s = Setup(kind, dim, 2, 1, page, [0, 1, 15, 16, 17, 63, 64, 65, 127, 128, 129, 500], [5, 1, 3, 16, 17, 2, 8, 17, 1, 4, 17, 9], seed=page)
    s.check(*s.run())


@pytest.mark.parametrize("group", [1, 2, 3, 4, 5, 8, 16])
@pytest.mark.parametrize("nodes", [1, 2, 7, 16, 33, 64])
def test_shapes(group, nodes):
    kind, dim = ("bf16", 128) if (group + nodes) % 2 else ("fp16", 64)
    s = Setup(kind, dim, 2, group, 16, [70, 0, 200], [nodes, nodes, max(1, nodes - 3)], seed=group * 100 + nodes)
    s.check(*s.run())


@pytest.mark.parametrize("kind,dim", [("bf16", 128), ("fp16", 64), ("bf16", 64), ("fp16", 128)])
@pytest.mark.parametrize("group,nodes", [(1, 1), (8, 1), (4, 16), (8, 64)])
def test_one_long_sequence_is_split(kind, dim, group, nodes):
    s = Setup(kind, dim, 1, group, 32, [9001], [nodes], seed=3)
    s.check(*s.run())


def test_many_short_sequences():
    rng = random.Random(5)
    lengths = [rng.choice((0, 1, 5, 40, 64, 100)) for _ in range(400)]
    s = Setup("bf16", 64, 2, 2, 8, lengths, [rng.randint(0, 4) for _ in lengths], seed=5, most=6)
    s.check(*s.run())


def test_mixed_lengths():
    s = Setup("bf16", 128, 4, 2, 64, [1, 3000, 0, 12, 700, 64], [3, 12, 4, 0, 1, 12], seed=6)
    s.check(*s.run())


@pytest.mark.parametrize("nodes", [5, 64])
@pytest.mark.parametrize("group", [1, 8])
def test_nodes_that_see_nothing(nodes, group):
    """Roots, and nodes that see no drafted node: with nothing committed these give zeros and -infinity."""
    s = Setup("bf16", 64, 2, group, 8, [0, 30, 0], [nodes, nodes, 1], seed=8, holes=True)
    s.parents[2][0] = -2
    out, lse = s.run()
    s.check(out, lse)
    assert (out[2, 0] == 0).all() and torch.isinf(lse[2, 0]).all()


@pytest.mark.parametrize("group", [1, 16])
@pytest.mark.parametrize("spread", [0.0, 1e-3, 8.0])
def test_flat_and_peaked_scores(spread, group):
    s = Setup("bf16", 128, 1, group, 16, [333, 64], [6, 9], seed=9, spread=spread)
    s.check(*s.run())


@pytest.mark.parametrize("scale", [0.0, -0.3, 1.0])
def test_scales(scale):
    s = Setup("fp16", 64, 2, 2, 16, [130, 3], [6, 2], seed=10)
    s.check(*s.run(scale=scale), scale=scale)


@pytest.mark.parametrize("kind", ["bf16", "fp16"])
@pytest.mark.parametrize("group,nodes", [(1, 6), (4, 6), (8, 40)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_values_that_are_not_finite_reach_only_rows_that_see_them(kind, group, nodes, bad):
    s = Setup(kind, 128, 2, group, 16, [90, 0], [nodes, nodes], seed=11)
    clean, clean_lse = s.run()
    before = s.pool.clone()
    marks = []
    for b in (0, 1):
        for which, node, head, column in ((0, 3, 0, 5), (1, 4, 1, 9), (1, 2, 1, 127)):
            at = s.lengths[b] + node
            s.pool[0, which, s.tables[b, at // 16], at % 16, head, column] = bad
            marks.append((b, which, node, head, column))
    s.cache.pool.copy_(s.pool)
    out, _ = s.run()
    hit = torch.zeros_like(out, dtype=torch.bool)
    for b, which, node, head, column in marks:
        for n, seen in enumerate(drafting.ancestors(s.parents[b], nodes)):
            if node in seen:
                rows = hit[b, n, head * group:(head + 1) * group]
                if which:
                    rows[:, column] = True
                else:
                    rows[:] = True
    # Rows that see none of the marked nodes are the same bits.  The finite columns of rows that see a
    # marked value row may be summed in another order (its products are taken apart from the others):
    # they are held to the bound against the formula, with the marked elements set aside.
    rows = torch.zeros_like(hit)
    for b, which, node, head, column in marks:
        for n, seen in enumerate(drafting.ancestors(s.parents[b], nodes)):
            rows[b, n, head * group:(head + 1) * group] |= node in seen
    assert torch.equal(out[~rows], clean[~rows]) and torch.isfinite(out[~hit]).all()
    damaged, s.pool = s.pool, before
    s.check(torch.where(hit, clean, out), clean_lse)
    s.pool = damaged
    # An infinite or undefined value that is seen shows; an infinite key gives NaN or takes or loses all the weight.
    for b, which, node, head, column in marks:
        if which:
            for n, seen in enumerate(drafting.ancestors(s.parents[b], nodes)):
                if node in seen:
                    assert not torch.isfinite(out[b, n, head * group:(head + 1) * group, column]).any()


def test_lists_layers_and_strides():
    s = Setup("bf16", 64, 2, 2, 16, [40, 100, 7, 64], [4, 9, 2, 5], seed=12, layers=3)
    order = [2, 0, 3]
    wide = torch.zeros((9, 3, 5, 72), dtype=torch.bfloat16, device="cuda")
    query = wide.permute(1, 0, 2, 3)[:, :, 1:, :64]
    query.copy_(s.query[order].cuda())
    big = torch.full((3, 4, 9, 80), 77.0, dtype=torch.bfloat16, device="cuda")
    out = big.transpose(1, 2)[..., 8:72]
    lse = torch.full((3, 9, 4), 77.0, device="cuda")
    s.cache.attention(2, query, ints([s.parents[b] for b in order]), out, nodes=ints([s.nodes[b] for b in order]),
                      sequences=ints(order), lse=lse)
    full, full_lse = (torch.full(t, 77.0, dtype=torch.float64) for t in ((4, 9, 4, 64), (4, 9, 4)))
    full[order], full_lse[order] = out.cpu().double(), lse.cpu().double()
    s.check(full, full_lse, layer=2, entries=order)
    assert (big[..., :8] == 77.0).all() and (big[..., 72:] == 77.0).all()


def test_the_same_sequence_twice_and_repeated_calls():
    s = Setup("bf16", 128, 2, 4, 16, [1500, 30], [12, 12], seed=13)
    out = s.cache.attention(0, s.query[[0, 0]].cuda(), ints([s.parents[0]] * 2), nodes=ints([12, 12]), sequences=ints([0, 0]))
    assert torch.equal(out[0], out[1]) or (out[0] - out[1]).abs().max() < 0.05  # the split may differ between entries
    again = s.cache.attention(0, s.query[[0, 0]].cuda(), ints([s.parents[0]] * 2), nodes=ints([12, 12]), sequences=ints([0, 0]))
    assert torch.equal(out, again)


def test_invalid_entries_are_reported_and_left():
    s = Setup("bf16", 64, 1, 2, 16, [40, 100, 7], [4, 9, 2], seed=14)
    s.cache.lengths[1] = 112  # with its nodes more than its pages hold
    errors = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = torch.full((5, 9, 2, 64), 77.0, dtype=torch.bfloat16, device="cuda")
    lse = torch.full((5, 9, 2), 77.0, device="cuda")
    query = s.query[[0, 1, 2, 2, 2]].cuda()
    trees = ints([s.parents[b] for b in (0, 1, 2, 2, 2)])
    s.cache.attention(0, query, trees, out, nodes=ints([4, 9, 2, 2, 2]), sequences=ints([0, 1, 2, 3, -1]), lse=lse, error_word=errors)
    assert errors.item() == 16
    got, got_lse = out.cpu().double(), lse.cpu().double()
    s.check(got, got_lse, entries=[0, 2])
    assert (got[[1, 3, 4]] == 77.0).all() and (got_lse[[1, 3, 4]] == 77.0).all()
    # A page that is none, and a parent behind its child: reported; every other entry is right.
    errors.zero_()
    s.cache.lengths[1] = 100
    s.cache.tables[1, 2] = 1 << 20
    trees[0, 2] = 3
    s.cache.attention(0, query[:3], trees[:3], out[:3], nodes=ints([4, 9, 2]), lse=lse[:3], error_word=errors)
    assert errors.item() == 16
    s.check(out.cpu().double(), lse.cpu().double(), entries=[2])


def test_captured_and_on_two_streams():
    """Two captured graphs of the same cache replayed at once: each has its own temporary memory."""
    s = Setup("bf16", 128, 2, 4, 16, [3000, 700], [16, 9], seed=15)
    want, _ = s.run()
    query, trees, nodes = s.query.cuda(), ints(s.parents), ints(s.nodes)
    torch.cuda.synchronize()
    streams, graphs, outs = [torch.cuda.Stream() for _ in range(2)], [], []
    for stream in streams:
        with torch.cuda.stream(stream):
            out = torch.full((2, 16, 8, 128), 77.0, dtype=torch.bfloat16, device="cuda")
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                s.cache.attention(0, query, trees, out, nodes=nodes)
            graphs.append(graph)
            outs.append(out)
    torch.cuda.synchronize()
    for _ in range(10):
        for stream, graph in zip(streams, graphs):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(out.cpu().double(), want) for out in outs)


def test_positions_past_two_gigabytes():
    """Pages whose byte offsets pass 32 bits."""
    cache = tsac_cuda.PagedCache.empty(1, 70, 1024, 256, 128, 1, 66, dtype=torch.bfloat16)  # 64 MiB a page
    torch.manual_seed(0)
    used = [69, 3, 68]
    cache.tables[0, :3] = ints(used)
    cache.counts[0] = 3
    cache.refs[used] = 1
    length = 2050
    cache.lengths[0] = length
    for page in used:
        cache.pool[0, :, page].normal_()
    parents = ints([[-1, 0, 0]])
    query = torch.randn(1, 3, 256, 128, device="cuda").to(torch.bfloat16)
    out = cache.attention(0, query, parents)
    keys, values = (cache.pool[0, i][used].flatten(0, 1)[:length + 3] for i in (0, 1))
    for head in (0, 255):
        want, _, size = drafting.attention(query[0, :, head:head + 1].cpu().double(), keys[:, head:head + 1].cpu().double(),
                                           values[:, head:head + 1].cpu().double(), length, [-1, 0, 0], 3, 1, 128 ** -0.5)
        # h (A + |out|) plus a thousandth of A for the 32-bit parts, as in Setup.check.
        assert ((out[0, :, head:head + 1].cpu().double() - want).abs() <= 2.0 ** -8 * (size + want.abs()) + 1e-3 * size).all()


def test_binding_refusals():
    s = Setup("bf16", 64, 1, 2, 16, [4], [2], seed=16)
    query, trees = s.query.cuda(), ints(s.parents)
    with pytest.raises(tsac_cuda.TsacError, match="query must be"):
        s.cache.attention(0, query.half(), trees)
    with pytest.raises(tsac_cuda.TsacError, match="parents must be"):
        s.cache.attention(0, query, trees.long())
    with pytest.raises(tsac_cuda.TsacError, match="out must be"):
        s.cache.attention(0, query, trees, torch.empty_like(query)[:, :1])
    with pytest.raises(tsac_cuda.TsacError, match="layer out of range"):
        s.cache.attention(1, query, trees)
    with pytest.raises(tsac_cuda.TsacError, match="16-byte aligned"):
        s.cache.attention(0, torch.empty(query.numel() + 8, dtype=query.dtype, device="cuda")[1:1 + query.numel()].view(query.shape), trees)


def test_a_whole_drafted_step():
    """reserve, append, attention, verification and keep together, twice, with a fork between: the cache that
    results is the one that plain decoding of the kept tokens gives."""
    torch.manual_seed(1)
    rng = random.Random(1)
    vocab, heads, dim, most = 50, 2, 64, 6
    cache = tsac_cuda.PagedCache.empty(2, 40, 8, heads, dim, 4, 10)
    embed = torch.randn(2, 2, vocab, heads, dim, device="cuda").to(torch.bfloat16)  # a token's row in each layer
    texts = {0: [3, 7, 9, 11, 2], 1: [5] * 11}
    for s, text in texts.items():
        cache.reserve(ints([len(text)]), sequences=ints([s]))
        for layer in range(2):
            rows = embed[layer][:, text]
            cache.append(layer, rows[0][None], rows[1][None], sequences=ints([s]))
        cache.keep(ints([list(range(len(text)))]), ints([len(text)]), sequences=ints([s]))
    last = {0: 1, 1: 4}
    for turn in range(3):
        if turn == 1:
            cache.fork(ints([1]), ints([3]))
            texts[3], last[3] = list(texts[1]), 8
        names = sorted(texts)
        tokens = [[last[s]] + [rng.randrange(vocab) for _ in range(most - 1)] for s in names]
        parents = [random_tree(rng, most) for _ in names]
        listed = ints(names)
        cache.reserve(ints([most] * len(names)), sequences=listed)
        rows = embed[:, :, ints(tokens).long()]
        outs = []
        for layer in range(2):
            cache.append(layer, rows[layer, 0], rows[layer, 1], sequences=listed)
            query = torch.randn(len(names), most, 2 * heads, dim, device="cuda").to(torch.bfloat16)
            outs.append((query, cache.attention(layer, query, ints(parents), sequences=listed)))
        # Attention over the pages is attention over the plain token lists.
        for layer, (query, out) in enumerate(outs):
            for i, s in enumerate(names):
                line = texts[s] + tokens[i]
                keys, values = (embed[layer, w][line].cpu().double() for w in (0, 1))
                want, _, size = drafting.attention(query[i].cpu().double(), keys, values, len(texts[s]), parents[i], most, 2, dim ** -0.5)
                assert ((out[i].cpu().double() - want).abs() <= 2.0 ** -8 * (size + want.abs()) + 1e-3 * size).all()
        target = torch.softmax(torch.randn(len(names), most, vocab, device="cuda") + 3 * torch.nn.functional.one_hot(
            ints(tokens).long().roll(-1, 1), vocab), -1)
        accepted, path, token = tsac_cuda.draft_verify(target, ints(tokens), ints(parents),
                                                       torch.rand(len(names), most, device="cuda") * 0.3, torch.rand(len(names), device="cuda"))
        cache.keep(path, accepted, sequences=listed)
        cache.release(sequences=listed, positions=cache.lengths[listed.long()])
        for i, s in enumerate(names):
            texts[s] += [tokens[i][n] for n in path[i].tolist()[:accepted[i].item()]]
            last[s] = token[i].item()
        assert cache.lengths.tolist() == [len(texts.get(s, [])) for s in range(4)]
        assert any(n > 1 for n in accepted.tolist())
    table = cache.tables.tolist()
    for s, text in texts.items():
        for i, token in enumerate(text):
            assert torch.equal(cache.pool[:, :, table[s][i // 8], i % 8], embed[:, :, token])
    cache.release()
    assert cache.refs.sum().item() == 0


@pytest.mark.parametrize("kind,dim,group,nodes", [("bf16", 128, 1, 9), ("fp16", 64, 2, 8), ("bf16", 64, 4, 17), ("fp16", 128, 8, 33)])
def test_output_in_place_of_the_query(kind, dim, group, nodes):
    """One buffer for query and output, items split over CTAs and whole ones alike."""
    s = Setup(kind, dim, 2, group, 16, [4000, 3, 90, 700], [nodes, nodes, 2, nodes], seed=17)
    buffer = s.query.cuda()
    lse = torch.full((4, nodes, 2 * group), 77.0, device="cuda")
    out = s.cache.attention(0, buffer, ints(s.parents), buffer, nodes=ints(s.nodes), lse=lse)
    assert out is buffer
    got = out.cpu().double()
    assert torch.equal(got[2, 2:], s.query[2, 2:].double())
    got[2, 2:] = 77.0
    s.check(got, lse.cpu().double())


@pytest.mark.parametrize("kind,dim,group,nodes", [("bf16", 128, 2, 7), ("fp16", 64, 1, 16), ("fp16", 128, 4, 20), ("bf16", 64, 8, 30)])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_queries_that_are_not_finite_stay_in_their_rows(kind, dim, group, nodes, bad):
    s = Setup(kind, dim, 2, group, 16, [300, 20], [nodes, nodes], seed=18)
    clean, clean_lse = s.run()
    finite = s.query.clone()
    spoiled = [(0, 0, 0), (0, nodes - 1, 2 * group - 1), (1, nodes // 2, group)]
    for b, n, h in spoiled:
        s.query[b, n, h, 5] = bad
    out, lse = s.run()
    s.query = finite
    for b, n, h in spoiled:
        assert not torch.isfinite(out[b, n, h]).any()
        out[b, n, h], lse[b, n, h] = clean[b, n, h], clean_lse[b, n, h]
    s.check(out, lse)


@pytest.mark.parametrize("dim,group,nodes", [(128, 1, 20), (64, 5, 40)])
def test_positions_past_two_gigabytes_for_many_rows(dim, group, nodes):
    """The same for the kernel of many rows, in the second of two layers: planes of more than 4 GiB."""
    heads = 32768 // dim
    cache = tsac_cuda.PagedCache.empty(2, 70, 1024, heads, dim, 2, 66, dtype=torch.float16)  # 64 MiB a page
    torch.manual_seed(1)
    used = [69, 3, 68]
    cache.tables[1, :3] = ints(used)
    cache.counts[1] = 3
    cache.refs[used] = 1
    length = 2050 - nodes
    cache.lengths[1] = length
    for page in used:
        cache.pool[1, :, page].normal_()
    parents = ints([[-1] + [n // 2 for n in range(nodes - 1)]])
    query = torch.randn(1, nodes, heads * group, dim, device="cuda").to(torch.float16)
    errors = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = cache.attention(1, query, parents, sequences=ints([1]), error_word=errors)
    assert errors.item() == 0
    keys, values = (cache.pool[1, i][used].flatten(0, 1)[:length + nodes] for i in (0, 1))
    for head in (0, heads - 1):
        mine = slice(head * group, (head + 1) * group)
        want, _, size = drafting.attention(query[0, :, mine].cpu().double(), keys[:, head:head + 1].cpu().double(),
                                           values[:, head:head + 1].cpu().double(), length, parents[0].tolist(), nodes, group, dim ** -0.5)
        # h (A + |out|) plus a thousandth of A for the 32-bit parts and subnormals, as in Setup.check.
        assert ((out[0, :, mine].cpu().double() - want).abs() <= 2.0 ** -11 * (size + want.abs()) + 1e-3 * size).all()


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("group,nodes", [(1, 24), (4, 33), (16, 20)])
@pytest.mark.parametrize("length", [1, 61, 63, 126, 131, 382])
def test_drafted_values_that_are_not_finite_at_any_start(dim, group, nodes, length):
    """Drafted rows that begin anywhere in a tile, so that the lanes that look at a row are not those that
    copied it, every fourth node with an undefined value."""
    s = Setup("bf16", dim, 2, group, 16, [length, length + 1], [nodes, nodes], seed=length)
    clean, clean_lse = s.run()
    damaged = s.cache.pool.clone()
    marks = [(b, node, (7 * node + b) % dim) for b in (0, 1) for node in range(0, nodes, 4)]
    for b, node, column in marks:
        at = s.lengths[b] + node
        damaged[0, 1, s.tables[b, at // 16], at % 16, 1, column] = math.nan
    s.cache.pool.copy_(damaged)
    hit = torch.zeros_like(clean, dtype=torch.bool)
    for b, node, column in marks:
        for n, seen in enumerate(drafting.ancestors(s.parents[b], nodes)):
            hit[b, n, group:, column] |= node in seen
    for _ in range(5):
        out, lse = s.run()
        assert torch.equal(torch.isnan(out), hit) and torch.equal(lse, clean_lse)
        s.check(torch.where(hit, clean, out), lse)


@pytest.mark.parametrize("kind,dim,group", [("bf16", 128, 8), ("fp16", 64, 5), ("bf16", 64, 2)])
def test_undefined_values_in_some_of_many_trees(kind, dim, group):
    """Several items one after another in each CTA, some with drafted values that are undefined: the marks
    of one never reach the next."""
    count, nodes = 60, 48
    s = Setup(kind, dim, 8, group, 16, [(37 * b) % 300 for b in range(count)], [nodes - b % 5 for b in range(count)], seed=4)
    clean, clean_lse = s.run()
    damaged = s.cache.pool.clone()
    hit = torch.zeros_like(clean, dtype=torch.bool)
    for b in range(0, count, 3):
        for head in range(8):
            node, column = (5 * b + 11 * head) % s.nodes[b], (b + 9 * head) % dim
            at = s.lengths[b] + node
            damaged[0, 1, s.tables[b, at // 16], at % 16, head, column] = math.nan
            for n, seen in enumerate(drafting.ancestors(s.parents[b], s.nodes[b])):
                hit[b, n, head * group:(head + 1) * group, column] |= node in seen
    s.cache.pool.copy_(damaged)
    for _ in range(5):
        out, lse = s.run()
        assert torch.equal(torch.isnan(out), hit) and torch.equal(lse, clean_lse)
    s.check(torch.where(hit, clean, out), lse, entries=[0, 1, 2, 27, 58])


@pytest.mark.parametrize("kind,dim,group,nodes", [("fp16", 64, 1, 1), ("fp16", 128, 4, 4), ("fp16", 64, 4, 32), ("fp16", 128, 3, 7),
                                                  ("fp16", 64, 8, 64), ("fp16", 128, 8, 64), ("bf16", 128, 4, 4), ("bf16", 64, 8, 20)])
@pytest.mark.parametrize("nats", [16.0, 18.0, 20.0])
@pytest.mark.parametrize("sink", [0, 19000])
def test_small_weights_beside_a_dominant_key(kind, dim, group, nodes, nats, sink):
    """One key far above 20,000 others, with zeros as its value: the others' weights are the output, and
    fp16 has to hold them.  A weight is rounded by half a step of itself, or by 2^-25 where it is subnormal;
    with the row's largest at 2^10 at least that is 2^-35 per key in units of the largest.  The sequence is
    listed often enough that no item is split over many CTAs, each of which would have a maximum of its own."""
    length, page, scale, count = 20_000, 64, dim ** -0.5, 296
    g = torch.Generator().manual_seed(dim + nodes)
    pages = -(-(length + nodes) // page)
    keys = torch.randn(pages * page, dim, generator=g) * 0.3
    values = 1.0 + 0.25 * torch.randn(pages * page, dim, generator=g)
    keys[sink], values[sink] = nats / math.sqrt(dim), 0.0
    query = (1.0 + 0.05 * torch.randn(1, nodes, group, dim, generator=g)).to(TYPES[kind]).cuda()
    pool = torch.stack((keys, values)).view(1, 2, pages, page, 1, dim).to(TYPES[kind]).cuda()
    cache = tsac_cuda.PagedCache(pool, torch.arange(pages, dtype=torch.int32, device="cuda")[None], ints([pages]), ints([length]),
                                 torch.ones(pages, dtype=torch.int32, device="cuda"))
    lse = torch.empty(count, nodes, group, device="cuda")
    out = cache.attention(0, query.expand(count, -1, -1, -1), ints([[-1] + [0] * (nodes - 1)] * count), lse=lse,
                          sequences=torch.zeros(count, dtype=torch.int32, device="cuda")).double()
    k, v = (pool[0, i].reshape(-1, dim)[:length + nodes].double() for i in (0, 1))
    z = torch.einsum("nhd,kd->nhk", query[0].double(), k) * scale
    for n in range(nodes):  # node 0 and children of it
        z[n, :, length + 1:length + max(1, n)] = -math.inf
        z[n, :, length + n + 1:] = -math.inf
    p = torch.softmax(z, -1)
    want, size, want_lse = p @ v, p @ v.abs(), torch.logsumexp(z, -1)
    half, total = torch.finfo(TYPES[kind]).eps / 2, length + nodes
    reach = (query[0].double().abs().amax((0, 1)) * k.abs().amax(0)).sum().item() * scale
    fine = (2 * (dim + 2) * reach + 2 * total) * 2.0 ** -23
    tiny = 2.0 ** -25 + total * 2.0 ** -35 * v.abs().max().item() if kind == "fp16" else 0.0
    assert ((out - want).abs() <= half * (1 + fine) * size + half * want.abs() + fine * size + tiny).all()
    assert ((lse.double() - want_lse).abs() <= fine + 4 * 2.0 ** -23 * (1 + want_lse.abs())).all()


@pytest.mark.parametrize("kind,dim,group,nodes", [("fp16", 64, 1, 3), ("bf16", 128, 2, 8), ("fp16", 64, 4, 17), ("fp16", 128, 8, 33), ("bf16", 64, 4, 40)])
def test_scores_of_any_size(kind, dim, group, nodes):
    """Scores of up to 2^36 in powers of two, exact in 32 bits before the scale and far apart: the largest keys
    share the row, and the log of the sum is their score."""
    s = Setup(kind, dim, 1, group, 16, [700, 5], [nodes, nodes], seed=20)
    g = torch.Generator().manual_seed(20)
    s.pool[:, 0] = 0.0
    s.pool[:, 0, ..., 3] = torch.randint(-100, 101, s.pool[:, 0, ..., 3].shape, generator=g).to(s.pool.dtype)
    s.cache.pool.copy_(s.pool)
    s.query[:] = 0.0
    s.query[..., 3] = 2.0 ** 15 * torch.where(torch.arange(nodes) % 3 == 2, -1, 1)[:, None]
    for power in range(0, 14):
        scale = 2.0 ** power * (1 + 0.07 * power)
        out, lse = s.run(scale=scale)
        for b in (0, 1):
            keys, values = s.rows(b)
            want, want_lse, size = drafting.attention(s.query[b].double(), keys, values, s.lengths[b], s.parents[b], nodes, group, scale)
            half = torch.finfo(TYPES[kind]).eps / 2
            # Weights of equal scores are equal but for their own rounding; the others are nothing.
            assert ((out[b] - want).abs() <= 2 * half * (size + want.abs()) + 2.0 ** -25).all(), (power, b)
            assert ((lse[b] - want_lse).abs() <= 4 * 2.0 ** -23 * (1 + want_lse.abs())).all(), (power, b)


@pytest.mark.parametrize("kind,dim,group,nodes", [("bf16", 128, 2, 7), ("fp16", 64, 1, 16), ("fp16", 128, 4, 20), ("bf16", 64, 8, 30)])
@pytest.mark.parametrize("length", [3, 20, 3000])
def test_rows_of_undefined_scores(kind, dim, group, nodes, length):
    """A query row with a NaN: its output and its log of the sum are NaN, whole items and shared ones alike."""
    s = Setup(kind, dim, 2, group, 16, [length, 20], [nodes, nodes], seed=21)
    clean, clean_lse = s.run()
    hit = torch.zeros_like(clean_lse, dtype=torch.bool)
    for b, n, h in ((0, 0, 0), (0, nodes - 1, 2 * group - 1), (1, nodes // 2, group)):
        s.query[b, n, h, 5] = math.nan
        hit[b, n, h] = True
    out, lse = s.run()
    assert torch.equal(torch.isnan(lse), hit) and torch.equal(torch.isnan(out), hit[..., None].expand_as(out))
    assert torch.equal(lse[~hit], clean_lse[~hit]) and torch.equal(out[~hit], clean[~hit])


@pytest.mark.parametrize("kind,dim,group,nodes", [("bf16", 128, 1, 5), ("fp16", 64, 2, 8), ("bf16", 64, 4, 17), ("fp16", 128, 8, 33)])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_a_scale_of_zero_hides_nothing(kind, dim, group, nodes, bad):
    """Zero times a score that is not finite is undefined, in a row of many keys and of one."""
    s = Setup(kind, dim, 2, group, 16, [300, 20, 0], [nodes, nodes, nodes], seed=18)
    hit = torch.zeros(3, nodes, 2 * group, dtype=torch.bool)
    for b, n, h in ((1, nodes - 1, 0), (2, 0, group), (2, 0, 0)):
        s.query[b, n, h, 3] = bad
        hit[b, n, h] = True
    out, lse = s.run(scale=0.0)
    assert torch.equal(torch.isnan(lse), hit) and torch.equal(torch.isnan(out), hit[..., None].expand_as(out))
    assert torch.isfinite(out[~hit]).all()


def test_scratch_is_sized_by_the_caches_device(monkeypatch):
    """Whichever device is current: here a second one is pretended, and every call of the library has to find
    the cache's own in its place."""
    s = Setup("bf16", 64, 1, 2, 16, [40], [4], seed=22)
    current, calls = [7], []

    class Guard:
        def __init__(self, index):
            self.index = index

        def __enter__(self):
            current.append(self.index)

        def __exit__(self, *exc):
            current.pop()

    class Library:
        def __getattr__(self, name):
            fn = getattr(tsac_cuda._drafting(), name)

            def called(*arguments):
                calls.append((name, current[-1]))
                return fn(*arguments)
            return called

    on = tsac_cuda._Device(s.cache.index)
    monkeypatch.setattr(on, "_current", lambda: current[-1])
    monkeypatch.setattr(on, "_cuda", type("Cuda", (), {"device": Guard}))
    monkeypatch.setattr(s.cache, "_on", on)
    monkeypatch.setattr(s.cache, "_lib", Library())
    s.check(*s.run())
    assert {name for name, _ in calls} == {"tsac_cuda_tree_attention", "tsac_cuda_tree_attention_scratch_bytes"}
    assert all(device == s.cache.index for _, device in calls), calls


def test_gradients_are_refused_not_dropped():
    s = Setup("bf16", 64, 1, 2, 16, [40], [4], seed=23)
    query, trees, rows = s.query.cuda(), ints(s.parents), torch.ones(1, 4, 1, 64, dtype=torch.bfloat16, device="cuda")
    s.cache.append(0, rows, rows)
    want = s.cache.attention(0, query, trees)
    learned, learned_rows = query.clone().requires_grad_(), rows.clone().requires_grad_()
    with pytest.raises(tsac_cuda.TsacError, match="query requires a gradient"):
        s.cache.attention(0, learned, trees)
    with pytest.raises(tsac_cuda.TsacError, match="out requires a gradient"):
        s.cache.attention(0, query, trees, learned)
    with pytest.raises(tsac_cuda.TsacError, match="keys requires a gradient"):
        s.cache.append(0, learned_rows, rows)
    with pytest.raises(tsac_cuda.TsacError, match="values requires a gradient"):
        s.cache.append(0, rows, learned_rows)
    with pytest.raises(tsac_cuda.TsacError, match="pool requires a gradient"):
        tsac_cuda.PagedCache(s.cache.pool.clone().requires_grad_(), s.cache.tables, s.cache.counts, s.cache.lengths, s.cache.refs)
    for block in (torch.no_grad, torch.inference_mode):
        with block():
            assert torch.equal(s.cache.attention(0, learned, trees), want)
            s.cache.append(0, learned_rows, learned_rows)
