"""Verification of drafted tokens on the GPU against the rule in 64 bits (tests/drafting.py).

All results are integers and have to be equal.  Random probabilities put a
coin or a draw within 1e-12 (the rounding of 64-bit sums) of a border with a
probability below 1e-8 over all cases here, so no tolerance is needed."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import drafting
import tsac_cuda

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def case(batch, nodes, vocab, kind, with_draft, seed, chain=False, sharp=3.0):
    g = torch.Generator().manual_seed(seed)
    logits = torch.randn((batch, nodes, vocab), generator=g) * sharp
    target = torch.softmax(logits, -1).to(TYPES[kind])
    draft = torch.softmax(logits + torch.randn((batch, nodes, vocab), generator=g), -1).to(TYPES[kind])
    index = torch.arange(nodes)
    if chain:
        parents = (index - 1).expand(batch, nodes).clone()
    else:
        parents = torch.maximum(index - torch.randint(1, 6, (batch, nodes), generator=g), torch.zeros(1, dtype=torch.long))
        parents[:, 0] = -1
    rows = draft[torch.arange(batch)[:, None], parents.clamp(min=0)].float()
    tokens = torch.multinomial(rows.flatten(0, 1), 1, generator=g).view(batch, nodes)
    coins = torch.rand((batch, nodes), generator=g) * torch.rand((batch, 1), generator=g)  # some batches accept more
    draws = torch.rand(batch, generator=g)
    return target, tokens.int(), parents.int(), coins, draws, draft if with_draft else None


def check(target, tokens, parents, coins, draws, draft, nodes=None, word=0):
    batch, most, _ = target.shape
    cuda = [None if t is None else t.cuda() for t in (target, tokens, parents, coins, draws, draft)]
    count = torch.tensor(nodes, dtype=torch.int32).cuda() if nodes is not None else None
    errors = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = tsac_cuda.draft_verify(*cuda[:5], draft=cuda[5], nodes=count, error_word=errors)
    accepted, path, token = (t.cpu().tolist() for t in got)
    for b in range(batch):
        n = min(most, nodes[b]) if nodes is not None else most
        want, next_token = drafting.verify(target[b].double().numpy(), tokens[b].tolist(), parents[b].tolist(),
                                           coins[b].double().tolist(), float(draws[b]),
                                           None if draft is None else draft[b].double().numpy(), n)
        assert accepted[b] == len(want) and path[b] == want + [-1] * (most - len(want)), b
        assert token[b] == next_token, b
    assert errors.item() == word
    return accepted, path, token


@pytest.mark.parametrize("kind", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("with_draft", [False, True])
@pytest.mark.parametrize("vocab", [1, 2, 31, 1024, 1025, 16383, 16384, 33333])
def test_trees(kind, with_draft, vocab):
    accepted = []
    for chain in (False, True):
        accepted += check(*case(9, 11, vocab, kind, with_draft, vocab + chain, chain))[0]
    assert vocab < 31 or len(set(accepted)) > 1  # both accepted and rejected first children occur


@pytest.mark.parametrize("with_draft", [False, True])
@pytest.mark.parametrize("nodes", [1, 2, 64])
def test_tree_sizes(nodes, with_draft):
    check(*case(17, nodes, 700, "fp32", with_draft, nodes))
    check(*case(3, nodes, 40000, "fp32", with_draft, nodes))


def test_large_vocabulary_and_batch():
    check(*case(5, 3, 131073, "fp32", True, 1, chain=True, sharp=1.0))
    check(*case(300, 4, 130, "bf16", True, 2, chain=True))


def test_padded_batches():
    for with_draft in (False, True):
        check(*case(6, 9, 500, "fp32", with_draft, 4), nodes=[9, 0, 1, 5, -2, 100])


def test_strided_rows_of_every_alignment():
    """Rows that start anywhere, and target and draft rows that start at different places of 16 bytes."""
    for kind, skip in (("fp32", 1), ("bf16", 3), ("fp16", 7)):
        target, tokens, parents, coins, draws, draft = case(4, 5, 999, kind, True, 8)
        for a, b in ((skip, skip), (0, skip), (skip, 0)):
            wide = [torch.full((4, 5, 999 + 2 * skip + 2), 7.0, dtype=TYPES[kind]) for _ in range(2)]
            wide[0][:, :, a:a + 999], wide[1][:, :, b:b + 999] = target, draft
            cuda = [w.cuda() for w in wide]
            got = tsac_cuda.draft_verify(cuda[0][:, :, a:a + 999], tokens.cuda(), parents.cuda(), coins.cuda(), draws.cuda(),
                                         draft=cuda[1][:, :, b:b + 999])
            want = tsac_cuda.draft_verify(target.cuda(), tokens.cuda(), parents.cuda(), coins.cuda(), draws.cuda(), draft=draft.cuda())
            assert all(torch.equal(x, y) for x, y in zip(got, want))
    check(target, tokens, parents, coins, draws, draft)


def _rows(*rows):
    return torch.tensor(rows, dtype=torch.float32)[None]


def test_borders():
    """Coins and draws exactly on a border, in numbers that every type holds."""
    p = [0.25, 0.5, 0.125, 0.125]
    q = [0.5, 0.25, 0.125, 0.125]
    tree = torch.tensor([[-1, 0, 0]], dtype=torch.int32)
    for with_draft in (False, True):
        draft = _rows(q, q, q) if with_draft else None
        for first in range(4):
            for second in range(4):
                tokens = torch.tensor([[0, first, second]], dtype=torch.int32)
                for u in (0.0, 0.25, 0.5, 0.75):
                    for v in (0.0, 0.5, 2 / 3):
                        for draw in (0.0, 0.25, 0.5, 0.75, 1 - 2.0 ** -24):
                            check(_rows(p, p, p), tokens, tree, torch.tensor([[0.5, u, v]]), torch.tensor([draw]), draft)


def test_draft_that_covers_the_target():
    """No excess over the draft leaves the target as it was; the same distribution is always accepted."""
    p = [0.5, 0.5, 0.0, 0.0]
    chain = torch.tensor([[-1, 0]], dtype=torch.int32)
    for coin in (0.25, 1 - 2.0 ** -24):
        got = check(_rows(p, p), torch.tensor([[0, 1]], dtype=torch.int32), chain, torch.tensor([[0.0, coin]]), torch.tensor([0.75]), _rows(p, p))
        assert got[0] == [2]
    cover = [0.75, 0.75, 0.0, 0.0]
    got = check(_rows(p, p), torch.tensor([[0, 2]], dtype=torch.int32), chain, torch.tensor([[0.0, 0.5]]), torch.tensor([0.75]), _rows(cover, p))
    assert got[0] == [1] and got[2] == [1]


def test_rejected_tokens_that_were_everything():
    """Without a draft and with nothing left, the target itself: a coin of 1 is outside [0, 1) but must not hang or fault."""
    p = [0.0, 1.0, 0.0, 0.0]
    tree = torch.tensor([[-1, 0, 0]], dtype=torch.int32)
    got = check(_rows(p, p, p), torch.tensor([[0, 1, 1]], dtype=torch.int32), tree, torch.tensor([[0.0, 1.0, 0.5]]), torch.tensor([0.5]), None)
    assert got[0] == [1] and got[2] == [1]


def test_tokens_and_parents_that_are_none():
    target, tokens, parents, coins, draws, draft = case(5, 6, 77, "fp32", True, 3)
    tokens[0, 1], tokens[1, 2], tokens[2, 1] = 77, -1, 2147483647
    parents[3, 2], parents[3, 4], parents[4, 1] = 5, 4, -9
    for d in (None, draft):
        check(target, tokens, parents, coins, draws, d)


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("vocab", [50, 20000])
def test_rows_that_are_no_distribution(bad, vocab):
    """A NaN, an infinity or nothing but zeros where a token is drawn: token -1 and bit 1; rows that no draw reads do not matter."""
    target, tokens, parents, coins, draws, draft = case(4, 2, vocab, "fp32", True, 5, chain=True)
    coins[:, 1] = torch.tensor([0.999, 0.999, 0.0, 0.0])
    for d in (None, draft):
        t = target.clone()
        t[0, 0, (int(tokens[0, 1]) + 1) % vocab] = bad
        got = check(t, tokens, parents, coins, draws, d, word=1 if drafted_rejects(t, tokens, coins, d) else 0)
        t = target.clone()
        t[2, 1] = 0.0
        t[2, 0, int(tokens[2, 1])] = 1.0
        got = check(t, tokens, parents, coins, draws, d, word=1)
        assert got[2][2] == -1 and got[0][2] == 2
    d = draft.clone()
    d[1, 0, (int(tokens[1, 1]) + 1) % vocab] = bad
    target[1, 0, int(tokens[1, 1])] = 0.0
    assert check(target, tokens, parents, coins, draws, d, word=1)[2][1] == -1 if bad != bad else True


def drafted_rejects(target, tokens, coins, draft):
    x = int(tokens[0, 1])
    return not float(coins[0, 1]) * (1.0 if draft is None else float(draft[0, 0, x])) < float(target[0, 0, x])


def test_empty_batch_and_reused_outputs():
    target, tokens, parents, coins, draws, _ = case(3, 4, 64, "fp32", False, 6)
    empty = tsac_cuda.draft_verify(target[:0].cuda(), tokens[:0].cuda(), parents[:0].cuda(), coins[:0].cuda(), draws[:0].cuda())
    assert [t.shape[0] for t in empty] == [0, 0, 0]
    out = tuple(torch.full(s, 99, dtype=torch.int32, device="cuda") for s in ((3,), (3, 4), (3,)))
    got = tsac_cuda.draft_verify(target.cuda(), tokens.cuda(), parents.cuda(), coins.cuda(), draws.cuda(), out=out)
    want = check(target, tokens, parents, coins, draws, None)
    assert [t.tolist() for t in got] == list(want) and got[0] is out[0]


def test_captured_and_on_another_stream():
    args = [t.cuda() for t in case(4, 5, 20000, "fp32", False, 7)[:5]]
    want = [t.clone() for t in tsac_cuda.draft_verify(*args)]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got = tsac_cuda.draft_verify(*args)
        for t in got:
            t.fill_(-5)
        graph.replay()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_binding_refusals():
    target, tokens, parents, coins, draws, draft = (None if t is None else t.cuda() for t in case(2, 3, 16, "fp32", True, 9))
    with pytest.raises(tsac_cuda.TsacError, match="draft must be"):
        tsac_cuda.draft_verify(target, tokens, parents, coins, draws, draft=draft.half())
    with pytest.raises(tsac_cuda.TsacError, match="tokens must be"):
        tsac_cuda.draft_verify(target, tokens.long(), parents, coins, draws)
    with pytest.raises(tsac_cuda.TsacError, match="coins must be"):
        tsac_cuda.draft_verify(target, tokens, parents, coins[:, :2], draws)
    with pytest.raises(tsac_cuda.TsacError, match="draws must be"):
        tsac_cuda.draft_verify(target, tokens, parents, coins, draws.cpu())


def test_binding_refuses_error_words_of_other_sizes():
    target, tokens, parents, coins, draws, _ = (None if t is None else t.cuda() for t in case(2, 3, 16, "fp32", False, 9))
    for word in (torch.zeros(4, dtype=torch.uint8, device="cuda"), torch.zeros(1, dtype=torch.int64, device="cuda"),
                 torch.zeros(0, dtype=torch.int32, device="cuda")):
        with pytest.raises(tsac_cuda.TsacError, match="32-bit word"):
            tsac_cuda.draft_verify(target, tokens, parents, coins, draws, error_word=word)


@pytest.mark.parametrize("with_draft", [False, True])
@pytest.mark.parametrize("vocab", [64, 9001])
@pytest.mark.parametrize("draw", [-0.25, -float("inf"), float("nan"), 1.0, 7.0])
def test_draws_outside_the_interval_give_a_token(with_draft, vocab, draw):
    """Every output is written, with a token of positive weight."""
    target, tokens, parents, coins, draws, draft = case(3, 4, vocab, "fp32", with_draft, 6)
    target[..., :5], target[..., -3:] = 0.0, 0.0
    draws[1] = draw
    out = tuple(torch.full(s, 99999, dtype=torch.int32, device="cuda") for s in ((3,), (3, 4), (3,)))
    tsac_cuda.draft_verify(target.cuda(), tokens.cuda(), parents.cuda(), coins.cuda(), draws.cuda(),
                           draft=None if draft is None else draft.cuda(), out=out)
    want = drafting.verify(target[1].double().numpy(), tokens[1].tolist(), parents[1].tolist(), coins[1].double().tolist(),
                           1.0 if draw >= 1 else 0.0, None if draft is None else draft[1].double().numpy(), 4)
    assert out[1][1].tolist() == want[0] + [-1] * (4 - len(want[0])) and out[2][1].item() == want[1]
    assert target[1, want[0][-1], want[1]] > 0


@pytest.mark.parametrize("kind", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("vocab", [50, 20000])
def test_infinite_draft_probabilities_at_a_rejection(kind, vocab):
    """An infinite q takes its token's excess to nothing and leaves the others'; one that is drafted is rejected."""
    target, tokens, parents, coins, draws, draft = case(4, 2, vocab, kind, True, 5, chain=True)
    coins[:, 1] = 0.75
    for b in (1, 2):
        target[b, 0, int(tokens[b, 1])] = 0.0  # rejected
    likely = int(torch.argmax(target[1, 0].float() - draft[1, 0].float()))
    draft[1, 0, likely] = float("inf")
    draft[3, 0, int(tokens[3, 1])] = float("inf")
    accepted, _, token = check(target, tokens, parents, coins, draws, draft)
    assert accepted[1:] == [1, 1, 1] and token[1] != likely and token[3] != int(tokens[3, 1])
