"""The operators of drafted decoding over a paged key/value cache, as measured cases.

A probability model that answers token by token is bound by the latency of its
steps.  Drafting several tokens and checking them together needs four things
beside the model's projections: pages for the keys and values (forked, copied,
compacted and freed as continuations come and go), the rows of the drafted
tokens stored into them and the accepted ones kept, attention of a whole tree
of drafted tokens over the cache, and the verification of the tree against the
target's probabilities.

Each case runs either in plain torch operations (`own` false) or through this
repository's entry points (`own` true).  Sizes: the repository's own model (4
heads of 128, 12 layers, 1,024 tokens, histories up to 1,024) and generic ones.
"""
import math
import sys

import torch

own = False

DEVICE = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


def listed():
    return [
        # One decode step of this repository's temporal stack: 3 entropy lanes, a chain's worth of drafts.
        {"name": "attention codec lanes", "op": "attention", "type": "bf16", "batch": 3, "kv_heads": 4, "group": 1,
         "head_dim": 128, "page": 64, "nodes": 12, "length": 1023},
        # A serving batch with a small tree for each sequence and shared key heads.
        {"name": "attention batch trees", "op": "attention", "type": "bf16", "batch": 64, "kv_heads": 8, "group": 4,
         "head_dim": 128, "page": 16, "nodes": 16, "length": 4096},
        # Plain decoding: the tree is the single last token.
        {"name": "attention single tokens", "op": "attention", "type": "fp16", "batch": 96, "kv_heads": 4, "group": 8,
         "head_dim": 64, "page": 32, "nodes": 1, "length": 8191},
        # Two long documents with a large tree each: as much arithmetic as memory traffic.
        {"name": "attention long trees", "op": "attention", "type": "bf16", "batch": 2, "kv_heads": 8, "group": 4,
         "head_dim": 128, "page": 64, "nodes": 64, "length": 131072},
        # The codec's vocabulary, a chain of drafts for each of 64 recordings: latency.
        {"name": "verify codec chains", "op": "verify", "type": "fp32", "batch": 64, "vocab": 1024, "nodes": 12,
         "draft": True},
        # A text-sized vocabulary of odd size, chains drafted by sampling a draft model.
        {"name": "verify chains", "op": "verify", "type": "bf16", "batch": 48, "vocab": 50001, "nodes": 6, "draft": True},
        # A large vocabulary, trees of a draft model's likeliest tokens.
        {"name": "verify trees", "op": "verify", "type": "fp32", "batch": 160, "vocab": 131072, "nodes": 24,
         "draft": False},
        # One step's rows into the cache of the repository's temporal stack, and the accepted ones kept.
        {"name": "step codec lanes", "op": "step", "type": "bf16", "batch": 3, "layers": 12, "kv_heads": 4,
         "head_dim": 128, "page": 64, "nodes": 12, "length": 1000},
        # The same of a serving batch.
        {"name": "step batch", "op": "step", "type": "bf16", "batch": 64, "layers": 24, "kv_heads": 8, "head_dim": 128,
         "page": 16, "nodes": 24, "length": 500},
        # Continuations of one prompt replaced by copies of the better ones.
        {"name": "pages fork few", "op": "pages", "do": "fork", "type": "bf16", "layers": 12, "kv_heads": 4,
         "head_dim": 128, "page": 64, "roots": 2, "children": 3, "length": 900},
        # A beam or a group of samples for each of many prompts.
        {"name": "pages fork many", "op": "pages", "do": "fork", "type": "fp16", "layers": 16, "kv_heads": 8,
         "head_dim": 128, "page": 32, "roots": 16, "children": 7, "length": 2021},
        # A scattered pool drawn together so that its upper part can be given back.
        {"name": "pages compact", "op": "pages", "do": "compact", "type": "bf16", "layers": 24, "kv_heads": 8,
         "head_dim": 128, "page": 16, "pages": 2000, "live": 900, "sequences": 40},
    ]


def _log(rng, low, high):
    """A whole number of [low, high], even over its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 1)) - 0.5 / (high + 1))))))


def draw(rng):
    op = rng.choice(("attention", "attention", "verify", "step", "pages"))
    if op == "attention":
        case = {"op": op, "type": rng.choice(("bf16", "fp16")), "batch": _log(rng, 1, 96), "kv_heads": rng.choice((1, 2, 3, 4, 8)),
                "group": rng.choice((1, 2, 4, 5, 8)), "head_dim": rng.choice((64, 128)), "page": rng.choice((8, 16, 32, 64, 128, 256)),
                "nodes": rng.choice((1, _log(rng, 1, 64), _log(rng, 1, 64))), "length": _log(rng, 1, 131072)}
        top = work(listed()[3])
        while work(case)["bytes"] > top["bytes"] or work(case)["flops"] > top["flops"]:
            case["length"] = max(1, case["length"] * 2 // 3)
        return case
    if op == "verify":
        case = {"op": op, "type": rng.choice(("bf16", "fp16", "fp32")), "batch": _log(rng, 1, 160), "vocab": _log(rng, 1000, 131072),
                "nodes": _log(rng, 1, 32), "draft": rng.random() < 0.5}
        while case["batch"] * case["vocab"] * case["nodes"] > 160 * 131072 * 24 // 2:
            case["batch"] = max(1, case["batch"] // 2)
        return case
    case = {"op": op, "type": rng.choice(("bf16", "fp16")), "layers": rng.choice((2, 3, 6, 12, 16)), "kv_heads": rng.choice((1, 2, 4, 8)),
            "head_dim": rng.choice((64, 128)), "page": rng.choice((8, 16, 32, 64, 128))}
    if op == "step":
        case.update(batch=_log(rng, 1, 64), nodes=_log(rng, 1, 24), length=_log(rng, 1, 500))
    elif rng.random() < 0.5:
        case.update(do="fork", roots=_log(rng, 1, 16), children=_log(rng, 1, 7), length=_log(rng, 1, 2021))
    else:
        live = _log(rng, 8, 500)
        case.update(do="compact", live=live, pages=live + _log(rng, 4, 900), sequences=_log(rng, 1, 40))
    return case


def _lengths(case):
    """Committed positions of each sequence: ragged between half of `length` and all of it."""
    return [max(1, int(case["length"] * (1.0 - 0.5 * ((i * 0.6180339887) % 1.0)))) for i in range(case["batch"])]


def _nodes(case):
    """Nodes of each sequence's tree: the largest has `nodes`, the batch is padded to it."""
    return [max(1, case["nodes"] - (i * 5) % (case["nodes"] // 3 + 1)) for i in range(case["batch"])]


def work(case):
    size = BYTES[case["type"]]
    if case["op"] == "attention":
        n, length = _nodes(case), _lengths(case)
        heads = case["kv_heads"] * case["group"]
        kv = sum(a + b for a, b in zip(n, length)) * case["kv_heads"] * case["head_dim"] * 2 * size
        rows = sum(n) * heads * case["head_dim"] * 2 * size
        return {"bytes": kv + rows, "flops": 4 * heads * case["head_dim"] * sum(a * (b + 1) for a, b in zip(n, length))}
    if case["op"] == "verify":
        # The target's row at the last accepted node, and the draft's beside it; a gather for each node.
        rows = 2 if case["draft"] else 1
        return {"bytes": case["batch"] * (rows * case["vocab"] * size + case["nodes"] * (rows * size + 16)),
                "flops": case["batch"] * case["vocab"] * (3 if case["draft"] else 1)}
    row = case["kv_heads"] * case["head_dim"] * size
    if case["op"] == "step":
        n = sum(_nodes(case))
        return {"bytes": case["layers"] * 2 * row * (2 * n + 2 * (n // 2)), "flops": 0}
    page = case["layers"] * 2 * case["page"] * row
    if case["do"] == "fork":
        # One private copy of the last page for each child, and the tables.
        held = -(-(case["length"] + 1) // case["page"])
        return {"bytes": case["roots"] * case["children"] * ((2 * page if case["length"] % case["page"] else 0) + 8 * held), "flops": 0}
    # Live pages that lie above where the last one will be, moved once.
    return {"bytes": 2 * page * case["live"] * (case["pages"] - case["live"]) / case["pages"] + 8 * case["pages"], "flops": 0}


def _pool(case, pages, generator):
    """[layers][keys, values][pages][page][heads][head_dim]"""
    shape = (case.get("layers", 1), 2, pages, case["page"], case["kv_heads"], case["head_dim"])
    return torch.randn(shape, generator=generator, device=DEVICE, dtype=TYPES[case["type"]])


def _trees(batch, nodes, generator):
    """Parents of random trees: node 0 is the last known token, each later node's parent one of the four before it."""
    back = torch.randint(1, 5, (batch, nodes), generator=generator, device=DEVICE)
    index = torch.arange(nodes, device=DEVICE)
    parents = torch.maximum(index - back, torch.zeros_like(back))
    parents[:, 0] = -1
    return parents.to(torch.int32)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def _tables(held, width, pages, generator):
    """Distinct random pages for each sequence, -1 behind them, and the pages' reference counts."""
    order = torch.randperm(pages, generator=generator, device=DEVICE)
    held = torch.tensor(held, device=DEVICE)
    start = torch.cumsum(held, 0) - held
    at = torch.arange(width, device=DEVICE)
    tables = torch.where(at < held[:, None], order[(start[:, None] + at).clamp(max=pages - 1)], -1).to(torch.int32)
    refs = torch.zeros(pages, dtype=torch.int32, device=DEVICE)
    refs[order[:int(held.sum())]] = 1
    return tables, held.to(torch.int32), refs


def prepare(case, seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    kind = TYPES[case["type"]]
    state = {"case": case}
    if case["op"] == "attention":
        lengths, nodes = _lengths(case), _nodes(case)
        held = [-(-(a + b) // case["page"]) for a, b in zip(lengths, nodes)]
        pages = sum(held) + 3
        shape = (case["batch"], case["nodes"], case["kv_heads"] * case["group"], case["head_dim"])
        tables, counts, refs = _tables(held, max(held) + 1, pages, g)
        state.update(pool=_pool(case, pages, g), tables=tables, counts=counts, refs=refs, lengths=_ints(lengths), nodes=_ints(nodes),
                     most=max(lengths), parents=_trees(case["batch"], case["nodes"], g),
                     query=torch.randn(shape, generator=g, device=DEVICE, dtype=kind),
                     out=torch.zeros(shape, device=DEVICE, dtype=kind))
        return state
    if case["op"] == "verify":
        batch, nodes, vocab = case["batch"], case["nodes"], case["vocab"]
        logits = torch.randn((batch, nodes, vocab), generator=g, device=DEVICE) * 2.5
        target = torch.softmax(logits, -1).to(kind)
        draft = torch.softmax(logits.add_(torch.randn((batch, nodes, vocab), generator=g, device=DEVICE), alpha=0.5), -1).to(kind)
        del logits
        index = torch.arange(nodes, device=DEVICE)
        if case["draft"]:
            parents = (index - 1).to(torch.int32).expand(batch, nodes).contiguous()
            u = torch.rand((batch, nodes, 1), generator=g, device=DEVICE)
            drawn = torch.searchsorted(torch.cumsum(draft.float(), -1), u).clamp(max=vocab - 1)[..., 0]
            tokens = torch.roll(drawn, 1, 1)
        else:
            parents = _trees(batch, nodes, g)
            same = (parents[:, :, None] == parents[:, None, :]) & (index[None, :] < index[:, None])
            rank = same.sum(-1)
            best = torch.topk(draft, 5, -1).indices
            tokens = best[torch.arange(batch, device=DEVICE)[:, None], parents.long().clamp(min=0), rank.clamp(max=4)]
            draft = None
        state.update(target=target, draft=draft, parents=parents, tokens=tokens.to(torch.int32).contiguous(), nodes=_ints(_nodes(case)),
                     coins=torch.rand((batch, nodes), generator=g, device=DEVICE), draws=torch.rand(batch, generator=g, device=DEVICE))
        return state
    if case["op"] == "step":
        lengths, nodes = _lengths(case), _nodes(case)
        held = [-(-a // case["page"]) for a in lengths]
        more = case["nodes"] // case["page"] + 2
        pages = sum(held) + more * case["batch"] + 5
        tables, counts, refs = _tables(held, max(held) + more, pages, g)
        batch, most = case["batch"], case["nodes"]
        rows = (case["layers"], 2, batch, most, case["kv_heads"], case["head_dim"])
        # The accepted nodes: the first, then about half of the others, in ascending order.
        n = _ints(nodes)[:, None]
        at = torch.arange(most, device=DEVICE)
        taken = ((torch.rand((batch, most), generator=g, device=DEVICE) < 0.5) | (at == 0)) & (at < n)
        path = torch.sort(torch.where(taken, at, most), -1).values
        state.update(pool=_pool(case, pages, g), tables=tables, counts=counts, refs=refs, lengths=_ints(lengths), nodes=_ints(nodes),
                     path=torch.where(path < most, path, -1).to(torch.int32), accepted=taken.sum(-1).to(torch.int32),
                     rows=torch.randn(rows, generator=g, device=DEVICE, dtype=kind), after=torch.zeros(batch, dtype=torch.int32, device=DEVICE))
        return state
    if case["do"] == "fork":
        roots, children, page = case["roots"], case["children"], case["page"]
        lengths = [max(1, case["length"] - (i * 7) % (case["length"] // 4 + 1)) for i in range(roots)]
        held = [-(-a // page) for a in lengths] + [0] * (roots * children)
        pages = sum(held) + 2 * roots * (children + 1) + 9
        tables, counts, refs = _tables(held, max(held) + 2, pages, g)
        state.update(pool=_pool(case, pages, g), tables=tables, counts=counts, refs=refs, lengths=_ints(lengths + [0] * (roots * children)),
                     parents=_ints([i for i in range(roots) for _ in range(children)]),
                     children=_ints(list(range(roots, roots + roots * children))),
                     # Continuations before the prompts, so that these keep their own last pages.
                     sequences=_ints(list(range(roots, roots + roots * children)) + list(range(roots))),
                     positions=_ints([1] * (roots + roots * children)))
        return state
    live, pages, sequences = case["live"], case["pages"], case["sequences"]
    base = [live // sequences + (i < live % sequences) for i in range(sequences)]
    tables, counts, refs = _tables(base, max(base), pages, g)
    # A continuation of each sequence that shares its pages.
    tables, counts, refs = torch.cat((tables, tables)), torch.cat((counts, counts)), refs * 2
    state.update(pool=_pool(case, pages, g), tables=tables.contiguous(), counts=counts, refs=refs, lengths=counts * case["page"],
                 tables_out=torch.full_like(tables, -1), refs_out=torch.zeros_like(refs), live=torch.zeros(1, dtype=torch.int32, device=DEVICE))
    return state


# ------------------------------------------------------------ plain forms --
def _ancestors(parents):
    """[batch][node][node]: whether the second node is the first or one of its ancestors."""
    nodes = parents.shape[1]
    index = torch.arange(nodes, device=parents.device)
    edge = (parents[:, :, None] == index).float() + torch.eye(nodes, device=parents.device)
    return torch.linalg.matrix_power(edge, max(1, nodes - 1)) > 0


def _plain_attention(s):
    case, pool = s["case"], s["pool"]
    batch, nodes, page = case["batch"], case["nodes"], case["page"]
    at = torch.arange(s["most"] + nodes, device=DEVICE)
    slots = s["tables"].long().gather(1, (at // page).clamp(max=s["tables"].shape[1] - 1).expand(batch, -1)).clamp(min=0) * page + at % page
    known = at < s["lengths"][:, None]
    drafted = at - s["lengths"][:, None]
    held = drafted < s["nodes"][:, None]
    keys, values = (pool[0, i].reshape(-1, case["kv_heads"], case["head_dim"])[slots].float().masked_fill_(~held[..., None, None], 0.0).transpose(1, 2)
                    for i in (0, 1))
    sees = _ancestors(s["parents"]).gather(2, drafted.clamp(0, nodes - 1)[:, None].expand(-1, nodes, -1)) & held[:, None] | known[:, None]
    query = s["query"].float().view(batch, nodes, case["kv_heads"], case["group"], -1).permute(0, 2, 3, 1, 4)
    scores = query.reshape(batch, case["kv_heads"], -1, case["head_dim"]) @ keys.transpose(2, 3)
    scores = scores.view(batch, case["kv_heads"], case["group"], nodes, -1).mul_(case["head_dim"] ** -0.5)
    scores.masked_fill_(~sees[:, None, None], -math.inf)
    scores.sub_(scores.amax(-1, keepdim=True)).exp_()
    total = scores.sum(-1, keepdim=True)
    out = (scores.view(batch, case["kv_heads"], -1, at.numel()) @ values).view(batch, case["kv_heads"], case["group"], nodes, -1) / total
    out = out.permute(0, 3, 1, 2, 4).reshape(s["out"].shape).to(s["out"].dtype)
    live = torch.arange(nodes, device=DEVICE) < s["nodes"][:, None]
    s["out"].copy_(torch.where(live[..., None, None], out, s["out"]))
    return s["out"]


def _plain_verify(s):
    target, draft, parents, tokens = s["target"], s["draft"], s["parents"].long(), s["tokens"].long()
    batch, nodes, vocab = target.shape
    at, rows = torch.arange(nodes, device=DEVICE), torch.arange(batch, device=DEVICE)
    live = at < s["nodes"][:, None]
    real = live & (at > 0)
    above = parents.clamp(min=0)
    p = target[rows[:, None], above, tokens].double().masked_fill(~real, 0.0)
    siblings = (parents[:, :, None] == parents[:, None, :]) & (at[None, :] < at[:, None]) & real[:, None, :]
    if draft is not None:  # chains: one child for each node
        passes = s["coins"].double() * draft[rows[:, None], above, tokens].double() < p
    else:  # the likeliest tokens of a draft: each child's share of what its earlier siblings left
        left = 1.0 - (siblings.double() @ p[..., None])[..., 0]
        passes = s["coins"].double() * left < p
    chosen = passes & real & ~(siblings & passes[:, None, :]).any(-1)
    chosen[:, 0] = live[:, 0]
    accepted = ~(_ancestors(s["parents"]) & ~chosen[:, None, :]).any(-1) & live
    count = accepted.sum(-1)
    last = torch.where(accepted, at, 0).amax(-1)
    weights = target[rows, last].double()
    rejected = (parents == last[:, None]) & real
    if draft is not None:
        left = (weights - draft[rows, last].double()).clamp_(min=0.0)
        use = rejected.any(-1) & (left.sum(-1) > 0)
        weights = torch.where(use[:, None], left, weights)
    else:
        weights.scatter_reduce_(1, torch.where(rejected, tokens, 0), torch.where(rejected, 0.0, math.inf).double(), "amin")
    sums = torch.cumsum(weights, -1)
    token = torch.searchsorted(sums, s["draws"].double()[:, None] * sums[:, -1:], right=True)[:, 0]
    path = torch.sort(torch.where(accepted, at, nodes), -1).values
    return count.to(torch.int32), torch.where(path < nodes, path, -1).to(torch.int32), token.to(torch.int32)


def _plain_reserve(s, sequences, positions):
    pool, tables, counts, refs, page = s["pool"], s["tables"], s["counts"], s["refs"], s["case"]["page"]
    width = tables.shape[1]
    length, more = s["lengths"][sequences].long(), positions.long()
    at = torch.arange(width, device=DEVICE)
    wanted = (at >= (length // page)[:, None]) & (at * page < (length + more)[:, None]) & (more > 0)[:, None]
    held = at < counts[sequences][:, None]
    now = tables[sequences].long()
    i, j = torch.nonzero(wanted & held, as_tuple=True)
    pages = now[i, j]
    earlier = (pages[None, :] == pages[:, None]).tril(-1).sum(-1)
    copy = refs[pages] - earlier > 1
    fresh = wanted & ~held
    fresh[i[copy], j[copy]] = True
    a, b = torch.nonzero(fresh, as_tuple=True)
    new = torch.nonzero(refs == 0)[:a.numel(), 0]
    old = now[a, b]
    source = held[a, b]
    pool[:, :, new[source]] = pool[:, :, old[source]]
    refs.index_add_(0, old[source], torch.full_like(old[source], -1, dtype=torch.int32))
    refs[new] = 1
    tables[sequences[a], b] = new.to(torch.int32)
    counts[sequences] = torch.maximum(counts[sequences].long(), torch.where(more > 0, (length + more + page - 1) // page, 0)).to(torch.int32)


def _plain_slots(s, positions):
    """Pool rows of [batch][n] positions."""
    page = s["case"]["page"]
    return s["tables"].long().gather(1, (positions // page).clamp(0, s["tables"].shape[1] - 1)) * page + positions % page


def _plain_step(s):
    case, pool = s["case"], s["pool"]
    batch, nodes = case["batch"], case["nodes"]
    every = torch.arange(batch, device=DEVICE)
    _plain_reserve(s, every, s["nodes"])
    flat = pool.view(case["layers"], 2, -1, case["kv_heads"], case["head_dim"])
    at = torch.arange(nodes, device=DEVICE)
    live = at < s["nodes"][:, None]
    slots = _plain_slots(s, s["lengths"].long()[:, None] + at)[live]
    flat[:, :, slots] = s["rows"][:, :, live]
    kept = at < s["accepted"][:, None]
    source = _plain_slots(s, s["lengths"].long()[:, None] + s["path"].long().clamp(min=0))[kept]
    place = _plain_slots(s, s["lengths"].long()[:, None] + at)[kept]
    flat[:, :, place] = flat[:, :, source]
    torch.add(s["lengths"], s["accepted"], out=s["after"])
    return s["after"], s["tables"], s["counts"], s["refs"], pool


def _plain_fork(s):
    tables, counts, lengths, refs = s["tables"], s["counts"], s["lengths"], s["refs"]
    page, children, parents = s["case"]["page"], s["children"].long(), s["parents"].long()
    at = torch.arange(tables.shape[1], device=DEVICE)
    gone = tables[children][at < counts[children][:, None]].long()
    refs.index_add_(0, gone, torch.full_like(gone, -1, dtype=torch.int32))
    share = torch.div(lengths[parents] + page - 1, page, rounding_mode="floor")
    shared = torch.where(at < share[:, None], tables[parents], -1)
    tables[children], counts[children], lengths[children] = shared, share, lengths[parents]
    pages = shared[shared >= 0].long()
    refs.index_add_(0, pages, torch.ones_like(pages, dtype=torch.int32))
    _plain_reserve(s, s["sequences"].long(), s["positions"])
    return s["tables"], s["counts"], s["lengths"], s["refs"], s["pool"]


def _plain_compact(s):
    tables, refs, pool = s["tables"], s["refs"], s["pool"]
    used = refs > 0
    at = torch.arange(refs.numel(), device=DEVICE)
    live = used.sum()
    moved, holes = torch.nonzero(used & (at >= live))[:, 0], torch.nonzero(~used & (at < live))[:, 0]
    pool[:, :, holes] = pool[:, :, moved]
    to = at.clone()
    to[moved] = holes
    held = torch.arange(tables.shape[1], device=DEVICE) < s["counts"][:, None]
    s["tables_out"].copy_(torch.where(held, to[tables.long().clamp(min=0)].to(torch.int32), -1))
    s["refs_out"].zero_()
    s["refs_out"][to[used]] = refs[used]
    s["live"].copy_(live)
    return s["tables_out"], s["refs_out"], s["live"], pool


# ------------------------------------------------------ the framework's own --
def _library():
    if "tsac_cuda" not in sys.modules:
        sys.path.insert(0, "tsac-metal_b200")
    import tsac_cuda
    return tsac_cuda


def _cache(s):
    """The handle that a program keeps beside the tensors it describes."""
    if "cache" not in s:
        s["cache"] = _library().PagedCache(s["pool"], s["tables"], s["counts"], s["lengths"], s["refs"])
    return s["cache"]


def _own(s):
    case = s["case"]
    if case["op"] == "attention":
        return _cache(s).attention(0, s["query"], s["parents"], s["out"], nodes=s["nodes"])
    if case["op"] == "verify":
        return _library().draft_verify(s["target"], s["tokens"], s["parents"], s["coins"], s["draws"], draft=s["draft"], nodes=s["nodes"])
    cache = _cache(s)
    if case["op"] == "step":
        cache.reserve(s["nodes"])
        rows = s["rows"]
        for layer in range(case["layers"]):
            cache.append(layer, rows[layer, 0], rows[layer, 1], nodes=s["nodes"])
        cache.keep(s["path"], s["accepted"], lengths_out=s["after"])
        return s["after"], s["tables"], s["counts"], s["refs"], s["pool"]
    if case["do"] == "fork":
        cache.release(sequences=s["children"])
        cache.fork(s["parents"], s["children"])
        cache.reserve(s["positions"], sequences=s["sequences"])
        return s["tables"], s["counts"], s["lengths"], s["refs"], s["pool"]
    cache.compact(tables_out=s["tables_out"], refs_out=s["refs_out"], live=s["live"])
    return s["tables_out"], s["refs_out"], s["live"], s["pool"]


def run(state):
    if own:
        return _own(state)
    case = state["case"]
    if case["op"] == "pages":
        return _plain_fork(state) if case["do"] == "fork" else _plain_compact(state)
    return {"attention": _plain_attention, "verify": _plain_verify, "step": _plain_step}[case["op"]](state)


# ----------------------------------------------------- definitions, 64 bits --
def _up(parents, node):
    """A node and its ancestors, ascending."""
    line = []
    while node >= 0:
        line.append(node)
        node = parents[node]
    return line[::-1]


def _exact_attention(case, s):
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device=DEVICE)
    tables, parents = s["tables"].tolist(), s["parents"].tolist()
    size = case["page"]
    for b, (length, nodes) in enumerate(zip(_lengths(case), _nodes(case))):
        held = torch.tensor(tables[b][:-(-(length + nodes) // size)], device=DEVICE)
        k = s["pool"][0, 0][held].flatten(0, 1)[:length + nodes]
        v = s["pool"][0, 1][held].flatten(0, 1)[:length + nodes]
        shut = torch.ones((nodes, length + nodes), dtype=torch.bool, device=DEVICE)
        shut[:, :length] = False
        for n in range(nodes):
            shut[n, [length + a for a in _up(parents[b], n)]] = False
        for h in range(case["kv_heads"] * case["group"]):
            q = s["query"][b, :nodes, h].double()
            z = torch.einsum("nd,ld->nl", q, k[:, h // case["group"]].double()) / math.sqrt(case["head_dim"])
            out[b, :nodes, h] = torch.softmax(z.masked_fill(shut, -math.inf), -1) @ v[:, h // case["group"]].double()
    return out


def _exact_verify(case, s):
    counts, paths, picks = [], [], []
    parents, tokens, coins, draws = (s[k].tolist() for k in ("parents", "tokens", "coins", "draws"))
    for b, nodes in enumerate(_nodes(case)):
        path, rejected = [0], []
        for n in range(1, nodes):
            if parents[b][n] != path[-1]:
                continue
            p = s["target"][b, path[-1], tokens[b][n]].item()
            if s["draft"] is not None:
                passed = coins[b][n] * s["draft"][b, path[-1], tokens[b][n]].item() < p
            else:
                passed = coins[b][n] * (1.0 - sum(s["target"][b, path[-1], t].item() for t in rejected)) < p
            if passed:
                path.append(n)
                rejected = []
            else:
                rejected.append(tokens[b][n])
        weights = s["target"][b, path[-1]].double()
        if rejected and s["draft"] is not None:
            rest = torch.relu(weights - s["draft"][b, path[-1]].double())
            weights = rest if rest.sum() > 0 else weights
        elif rejected:
            weights[rejected] = 0.0
        sums = weights.cumsum(0)
        picks.append(int((sums <= draws[b] * sums[-1]).sum()))
        counts.append(len(path))
        paths.append(path + [-1] * (case["nodes"] - len(path)))
    return torch.tensor(counts, dtype=torch.float64), torch.tensor(paths, dtype=torch.float64), torch.tensor(picks, dtype=torch.float64)


class _Pages:
    """The page bookkeeping, one table entry after another, in lists."""

    def __init__(self, case, s):
        self.size, self.pool = case["page"], s["pool"].double()
        self.width = s["tables"].shape[1]
        self.lengths, self.refs = s["lengths"].tolist(), s["refs"].tolist()
        self.held = [row[:n] for row, n in zip(s["tables"].tolist(), s["counts"].tolist())]

    def room(self, sequence, more):
        first = self.lengths[sequence] // self.size
        last = (self.lengths[sequence] + more - 1) // self.size
        for j in range(first, last + 1):
            pages = self.held[sequence]
            if j < len(pages) and self.refs[pages[j]] == 1:
                continue
            page = min(p for p in range(len(self.refs)) if self.refs[p] == 0 and p not in self.taken)
            self.taken.add(page)
            if j < len(pages):
                self.pool[:, :, page] = self.pool[:, :, pages[j]]
                self.refs[pages[j]] -= 1
                pages[j] = page
            else:
                pages.append(page)

    def reserve(self, wants):
        self.taken = set()
        for sequence, more in wants:
            self.room(sequence, more)
        for page in self.taken:
            self.refs[page] = 1

    def row(self, sequence, position):
        return self.held[sequence][position // self.size], position % self.size

    def tables(self):
        return torch.tensor([row + [-1] * (self.width - len(row)) for row in self.held], dtype=torch.float64)


def _numbers(values):
    return torch.tensor(values, dtype=torch.float64)


def _exact_step(case, s):
    book = _Pages(case, s)
    nodes = _nodes(case)
    book.reserve(list(enumerate(nodes)))
    path, accepted = s["path"].tolist(), s["accepted"].tolist()
    for b, n in enumerate(nodes):
        start = book.lengths[b]
        at = [book.row(b, start + i) for i in range(n)]
        page, slot = (torch.tensor(x, device=DEVICE) for x in zip(*at))
        book.pool[:, :, page, slot] = s["rows"][:, :, b, :n].double()
        kept = book.pool[:, :, page, slot][:, :, path[b][:accepted[b]]]
        book.pool[:, :, page[:accepted[b]], slot[:accepted[b]]] = kept
    after = [a + b for a, b in zip(book.lengths, accepted)]
    return _numbers(after), book.tables(), _numbers([len(x) for x in book.held]), _numbers(book.refs), book.pool


def _exact_fork(case, s):
    book = _Pages(case, s)
    for parent, child in zip(s["parents"].tolist(), s["children"].tolist()):
        for page in book.held[child]:
            book.refs[page] -= 1
        book.lengths[child] = book.lengths[parent]
        book.held[child] = book.held[parent][:-(-book.lengths[parent] // book.size)]
        for page in book.held[child]:
            book.refs[page] += 1
    book.reserve([(i, 1) for i in s["sequences"].tolist()])
    return book.tables(), _numbers([len(x) for x in book.held]), _numbers(book.lengths), _numbers(book.refs), book.pool


def _exact_compact(case, s):
    book = _Pages(case, s)
    live = sum(r > 0 for r in book.refs)
    holes = [p for p in range(live) if book.refs[p] == 0]
    to = {}
    for page in range(len(book.refs)):
        if book.refs[page]:
            to[page] = page if page < live else holes.pop(0)
            book.pool[:, :, to[page]] = book.pool[:, :, page]
    refs = [0] * len(book.refs)
    for page, place in to.items():
        refs[place] = book.refs[page]
    book.held = [[to[p] for p in row] for row in book.held]
    return book.tables(), _numbers(refs), _numbers([live]), book.pool


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "pages":
        return _exact_fork(case, s) if case["do"] == "fork" else _exact_compact(case, s)
    return {"attention": _exact_attention, "verify": _exact_verify, "step": _exact_step}[case["op"]](case, s)
