"""The operators of decoding with beams over caches of a fixed budget, and what they are measured on.

A case names an operator (``op``) and its sizes:

``tallied``   attention of each request's one new token over its pages; what the token gives every slot, summed over the query heads of a
              key/value head, is added to the slots' weights, and the token's own slot enters them with its position
``queries``   the weights that many queries (a prompt, or its last tokens) give the slots they see, added to the slots' weights, without a result
``evict``     keeps the ``keep`` slots of each key/value head that weigh most (the first and the latest positions always) and moves their records
              into the first ``keep`` slots, for all layers
``select``    the best continuations of a group's beams over beams and vocabulary, by the sum of log probabilities
``reorder``   beams take over what their parents hold: pages, the records of the page that is not full yet, state records

Where ``own`` is false the operators run in their plain form, where it is true through the package.
"""
from __future__ import annotations

import math

import torch

own = False

DEVICE = "cuda"


# ------------------------------------------------------------------------------------------ the cases
def listed() -> list[dict]:
    return [
        # one user's next token on the smallest shape: a launch and its latency
        _tallied("tallied 1 token", heads=14, kv_heads=2, dim=64, page=16, requests=1, context=512),
        # a server's steady state: sixteen conversations of different lengths
        _tallied("tallied 16 conversations", heads=28, kv_heads=4, dim=128, page=16, requests=16, context=4099),
        # a full batch of long conversations, just before their caches are cut back
        _tallied("tallied 64 at 8192", heads=28, kv_heads=4, dim=128, page=64, requests=64, context=8192),
        # a short question: its last tokens decide what stays
        _queries("queries 8 of 300", heads=14, kv_heads=2, dim=64, page=16, requests=1, context=300, count=8),
        # a long document whose last 32 tokens decide what stays of it
        _queries("queries 32 of 8192", heads=28, kv_heads=4, dim=128, page=16, requests=1, context=8192, count=32),
        # three whole prompts of different lengths in one step
        _queries("queries of three prompts", heads=32, kv_heads=8, dim=128, page=32, requests=3, context=2047, count=2047),
        # one conversation at its budget gives up a slot per layer and head at every token
        _evict("evict 1 slot", layers=24, kv_heads=2, dim=64, page=16, requests=1, context=1025, keep=1024, first=4, recent=64),
        # a long document is cut to its budget once its prompt has been read
        _evict("evict 28675 of 32771", layers=4, kv_heads=8, dim=128, page=64, requests=1, context=32771, keep=4096, first=4, recent=256),
        # one user's four beams: latency over a large vocabulary
        _select("select 1 group", groups=1, beams=4, vocab=151936, take=8),
        # a full batch of beams
        _select("select 32 groups", groups=32, beams=8, vocab=152064, take=16, logits="bfloat16"),
        # one user's four beams
        _reorder("reorder 1 group", groups=1, beams=4, layers=24, kv_heads=2, dim=64, page=16, context=517),
        # a full batch of beams of a decoder with state records beside its pages
        _reorder("reorder 16 groups", groups=16, beams=8, layers=28, kv_heads=4, dim=128, page=64, context=1061, states=4, record=32768),
    ]


def draw(rng) -> dict:
    op = rng.choice(["tallied", "tallied", "queries", "queries", "evict", "evict", "select", "select", "reorder"])
    heads, kv_heads, dim = rng.choice([(14, 2, 64), (28, 4, 128), (16, 4, 128), (32, 8, 128), (16, 16, 64), (24, 1, 128)])
    page = rng.choice([8, 16, 32, 64])
    if op == "tallied":
        requests = _spread(rng, 1, 96)
        return _tallied(None, heads=heads, kv_heads=kv_heads, dim=dim, page=page, requests=requests, context=min(_spread(rng, 1, 65536), (1 << 20) // (requests * kv_heads) + 1))
    if op == "queries":
        if rng.random() < 0.5:  # the last tokens of prompts
            requests, count = _spread(rng, 1, 8), _spread(rng, 1, 64)
            return _queries(None, heads=heads, kv_heads=kv_heads, dim=dim, page=page, requests=requests, context=count + _spread(rng, 1, 16384 // requests), count=count)
        requests = rng.choice([1, 1, 2, 3])  # prompts, or their portions
        count = _spread(rng, 65, 1500 if requests == 1 else 1000)
        return _queries(None, heads=heads, kv_heads=kv_heads, dim=dim, page=page, requests=requests, context=count + rng.choice([0, 0, _spread(rng, 1, 600)]), count=count)
    if op == "evict":
        requests, layers = _spread(rng, 1, 16), rng.choice([1, 2, 4, 8])
        context = max(2, min(_spread(rng, 16, 32768), 1000000 // (requests * layers * kv_heads)))
        keep = max(1, context - _spread(rng, 1, context))
        return _evict(None, layers=layers, kv_heads=kv_heads, dim=dim, page=page, requests=requests, context=context, keep=keep, first=rng.choice([0, 1, 4]), recent=min(keep, rng.choice([0, 1, 32, 256])))
    beams = rng.choice([1, 2, 3, 4, 5, 8, 16, 32])
    groups = max(1, min(_spread(rng, 1, 64), 256 // beams))
    if op == "select":
        return _select(None, groups=groups, beams=beams, vocab=rng.choice([32000, 151936, 152064, rng.randint(1000, 160000), rng.randint(1000, 160000)]), take=min(64, rng.choice([beams, 2 * beams])),
                       logits=rng.choice(["float32", "bfloat16"]))
    groups = max(1, min(groups, 128 // beams))
    return _reorder(None, groups=groups, beams=beams, layers=rng.choice([1, 4, 24, 28]), kv_heads=kv_heads, dim=dim, page=page, context=_spread(rng, 1, 2000), states=rng.choice([0, 0, 1, 4]),
                    record=rng.choice([1024, 4096, 32768, rng.randint(1, 20000)]))


def _tallied(name, *, heads, kv_heads, dim, page, requests, context) -> dict:
    """``context``: the most slots that a request holds, its new token's among them (they hold between half of it and all)."""
    return _named(name, op="tallied", heads=heads, kv_heads=kv_heads, dim=dim, page=page, requests=requests, context=context)


def _queries(name, *, heads, kv_heads, dim, page, requests, context, count) -> dict:
    """``count``: the most queries of a request; they stand in the last of its slots."""
    return _named(name, op="queries", heads=heads, kv_heads=kv_heads, dim=dim, page=page, requests=requests, context=max(context, count), count=count)


def _evict(name, *, layers, kv_heads, dim, page, requests, context, keep, first, recent) -> dict:
    return _named(name, op="evict", layers=layers, kv_heads=kv_heads, dim=dim, page=page, requests=requests, context=context, keep=keep, first=first, recent=recent)


def _select(name, *, groups, beams, vocab, take, logits="float32") -> dict:
    return _named(name, op="select", groups=groups, beams=beams, vocab=vocab, take=take, logits=logits)


def _reorder(name, *, groups, beams, layers, kv_heads, dim, page, context, states=0, record=1024) -> dict:
    """``states``: layers that hold a state record of ``record`` float32 entries per beam instead of pages."""
    return _named(name, op="reorder", groups=groups, beams=beams, layers=layers, kv_heads=kv_heads, dim=dim, page=page, context=context, states=states, record=record)


def _named(name, **case) -> dict:
    return {**({"name": name} if name else {}), **case}


def _spread(rng, low: int, high: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(low), math.log(max(low, high))))))


def _lengths(case) -> list[int]:
    n, most = case["requests"], case["context"]
    return [max(1, most - i * most // (2 * n)) for i in range(n)]


def _counts(case) -> list[int]:
    """Queries of each request: whole prompts stay whole, the last tokens of prompts are as many for all of them."""
    return [min(case["count"], length) for length in _lengths(case)]


# ------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case) -> dict:
    op = case["op"]
    if op == "select":
        rows = case["groups"] * case["beams"]
        return {"bytes": rows * case["vocab"] * {"bfloat16": 2, "float32": 4}[case["logits"]] + rows * 4 + case["groups"] * case["take"] * 12, "flops": rows * case["vocab"] * 3}
    if op == "reorder":
        beams, groups, page = case["beams"], case["groups"], case["page"]
        moved = (case["context"] % page) * case["layers"] * 2 * case["kv_heads"] * case["dim"] * 2 + case["states"] * case["record"] * 4 + case["context"] // page * 4
        # beams whose parent is another one are written; beams that are another one's parent are read (parents are drawn evenly)
        written, read = beams - 1, beams * (1 - (1 - 1 / beams) ** (beams - 1))
        return {"bytes": groups * moved * (written + read) + groups * beams * 4, "flops": 0}
    lengths, kv, dim = _lengths(case), case["kv_heads"], case["dim"]
    if op == "tallied":
        slots = sum(lengths) * kv
        return {"bytes": slots * (4 * dim + 8) + 4 * len(lengths) * (case["heads"] * dim + kv), "flops": 4 * sum(lengths) * case["heads"] * dim}
    if op == "queries":
        counts = _counts(case)
        seen = sum(n * length - n * (n - 1) // 2 for n, length in zip(counts, lengths))  # query i of n sees length - n + i + 1 slots
        return {"bytes": sum(lengths) * kv * (2 * dim + 8) + sum(counts) * case["heads"] * dim * 2, "flops": 2 * seen * case["heads"] * dim}
    keep, first, recent, total = case["keep"], case["first"], case["recent"], 0
    capacity = _blocks(case) * case["page"]
    for n in lengths:
        later = max(0, n - keep)  # slots behind the first `keep`
        fixed = min(recent, later, keep)
        free = max(1, n - first - recent)
        moves = (fixed + max(0, keep - first - recent) * max(0, later - recent) / free) if later else 0
        total += kv * case["layers"] * (n * 8 + capacity * 8 + moves * 2 * 4 * dim)
    return {"bytes": total + 4 * 3 * len(lengths), "flops": 0}


# ------------------------------------------------------------------------------------------ inputs
def prepare(case, seed: int) -> dict:
    random = torch.Generator(DEVICE).manual_seed(seed)
    return {"tallied": _prepare_tallied, "queries": _prepare_queries, "evict": _prepare_evict, "select": _prepare_select, "reorder": _prepare_reorder}[case["op"]](case, random)


def _integers(values) -> torch.Tensor:
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def _records(random, *shape) -> torch.Tensor:
    """Keys and values [..., dim] as projections give them: normal, of another size from record to record, a few channels larger."""
    x = torch.randn(*shape, device=DEVICE, generator=random)
    x *= torch.exp2(0.5 * torch.randn(*shape[:-1], 1, device=DEVICE, generator=random))
    channels = torch.ones(shape[-1], device=DEVICE)
    channels[:: max(1, shape[-1] // 4)] = 4.0
    return (x * channels).to(torch.bfloat16)


def _pages(random, requests: int, blocks: int) -> torch.Tensor:
    """A block table [requests, blocks] of pages in no order, none of them twice."""
    return torch.randperm(requests * blocks, device=DEVICE, generator=random).to(torch.int32).view(requests, blocks)


def _blocks(case) -> int:
    return -(-case["context"] // case["page"])


def _history(random, lengths, kv, capacity, layers=None):
    """Slots' weights as the tokens before have left them (a few slots hold most), and their positions; none behind a request's length."""
    shape = (*([layers] if layers else []), len(lengths), kv, capacity)
    slot = torch.arange(capacity, dtype=torch.int32, device=DEVICE)
    held = (slot < _integers(lengths)[:, None])[:, None]
    weights = torch.exp(1.5 * torch.randn(shape, device=DEVICE, generator=random)) * held
    return weights, torch.where(held, slot, -1).expand(shape).contiguous()


def _prepare_pages(case, random) -> dict:
    lengths, kv, dim, page = _lengths(case), case["kv_heads"], case["dim"], case["page"]
    table = _pages(random, len(lengths), _blocks(case))
    weights, positions = _history(random, lengths, kv, table.shape[1] * page)
    return {"op": case["op"], "heads": case["heads"], "cache": _records(random, table.numel(), 2, kv, page, dim), "table": table, "lengths": _integers(lengths), "longest": max(lengths),
            "weights": weights, "positions": positions, "scale": dim ** -0.5}


def _queries_of(random, tokens, case) -> torch.Tensor:
    return (2.0 * torch.randn(tokens, case["heads"] * case["dim"], device=DEVICE, generator=random)).to(torch.bfloat16)


def _prepare_tallied(case, random) -> dict:
    s = _prepare_pages(case, random)
    s["weights"].masked_fill_(torch.arange(s["weights"].shape[2], device=DEVICE) == s["lengths"][:, None, None] - 1, 0.0)  # the new token's slot is yet to enter
    return {**s, "q": _queries_of(random, case["requests"], case), "newest": s["lengths"] + 5}


def _prepare_queries(case, random) -> dict:
    s, counts, lengths = _prepare_pages(case, random), _counts(case), _lengths(case)
    # slots of the queries' own tokens come without a history
    s["weights"].masked_fill_(torch.arange(s["weights"].shape[2], device=DEVICE) >= (s["lengths"] - _integers(counts))[:, None, None], 0.0)
    starts = [sum(counts[:i]) for i in range(len(counts) + 1)]
    most = max(counts)
    # for the plain form: a request's queries side by side, and the last slot that each of them sees (-1: no query)
    place = [[min(starts[i] + j, starts[i + 1] - 1) for j in range(most)] for i in range(len(counts))]
    last = [[lengths[i] - counts[i] + j if j < counts[i] else -1 for j in range(most)] for i in range(len(counts))]
    return {**s, "q": _queries_of(random, starts[-1], case), "starts": _integers(starts), "most": most, "place": torch.tensor(place, device=DEVICE), "last": torch.tensor(last, device=DEVICE)}


def _prepare_evict(case, random) -> dict:
    lengths, kv, dim, page, layers = _lengths(case), case["kv_heads"], case["dim"], case["page"], case["layers"]
    table = _pages(random, len(lengths), _blocks(case))
    weights, positions = _history(random, lengths, kv, table.shape[1] * page, layers)
    cache = torch.empty(layers, table.numel(), 2, kv, page, dim, dtype=torch.bfloat16, device=DEVICE)
    for layer in cache:
        layer.copy_(_records(random, *layer.shape))
    return {"op": "evict", "cache": cache, "table": table, "lengths": _integers(lengths), "newest": _integers(lengths) - 1, "weights": weights, "positions": positions,
            "after": (torch.empty_like(weights), torch.empty_like(positions)), "keep": case["keep"], "first": case["first"], "recent": case["recent"], "longest": max(lengths)}


def _prepare_select(case, random) -> dict:
    groups, beams, vocab = case["groups"], case["beams"], case["vocab"]
    # a language model's logits: a wide bulk and a few tokens that stand out
    logits = 2.0 * torch.randn(groups * beams, vocab, device=DEVICE, generator=random)
    few = torch.randint(0, vocab, (groups * beams, 8), device=DEVICE, generator=random)
    logits.scatter_(1, few, 12.0 + 2.0 * torch.randn(groups * beams, 8, device=DEVICE, generator=random))
    scores = -20.0 - 1.5 * torch.rand(groups, beams, device=DEVICE, generator=random)
    return {"op": "select", "logits": logits.to(getattr(torch, case["logits"])), "scores": scores, "take": case["take"]}


def _prepare_reorder(case, random) -> dict:
    groups, beams, page, kv, dim, layers = (case[name] for name in ("groups", "beams", "page", "kv_heads", "dim", "layers"))
    rows, blocks = groups * beams, case["context"] // page + 1
    # full pages are only pointed to, by whichever beams came from them; the pages that are not full yet are each beam's own
    table = torch.randint(0, rows, (rows, blocks), device=DEVICE, generator=random).to(torch.int32)
    table[:, -1] = torch.randperm(rows, device=DEVICE, generator=random)
    cache = torch.empty(layers, rows, 2 * kv, page, dim, dtype=torch.bfloat16, device=DEVICE)
    for layer in cache:
        layer.copy_(_records(random, *layer.shape))
    states = [torch.randn(case["states"], rows, case["record"], device=DEVICE, generator=random)] if case["states"] else []
    parents = torch.randint(0, beams, (groups, beams), device=DEVICE, generator=random).to(torch.int32)
    return {"op": "reorder", "parents": parents, "lengths": torch.full((groups,), case["context"], dtype=torch.int32, device=DEVICE), "table": table, "caches": [cache], "states": states}


# ------------------------------------------------------------------------------------------ one pass
def run(state: dict):
    return (_own if own else _plain)[state["op"]](state)


def _own_tallied(s):
    from hyperion_b200 import ops

    out = ops.attention_tallied(s["q"], s["heads"], s["cache"], s["table"], s["lengths"], s["newest"], ops.Tally(s["weights"], s["positions"]), s["scale"], longest=s["longest"])
    return out, s["weights"], s["positions"]


def _own_queries(s):
    from hyperion_b200 import ops

    ops.tally_queries(s["q"], s["heads"], s["cache"], s["table"], s["starts"], s["lengths"], ops.Tally(s["weights"], s["positions"]), s["scale"], most=s["most"], longest=s["longest"])
    return s["weights"]


def _own_evict(s):
    from hyperion_b200 import ops

    left = ops.evict(s["cache"], s["table"], s["lengths"], s["newest"], ops.Tally(s["weights"], s["positions"]), s["keep"], first=s["first"], recent=s["recent"], longest=s["longest"],
                     out=ops.Tally(*s["after"]))
    return left, s["cache"], s["after"]


def _own_select(s):
    from hyperion_b200.sampling import beam_select

    return tuple(beam_select(s["logits"], s["scores"], s["take"]))


def _own_reorder(s):
    from hyperion_b200 import ops

    ops.beam_reorder(s["parents"], s["lengths"], s["table"], s["caches"], s["states"])
    return s["table"], s["caches"], s["states"]


def _held(s, which):
    """Keys (0) or values (1) of every request [requests, kv, slots, dim], in 32 bits."""
    x = s["cache"][:, which][s["table"].long()].float()
    requests, blocks, kv, page, dim = x.shape
    return x.transpose(1, 2).reshape(requests, kv, blocks * page, dim)


def _weights_of(scores, visible):
    """Softmax over the visible slots; a query that sees none gives nothing."""
    scores = torch.where(visible, scores, -math.inf)
    top = scores.amax(-1, keepdim=True)
    weight = torch.exp(scores - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = weight.sum(-1, keepdim=True)
    return weight / torch.where(total > 0, total, torch.ones_like(total))


def _plain_tallied(s):
    k, kv = _held(s, 0), s["weights"].shape[1]
    q = s["q"].float().view(s["q"].shape[0], kv, s["heads"] // kv, -1)
    slot = torch.arange(k.shape[2], device=DEVICE)
    visible = slot < s["lengths"][:, None, None, None]
    weight = _weights_of((q @ k.transpose(2, 3)) * s["scale"], visible)
    v = torch.where(visible.transpose(2, 3), _held(s, 1), 0.0)
    out = (weight @ v).reshape(s["q"].shape).to(torch.bfloat16)
    given, entering = weight.sum(2), slot == s["lengths"][:, None, None] - 1
    s["weights"].copy_(torch.where(entering, given, s["weights"] + given))
    s["positions"].copy_(torch.where(entering, s["newest"][:, None, None], s["positions"]))
    return out, s["weights"], s["positions"]


def _plain_queries(s):
    k, kv, (requests, most) = _held(s, 0), s["weights"].shape[1], s["place"].shape
    q = s["q"].float().view(s["q"].shape[0], kv, s["heads"] // kv, -1)[s["place"]].permute(0, 2, 3, 1, 4)  # [requests, kv, group, queries, dim]
    visible = torch.arange(k.shape[2], device=DEVICE) <= s["last"][:, None, None, :, None]
    s["weights"] += _weights_of((q @ k.unsqueeze(2).transpose(3, 4)) * s["scale"], visible).sum((2, 3))
    return s["weights"]


def _plain_evict(s):
    weights, positions, keep, page = s["weights"], s["positions"], s["keep"], s["cache"].shape[4]
    layers, rows, kv, capacity = weights.shape
    slot = torch.arange(capacity, device=DEVICE)
    length = s["lengths"].long()[:, None, None]
    held, cut = slot < length, length > keep
    fixed = (positions < s["first"]) | (positions > s["newest"][:, None, None] - s["recent"])
    rank = torch.where(held, torch.where(fixed, math.inf, torch.nan_to_num(weights, nan=-3e38, posinf=math.inf, neginf=-3e38)), -math.inf)
    best = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :keep]
    kept = torch.zeros_like(rank, dtype=torch.bool).scatter_(-1, best, True) & held
    mover, hole = kept & (slot >= keep) & cut, ~kept & (slot < keep) & cut
    # the i-th slot that moves goes to the i-th free one
    place = torch.where(mover, mover.cumsum(-1) - 1, -1)
    holes = torch.sort(torch.where(hole, slot, capacity), dim=-1).values
    layer, row, head, source = mover.nonzero(as_tuple=True)
    target = holes[layer, row, head, place[layer, row, head, source]]
    table = s["table"].long()
    cache = s["cache"]
    cache[layer, table[row, target // page], :, head, target % page] = cache[layer, table[row, source // page], :, head, source % page]
    after, at = s["after"]
    stays = held & (slot < keep)
    after.copy_(torch.where(stays, weights, 0.0))
    at.copy_(torch.where(stays, positions, -1))
    after[layer, row, head, target] = weights[layer, row, head, source]
    at[layer, row, head, target] = positions[layer, row, head, source]
    return s["lengths"].clamp(max=keep), cache, s["after"]


def _plain_select(s):
    groups, beams = s["scores"].shape
    logits = s["logits"].double()
    score = torch.log_softmax(logits, 1) + s["scores"].double().view(-1, 1)
    # a row's best by one key of its logit's order and its index, so that ties go to the lowest; then the group's best among the rows' best
    bits = s["logits"].float().view(torch.int32)
    order = (bits ^ ((bits >> 31) & 0x7FFFFFFF)).long()
    vocab, few = logits.shape[1], min(s["take"], logits.shape[1])
    key = torch.topk((order << 32) | torch.arange(vocab - 1, -1, -1, device=DEVICE), few, dim=1).values
    token = vocab - 1 - (key & 0xFFFFFFFF)
    value, at = torch.sort(score.gather(1, token).view(groups, -1), dim=1, descending=True, stable=True)
    value, at = value[:, : s["take"]], at[:, : s["take"]]
    return (at // few).to(torch.int32), token.view(groups, -1).gather(1, at).to(torch.int32), value.float()


def _plain_reorder(s):
    groups, beams = s["parents"].shape
    table, page = s["table"], s["caches"][0].shape[3]
    source = (s["parents"].long() + torch.arange(groups, device=DEVICE)[:, None] * beams).view(-1)
    length = s["lengths"].long().repeat_interleave(beams)
    full, filled = length // page, length % page
    # the first records of the page that is not full: from the parent's page to the beam's own
    own_page = table.gather(1, full.clamp(max=table.shape[1] - 1)[:, None])[:, 0].long()
    for cache in s["caches"]:
        moved = torch.arange(page, device=DEVICE)[:, None] < filled[:, None, None, None]
        cache[:, own_page] = torch.where(moved, cache[:, own_page[source]], cache[:, own_page])
    for state in s["states"]:
        state.copy_(state[:, source])
    table.copy_(torch.where(torch.arange(table.shape[1], device=DEVICE) < full[:, None], table[source], table))
    return table, s["caches"], s["states"]


_own = {"tallied": _own_tallied, "queries": _own_queries, "evict": _own_evict, "select": _own_select, "reorder": _own_reorder}
_plain = {"tallied": _plain_tallied, "queries": _plain_queries, "evict": _plain_evict, "select": _plain_select, "reorder": _plain_reorder}


# ------------------------------------------------------------------------------------------ the definitions, in 64 bits
def exact(case, seed: int):
    s = prepare(case, seed)
    return {"tallied": _exact_tallied, "queries": _exact_queries, "evict": _exact_evict, "select": _exact_select, "reorder": _exact_reorder}[case["op"]](case, s)


def _exact_attention(case, s, counts, after):
    """Per request: the weights [kv, group, queries, slots] that its queries give, and its values; handed to ``after``."""
    kv, page, first = case["kv_heads"], case["page"], 0
    for r, (count, length) in enumerate(zip(counts, _lengths(case))):
        k, v = s["cache"][s["table"][r, : -(-length // page)].long()].double().permute(1, 2, 0, 3, 4).reshape(2, kv, -1, case["dim"])[:, :, :length]
        q = s["q"][first: first + count].double().view(count, kv, -1, case["dim"]).permute(1, 2, 0, 3)
        rows = max(1, (1 << 27) // (case["heads"] * length))  # queries at a time: a gigabyte of scores
        for i in range(0, count, rows):
            part = q[:, :, i: i + rows]
            last = torch.arange(length - count + i, length - count + i + part.shape[2], device=DEVICE)
            scores = (part @ k.unsqueeze(1).transpose(2, 3)) * case["dim"] ** -0.5
            scores.masked_fill_(torch.arange(length, device=DEVICE) > last[:, None], -math.inf)
            after(r, length, torch.softmax(scores, -1), v)
        first += count


def _exact_tallied(case, s):
    weights, out = s["weights"].double(), []

    def after(r, length, p, v):
        weights[r, :, length - 1] = 0
        weights[r, :, :length] += p.sum((1, 2))
        out.append((p @ v.unsqueeze(1)).reshape(1, -1))

    _exact_attention(case, s, [1] * case["requests"], after)
    return torch.cat(out), weights, None


def _exact_queries(case, s):
    weights = s["weights"].double()

    def after(r, length, p, v):
        weights[r, :, :length] += p.sum((1, 2))

    _exact_attention(case, s, _counts(case), after)
    return weights


def _exact_evict(case, s):
    return None  # nothing is computed: records and weights are moved


def _exact_select(case, s):
    groups, beams, take = case["groups"], case["beams"], case["take"]
    found = []
    for g in range(groups):  # a group at a time
        z = s["logits"][g * beams: (g + 1) * beams].double()
        z = z - torch.logsumexp(z, 1, keepdim=True) + s["scores"][g].double()[:, None]
        found.append(torch.topk(z.view(-1), take).values)
    return None, None, torch.stack(found)


def _exact_reorder(case, s):
    return None
