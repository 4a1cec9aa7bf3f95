"""The operators that serve many requests from one 8-bit cache, and what they are measured on.

A case names an operator (``op``) and its sizes:

``store``      quantises the keys and values of a step's tokens and writes them to their pages: a record (a key or a value of one
               head) becomes codes of 8-bit floating point (e4m3) and one exponent e, the smallest in [-40, 40] with max|x| <= 448 * 2^e
``load``       reads records back from their pages as bfloat16
``attention``  the step's queries over their requests' pages, 8-bit or bfloat16; the first ``shared`` positions are the same pages for
               all requests of a group
``verify``     drafted tokens against the target's logits, from given random numbers: how many stand, and the token that follows them

Where ``own`` is false the operators run in their plain form, where it is true through the package.
"""
from __future__ import annotations

import math

import torch

own = False

LARGEST = 448.0           # of e4m3
EXPONENTS = (-40, 40)
DEVICE = "cuda"


# ------------------------------------------------------------------------------------------ the cases
def listed() -> list[dict]:
    return [
        # one user's next token on the smallest shape: a launch and its latency
        _store("store 1 token", tokens=1, heads=14, kv_heads=2, dim=64, page=16),
        # a long prompt's keys and values, out of the product's [queries | keys | values] rows, an odd number of them
        _store("store 8191 tokens", tokens=8191, heads=32, kv_heads=8, dim=128, page=64),
        # a short conversation handed on in bfloat16
        _load("load 700 tokens", tokens=700, kv_heads=4, dim=128, page=16),
        # 64 conversations of 2,048 positions leave the 8-bit cache (to another engine, to a host copy)
        _load("load 131072 tokens", tokens=131072, kv_heads=4, dim=128, page=32),
        # one user's next token: latency
        _attention("attend 1 token", heads=14, kv_heads=2, dim=64, page=16, requests=1, context=512),
        # a server's steady state: eight conversations that share nothing
        _attention("attend 8 conversations", heads=28, kv_heads=4, dim=128, page=16, requests=8, context=2048),
        # 64 conversations behind one system prompt
        _attention("attend 64 behind 4096", heads=28, kv_heads=4, dim=128, page=16, requests=64, groups=1, shared=4096, context=512),
        # drafted tokens of requests behind two prefixes of odd length, bfloat16 pages
        _attention("attend drafts, two prefixes", heads=32, kv_heads=8, dim=128, page=32, requests=16, groups=2, shared=1999, context=300, count=5, bits=16),
        # 256 questions about one long document: the largest
        _attention("attend 256 behind 16384", heads=28, kv_heads=4, dim=128, page=64, requests=256, groups=1, shared=16384, context=1024),
        # a portion of a prompt that goes on from what is cached
        _attention("attend a prompt's portion", heads=16, kv_heads=4, dim=128, page=16, requests=1, context=5000, count=1000),
        # one user's four drafts: latency over a large vocabulary
        _verify("verify 1 request", requests=1, drafts=4, vocab=151936),
        # a full batch's drafts over bfloat16 logits
        _verify("verify 64 requests", requests=64, drafts=5, vocab=152064, logits="bfloat16"),
    ]


def draw(rng) -> dict:
    op = rng.choice(["store", "load", "attention", "attention", "attention", "verify"])
    heads, kv_heads, dim = rng.choice([(14, 2, 64), (28, 4, 128), (16, 4, 128), (32, 8, 128), (16, 16, 64), (8, 1, 128)])
    page = rng.choice([8, 16, 32, 64])
    if op == "store":
        return _store(None, tokens=_spread(rng, 1, 8192), heads=heads, kv_heads=kv_heads, dim=dim, page=page, source=rng.choice(["bfloat16", "bfloat16", "float32"]))
    if op == "load":
        return _load(None, tokens=_spread(rng, 1, 65536), kv_heads=kv_heads, dim=dim, page=page, result=rng.choice(["bfloat16", "bfloat16", "float32"]))
    if op == "verify":
        return _verify(None, requests=_spread(rng, 1, 64), drafts=rng.randint(1, 7), vocab=rng.choice([32000, 151936, 152064, rng.randint(1000, 160000)]),
                       logits=rng.choice(["float32", "bfloat16"]), probabilities=rng.random() < 0.75, greedy=rng.random() < 0.25)
    bits = rng.choice([8, 8, 8, 16])
    kind = rng.choice(["alone", "shared", "shared", "drafts", "portion"])
    if kind == "portion":
        count = _spread(rng, 9, 1500)
        return _attention(None, heads=heads, kv_heads=kv_heads, dim=dim, page=page, requests=rng.choice([1, 1, 2, 3]), context=count + _spread(rng, 1, 6000), count=count, bits=bits)
    each = rng.randint(2, 8) if kind == "drafts" else 1
    if kind == "alone":
        requests = _spread(rng, 1, 64)
        return _attention(None, heads=heads, kv_heads=kv_heads, dim=dim, page=page, requests=requests, context=min(_spread(rng, 1, 16384), 131072 // requests + 1), bits=bits)
    groups = rng.choice([1, 1, 1, 2, 3])
    requests = groups * max(1, _spread(rng, 2, 192 if each == 1 else 32) // groups)
    return _attention(None, heads=heads, kv_heads=kv_heads, dim=dim, page=page, requests=requests, groups=groups, shared=_spread(rng, 64, 8192),
                      context=_spread(rng, 8, 1024), count=each, bits=bits)


def _store(name, *, tokens, heads, kv_heads, dim, page, source="bfloat16") -> dict:
    return _named(name, op="store", tokens=tokens, heads=heads, kv_heads=kv_heads, dim=dim, page=page, source=source)


def _load(name, *, tokens, kv_heads, dim, page, result="bfloat16") -> dict:
    return _named(name, op="load", tokens=tokens, kv_heads=kv_heads, dim=dim, page=page, result=result)


def _attention(name, *, heads, kv_heads, dim, page, requests, context, groups=0, shared=0, count=1, bits=8) -> dict:
    """``context``: the most positions that a request holds beyond the shared ones (they have between half of it and all), its new
    tokens among them; ``count``: the most new tokens of a request."""
    return _named(name, op="attention", heads=heads, kv_heads=kv_heads, dim=dim, page=page, requests=requests, groups=groups, shared=shared if groups else 0,
                  context=max(context, count), count=count, bits=bits)


def _verify(name, *, requests, drafts, vocab, logits="float32", probabilities=True, greedy=False) -> dict:
    """``probabilities``: the drafter gives its own; otherwise its tokens stand for themselves.  ``greedy``: every third request has temperature 0."""
    return _named(name, op="verify", requests=requests, drafts=drafts, vocab=vocab, logits=logits, probabilities=probabilities, greedy=greedy)


def _named(name, **case) -> dict:
    return {**({"name": name} if name else {}), **case}


def _spread(rng, low: int, high: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _counts(case) -> list[int]:
    """New tokens of each request; a batch's drafts differ in number."""
    n, most = case["requests"], case["count"]
    return [most if n == 1 or i == 0 else max(1, most - i % min(most, 4)) for i in range(n)]


def _contexts(case) -> list[int]:
    """Positions that each request holds beyond the shared ones, new tokens included."""
    n, counts = case["requests"], _counts(case)
    return [max(counts[i], case["context"] - i * case["context"] // (2 * n)) for i in range(n)]


def _draft_counts(case) -> list[int]:
    return [case["drafts"] - (i * 3) % (case["drafts"] + 1) for i in range(case["requests"])]


# ------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case) -> dict:
    op = case["op"]
    if op in ("store", "load"):
        records = case["tokens"] * 2 * case["kv_heads"]
        wide = {"bfloat16": 2, "float32": 4}[case["source" if op == "store" else "result"]]
        return {"bytes": records * (case["dim"] * (wide + 1) + 1), "flops": records * case["dim"] * 3}
    if op == "attention":
        counts, contexts, shared, dim = _counts(case), _contexts(case), case["shared"], case["dim"]
        keys = case["groups"] * shared + sum(contexts)
        record = dim + 1 if case["bits"] == 8 else 2 * dim
        seen = sum(n * (shared + c) - n * (n - 1) // 2 for n, c in zip(counts, contexts))  # token i of n sees c - n + i + 1 own positions
        return {"bytes": 2 * keys * case["kv_heads"] * record + 2 * sum(counts) * case["heads"] * dim * 2, "flops": 4 * seen * case["heads"] * dim}
    counts, vocab = _draft_counts(case), case["vocab"]
    rows, requests = sum(counts) + len(counts), len(counts)
    element = {"bfloat16": 2, "float32": 4}[case["logits"]]
    # every row's logits; the drafter's probabilities and the random numbers of the row at which a request ends
    return {"bytes": rows * vocab * element + requests * vocab * 4 * (2 if case["probabilities"] else 1), "flops": rows * vocab * 4 + requests * vocab * 3}


# ------------------------------------------------------------------------------------------ inputs
def prepare(case, seed: int) -> dict:
    random = torch.Generator(DEVICE).manual_seed(seed)
    return {"store": _prepare_store, "load": _prepare_load, "attention": _prepare_attention, "verify": _prepare_verify}[case["op"]](case, random)


def _integers(values) -> torch.Tensor:
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def _records(random, *shape) -> torch.Tensor:
    """Keys and values [..., dim] as projections give them: normal, of another size from record to record, a few channels larger."""
    x = torch.randn(*shape, device=DEVICE, generator=random)
    size = torch.exp2(0.5 * torch.randn(*shape[:-1], 1, device=DEVICE, generator=random))
    channels = torch.ones(shape[-1], device=DEVICE)
    channels[:: max(1, shape[-1] // 4)] = 4.0
    return x * size * channels


def _pages(random, requests: int, blocks: int) -> torch.Tensor:
    """A block table [requests, blocks] of pages in no order, none of them twice."""
    return torch.randperm(requests * blocks, device=DEVICE, generator=random).to(torch.int32).view(requests, blocks)


def _token_places(case, random):
    """Tokens of a few requests, one behind the other from position 0 on: (block table, token's row, token's position, pages)."""
    tokens, page = case["tokens"], case["page"]
    rows = max(1, min(64, tokens // 512))
    each = -(-tokens // rows)
    table = _pages(random, rows, -(-each // page))
    flat = torch.arange(tokens, device=DEVICE)
    return table, (flat // each).to(torch.int32), (flat % each).to(torch.int32), table.numel()


def _prepare_store(case, random) -> dict:
    kv, dim, heads = case["kv_heads"], case["dim"], case["heads"]
    table, row, position, pages = _token_places(case, random)
    source = torch.randn(case["tokens"], (heads + 2 * kv) * dim, device=DEVICE, generator=random)
    source[:, heads * dim:] = _records(random, case["tokens"], 2 * kv, dim).view(case["tokens"], -1)
    return {"op": "store", "source": source.to(getattr(torch, case["source"])), "k": heads * dim, "v": (heads + kv) * dim, "cache": _empty_cache(pages, case),
            "table": table, "row": row, "position": position}


def _empty_cache(pages, case):
    shape = (pages, 2, case["kv_heads"], case["page"])
    return torch.zeros(*shape, case["dim"], dtype=torch.uint8, device=DEVICE).view(torch.float8_e4m3fn), torch.zeros(shape, dtype=torch.int8, device=DEVICE)


def _prepare_load(case, random) -> dict:
    table, row, position, pages = _token_places(case, random)
    cache = _quantise(_records(random, pages, 2, case["kv_heads"], case["page"], case["dim"]))
    return {"op": "load", "cache": cache, "table": table, "row": row, "position": position, "dtype": getattr(torch, case["result"])}


def _prepare_attention(case, random) -> dict:
    counts, contexts, page, shared, groups = _counts(case), _contexts(case), case["page"], case["shared"], case["groups"]
    requests, heads, dim = case["requests"], case["heads"], case["dim"]
    each, whole = (requests // groups if groups else 1), shared // page
    own_blocks = -(-(shared + max(contexts)) // page) - whole
    # a group's requests hold the same pages for the shared positions, and pages of their own from there on, in no order; a page in which the shared
    # positions end is copied for each of them, as an engine does
    pages = torch.randperm(groups * whole + requests * own_blocks, device=DEVICE, generator=random).to(torch.int32)
    table = pages[groups * whole:].view(requests, own_blocks)
    if whole:
        table = torch.cat([pages[: groups * whole].view(groups, whole).repeat_interleave(each, 0), table], 1)
    x = _records(random, pages.numel(), 2, case["kv_heads"], page, dim)
    if shared % page:
        at = table[:, whole].long()
        x[at, :, :, : shared % page] = x[at[::each].repeat_interleave(each)][:, :, :, : shared % page]
    cache = _quantise(x) if case["bits"] == 8 else x.to(torch.bfloat16)
    del x
    tokens, most = sum(counts), max(counts)
    starts = [sum(counts[:i]) for i in range(requests)]
    q = (2.0 * torch.randn(tokens, heads * dim, device=DEVICE, generator=random)).to(torch.bfloat16)
    state = {"op": "attention", "q": q, "heads": heads, "kv": case["kv_heads"], "dim": dim, "page": page, "cache": cache, "table": table, "scale": dim ** -0.5,
             "shared": shared, "groups": groups, "counts": counts, "lengths": [shared + c for c in contexts],
             # for the plain form: a request's tokens side by side, and how many positions beyond the shared ones each of them sees
             "place": torch.tensor([[starts[i] + min(j, counts[i] - 1) for j in range(most)] for i in range(requests)], device=DEVICE),
             "seen": torch.tensor([[contexts[i] - counts[i] + 1 + min(j, counts[i] - 1) for j in range(most)] for i in range(requests)], device=DEVICE),
             "back": torch.tensor([i * most + j for i in range(requests) for j in range(counts[i])], device=DEVICE)}
    if own:
        from hyperion_b200.ops.shared import plan_shared

        state["plan"] = plan_shared(counts, state["lengths"], heads, case["kv_heads"], dim, shared=[(g * each, each, shared) for g in range(groups)], device=q.device)
    return state


def _prepare_verify(case, random) -> dict:
    counts, vocab = _draft_counts(case), case["vocab"]
    rows, requests = sum(counts) + len(counts), len(counts)
    starts = [sum(counts[:i]) + i for i in range(requests + 1)]
    # a language model's logits: a wide bulk and a few tokens that stand out
    logits = 2.0 * torch.randn(rows, vocab, device=DEVICE, generator=random)
    few = torch.randint(0, vocab, (rows, 8), device=DEVICE, generator=random)
    logits.scatter_(1, few, 12.0 + 2.0 * torch.randn(rows, 8, device=DEVICE, generator=random))
    guess = logits + 0.4 * torch.randn(rows, vocab, device=DEVICE, generator=random)
    guess = guess.sub_(guess.amax(1, keepdim=True)).exp_()
    guess = guess.div_(guess.sum(1, keepdim=True))
    drafts = (guess / _exponential(random, rows, vocab)).argmax(1).to(torch.int32)
    temperature = [0.0 if case["greedy"] and i % 3 == 0 else (1.0, 0.8, 0.6)[i % 3] for i in range(requests)]
    owner = [i for i, n in enumerate(counts) for _ in range(n + 1)]
    most = max(counts) + 1
    return {"op": "verify", "logits": logits.to(getattr(torch, case["logits"])), "start": _integers(starts), "drafts": drafts, "most": most,
            "probabilities": guess if case["probabilities"] else None, "uniform": torch.rand(rows, device=DEVICE, generator=random),
            "noise": _exponential(random, requests, vocab), "temperature": torch.tensor(temperature, device=DEVICE),
            # for the plain form: each row's request, and each request's rows side by side
            "owner": torch.tensor(owner, device=DEVICE), "counts": torch.tensor(counts, device=DEVICE),
            "place": torch.tensor([[min(starts[i] + j, starts[i + 1] - 1) for j in range(most)] for i in range(requests)], device=DEVICE)}


def _exponential(random, *shape) -> torch.Tensor:
    return torch.empty(*shape, device=DEVICE).exponential_(generator=random).clamp_(min=1e-30)


# ------------------------------------------------------------------------------------------ one pass
def run(state: dict):
    return (_own if own else _plain)[state["op"]](state)


def _own_store(s):
    from hyperion_b200.ops.cache8 import Cache8, cache8_store

    cache8_store(s["source"], s["k"], s["v"], Cache8(*s["cache"]), s["table"], s["row"], s["position"])
    return s["cache"]


def _own_load(s):
    from hyperion_b200.ops.cache8 import Cache8, cache8_load

    return cache8_load(Cache8(*s["cache"]), s["table"], s["row"], s["position"], dtype=s["dtype"])


def _own_attention(s):
    from hyperion_b200.ops.cache8 import Cache8
    from hyperion_b200.ops.shared import attention_shared

    return attention_shared(s["q"], s["heads"], Cache8(*s["cache"]) if isinstance(s["cache"], tuple) else s["cache"], s["table"], s["plan"], s["scale"])


def _own_verify(s):
    from hyperion_b200.sampling.verify import verify_drafts

    return verify_drafts(s["logits"], s["start"], s["drafts"], s["uniform"], s["noise"], s["temperature"], most=s["most"], probabilities=s["probabilities"])


def _quantise(x):
    """Codes and exponents of records [..., dim] in 32 bits."""
    x = x.float()
    size = torch.where(torch.isnan(x), torch.zeros_like(x), x.abs()).amax(-1)
    fraction, exponent = torch.frexp(size)  # size = fraction * 2^exponent; 448 = 0.875 * 2^9
    e = exponent - 9 + (fraction > 0.875)
    e = torch.where(size == 0, EXPONENTS[0], torch.where(torch.isinf(size), EXPONENTS[1], e)).clamp(*EXPONENTS)
    return (x * _power(-e).unsqueeze(-1)).clamp(-LARGEST, LARGEST).to(torch.float8_e4m3fn), e.to(torch.int8)


def _power(e):
    """2^e of whole numbers as float32, from its bits."""
    return ((e.int() + 127) << 23).view(torch.float32)


def _values(codes, exponents):
    return codes.float() * _power(exponents).unsqueeze(-1)


def _plain_store(s):
    codes, exponents = s["cache"]
    kv, page, dim = codes.shape[2:]
    x = torch.stack([s["source"][:, s["k"]: s["k"] + kv * dim], s["source"][:, s["v"]: s["v"] + kv * dim]], 1).view(-1, 2, kv, dim)
    c, e = _quantise(x)
    position = s["position"].long()
    at = (s["table"][s["row"].long(), position // page].long()[:, None, None], torch.arange(2, device=DEVICE)[:, None], torch.arange(kv, device=DEVICE), (position % page)[:, None, None])
    codes.view(torch.uint8)[at] = c.view(torch.uint8)
    exponents[at] = e
    return s["cache"]


def _plain_load(s):
    codes, exponents = s["cache"]
    page, position = codes.shape[3], s["position"].long()
    of, slot = s["table"][s["row"].long(), position // page].long(), position % page
    return _values(codes.view(torch.uint8)[of, :, :, slot].view(torch.float8_e4m3fn), exponents[of, :, :, slot]).to(s["dtype"])


def _dense(s, blocks):
    """Keys and values [n, positions, kv, dim] of the pages ``blocks`` [n, b], in 32 bits."""
    blocks = blocks.long()
    if isinstance(s["cache"], tuple):
        x = _values(s["cache"][0].view(torch.uint8)[blocks].view(torch.float8_e4m3fn), s["cache"][1][blocks])
    else:
        x = s["cache"][blocks].float()
    n, b, _, kv, page, dim = x.shape
    x = x.permute(2, 0, 1, 4, 3, 5).reshape(2, n, b * page, kv, dim)
    return x[0], x[1]


def _plain_attention(s):
    shared, groups, page, kv, dim = s["shared"], s["groups"], s["page"], s["kv"], s["dim"]
    requests, most = s["place"].shape
    group = s["heads"] // kv
    q = s["q"].float().view(-1, kv, group, dim)[s["place"]]  # [requests, tokens, kv, group, dim]
    first = shared // page                                    # the page that holds the first position of a request's own
    k, v = _dense(s, s["table"][:, first:])
    at = torch.arange(first * page, first * page + k.shape[1], device=DEVICE) - shared
    visible = (at >= 0) & (at < s["seen"].unsqueeze(-1))      # [requests, tokens, positions]
    scores = torch.einsum("rnhgd,rlhd->rhgnl", q, k) * s["scale"]
    scores = torch.where(visible[:, None, None], scores, -math.inf)
    if groups:
        each = requests // groups
        pk, pv = _dense(s, s["table"][::each, : -(-shared // page)])
        pk, pv = pk[:, :shared], pv[:, :shared]
        before = torch.einsum("arnhgd,aphd->arhgnp", q.view(groups, each, most, kv, group, dim), pk).reshape(requests, kv, group, most, shared) * s["scale"]
        scores = torch.cat([before, scores], -1)
        del before
    top = scores.amax(-1, keepdim=True)
    weight = torch.exp(scores - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    del scores
    total = weight.sum(-1, keepdim=True)
    weight = weight / torch.where(total > 0, total, torch.ones_like(total))
    out = torch.einsum("rhgnl,rlhd->rnhgd", weight[..., shared:], torch.where(visible.any(1)[:, :, None, None], v, torch.zeros_like(v)))
    if groups:
        out = out + torch.einsum("arhgnp,aphd->arnhgd", weight[..., :shared].reshape(groups, each, kv, group, most, shared), pv).reshape(out.shape)
    return out.reshape(requests * most, kv * group * dim)[s["back"]].to(torch.bfloat16)


def _plain_verify(s):
    logits = s["logits"].float()
    logits = torch.where(torch.isnan(logits), -math.inf, logits).clamp(max=torch.finfo(torch.float32).max)
    temperature = s["temperature"][s["owner"]]
    greedy = temperature == 0
    scaled = logits / torch.where(greedy, torch.ones_like(temperature), temperature).unsqueeze(1)
    top = scaled.amax(1, keepdim=True)
    p = torch.exp(scaled - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = p.sum(1, keepdim=True)
    p = p / torch.where(total > 0, total, torch.ones_like(total))
    best = logits.argmax(1)
    drafts = s["drafts"].long().unsqueeze(1)
    chance = s["probabilities"].gather(1, drafts)[:, 0] if s["probabilities"] is not None else torch.ones_like(temperature)
    stands = torch.where(greedy, drafts[:, 0] == best, s["uniform"] * chance < p.gather(1, drafts)[:, 0])
    column = torch.arange(s["most"], device=DEVICE)
    accepted = (stands[s["place"]] & (column < s["counts"][:, None])).long().cumprod(1).sum(1)
    at = s["start"][:-1].long() + accepted
    more = accepted < s["counts"]  # a draft was refused: what is left of the target's probabilities beside the drafter's
    left = p[at]
    if s["probabilities"] is not None:
        rest = (left - s["probabilities"][at]).clamp(min=0)
    else:
        rest = left.scatter(1, drafts[at], 0.0)
    rest = torch.where((more & (rest.sum(1) > 0)).unsqueeze(1), rest, left)
    last = torch.where(greedy[at], best[at], (rest / s["noise"]).argmax(1))
    tokens = torch.where(column < accepted[:, None], s["drafts"].long()[s["place"]], torch.where(column == accepted[:, None], last[:, None], -1))
    return accepted.to(torch.int32), tokens.to(torch.int32)


_own = {"store": _own_store, "load": _own_load, "attention": _own_attention, "verify": _own_verify}
_plain = {"store": _plain_store, "load": _plain_load, "attention": _plain_attention, "verify": _plain_verify}


# ------------------------------------------------------------------------------------------ the definitions, in 64 bits
def _powers(low, high):
    return torch.tensor([2.0 ** i for i in range(low, high + 1)], dtype=torch.float64, device=DEVICE)


def exact(case, seed: int):
    if case["op"] == "verify":
        return None  # whole numbers
    s = prepare(case, seed)
    if case["op"] == "store":
        return _exact_store(s)
    if case["op"] == "load":
        codes, exponents = (t.double() for t in s["cache"])
        at, slot = s["position"].long() // case["page"], s["position"].long() % case["page"]
        page = s["table"].long()[s["row"].long(), at]
        return codes[page, :, :, slot] * _powers(*EXPONENTS)[exponents[page, :, :, slot].long() - EXPONENTS[0]][..., None]
    if isinstance(s["cache"], tuple):
        codes, exponents = s["cache"]
        records = lambda pages: codes.view(torch.uint8)[pages].view(torch.float8_e4m3fn).double() * _powers(*EXPONENTS)[exponents[pages].long() - EXPONENTS[0]][..., None]  # noqa: E731
    else:
        records = lambda pages: s["cache"][pages].double()  # noqa: E731
    heads, kv, dim, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    out, first = [], 0
    for count, length, pages in zip(s["counts"], s["lengths"], s["table"].long()):
        k, v = records(pages[: -(-length // page)]).permute(1, 2, 0, 3, 4).reshape(2, kv, -1, dim)[:, :, :length]
        q = s["q"][first: first + count].double().view(count, kv, heads // kv, dim).permute(1, 2, 0, 3)
        rows = max(1, (1 << 27) // (heads * length))  # queries at a time: a gigabyte of scores
        for i in range(0, count, rows):
            part = q[:, :, i: i + rows]
            last = torch.arange(length - count + i, length - count + i + part.shape[2], device=DEVICE)
            scores = (part @ k.unsqueeze(1).transpose(2, 3)) * dim ** -0.5
            scores.masked_fill_(torch.arange(length, device=DEVICE) > last[:, None], -math.inf)
            out.append((torch.softmax(scores, -1) @ v.unsqueeze(1)).permute(2, 0, 1, 3).reshape(-1, heads * dim))
        first += count
    return torch.cat(out)


def _exact_store(s):
    codes, exponents = (t.double() for t in s["cache"])
    kv, page, dim = codes.shape[2:]
    powers = _powers(*EXPONENTS)
    for which, column in enumerate((s["k"], s["v"])):
        x = s["source"][:, column: column + kv * dim].double().view(-1, kv, dim)
        e = torch.searchsorted(LARGEST * powers, x.abs().amax(-1).contiguous()).clamp(max=len(powers) - 1)  # counted from the smallest
        y = (x / powers[e].unsqueeze(-1)).clamp(-LARGEST, LARGEST)
        e = e + EXPONENTS[0]
        step = _powers(-9, 5)[torch.searchsorted(_powers(-6, 8), y.abs().clamp(min=2.0 ** -6), right=True) - 1]  # three bits behind the leading one, none below 2^-9
        position = s["position"].long()
        at = s["table"].long()[s["row"].long(), position // page]
        codes[at, which, :, position % page] = torch.round(y / step) * step
        exponents[at, which, :, position % page] = e.double()
    return codes, exponents
