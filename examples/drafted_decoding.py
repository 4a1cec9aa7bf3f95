"""Drafted decoding of several requests behind one system prompt, over an 8-bit cache.

A small decoder with seeded random weights, built from the package's operators: keys and values go into paged 8-bit records (``cache8_store``),
all requests read the system prompt's pages together (``plan_shared``, ``attention_shared``), the decoder's first layers draft a few tokens per
request, one pass of the whole decoder sees them all, and ``verify_drafts`` keeps those that stand.  A finished request's records are read back as
bfloat16 (``cache8_load``), as one would move them to another cache.

    python examples/drafted_decoding.py --requests 6 --tokens 32 --drafts 4 --temperature 0.8
"""
from __future__ import annotations

import argparse
import sys
import time
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

from hyperion_b200 import ops  # noqa: E402
from hyperion_b200.parts.rope import rotary_table  # noqa: E402
from hyperion_b200.sampling import verify_drafts  # noqa: E402

PAGE = 16


class Decoder:
    """``layers`` blocks of grouped-query attention and a gated feed-forward, bfloat16 weights, float32 residual stream.  The later layers add less
    than the first ``drafting`` ones, so that what those would answer is often what all of them answer."""

    def __init__(self, *, vocab=4096, hidden=512, heads=8, kv_heads=2, head_dim=64, inner=1024, layers=4, drafting=2, positions=4096, seed=0, device="cuda"):
        self.vocab, self.heads, self.kv_heads, self.head_dim, self.layers, self.drafting, self.device = vocab, heads, kv_heads, head_dim, layers, drafting, torch.device(device)
        random = torch.Generator().manual_seed(seed)

        def matrix(rows, columns, size=1.0):
            return (torch.randn(rows, columns, generator=random) * size * columns ** -0.5).to(torch.bfloat16).to(device)

        self.width = (heads + 2 * kv_heads) * head_dim
        later = [1.0 if i < drafting else 0.25 for i in range(layers)]
        self.qkv = [matrix(self.width, hidden) for _ in range(layers)]
        self.o = [matrix(hidden, heads * head_dim, later[i]) for i in range(layers)]
        self.gate_up = [matrix(2 * inner, hidden) for _ in range(layers)]
        self.down = [matrix(hidden, inner, 2 * later[i]) for i in range(layers)]
        self.table = matrix(vocab, hidden, hidden ** 0.5)
        self.head = matrix(vocab, hidden, 3.0)
        self.norm = torch.ones(hidden, device=device)
        self.rotations = rotary_table(head_dim, 10000.0, positions).to(device)

    def new_cache(self, pages: int) -> list[ops.Cache8]:
        return [ops.new_cache8(pages, self.kv_heads, PAGE, self.head_dim, self.device) for _ in range(self.layers)]

    def forward(self, ids, positions, rows, cache, block_table, plan, *, layers=None, last=None):
        """Logits of the step's tokens (of those at ``last`` only), whose keys and values go to row ``rows`` of the block table at ``positions``."""
        h, delta, turned = ops.embedding(self.table, ids), None, self.heads + self.kv_heads
        for i in range(layers or self.layers):
            x = ops.add_rmsnorm(h, delta, self.norm, 1e-6, torch.bfloat16)
            qkv = ops.linear(x, self.qkv[i])
            ops.rope_(qkv, turned, self.head_dim, positions, self.rotations)
            ops.cache8_store(qkv, self.heads * self.head_dim, turned * self.head_dim, cache[i], block_table, rows, positions)
            attended = ops.attention_shared(qkv, self.heads, cache[i], block_table, plan, self.head_dim ** -0.5)
            x = ops.add_rmsnorm(h, ops.linear(attended, self.o[i]), self.norm, 1e-6, torch.bfloat16)
            delta = ops.linear(ops.gated_linear(x, self.gate_up[i], None), self.down[i])
        x = ops.add_rmsnorm(h, delta, self.norm, 1e-6, torch.bfloat16, rows=last)
        return ops.linear(x, self.head, out_dtype=torch.float32)


class Conversations:
    """Requests behind one system prompt: whole pages of it are held once, every request's block table begins with them."""

    def __init__(self, model: Decoder, system: list[int], prompts: list[list[int]], *, tokens: int, drafts: int, temperature: float, seed: int = 0):
        self.model, self.drafts, self.tokens, self.requests, device = model, drafts, tokens, len(prompts), model.device
        self.shared = len(system) // PAGE * PAGE  # what is left of the system prompt belongs to each request
        prompts = [system[self.shared:] + prompt for prompt in prompts]
        common, own = self.shared // PAGE, -(-(max(map(len, prompts)) + tokens + drafts) // PAGE)
        table = torch.arange(self.requests * own).view(self.requests, own) + common
        self.block_table = torch.cat([torch.arange(common).expand(self.requests, common), table], 1).to(torch.int32).to(device)
        self.cache = model.new_cache(common + self.requests * own)
        self.random = torch.Generator(device=device).manual_seed(seed)
        self.temperature = torch.full((self.requests,), temperature, device=device)
        self.lengths = [self.shared + len(prompt) for prompt in prompts]
        self.said: list[list[int]] = [[] for _ in prompts]
        self.passes = 0
        if self.shared:  # the pages of all, filled once
            self._pass([0], [system[: self.shared]], [self.shared], shared=False)
        logits = self._pass(range(self.requests), prompts, self.lengths, last=True)
        _, first = self._choose(logits, torch.arange(self.requests + 1, dtype=torch.int32, device=device), torch.zeros(self.requests, dtype=torch.int32, device=device), None, self.temperature, 1)
        for said, token in zip(self.said, first.flatten().tolist()):
            said.append(token)

    def _pass(self, who, ids, lengths, *, shared=True, layers=None, last=False):
        """The model over ``ids`` (a list per request, or a tensor [requests, tokens]), the last of which is position ``lengths[i] - 1`` of its request."""
        device, counts = self.model.device, [len(row) for row in ids]
        flat = ids.flatten() if isinstance(ids, torch.Tensor) else torch.tensor([t for row in ids for t in row], dtype=torch.int32).to(device)
        positions = torch.cat([torch.arange(length - n, length) for n, length in zip(counts, lengths)]).to(torch.int32).to(device)
        rows = torch.repeat_interleave(torch.arange(len(counts)), torch.tensor(counts)).to(torch.int32).to(device)
        ends = (torch.tensor(counts).cumsum(0) - 1).to(torch.int32).to(device) if last else None
        plan = ops.plan_shared(counts, lengths, self.model.heads, self.model.kv_heads, self.model.head_dim,
                               shared=[(0, len(counts), self.shared)] if shared and self.shared else (), device=device)
        return self.model.forward(flat, positions, rows, self.cache, self.block_table[list(who)], plan, layers=layers, last=ends)

    def _choose(self, logits, row_start, drafted, probabilities, temperature, most):
        requests, (rows, vocab) = len(temperature), logits.shape
        uniform = torch.rand(rows, device=logits.device, generator=self.random)
        noise = torch.empty(requests, vocab, device=logits.device).exponential_(generator=self.random)
        return verify_drafts(logits, row_start, drafted, uniform, noise, temperature, most=most, probabilities=probabilities)

    def round(self, who: list[int]) -> list[int]:
        """Drafts and one pass of the whole model for the requests ``who``; how many drafts of each stood."""
        model, n, device = self.model, self.drafts, self.model.device
        lengths, temperature = [self.lengths[r] for r in who], self.temperature[who]
        ids = torch.tensor([[self.said[r][-1]] for r in who], dtype=torch.int32, device=device)
        greedy = float(temperature[0]) == 0
        probabilities = None if greedy else torch.zeros(len(who), n + 1, model.vocab, device=device)
        ones = torch.arange(len(who) + 1, dtype=torch.int32, device=device)
        for i in range(n):  # the first layers draft; what they store there is what the whole model stores again
            logits = self._pass(who, ids[:, -1:], [length + i + 1 for length in lengths], layers=model.drafting)
            if not greedy:
                probabilities[:, i] = torch.softmax(logits / temperature[:, None], 1)
            _, token = self._choose(logits, ones, torch.zeros(len(who), dtype=torch.int32, device=device), None, temperature, 1)
            ids = torch.cat([ids, token], 1)
        logits = self._pass(who, ids, [length + n + 1 for length in lengths])
        drafted = torch.cat([ids[:, 1:], torch.zeros_like(ids[:, :1])], 1).flatten().contiguous()
        row_start = ones * (n + 1)
        accepted, tokens = self._choose(logits, row_start, drafted, None if greedy else probabilities.view(-1, model.vocab), temperature, n + 1)
        self.passes += 1
        stood = accepted.tolist()
        for r, count, row in zip(who, stood, tokens.tolist()):
            self.said[r] += row[: count + 1]
            self.lengths[r] += count + 1
        ops.raise_on_status(device)
        return stood

    def run(self) -> list[int]:
        """Rounds until every request has said its tokens; how many drafts stood, by round and request."""
        stood = []
        while waiting := [r for r in range(self.requests) if len(self.said[r]) < self.tokens]:
            stood += self.round(waiting)
        self.said = [said[: self.tokens] for said in self.said]
        return stood

    def records(self, r: int) -> list[torch.Tensor]:
        """A request's keys and values, layer by layer, as bfloat16 [positions, 2, kv_heads, d]."""
        positions = torch.arange(self.lengths[r], dtype=torch.int32, device=self.model.device)
        return [ops.cache8_load(cache, self.block_table, torch.full_like(positions, r), positions) for cache in self.cache]


def main(argv=None) -> Conversations:
    options = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    options.add_argument("--requests", type=int, default=6)
    options.add_argument("--system", type=int, default=500, help="tokens of the system prompt")
    options.add_argument("--tokens", type=int, default=32, help="to be generated by each request")
    options.add_argument("--drafts", type=int, default=4)
    options.add_argument("--temperature", type=float, default=0.0)
    options.add_argument("--seed", type=int, default=0)
    a = options.parse_args(argv)
    model = Decoder(seed=a.seed)
    random = torch.Generator().manual_seed(a.seed + 1)
    draw = lambda n: torch.randint(model.vocab, (n,), generator=random).tolist()  # noqa: E731
    talk = Conversations(model, draw(a.system), [draw(5 + 3 * r) for r in range(a.requests)], tokens=a.tokens, drafts=a.drafts, temperature=a.temperature, seed=a.seed)
    start = time.perf_counter()
    stood = talk.run()
    took = time.perf_counter() - start
    for r, said in enumerate(talk.said):
        print(f"request {r}: {' '.join(map(str, said))}")
    record = sum(t.nbytes for t in talk.records(0))
    print(f"{talk.passes} passes of the whole model for {a.tokens - 1} tokens a request, {sum(stood) / max(1, len(stood)):.2f} of {a.drafts} drafts stood, "
          f"{took * 1e3:.0f} ms; request 0's records are {record // 1024} KB as bfloat16, a little over half of that in their pages")
    return talk


if __name__ == "__main__":
    main()
