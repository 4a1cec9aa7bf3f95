"""Beam search of several requests behind long prompts whose caches are cut back to a budget.

A small decoder with seeded random weights, built from the package's operators.  A prompt's keys and values go into pages (``kv_store``), its last tokens say what of it they look at (``tally_queries``), and what weighs
least is given up (``evict``) before the beams begin.  Then every beam of a request goes on from the same pages: a step attends and tallies (``attention_tallied``), the best continuations are chosen over beams and
vocabulary (``beam_select``), and beams take over what their parents hold (``beam_reorder``: tables, the page that is not full yet, tallies).  With one beam a request's pages are its own, and it is held to its budget
at every token.

    python examples/beams_on_a_budget.py --requests 3 --beams 4 --tokens 24 --prompt 700 --budget 256
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
from hyperion_b200.sampling import beam_select  # noqa: E402

PAGE = 16
FIRST, RECENT, LOOKING = 4, 32, 16  # positions that always stay, and how many of a prompt's last tokens say what stays


class Decoder:
    """``layers`` blocks of grouped-query attention and a gated feed-forward, bfloat16 weights, float32 residual stream."""

    def __init__(self, *, vocab=4096, hidden=512, heads=8, kv_heads=2, head_dim=64, inner=1024, layers=3, positions=4096, seed=0, device="cuda"):
        self.vocab, self.heads, self.kv_heads, self.head_dim, self.layers, self.device = vocab, heads, kv_heads, head_dim, layers, torch.device(device)
        random = torch.Generator().manual_seed(seed)

        def matrix(rows, columns, size=1.0):
            return (torch.randn(rows, columns, generator=random) * size * columns ** -0.5).to(torch.bfloat16).to(device)

        self.qkv = [matrix((heads + 2 * kv_heads) * head_dim, hidden) for _ in range(layers)]
        self.o = [matrix(hidden, heads * head_dim) for _ in range(layers)]
        self.gate_up = [matrix(2 * inner, hidden) for _ in range(layers)]
        self.down = [matrix(hidden, inner, 2.0) for _ in range(layers)]
        self.table = matrix(vocab, hidden, hidden ** 0.5)
        self.head = matrix(vocab, hidden, 3.0)
        self.norm = torch.ones(hidden, device=device)
        self.rotations = rotary_table(head_dim, 10000.0, positions).to(device)

    def new_cache(self, pages: int) -> torch.Tensor:
        return torch.zeros(self.layers, pages, 2, self.kv_heads, PAGE, self.head_dim, dtype=torch.bfloat16, device=self.device)

    def forward(self, ids, positions, slots, rows, cache, block_table, attend, *, last=None):
        """Logits of the step's tokens (of those at ``last`` only): each is at a position of its own, and its key and value go to a slot of row ``rows`` of the block table.  ``attend(layer, qkv)`` gives what the layer's
        queries see."""
        h, delta, turned = ops.embedding(self.table, ids), None, self.heads + self.kv_heads
        for i in range(self.layers):
            x = ops.add_rmsnorm(h, delta, self.norm, 1e-6, torch.bfloat16)
            qkv = ops.linear(x, self.qkv[i])
            ops.rope_(qkv, turned, self.head_dim, positions, self.rotations)
            ops.kv_store(qkv, self.heads * self.head_dim, turned * self.head_dim, cache[i], block_table, rows, slots)
            x = ops.add_rmsnorm(h, ops.linear(attend(i, qkv), self.o[i]), self.norm, 1e-6, torch.bfloat16)
            delta = ops.linear(ops.gated_linear(x, self.gate_up[i], None), self.down[i])
        x = ops.add_rmsnorm(h, delta, self.norm, 1e-6, torch.bfloat16, rows=last)
        return ops.linear(x, self.head, out_dtype=torch.float32)


class Search:
    """``beams`` beams of each prompt, group by group; row g * beams + j of the block table is beam j of request g."""

    def __init__(self, model: Decoder, prompts: list[list[int]], *, beams: int, tokens: int, budget: int):
        self.model, self.beams, self.tokens, self.budget, self.groups = model, beams, tokens, budget, len(prompts)
        device, lengths = model.device, [len(prompt) for prompt in prompts]
        rows = self.groups * beams
        # every beam has pages of its own for all that may come; a beam that takes over a parent's full pages points to them instead
        most = max(lengths) + tokens
        self.blocks = -(-most // PAGE)
        self.own = torch.arange(rows * self.blocks, dtype=torch.int32, device=device).view(rows, self.blocks)
        self.block_table = self.own.clone()
        self.cache = model.new_cache(rows * self.blocks)
        self.tally = ops.new_tally(rows, model.kv_heads, self.blocks * PAGE, layers=model.layers, device=device)
        self.held = torch.tensor(lengths, dtype=torch.int32, device=device)       # slots of each request's beams
        self.came = self.held.clone()                                             # tokens, those whose slots were given up among them
        self.scores = torch.full((self.groups, beams), float("-inf"), device=device)
        self.scores[:, 0] = 0
        self.said = torch.zeros(rows, 0, dtype=torch.int32, device=device)
        self.step(self._prompts(prompts, lengths))

    def _ints(self, values) -> torch.Tensor:
        return torch.tensor(values, dtype=torch.int32, device=self.model.device)

    def _prompts(self, prompts, lengths) -> torch.Tensor:
        """The prompts, read into the pages of each request's first beam and cut back to the budget; logits [rows, vocab] of what may follow, in the rows of the first beams."""
        model, first = self.model, torch.arange(0, self.groups * self.beams, self.beams, device=self.model.device)
        table, counts = self.block_table[first].contiguous(), torch.tensor(lengths)
        positions = self._ints([p for n in lengths for p in range(n)])
        rows = torch.repeat_interleave(torch.arange(self.groups), counts).to(torch.int32).to(model.device)
        ends = counts.cumsum(0)
        looking = [min(n, LOOKING) for n in lengths]
        picked = torch.cat([torch.arange(end - n, end) for end, n in zip(ends.tolist(), looking)]).to(model.device)
        starts = self._ints([0, *torch.tensor(looking).cumsum(0).tolist()])
        plan = ops.plan_shared(lengths, lengths, model.heads, model.kv_heads, model.head_dim, device=model.device)
        tally = ops.Tally(self.tally.weights[:, first].contiguous(), self.tally.positions[:, first].contiguous())
        scale = model.head_dim ** -0.5

        def attend(layer, qkv):
            ops.tally_queries(qkv[picked], model.heads, self.cache[layer], table, starts, self.held, ops.Tally(tally.weights[layer], tally.positions[layer]), scale, most=max(looking))
            return ops.attention_shared(qkv, model.heads, self.cache[layer], table, plan, scale)

        logits = model.forward(self._ints([t for prompt in prompts for t in prompt]), positions, positions, rows, self.cache, table, attend, last=(ends - 1).to(torch.int32).to(model.device))
        self.held = ops.evict(self.cache, table, self.held, self.came - 1, tally, self.budget, first=FIRST, recent=RECENT)
        self.tally.weights[:, first], self.tally.positions[:, first] = tally
        spread = torch.zeros(self.groups * self.beams, model.vocab, device=model.device)
        spread[first] = logits
        return spread

    def step(self, logits: torch.Tensor) -> None:
        """The best continuations of every request's beams, which take over what their parents hold."""
        choice = beam_select(logits, self.scores, self.beams)
        self.scores = choice.scores
        model, pages = self.model, self.cache.shape[1]
        states = [self.tally.weights, self.tally.positions, self.said[None]] if self.said.shape[1] else list(self.tally)
        ops.beam_reorder(choice.parents, self.held, self.block_table, [self.cache.view(model.layers, pages, 2 * model.kv_heads, PAGE, model.head_dim)], states)
        self.said = torch.cat([self.said, choice.tokens.view(-1, 1)], 1)

    def more(self) -> None:
        """One more token of every beam."""
        model, beams = self.model, self.beams
        slots, came = self.held.repeat_interleave(beams), self.came.repeat_interleave(beams)
        rows = torch.arange(self.groups * beams, dtype=torch.int32, device=model.device)
        lengths, scale = slots + 1, model.head_dim ** -0.5

        def attend(layer, qkv):
            return ops.attention_tallied(qkv, model.heads, self.cache[layer], self.block_table, lengths, came, ops.Tally(self.tally.weights[layer], self.tally.positions[layer]), scale)

        logits = model.forward(self.said[:, -1].contiguous().clamp(min=0), came, slots, rows, self.cache, self.block_table, attend)
        self.held, self.came = self.held + 1, self.came + 1
        if beams == 1:
            self.held = ops.evict(self.cache, self.block_table, self.held, self.came - 1, self.tally, self.budget, first=FIRST, recent=RECENT)
        self.step(logits)

    def run(self) -> list[list[list[int]]]:
        """Every beam's tokens, the best beam of a request first."""
        while self.said.shape[1] < self.tokens:
            self.more()
        ops.raise_on_status(self.model.device)
        return self.said.view(self.groups, self.beams, -1).tolist()


def main(argv=None) -> Search:
    options = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    options.add_argument("--requests", type=int, default=3)
    options.add_argument("--beams", type=int, default=4)
    options.add_argument("--tokens", type=int, default=24, help="to be generated by each beam")
    options.add_argument("--prompt", type=int, default=700, help="tokens of the longest prompt")
    options.add_argument("--budget", type=int, default=256, help="slots that stay of a prompt")
    options.add_argument("--seed", type=int, default=0)
    a = options.parse_args(argv)
    model, random = Decoder(seed=a.seed), torch.Generator().manual_seed(a.seed + 1)
    prompts = [torch.randint(model.vocab, (max(1, a.prompt - 57 * r),), generator=random).tolist() for r in range(a.requests)]
    start = time.perf_counter()
    search = Search(model, prompts, beams=a.beams, tokens=a.tokens, budget=a.budget)
    said = search.run()
    took = time.perf_counter() - start
    for r, beams in enumerate(said):
        print(f"request {r}: {search.scores[r, 0].item():.2f}  {' '.join(map(str, beams[0]))}")
    held, came = search.held.tolist(), search.came.tolist()
    print(f"{a.requests} requests of {a.beams} beams, {a.tokens} tokens each, {took * 1e3:.0f} ms; slots held of tokens that came: " + ", ".join(f"{h} of {c}" for h, c in zip(held, came)))
    return search


if __name__ == "__main__":
    main()
