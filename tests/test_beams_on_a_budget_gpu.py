"""The example of beams on a budget: all operators of the set together, against one pass of the same decoder over the whole sequences."""
from __future__ import annotations

import importlib.util
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu


def example():
    spec = importlib.util.spec_from_file_location("beams_on_a_budget", Path(__file__).resolve().parents[1] / "examples" / "beams_on_a_budget.py")
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def search(beams, tokens=14, budget=10_000, prompts=(61, 40, 7), seed=0):
    e = example()
    random = torch.Generator().manual_seed(seed + 5)
    said = [torch.randint(4096, (n,), generator=random).tolist() for n in prompts]
    return e, e.Search(e.Decoder(seed=3), said, beams=beams, tokens=tokens, budget=budget), said


def whole(e, model, ids):
    """Logits of every token of ``ids`` by one pass."""
    ops, n = e.ops, len(ids)
    ints = lambda values: torch.tensor(values, dtype=torch.int32, device="cuda")  # noqa: E731
    table = torch.arange(-(-n // e.PAGE), dtype=torch.int32, device="cuda")[None].contiguous()
    cache, plan = model.new_cache(table.shape[1]), ops.plan_shared([n], [n], model.heads, model.kv_heads, model.head_dim)
    positions = ints(list(range(n)))
    return model.forward(ints(ids), positions, positions, torch.zeros_like(positions), cache, table,
                         lambda layer, qkv: ops.attention_shared(qkv, model.heads, cache[layer], table, plan, model.head_dim ** -0.5)).double()


@pytest.mark.parametrize("beams", [1, 2, 5, 8])
def test_scores_are_those_of_the_whole_sequences(beams):
    """While nothing has to be given up, a beam's score is the sum of the log probabilities of its tokens.  Both ways round activations to bfloat16 (2^-8 of a value) at other places of the arithmetic, so a logit (standard
    deviation 3) may differ by some hundredths and a log probability by twice that: a tenth is allowed a token.  A token of another beam's history would be off by several."""
    e, found, prompts = search(beams)
    said = found.run()
    for g, prompt in enumerate(prompts):
        scores = found.scores[g].tolist()
        assert scores == sorted(scores, reverse=True) and len({tuple(beam) for beam in said[g]}) == beams
        for beam, score in zip(said[g], scores):
            logits = torch.log_softmax(whole(e, found.model, prompt + beam)[len(prompt) - 1: -1], 1)
            want = logits.gather(1, torch.tensor(beam, device="cuda")[:, None]).sum().item()
            assert abs(score - want) <= 0.1 * len(beam), (g, score, want)


def test_one_beam_is_the_greedy_search():
    e, found, prompts = search(1)
    for prompt, (beam,) in zip(prompts, found.run()):
        rows = whole(e, found.model, prompt + beam)[len(prompt) - 1: -1]
        behind = rows.max(1).values - rows.gather(1, torch.tensor(beam, device="cuda")[:, None])[:, 0]
        assert bool((behind <= 0.25).all())  # as above: two logits, a tenth each, and the one that may have been on the other side


@pytest.mark.parametrize("beams", [1, 4])
def test_on_a_budget(beams):
    """Requests are held to their budget, keep what always stays, and say the same again."""
    e, found, _ = search(beams, tokens=40, budget=64, prompts=(300, 64, 20, 129))
    said = found.run()
    held, came = found.held.tolist(), found.came.tolist()
    assert came == [339, 103, 59, 168]
    assert held == ([64, 64, 59, 64] if beams == 1 else [64 + 39, 64 + 39, 59, 64 + 39])
    weights, positions = found.tally
    for g in range(4):
        for row in range(g * beams, (g + 1) * beams):
            for layer in range(found.model.layers):
                for head in range(found.model.kv_heads):
                    here = positions[layer, row, head, : held[g]].tolist()
                    assert len(set(here)) == held[g] and max(here) == came[g] - 1 and set(range(e.FIRST)) <= set(here)
                    assert beams > 1 or set(range(came[g] - e.RECENT, came[g])) <= set(here)
    assert bool(torch.isfinite(weights).all()) and bool((weights >= 0).all())
    _, again, _ = search(beams, tokens=40, budget=64, prompts=(300, 64, 20, 129))
    assert again.run() == said


def test_a_beams_pages_hold_its_own_history():
    """Every beam's keys, read through its table, are those of one pass over its prompt and tokens, up to the rounding of activations."""
    e, found, prompts = search(4, tokens=30)
    said = found.run()
    model = found.model
    for g, prompt in enumerate(prompts):
        for j in (0, 3):
            row, n = g * 4 + j, int(found.held[g])
            ids = prompt + said[g][j][:-1]
            assert len(ids) == n
            keys = found.cache[0][found.block_table[row].long(), 0].transpose(1, 2).reshape(-1, model.kv_heads, model.head_dim)[:n].float()
            table = torch.arange(-(-n // e.PAGE), dtype=torch.int32, device="cuda")[None].contiguous()
            cache = model.new_cache(table.shape[1])
            positions = torch.arange(n, dtype=torch.int32, device="cuda")
            plan = e.ops.plan_shared([n], [n], model.heads, model.kv_heads, model.head_dim)
            model.forward(torch.tensor(ids, dtype=torch.int32, device="cuda"), positions, positions, torch.zeros_like(positions), cache, table,
                          lambda layer, qkv: e.ops.attention_shared(qkv, model.heads, cache[layer], table, plan, model.head_dim ** -0.5))
            want = cache[0][:, 0].transpose(1, 2).reshape(-1, model.kv_heads, model.head_dim)[:n].float()
            # the first layer's keys hang on the token and its position alone: products of other row counts may add up in another order and round to the neighbouring bfloat16, 2^-7 of the value, before and behind the rotation
            assert bool(((keys - want).abs() <= 2.0 ** -5 * want.abs().amax(-1, keepdim=True)).all())


def test_the_command():
    assert example().main(["--requests", "2", "--beams", "3", "--tokens", "5", "--prompt", "100", "--budget", "48"]).said.shape == (6, 5)
