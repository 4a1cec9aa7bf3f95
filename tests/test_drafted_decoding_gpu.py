"""The example of drafted decoding: all operators of a drafted step over an 8-bit cache together."""
import importlib.util
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu


def example():
    spec = importlib.util.spec_from_file_location("drafted_decoding", Path(__file__).resolve().parents[1] / "examples" / "drafted_decoding.py")
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def conversations(drafts, temperature, tokens=20, seed=0, requests=4):
    e = example()
    random = torch.Generator().manual_seed(7)
    draw = lambda n: torch.randint(4096, (n,), generator=random).tolist()  # noqa: E731
    system, prompts = draw(123), [draw(3 + 5 * r) for r in range(requests)]
    return e, e.Conversations(e.Decoder(seed=3), system, prompts, tokens=tokens, drafts=drafts, temperature=temperature, seed=seed), system, prompts


@pytest.mark.parametrize("drafts", [0, 1, 4])
def test_greedy_tokens_are_the_whole_models(drafts):
    """Every token said is, up to rounding, the largest logit of one pass over all that was said.  The keys and values of both are rounded to 8 bits (2^-4 of an entry) from
    bfloat16 entries that may differ in their last bit, so logits may differ a little; a token that does not belong there would be some three standard deviations of a
    row's logits behind, a quarter of one is allowed."""
    e, talk, system, prompts = conversations(drafts, 0.0)
    stood = talk.run()
    assert all(len(said) == 20 for said in talk.said) and all(0 <= s <= drafts for s in stood)
    if drafts:
        assert sum(stood) > 0 and talk.passes < 19  # the first layers often answer as all of them do
    for prompt, said in zip(prompts, talk.said):
        again = e.Conversations(talk.model, [], [system + prompt + said], tokens=1, drafts=0, temperature=0.0)
        logits = again._pass([0], [system + prompt + said], [len(system + prompt + said)]).double()
        rows = logits[len(system + prompt) - 1 : -1]
        behind = rows.max(1).values - rows.gather(1, torch.tensor(said, device=rows.device)[:, None])[:, 0]
        assert (behind <= 0.25 * rows.std(1)).all(), behind.max()


def test_drawn_tokens():
    _, talk, _, _ = conversations(3, 0.8, seed=5)
    stood = talk.run()
    _, same, _, _ = conversations(3, 0.8, seed=5)
    same.run()
    assert talk.said == same.said and sum(stood) > 0 and all(0 <= t < 4096 for said in talk.said for t in said)


def test_records_go_back_unchanged():
    """Records read as bfloat16 and stored in another request's pages are read there as they were."""
    e, talk, _, _ = conversations(2, 0.0, tokens=6, requests=2)
    talk.run()
    before = talk.records(0)
    cache = talk.model.new_cache(talk.cache[0].codes.shape[0])
    table = talk.block_table.flip(1).contiguous()
    positions = torch.arange(talk.lengths[0], dtype=torch.int32, device=talk.model.device)
    row = torch.zeros_like(positions)
    width = talk.model.kv_heads * talk.model.head_dim
    for old, new in zip(before, cache):
        e.ops.cache8_store(old.view(len(positions), 2 * width), 0, width, new, table, row, positions)
        assert torch.equal(e.ops.cache8_load(new, table, row, positions), old)
    e.ops.raise_on_status(talk.model.device)
