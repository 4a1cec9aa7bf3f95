"""Drafts verified at low temperatures, and over logits far from zero: the weights of a row are powers of the difference to its largest logit, however large that is beside the
temperature.

Answers are whole numbers and have to be equal.  An entry's probability is off by some 2^-18 of itself where it counts at all (its exponent, up to 30, is rounded to 2^-23 of itself
three times), so the 1,300 decisions of this file fall the other way with a probability of some 0.01 in all."""
from __future__ import annotations

import pytest
import torch
from test_verify_drafts_gpu import case, compare, expected

from hyperion_b200.sampling import verify_drafts

pytestmark = pytest.mark.gpu
LARGEST = torch.finfo(torch.float32).max


def peaked(temperature, dtype, vocab, offset=0.0, seed=0, probabilities=True):
    """Requests whose rows have a largest logit of 16 to 18 (before ``offset``), which is the draft of all rows but every fifth one, and a second one close to it."""
    c = case([4] * 6, vocab, seed, dtype, probabilities, temperatures=(temperature,))
    random = torch.Generator("cuda").manual_seed(seed + 1)
    logits = 3.0 * torch.randn(c["logits"].shape, device="cuda", generator=random).clamp(-4, 4)
    top = 16.0 + 2.0 * torch.rand(len(logits), 1, device="cuda", generator=random)
    where = torch.stack([torch.randperm(vocab, device="cuda", generator=random)[:2] for _ in range(len(logits))])
    logits.scatter_(1, where, torch.cat([top, top - 3.0 * temperature], 1))
    c["logits"] = (logits + offset).to(dtype)
    c["drafts"] = c["logits"].float().argmax(1).to(torch.int32)
    c["drafts"][::5] = where[::5, 1].to(torch.int32)
    if probabilities:
        c["probabilities"] = torch.softmax((c["logits"].double() - c["logits"].double().amax(1, keepdim=True)) / (1.5 * temperature), 1).float()
    return c


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("temperature", [0.3, 1e-1, 1e-2, 1e-3, 1e-4, 1e-5, 1e-6, 1e-7, 1e-8, 1e-20, 1e-37])
def test_low_temperatures(temperature, dtype):
    for seed, (vocab, probabilities) in enumerate([(4096, True), (4097, False), (40001, True)]):
        compare(peaked(temperature, dtype, vocab, seed=seed, probabilities=probabilities))


@pytest.mark.parametrize("temperature", [1.0, 0.6, 1e-2])
@pytest.mark.parametrize("offset", [1e4, -1e4, 1e6, -1e9])
def test_logits_with_a_common_offset(offset, temperature):
    for seed, (vocab, probabilities) in enumerate([(4096, True), (40001, False)]):
        compare(peaked(temperature, torch.float32, vocab, offset, seed, probabilities))


@pytest.mark.parametrize("temperature", [1.0, 0.7, 1e-3])
@pytest.mark.parametrize("value", [LARGEST, 1e38, 3e37])
def test_a_forced_token(value, temperature):
    """One finite logit that leaves nothing to the others."""
    c = case([2, 0], 9000, 3, temperatures=(temperature,), probabilities=False)
    c["logits"][:, 4321] = value
    c["drafts"].fill_(4321)
    compare(c)
    accepted, tokens = verify_drafts(**c)
    assert accepted.tolist() == [2, 0] and tokens.tolist() == [[4321] * 3, [4321, -1, -1]]


@pytest.mark.parametrize("temperature", [1.0, 0.7, 1e-3])
@pytest.mark.parametrize("value", [-LARGEST, -1e38])
def test_rows_of_the_lowest_number(value, temperature):
    """Rows in which everything has the type's lowest value have equal probabilities: the noise decides."""
    c = case([1, 0], 5000, 4, temperatures=(temperature,))
    c["logits"][:] = value
    compare(c)
    c["probabilities"].fill_(0.0)  # the draft stands, and one is drawn from the row behind it
    compare(c)
    assert [a for a, _ in expected(c)] == [1, 0]
