"""Drafted tokens against the target's logits: the device's answer against the rule in 64 bits.

Answers are whole numbers and have to be equal.  A decision that is closer than float32's rounding may go either way; with the seeds below the expected number of such
decisions over the whole file is under 0.01 (some 400 decisions, each within some 2^-18 of a tie with a probability of about as much)."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from hyperion_b200 import ops
from hyperion_b200.sampling import reference_verify, verify_drafts

pytestmark = pytest.mark.gpu


def case(counts, vocab, seed, dtype=torch.float32, probabilities=True, temperatures=(1.0, 0.7, 0.0), spread=2.0):
    random = torch.Generator("cuda").manual_seed(seed)
    rows, requests = sum(counts) + len(counts), len(counts)
    logits = (spread * torch.randn(rows, vocab, device="cuda", generator=random)).to(dtype)
    guess = torch.softmax(logits.float() + 0.5 * torch.randn(rows, vocab, device="cuda", generator=random), 1)
    noise = torch.empty(requests, vocab, device="cuda").exponential_(generator=random).clamp_(min=1e-20)
    drafts = (guess / torch.empty_like(guess).exponential_(generator=random)).argmax(1).to(torch.int32)
    start = np.concatenate([[0], np.cumsum(np.array(counts) + 1)])
    temperature = [temperatures[i % len(temperatures)] for i in range(requests)]
    for i, t in enumerate(temperature):  # greedy requests whose first drafts are the largest
        if t == 0:
            for row in range(start[i], start[i] + 1 + i % 3):
                drafts[row] = logits[row].argmax()
    return dict(logits=logits, row_start=torch.tensor(start, dtype=torch.int32, device="cuda"), drafts=drafts, uniform=torch.rand(rows, device="cuda", generator=random),
                noise=noise, temperature=torch.tensor(temperature, dtype=torch.float32, device="cuda"), most=max(counts) + 1, probabilities=guess if probabilities else None)


def expected(c):
    start, answers = c["row_start"].tolist(), []
    for r in range(len(start) - 1):
        rows = slice(start[r], start[r + 1])
        n = start[r + 1] - start[r] - 1
        q = c["probabilities"][rows].cpu().numpy() if c["probabilities"] is not None else None
        answers.append(reference_verify(c["logits"][rows].float().cpu().numpy(), c["drafts"][rows].tolist()[:n], c["uniform"][rows].cpu().numpy().astype(np.float64),
                                        c["noise"][r].cpu().numpy().astype(np.float64), float(c["temperature"][r]), q))
    return answers


def compare(c):
    accepted, tokens = verify_drafts(**c)
    ops.raise_on_status(tokens.device)
    want = expected(c)
    assert accepted.tolist() == [a for a, _ in want]
    assert tokens.tolist() == [t + [-1] * (c["most"] - len(t)) for _, t in want]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("probabilities", [True, False])
@pytest.mark.parametrize("counts,vocab", [([0], 1), ([3], 2), ([4], 4096), ([2, 0, 5, 1, 3, 7], 4097), ([1, 2, 3], 31), ([5] * 9, 12289), ([4], 151936), ([11, 40], 1000)])
def test_against_the_rule(counts, vocab, probabilities, dtype):
    for seed in range(3):
        compare(case(counts, vocab, 100 * seed + vocab, dtype, probabilities))


def test_every_draft_stands_and_none_does():
    c = case([3, 3, 2], 5000, 1, temperatures=(1.0,))
    c["probabilities"] = torch.softmax(c["logits"], 1)
    c["uniform"].fill_(0.9999)
    compare(c)
    assert verify_drafts(**c)[0].tolist() == [3, 3, 2]
    c["uniform"].fill_(1.0)
    c["probabilities"][:, :] = 1.0  # more than any p: nothing stands and nothing is left beside it, so the target's own probabilities decide
    compare(c)
    assert verify_drafts(**c)[0].tolist() == [0, 0, 0]


def test_masked_logits():
    c = case([2, 2, 2, 2], 9000, 3, temperatures=(1.0, 0.0))
    c["logits"][:, 100:8950] = -float("inf")
    c["logits"][4, 5] = float("nan")
    c["logits"][7, :] = torch.finfo(torch.float32).min
    c["drafts"].clamp_(max=99)
    compare(c)


@pytest.mark.parametrize("value", [-float("inf"), float("nan")])
@pytest.mark.parametrize("temperature", [0.0, 1.0])
def test_a_row_without_any_logit(value, temperature):
    c = case([2], 5000, 4, temperatures=(temperature,))
    c["logits"][:] = value
    c["drafts"].fill_(7)
    accepted, tokens = verify_drafts(**c)
    assert accepted.tolist() == [0] and tokens.tolist() == [[0, -1, -1]]


def test_infinite_logits_share_the_row():
    c = case([0], 6000, 5, temperatures=(1.0,))
    c["logits"][0, 17] = c["logits"][0, 5000] = float("inf")
    c["noise"][0, 17], c["noise"][0, 5000] = 2.0, 1.0
    assert verify_drafts(**c)[1].tolist() == [[5000]]


def test_ties_go_to_the_lowest_index():
    c = case([1, 1], 9000, 6, temperatures=(0.0, 1.0))
    c["logits"][:] = 0.5
    c["noise"][:] = 1.0
    c["drafts"][0] = 0
    c["uniform"].fill_(1.0)
    accepted, tokens = verify_drafts(**{**c, "probabilities": None})
    assert accepted.tolist() == [1, 0]
    assert tokens.tolist() == [[0, 0], [0 if int(c["drafts"][2]) else 1, -1]]


def test_requests_without_rows_and_rows_beside_requests():
    c = case([2, 1, 3], 3000, 7, temperatures=(1.0,))
    whole = verify_drafts(**c)
    start = c["row_start"].tolist()
    start = [start[0], start[1], start[1], start[2], start[3]]  # the second of four has none
    noise = c["noise"][[0, 0, 1, 2]].contiguous()
    accepted, tokens = verify_drafts(**{**c, "row_start": torch.tensor(start, dtype=torch.int32, device="cuda"), "noise": noise, "temperature": torch.ones(4, device="cuda")})
    assert accepted.tolist() == [whole[0][0], 0, whole[0][1], whole[0][2]] and tokens[1].tolist() == [-1] * 4 and torch.equal(tokens[[0, 2, 3]], whole[1])


def test_rows_with_strides_and_off_boundaries():
    c = case([3, 2], 4099, 8)
    want = verify_drafts(**c)
    wide = {k: torch.zeros(c[k].shape[0], 4099 + 14, device="cuda") for k in ("logits", "noise", "probabilities")}
    for k, at in (("logits", 3), ("noise", 1), ("probabilities", 2)):
        wide[k] = wide[k][:, at: at + 4099]
        wide[k].copy_(c[k])
    got = verify_drafts(**{**c, **wide})
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_a_draft_outside_the_vocabulary_is_reported():
    c = case([2], 500, 9, temperatures=(1.0,))
    c["drafts"][0] = 500
    accepted, _ = verify_drafts(**c)
    assert accepted.tolist() == [0]
    with pytest.raises(ops.KernelError, match="token id"):
        ops.raise_on_status(c["logits"].device)


def test_tokens_are_distributed_as_the_target_s():
    """40,000 requests of one draft each over eight tokens: shares within five standard deviations of the target's probabilities."""
    n, vocab, random = 40000, 8, torch.Generator("cuda").manual_seed(10)
    target, guess = torch.tensor([2.0, 1.0, 0.5, 0.0, -1.0, 1.5, -3.0, 0.2], device="cuda"), torch.tensor([0.0, 2.0, 0.5, 1.0, -1.0, 0.0, -3.0, 1.2], device="cuda")
    q, p = torch.softmax(guess, 0), torch.softmax(target, 0)
    first = torch.zeros(vocab, dtype=torch.float64)
    for part in range(4):
        m = n // 4
        exponential = lambda *shape: torch.empty(*shape, device="cuda").exponential_(generator=random).clamp_(min=1e-20)  # noqa: E731
        drafts = torch.zeros(m, 2, dtype=torch.int32, device="cuda")
        drafts[:, 0] = (q / exponential(m, vocab)).argmax(1)
        _, tokens = verify_drafts(target.expand(2 * m, vocab).contiguous(), torch.arange(0, 2 * m + 1, 2, dtype=torch.int32, device="cuda"), drafts.view(-1),
                                  torch.rand(2 * m, device="cuda", generator=random), exponential(m, vocab), torch.ones(m, device="cuda"), most=2,
                                  probabilities=q.expand(2 * m, vocab).contiguous())
        first += torch.bincount(tokens[:, 0].long(), minlength=vocab).double().cpu()
    p = p.double().cpu()
    assert ((first / n - p).abs() <= 5 * (p * (1 - p) / n).sqrt()).all()


def test_refusals():
    c = case([1, 2], 100, 11)
    for bad in (dict(logits=c["logits"].half()), dict(logits=c["logits"][0]), dict(row_start=c["row_start"].long()), dict(drafts=c["drafts"][1:]), dict(uniform=c["uniform"].double()),
                dict(noise=c["noise"][:1]), dict(noise=c["noise"].double()), dict(temperature=c["temperature"][:1]), dict(most=0), dict(probabilities=c["probabilities"][:, 1:]),
                dict(logits=c["logits"].t().contiguous().t()), dict(logits=c["logits"].cpu())):
        with pytest.raises(ops.KernelError):
            verify_drafts(**{**c, **bad})
    none = verify_drafts(c["logits"][:0], c["row_start"][:1], c["drafts"][:0], c["uniform"][:0], c["noise"][:0], c["temperature"][:0], most=3)
    assert none[0].shape == (0,) and none[1].shape == (0, 3)
