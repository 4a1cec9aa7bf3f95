"""A beam search's selection against the rule in float64, and the reordering of what beams hold, to the bit."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from hyperion_b200 import ops
from hyperion_b200.ops.beams import beam_reorder
from hyperion_b200.sampling import beam_select, reference_beam_select

pytestmark = pytest.mark.gpu


UNDECIDED = 2.0 ** -20


def check_selection(logits, scores, take):
    """Every place holds the continuation that the rule puts there.  A row's sum is made of terms that are off by 2^-22 each at most (the exponential of the hardware) and float sums of 16 of them (2^-22 on top, at the
    very most), so its logarithm is off by less than 2^-21, and scores of two rows that lie closer than 2^-20 come in either order; within a row the order is that of the logits, to the bit."""
    choice = beam_select(logits, scores, take)
    groups, beams = scores.shape
    z = logits.float().cpu().numpy().reshape(groups, beams, -1)
    for g in range(groups):
        more = reference_beam_select(z[g], scores[g].cpu().numpy(), take + 64)
        want, score_of = more[:take], {(b, v): score for b, v, score in more}
        got = list(zip(choice.parents[g].tolist(), choice.tokens[g].tolist()))
        assert got[len(want):] == [(-1, -1)] * (take - len(want)) and len(set(got[: len(want)])) == len(want)
        for (b, v), (wanted_b, wanted_v, score) in zip(got, want):
            assert (b, v) == (wanted_b, wanted_v) or (b != wanted_b and abs(score_of[b, v] - score) < UNDECIDED) or abs(score_of[b, v] - score) < UNDECIDED and any(
                x != b and abs(s - score) < UNDECIDED for (x, _), s in score_of.items()), (got, want)
        for beam in range(beams):  # within a beam: the best of its own, in their order
            mine = [v for b, v in got if b == beam]
            assert mine == [v for b, v, _ in more if b == beam][: len(mine)]
        for place, (b, v) in enumerate(got[: len(want)]):
            # the score is rounded once to float32
            score = score_of[b, v]
            assert abs(choice.scores[g, place].item() - score) <= abs(score) * 2.0 ** -24 + 2.0 ** -21
        assert all(s == float("-inf") for s in choice.scores[g, len(want):].tolist())
    return choice


def some_logits(groups, beams, vocab, dtype=torch.float32, seed=0, more=0):
    random = torch.Generator("cuda").manual_seed(seed)
    x = torch.randn(groups * beams, vocab + more, device="cuda", generator=random) * 2
    x[:, : vocab // 50 + 1] *= 3
    scores = -10 - 3 * torch.rand(groups, beams, device="cuda", generator=random)
    return x.to(dtype)[:, :vocab], scores


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("groups,beams,vocab,take", [(1, 1, 1, 1), (1, 4, 1000, 8), (3, 5, 4097, 10), (2, 32, 5000, 64), (1, 8, 151936, 16), (40, 4, 12289, 4), (1, 3, 7, 21), (1, 2, 20, 64), (7, 1, 32000, 2)])
def test_selection(groups, beams, vocab, take, dtype):
    check_selection(*some_logits(groups, beams, vocab, dtype, seed=vocab), take)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("more,offset", [(1, 0), (3, 1), (8, 0), (7, 5)])
def test_rows_of_any_stride_and_alignment(more, offset, dtype):
    logits, scores = some_logits(2, 3, 9001, dtype, more=more + offset)
    wide = torch.empty(6, 9001 + more + offset, dtype=dtype, device="cuda")
    wide[:, offset: offset + 9001] = logits
    check_selection(wide[:, offset: offset + 9001], scores, 6)


def test_equal_scores_go_to_the_lowest_beam_and_token():
    logits = torch.zeros(6, 5000, device="cuda")
    scores = torch.zeros(2, 3, device="cuda")
    choice = check_selection(logits, scores, 20)
    assert choice.parents.tolist() == [[0] * 20] * 2 and choice.tokens.tolist() == [list(range(20))] * 2
    choice = check_selection(torch.full((4, 70000), -3.5, device="cuda"), torch.tensor([[-2.0, -1.0, -1.0, -3.0]], device="cuda"), 64)
    assert choice.parents.tolist() == [[1] * 64] and choice.tokens.tolist() == [list(range(64))]
    logits, _ = some_logits(1, 1, 9001)  # beams that hold the same, at addresses that are aligned differently
    same = torch.empty(4, 9001, device="cuda").copy_(logits)
    choice = check_selection(same, torch.zeros(1, 4, device="cuda"), 8)
    assert choice.parents.tolist() == [[0, 1, 2, 3] * 2]


def test_few_values_many_ties():
    random = torch.Generator("cuda").manual_seed(3)
    logits = torch.randint(0, 3, (8, 20000), device="cuda", generator=random).float()
    check_selection(logits, torch.tensor([[0.0, -1.0, -2.0, 0.0], [0.0, 0.0, 0.0, 0.0]], device="cuda"), 64)


def test_rising_and_falling_rows():
    """Every batch beats the one before; only the first one counts."""
    up = torch.arange(30000, device="cuda").float() / 1000
    check_selection(torch.stack([up, up.flip(0)]), torch.zeros(1, 2, device="cuda"), 64)
    check_selection(torch.stack([up, up]), torch.tensor([[0.0], [-1.0]], device="cuda"), 33)


def test_masked_logits_and_dead_beams():
    inf, nan = float("inf"), float("nan")
    logits, scores = some_logits(2, 4, 6000, seed=9)
    logits[0, :] = -inf          # nothing is allowed
    logits[1, 10:] = -inf        # few are
    logits[2, 5] = nan
    logits[3, 100] = inf
    scores[1] = torch.tensor([0.0, -inf, nan, -inf], device="cuda")
    check_selection(logits, scores, 16)
    logits[4, 3:] = -inf
    choice = check_selection(logits, scores, 16)
    assert choice.parents[1].tolist() == [0] * 3 + [-1] * 13
    logits[4, :] = nan
    assert check_selection(logits, scores, 16).parents[1].tolist() == [-1] * 16
    logits.fill_(torch.finfo(torch.float32).min)  # a mask of the lowest number: allowed, and equal
    assert check_selection(logits[:4], scores[:1].zero_(), 4).tokens.tolist() == [[0, 1, 2, 3]]


def test_a_first_step_of_one_beam():
    logits, _ = some_logits(3, 4, 8000, seed=11)
    scores = torch.full((3, 4), float("-inf"), device="cuda")
    scores[:, 0] = 0
    assert check_selection(logits, scores, 4).parents.tolist() == [[0] * 4] * 3


@pytest.mark.parametrize("vocab,take", [(10, 30), (1, 4), (40, 64), (300, 64)])
def test_dead_beams_have_no_continuations(vocab, take):
    """Not even where there are places left."""
    logits, scores = some_logits(2, 3, vocab, seed=vocab)
    scores[0, 1:] = -float("inf")
    scores[1, 0], scores[1, 2] = float("nan"), -float("inf")
    choice = check_selection(logits, scores, take)
    there = min(take, vocab)
    assert choice.parents.tolist() == [[0] * there + [-1] * (take - there), [1] * there + [-1] * (take - there)]


@pytest.mark.parametrize("beams,take", [(8, 16), (16, 16), (16, 32), (32, 64)])
@pytest.mark.parametrize("step", [float("inf"), 40.0, 3.0, 0.01])
def test_a_few_beams_hold_all_that_is_best(beams, take, step):
    logits, _ = some_logits(2, beams, 40001, torch.bfloat16, seed=beams)
    scores = torch.stack([-torch.arange(beams).float().mul(step).nan_to_num(0.0), -torch.arange(beams).flip(0).float().mul(step).nan_to_num(0.0)]).cuda()
    check_selection(logits, scores, take)


def test_scores_beyond_what_float_adds_up():
    """Sums of a score and a logit that pass the largest number, and scores beside which a logit is lost."""
    logits, _ = some_logits(1, 4, 3000, seed=5)
    for score in ([0.0, -3e38, -1e9, -3.4e38], [3e38, 3.4e38, 1e9, 0.0], [-3.4e38, -3.4e38, -float("inf"), -3.4e38]):
        choice = beam_select(logits, torch.tensor([score], device="cuda"), 8)
        best = max(range(4), key=lambda b: score[b])
        want = logits[best].double().sort(descending=True, stable=True).indices[:8]
        assert choice.parents.tolist() == [[best] * 8]
        if abs(score[best]) < 1e8:  # above, logits of different size are one score in float64, too
            assert choice.tokens.tolist() == [want.tolist()]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [1, 255, 256, 257, 511, 513, 8191, 8193, 33000])
def test_every_alignment_gives_the_same(vocab, dtype):
    """To the bit, for the rows of a call: eight bfloat16 or four float fit between two boundaries of 16 bytes."""
    logits, _ = some_logits(1, 1, vocab, dtype, seed=vocab)
    stride = (vocab + 7) // 8 * 8 + 9
    memory = torch.full((stride * 8,), float("inf"), dtype=dtype, device="cuda")  # what is beside a row is not looked at
    rows = memory.view(8, stride)[:, :vocab]
    rows.copy_(logits.expand(8, vocab))
    choice = check_selection(rows, torch.full((8, 1), -2.5, device="cuda"), 3)
    assert all((x == x[:1]).all() for x in choice)


def reordered(parents, lengths, table, caches, states, rows=None):
    """Plain: everything is read before anything is written."""
    groups, beams = parents.shape
    old_table, old_caches, old_states = table.clone(), [c.clone() for c in caches], [s.clone() for s in states]
    for g in range(groups):
        for j in range(beams):
            p, i = int(parents[g, j]), g * beams + j
            source = g * beams + (p if p >= 0 else j)
            if table.numel():
                page = caches[0].shape[3]
                full, filled = divmod(int(lengths[g]), page)
                table[i, :full] = old_table[source, :full]
                for cache, old in zip(caches, old_caches):
                    if filled:
                        cache[:, old_table[i, full], :, :filled] = old[:, old_table[source, full], :, :filled]
            for state, old in zip(states, old_states):
                a, b = (i, source) if rows is None else (int(rows[i]), int(rows[source]))
                state[:, a] = old[:, b]


def check_reordering(parents, lengths, *, page=16, outer=4, inner=64, layers=3, dtype=torch.bfloat16, records=(), rows=False, seed=0, caches=1):
    random = torch.Generator().manual_seed(seed)
    parents = torch.tensor(parents, dtype=torch.int32)
    groups, beams = parents.shape
    n = groups * beams
    width = max(lengths) // page + 1 + seed % 2
    pages = n * width + 3
    table = torch.randperm(pages, generator=random)[: n * width].to(torch.int32).view(n, width)

    def bytes_of(*shape):
        return torch.randint(0, 256, shape, dtype=torch.uint8, generator=random)

    size = torch.empty(0, dtype=dtype).element_size()
    pool = [bytes_of(layers, pages, outer, page, inner * size) for _ in range(caches)]
    places = n + 5 if rows else n
    at = torch.randperm(places, generator=random)[:n].to(torch.int32) if rows else None
    states = [bytes_of(2, places, r) for r in records]
    moved = [x.clone().cuda() for x in (table, *pool, *states)]
    lengths_there = torch.tensor(lengths, dtype=torch.int32).cuda()
    beam_reorder(parents.cuda(), lengths_there, moved[0] if caches else None, [c.view(dtype) for c in moved[1: 1 + caches]], moved[1 + caches:], state_rows=at.cuda() if rows else None)
    ops.raise_on_status(lengths_there.device)
    if not caches:
        table = table[:0]
    reordered(parents, lengths, table, pool, states, at)
    for got, want in zip(moved[0 if caches else 1:], ([table] if caches else []) + pool + states):
        assert torch.equal(got.cpu(), want)


@pytest.mark.parametrize("parents,lengths", [([[0]], [5]), ([[0, 0, 0, 0]], [37]), ([[3, 2, 1, 0]], [16]), ([[1, 2, 0]], [0]), ([[2, 2, 0, 3, 3], [0, 1, 2, 3, 4], [4, 3, 3, 1, 1]], [100, 31, 1]),
                                             ([[-1, 0, 0, -1]], [50])])
def test_reordering(parents, lengths):
    check_reordering(parents, lengths, seed=len(lengths), records=(4, 1000))


@pytest.mark.parametrize("beams", [2, 6, 8, 9, 16, 17, 32])
def test_any_number_of_beams(beams):
    random = np.random.default_rng(beams)
    check_reordering(random.integers(0, beams, (3, beams)).tolist(), [33, 64, 47], seed=beams, records=(160,), rows=True)


@pytest.mark.parametrize("page,outer,inner,layers,dtype,caches", [(8, 2, 128, 28, torch.bfloat16, 1), (64, 8, 128, 2, torch.float32, 1), (32, 1, 576, 3, torch.bfloat16, 1), (16, 4, 1, 2, torch.int8, 1),
                                                                  (16, 4, 3, 2, torch.uint8, 1), (5, 4, 6, 2, torch.bfloat16, 1), (16, 6, 64, 2, torch.float8_e4m3fn, 3)])
def test_pages_of_any_kind(page, outer, inner, layers, dtype, caches):
    check_reordering([[1, 1, 0, 2], [3, 3, 3, 3]], [page * 3 + page // 2, 2 * page - 1], page=page, outer=outer, inner=inner, layers=layers, dtype=dtype, caches=caches, records=(8,))


@pytest.mark.parametrize("record", [1, 2, 3, 4, 12, 16, 4096, 4097, 100000])
def test_records_of_any_size(record):
    check_reordering([[1, 2, 2, 0], [0, 0, 1, 3]], [9, 9], records=(record, 32), caches=0)


def test_a_page_of_codes_and_one_of_exponents():
    cache = ops.new_cache8(9, 2, 16, 64)
    random = torch.Generator("cuda").manual_seed(1)
    cache.codes.view(torch.uint8).random_(0, 256, generator=random)
    cache.exponents.random_(-40, 40, generator=random)
    codes, exponents = cache.codes.view(torch.uint8).clone(), cache.exponents.clone()
    table = torch.tensor([[0, 1], [0, 2], [0, 3]], dtype=torch.int32, device="cuda")
    beam_reorder(torch.tensor([[2, 0, 0]], dtype=torch.int32, device="cuda"), torch.tensor([21], dtype=torch.int32, device="cuda"), table,
                 [cache.codes.view(1, 9, 4, 16, 64), cache.exponents.view(1, 9, 4, 16, 1)])
    ops.raise_on_status(codes.device)
    old = [codes.clone(), exponents.clone()]
    for to, source in ((1, 3), (2, 1), (3, 1)):
        codes[to, :, :, :5], exponents[to, :, :, :5] = old[0][source, :, :, :5], old[1][source, :, :, :5]
    assert torch.equal(codes, cache.codes.view(torch.uint8)) and torch.equal(exponents, cache.exponents) and table[:, 0].tolist() == [0, 0, 0]


def test_what_is_not_there_is_reported_and_stays():
    cache, state = torch.randn(1, 4, 2, 8, 64, device="cuda"), torch.randn(1, 3, 5, device="cuda")
    length = torch.tensor([5], dtype=torch.int32, device="cuda")
    for parents, table, rows, match in (([[3, 0, 1]], [[0], [1], [2]], [0, 1, 2], "position"), ([[1, 0, 2]], [[0], [-1], [2]], [0, 1, 2], "block-table"), ([[2, 1, 1]], [[0], [4], [2]], [0, 1, 2], "block-table"),
                                        ([[1, 0, 0]], [[0], [1], [2]], [0, 5, -1], "position")):
        pages, records = cache.clone(), state.clone()
        beam_reorder(torch.tensor(parents, dtype=torch.int32, device="cuda"), length, torch.tensor(table, dtype=torch.int32, device="cuda"), [pages], [records],
                     state_rows=torch.tensor(rows, dtype=torch.int32, device="cuda"))
        with pytest.raises(ops.KernelError, match=match):
            ops.raise_on_status(cache.device)
        assert torch.equal(pages[0, 0], cache[0, 0]) or parents[0][0] in (1, 2) and 0 <= table[parents[0][0]][0] < 4


def test_a_tensor_comes_once():
    state = torch.zeros(1, 4, 8, device="cuda")
    with pytest.raises(ops.KernelError, match="once"):
        beam_reorder(torch.zeros(1, 4, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda"), None, [], [state, state])
