"""Arguments of the operators of beams and of caches of a fixed budget that are refused although their types and shapes are right; no GPU."""
from __future__ import annotations

import pytest
import torch
from test_beams_and_tally_refusals import bf16, evicted, ints, queried, refuses, reordered, tallied

from hyperion_b200.ops import Tally


@pytest.mark.parametrize("scale,fits", [(float("inf"), False), (1e39, False), (2.0 ** 128, False), (2.0 ** 127, True), (2.0 ** -100, True), (2.0 ** -101, False)])
def test_scales_beyond_float(scale, fits):
    refuses(tallied(scale=scale), fits)
    refuses(queried(scale=scale), fits)


@pytest.mark.parametrize("requests,out,fits", [(2, torch.zeros(1, 256, dtype=bf16).expand(2, 256), False), (2, torch.zeros(600, dtype=bf16).as_strided((2, 256), (252, 1)), False),
                                               (2, torch.zeros(600, dtype=bf16).as_strided((2, 256), (256, 1)), True), (2, torch.zeros(2, 300, dtype=bf16), True), (1, torch.zeros(1, 256, dtype=bf16).expand(1, 256), True),
                                               (1, torch.zeros(600, dtype=bf16).as_strided((1, 256), (4, 1)), True)])
def test_results_whose_rows_overlap(requests, out, fits):
    """Two requests would write the same place."""
    change = dict(out=out)
    if requests == 1:
        change |= dict(q=torch.zeros(1, 256, dtype=bf16), lengths=ints(1), newest=ints(1), tally=Tally(torch.zeros(1, 2, 48), ints(1, 2, 48)))
    refuses(tallied(**change), fits)


@pytest.mark.parametrize("shift,fits", [(0, True), (1, False), (48, False), (575, False), (576, True)])
@pytest.mark.parametrize("which", ["weights", "positions"])
def test_a_new_tally_that_overlaps_the_old_one(which, shift, fits):
    """It takes the place of the old one, or stands beside it: what is partly in its place would be written before it is read."""
    memory, numbers = torch.zeros(2 * 576), ints(2 * 576)
    old = Tally(memory[:576].view(3, 2, 2, 48), numbers[:576].view(3, 2, 2, 48))
    new = Tally(memory[shift: shift + 576].view(3, 2, 2, 48), numbers[shift: shift + 576].view(3, 2, 2, 48))
    if shift:  # the other of the two is beside the old one
        new = new._replace(**{"positions": ints(3, 2, 2, 48)} if which == "weights" else {"weights": torch.zeros(3, 2, 2, 48)})
    refuses(evicted(tally=old, out=new), fits)
    refuses(evicted(tally=new, out=old), fits)


def test_what_beams_hold_comes_once():
    """Parts of a tensor that is there already would move twice, one move beside the other."""
    pages, states = torch.zeros(3, 30, 4, 16, 64), torch.zeros(4, 6, 9)
    for caches, others, fits in (([pages[:2], pages[1:]], [states], False), ([pages[1:], pages[:2]], [], False), ([pages[:1], pages[1:]], [states], True), ([pages], [states[:2], states[2:], states[:1]], False),
                                 ([pages], [states[:2], states[2:]], True), ([pages], [states[:0], states], True), ([pages], [pages.view(-1)[64: 64 + 6 * 9].view(1, 6, 9)], False),
                                 ([pages], [states, states.view(torch.uint8)[3:]], False)):
        refuses(reordered(caches=caches, states=others), fits)
