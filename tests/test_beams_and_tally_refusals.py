"""What the operators of beams and of caches of a fixed budget refuse, and the selection's host reference; no GPU."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from hyperion_b200 import ops
from hyperion_b200.ops import KernelError, Tally, native
from hyperion_b200.sampling import beam_select, reference_beam_select


def ints(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def refuses(call, for_its_device):
    """The arguments are refused for what they are; those that are right, only because they are not on a GPU."""
    with pytest.raises(KernelError) as refusal:
        call()
    assert ("CUDA device" in str(refusal.value)) == for_its_device, str(refusal.value)


def tallied(**change):
    given = dict(q=torch.zeros(2, 4 * 64, dtype=torch.bfloat16), heads=4, cache=torch.zeros(5, 2, 2, 16, 64, dtype=torch.bfloat16), block_table=ints(2, 3), lengths=ints(2), newest=ints(2),
                 tally=Tally(torch.zeros(2, 2, 48), ints(2, 2, 48)), scale=0.125)
    given.update(change)
    return lambda: ops.attention_tallied(**given)


def queried(**change):
    given = dict(q=torch.zeros(7, 4 * 64, dtype=torch.bfloat16), heads=4, cache=torch.zeros(5, 2, 2, 16, 64, dtype=torch.bfloat16), block_table=ints(2, 3), starts=ints(3), lengths=ints(2),
                 tally=Tally(torch.zeros(2, 2, 48), ints(2, 2, 48)), scale=0.125, most=4)
    given.update(change)
    return lambda: ops.tally_queries(**given)


def evicted(**change):
    given = dict(cache=torch.zeros(3, 5, 2, 2, 16, 64, dtype=torch.bfloat16), block_table=ints(2, 3), lengths=ints(2), newest=ints(2), tally=Tally(torch.zeros(3, 2, 2, 48), ints(3, 2, 2, 48)), keep=8)
    given.update(change)
    return lambda: ops.evict(**given)


def reordered(**change):
    given = dict(parents=ints(2, 3), lengths=ints(2), block_table=ints(6, 4), caches=[torch.zeros(2, 30, 4, 16, 64)], states=[torch.zeros(2, 6, 9)])
    given.update(change)
    return lambda: ops.beam_reorder(**given)


def selected(logits=torch.zeros(6, 50), scores=torch.zeros(2, 3), take=4):
    return lambda: beam_select(logits, scores, take)


bf16 = torch.bfloat16
ATTENTION = [dict(cache=torch.zeros(5, 2, 2, 16, 64)), dict(cache=torch.zeros(5, 2, 2, 16, 80, dtype=bf16)), dict(cache=torch.zeros(5, 2, 2, 12, 64, dtype=bf16)), dict(cache=torch.zeros(5, 3, 2, 16, 64, dtype=bf16)),
             dict(cache=torch.zeros(5, 2, 2, 64, 16, dtype=bf16).transpose(3, 4)), dict(cache=torch.zeros(2, 2, 16, 64, dtype=bf16)), dict(heads=3), dict(heads=0), dict(heads=6), dict(block_table=ints(1, 3)),
             dict(block_table=ints(2, 3).long()), dict(block_table=ints(3, 2).t()), dict(lengths=ints(3)), dict(lengths=ints(2).long()), dict(lengths=ints(4)[::2]), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")),
             dict(longest=49), dict(longest=-1), dict(tally=Tally(torch.zeros(2, 2, 48), ints(2, 2, 47))), dict(tally=Tally(torch.zeros(2, 2, 48).double(), ints(2, 2, 48))),
             dict(tally=Tally(torch.zeros(1, 2, 48), ints(1, 2, 48))), dict(tally=Tally(torch.zeros(2, 48, 2).transpose(1, 2), ints(2, 2, 48))), dict(tally=Tally(torch.zeros(3, 2, 2, 48), ints(3, 2, 2, 48)))]


@pytest.mark.parametrize("change", ATTENTION + [dict(q=torch.zeros(2, 256)), dict(q=torch.zeros(2, 255, dtype=bf16)), dict(q=torch.zeros(256, 2, dtype=bf16).t()), dict(newest=ints(1)), {}])
def test_attention_tallied(change):
    refuses(tallied(**change), not change)


@pytest.mark.parametrize("change", ATTENTION + [dict(starts=ints(2)), dict(starts=ints(3).long()), dict(most=-1), dict(q=torch.zeros(7, 256)), {}])
def test_tally_queries(change):
    refuses(queried(**change), not change)


@pytest.mark.parametrize("change", [dict(keep=0), dict(first=-1), dict(recent=-1), dict(cache=torch.zeros(5, 2, 2, 16, 64)), dict(cache=torch.zeros(3, 5, 2, 2, 12, 64)), dict(cache=torch.zeros(3, 5, 2, 2, 16, 3)),
                                    dict(cache=torch.zeros(3, 5, 1, 2, 16, 64)), dict(cache=torch.zeros(3, 5, 2, 2, 64, 16).transpose(4, 5)), dict(block_table=ints(1, 3)), dict(newest=ints(3)), dict(lengths=ints(2).long()),
                                    dict(longest=49), dict(out=Tally(torch.zeros(3, 2, 2, 40), ints(3, 2, 2, 40))), dict(tally=Tally(torch.zeros(2, 2, 48), ints(2, 2, 48))), {}])
def test_evict(change):
    refuses(evicted(**change), not change)


def test_evict_half_in_place():
    tally = Tally(torch.zeros(3, 2, 2, 48), ints(3, 2, 2, 48))
    with pytest.raises(KernelError, match="takes the place of all of the old one"):
        evicted(tally=tally, out=Tally(tally.weights, ints(3, 2, 2, 48)))()


@pytest.mark.parametrize("change", [dict(parents=ints(2, 33), block_table=ints(66, 4)), dict(parents=ints(2, 3).long()), dict(parents=ints(6)), dict(lengths=ints(3)), dict(block_table=ints(5, 4)), dict(block_table=None),
                                    dict(caches=[]), dict(caches=[torch.zeros(2, 30, 4, 16)]), dict(caches=[torch.zeros(2, 30, 4, 16, 64), torch.zeros(2, 30, 4, 8, 64)]), dict(caches=[torch.zeros(2, 30, 16, 4, 64).transpose(2, 3)]),
                                    dict(states=[torch.zeros(2, 5, 9)]), dict(states=[torch.zeros(6)]), dict(states=[torch.zeros(2, 9, 6).transpose(1, 2)]), dict(states=[torch.zeros(2, 6, 9)] * 24), dict(state_rows=ints(5)), {}])
def test_beam_reorder(change):
    refuses(reordered(**change), not change)


@pytest.mark.parametrize("call", [selected(take=0), selected(take=65), selected(logits=torch.zeros(5, 50)), selected(logits=torch.zeros(6, 50).half()), selected(logits=torch.zeros(50, 6).t()), selected(logits=torch.zeros(1, 50).expand(6, 50)),
                                  selected(logits=torch.zeros(6, 0)), selected(scores=torch.zeros(2, 3).double()), selected(scores=torch.zeros(3, 2).t()), selected(torch.zeros(33, 50), torch.zeros(1, 33))])
def test_beam_select(call):
    refuses(call, False)


def test_beam_select_on_the_host():
    refuses(selected(), True)


def test_the_reference_selection():
    z = np.log(np.array([[0.5, 0.25, 0.25], [0.1, 0.6, 0.3]]))
    found = reference_beam_select(z, np.log(np.array([0.5, 0.4])), 4)
    assert [(b, v) for b, v, _ in found] == [(0, 0), (1, 1), (0, 1), (0, 2)]
    assert np.allclose([s for _, _, s in found], np.log([0.25, 0.24, 0.125, 0.125]), rtol=0, atol=1e-7)
    z[0, 1] = -np.inf
    assert [(b, v) for b, v, _ in reference_beam_select(z, np.array([0.0, -np.inf]), 4)] == [(0, 0), (0, 2)]
    assert reference_beam_select(np.full((2, 3), np.nan), np.zeros(2), 2) == []


def test_a_launchers_arguments_come_as_one_structure():
    """In their order and sizes: the launcher refuses what is wrong with any one of them, before it looks at the device."""
    evict = native.entry("evict", "hb_evict", "piiiiipippiippppiiiipppip", packed=True)
    names = ("cache layers pages kv_heads page_size record block_table width lengths newest requests longest weights positions to_weights to_positions capacity keep first recent left scratch status sms "
             "stream").split()
    sound = dict.fromkeys(names, 1 << 40) | dict(layers=1, pages=4, kv_heads=2, page_size=16, record=128, width=4, requests=70000, longest=64, capacity=64, keep=32, first=0, recent=0, sms=148, stream=0)

    def call(**changed):
        return evict(*(sound | changed).values())

    assert call(requests=0) == 0 and call(layers=0) == 0
    assert call() == -2  # more requests than a grid has room for
    for name in ("cache", "block_table", "lengths", "newest", "weights", "positions", "to_weights", "to_positions", "left", "scratch", "status"):
        assert call(**{name: 0}) == -1, name
    for name, wrong in (("pages", 0), ("kv_heads", 0), ("page_size", 24), ("record", 24), ("width", 3), ("longest", 65), ("capacity", 63), ("keep", 0), ("recent", -1), ("sms", 0), ("cache", (1 << 40) + 8), ("scratch", (1 << 40) + 8)):
        assert call(**{name: wrong}) == -1, name
    with pytest.raises(KernelError, match="hb_evict"):
        call(capacity=1 << 31)
