"""Waits inside the kernels that run out: the call reports it, the kernels leave (with what they had on its way arrived, and tensor memory freed), and the next call is right.

The kernels are built with a limit of their own: 0 looks at a barrier, so that every wait runs out at once, or 1, so that some may, with copies on their way."""
from __future__ import annotations

import pytest
import torch
from test_tally_gpu import pages_of, queries

from hyperion_b200 import ops
from hyperion_b200.ops import native
from hyperion_b200.ops.tally import attention_tallied, new_tally, tally_queries

pytestmark = pytest.mark.gpu


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def tallied(lengths, slack=1, heads=8, kv=2, dim=64):
    cache, table, random = pages_of(lengths, kv, dim, 16, seed=len(lengths), slack=slack)
    q, tally = queries(random, len(lengths), heads * dim), new_tally(len(lengths), kv, table.shape[1] * 16)

    def call():
        tally.weights.zero_()
        out = attention_tallied(q, heads, cache, table, ints(lengths), ints(lengths), tally, 0.125)
        return out, tally.weights.clone()
    return call


def many(counts, lengths):
    cache, table, random = pages_of(lengths, 2, 64, 16, seed=len(lengths) + 7)
    q, tally = queries(random, sum(counts), 8 * 64), new_tally(len(lengths), 2, table.shape[1] * 16)
    starts = ints([sum(counts[:i]) for i in range(len(counts) + 1)])

    def call():
        tally.weights.zero_()
        tally_queries(q, 8, cache, table, starts, ints(lengths), tally, 0.125, most=max(counts))
        return (tally.weights.clone(),)
    return call


@pytest.mark.parametrize("limit", [0, 1])
def test_waits_that_run_out(limit, monkeypatch):
    calls = {"hb_attention_tallied": [tallied([1500, 3, 1, 130, 800]), tallied([5000]), tallied([300] * 30), tallied([1500, 3, 1, 130, 800], 600), tallied([9000])], "hb_tally_queries": [many([20], [3000]), many([700, 1, 300], [700, 50, 900]), many([1], [1])]}
    want = {name: [call() for call in some] for name, some in calls.items()}
    ops.raise_on_status(torch.device("cuda", torch.cuda.current_device()))
    with monkeypatch.context() as patch:
        for name in calls:
            found = native._entries[name, 64]
            short = getattr(native.library(name[3:], HB_HEAD_DIM=64, HB_WAIT_LIMIT=limit), name)
            short.argtypes = found.argtypes
            patch.setitem(native._entries, (name, 64), short)
        for name, some in calls.items():
            for call, right in zip(some, want[name]):
                got = call()
                if limit == 0:
                    with pytest.raises(ops.KernelError, match="bounded wait"):
                        ops.raise_on_status(got[0].device)
                    continue
                try:
                    ops.raise_on_status(got[0].device)
                    assert all(torch.equal(a, b) for a, b in zip(got, right))
                except ops.KernelError as error:
                    assert "bounded wait" in str(error)
    for name, some in calls.items():
        for call, right in zip(some, want[name]):
            assert all(torch.equal(a, b) for a, b in zip(call(), right))
    ops.raise_on_status(torch.device("cuda", torch.cuda.current_device()))


@pytest.mark.parametrize("limit", [0, 1])
def test_waits_of_three_sets_that_run_out(limit, monkeypatch):
    calls = [tallied([1500, 3, 1, 130, 800], heads=24, kv=1, dim=128), tallied([30000], heads=20, kv=1, dim=128)]
    want, name = [call() for call in calls], "hb_attention_tallied"
    ops.raise_on_status(torch.device("cuda", torch.cuda.current_device()))
    found = native._entries[name, 128]
    with monkeypatch.context() as patch:
        short = getattr(native.library(name[3:], HB_HEAD_DIM=128, HB_WAIT_LIMIT=limit), name)
        short.argtypes = found.argtypes
        patch.setitem(native._entries, (name, 128), short)
        for call in calls:
            got = call()
            if limit == 0:
                with pytest.raises(ops.KernelError, match="bounded wait"):
                    ops.raise_on_status(got[0].device)
            else:
                try:
                    ops.raise_on_status(got[0].device)
                except ops.KernelError:
                    pass
    for call, right in zip(calls, want):
        assert all(torch.equal(a, b) for a, b in zip(call(), right))
        ops.raise_on_status(right[0].device)


@pytest.mark.parametrize("limit", [0, 1])
def test_waits_of_a_few_queries_of_long_contexts(limit, monkeypatch):
    call, name = many([4, 3, 0], [9000, 5000, 300]), "hb_tally_queries"
    want = call()
    ops.raise_on_status(want[0].device)
    found = native._entries[name, 64]
    with monkeypatch.context() as patch:
        short = getattr(native.library(name[3:], HB_HEAD_DIM=64, HB_WAIT_LIMIT=limit), name)
        short.argtypes = found.argtypes
        patch.setitem(native._entries, (name, 64), short)
        got = call()
        if limit == 0:
            with pytest.raises(ops.KernelError, match="bounded wait"):
                ops.raise_on_status(got[0].device)
        else:
            try:
                ops.raise_on_status(got[0].device)
            except ops.KernelError:
                pass
    assert torch.equal(call()[0], want[0])
    ops.raise_on_status(want[0].device)
