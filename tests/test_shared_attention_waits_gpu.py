"""Waits inside the kernels that run out: the step reports it, the kernels leave (with what they had on its way arrived, and tensor memory freed), and the next step is right.

The kernels are built with a limit of their own: 0 looks at a barrier, so that every wait runs out at once, or 1, so that some may, with copies on their way."""
from __future__ import annotations

import pytest
import torch
from test_shared_attention_gpu import agree, plain, step

from hyperion_b200 import ops
from hyperion_b200.ops import native
from hyperion_b200.ops.shared import attention_shared, plan_shared

pytestmark = pytest.mark.gpu
STEPS = [([1] * 5, [1500, 3, 1, 130, 800], ()), ([1] * 30, [300] * 30, ((0, 30, 200),)), ([3], [7000], ()), ([60, 1], [700, 500], ())]  # a cluster's; strips and tiles; strips; tiles


@pytest.mark.parametrize("limit", [0, 1])
@pytest.mark.parametrize("bits", [8, 16])
def test_waits_that_run_out(bits, limit, monkeypatch):
    calls = []
    for counts, lengths, groups in STEPS:
        q, cache, table = step(counts, lengths, 8, 2, 64, 16, bits, groups)
        calls.append(((q, 8, cache, table, plan_shared(counts, lengths, 8, 2, 64, shared=groups), 0.125), plain(q, 8, cache, table, counts, lengths, 0.125)))
    for call, want in calls:
        agree(attention_shared(*call), *want)
    with monkeypatch.context() as patch:
        for (name, dim), found in list(native._entries.items()):
            if name in ("hb_attention_strips", "hb_attention_shared_tiles") and dim == 64:
                module = "attention_shared" if name == "hb_attention_strips" else "attention_shared_tiles"
                short = getattr(native.library(module, HB_HEAD_DIM=64, HB_WAIT_LIMIT=limit), name)
                short.argtypes = found.argtypes
                patch.setitem(native._entries, (name, dim), short)
        for call, want in calls:
            got = attention_shared(*call)
            if limit == 0:
                with pytest.raises(ops.KernelError, match="bounded wait"):
                    ops.raise_on_status(got.device)
                continue
            try:
                agree(got, *want)
            except ops.KernelError as error:
                assert "bounded wait" in str(error)
    for call, want in calls:
        agree(attention_shared(*call), *want)
    torch.cuda.synchronize()


@pytest.mark.parametrize("bits", [8, 16])
def test_strips_that_leave_early_still_end_behind_the_tiles(bits, monkeypatch):
    """Strips start beside the tiles of their step, and whoever comes next waits for the strips alone: also where their waits run out, they end when the tiles have."""
    counts, lengths, groups = [1] * 60, [8100] * 60, ((0, 60, 8000),)
    q, cache, table = step(counts, lengths, 8, 2, 64, 16, bits, groups)
    plan = plan_shared(counts, lengths, 8, 2, 64, shared=groups)
    assert plan.tile_blocks and plan.strip_blocks
    call = (q, 8, cache, table, plan, 0.125)
    want = attention_shared(*call)
    short = native.library("attention_shared", HB_HEAD_DIM=64, HB_WAIT_LIMIT=0).hb_attention_strips
    short.argtypes = native._entries["hb_attention_strips", 64].argtypes
    for _ in range(20):
        with monkeypatch.context() as patch:
            patch.setitem(native._entries, ("hb_attention_strips", 64), short)
            attention_shared(*call)
        assert torch.equal(attention_shared(*call), want)  # over the same scratch memory
    with pytest.raises(ops.KernelError, match="bounded wait"):
        ops.raise_on_status(q.device)
