"""Waits that run out, where a block's heads are three sets' and where a few queries look at long contexts: a call whose waits have run out says so, and one that does not say so is right."""
from __future__ import annotations

import pytest
import torch
from test_tally_waits_gpu import many, tallied

from hyperion_b200 import ops
from hyperion_b200.ops import native

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("limit", [0, 1])
@pytest.mark.parametrize("name,dim,make", [("hb_attention_tallied", 128, lambda: tallied([1500, 3, 1, 130, 800], heads=24, kv=1, dim=128)), ("hb_attention_tallied", 128, lambda: tallied([30000], heads=20, kv=1, dim=128)),
                                           ("hb_tally_queries", 64, lambda: many([4, 3, 0], [9000, 5000, 300]))])
def test_waits_that_run_out_are_reported(name, dim, make, limit, monkeypatch):
    call = make()
    want = call()
    device = want[0].device
    ops.raise_on_status(device)
    found = native._entries[name, dim]
    with monkeypatch.context() as patch:
        short = getattr(native.library(name[3:], HB_HEAD_DIM=dim, HB_WAIT_LIMIT=limit), name)
        short.argtypes = found.argtypes
        patch.setitem(native._entries, (name, dim), short)
        for _ in range(3):
            got, said = call(), None
            try:
                ops.raise_on_status(device)
            except ops.KernelError as error:
                said = str(error)
            assert said is not None or limit == 1
            if said is None:
                assert all(torch.equal(a, b) for a, b in zip(got, want))
            else:
                assert "bounded wait" in said
    assert all(torch.equal(a, b) for a, b in zip(call(), want))
    ops.raise_on_status(device)
