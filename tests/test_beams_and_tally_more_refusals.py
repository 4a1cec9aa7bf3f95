"""Arguments of the operators of beams and of caches of a fixed budget that are refused although their types and shapes are right; no GPU."""
from __future__ import annotations

import pytest
from test_beams_and_tally_refusals import queried, refuses, tallied


@pytest.mark.parametrize("scale,fits", [(float("inf"), False), (1e39, False), (2.0 ** 128, False), (2.0 ** 127, True), (2.0 ** -100, True), (2.0 ** -101, False)])
def test_scales_beyond_float(scale, fits):
    refuses(tallied(scale=scale), fits)
    refuses(queried(scale=scale), fits)
