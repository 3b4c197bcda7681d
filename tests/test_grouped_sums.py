"""Grouped products: how far a long sum may be off."""
import importlib

import pytest

grouped = importlib.import_module("3deecelltracker_amd.grouped")
from test_grouped import UNIT

# what a wave adds up before it joins the total, and how many waves share a sum at least where it is that much
CHAIN, SHARED = 2048, 4


@pytest.mark.gpu
@pytest.mark.parametrize("case", ["dw", "wide", "narrow", "few"])
def test_a_long_sum_is_not_one_chain(case):
    """Equal values: an addition to a sum of s is off by up to half a unit of s, each time the same way, so one chain over n steps is off by n units
    in the end.  In chains of CHAIN steps it is CHAIN + n / (CHAIN * SHARED) units and the few that join the waves."""
    import torch as t
    third = float(t.tensor(1.0 / 3.0))
    if case == "dw":
        n = 1 << 20
        x, dy = t.ones(n, 512, device="cuda"), t.full((n, 512), third, device="cuda")
        got = grouped.product_grad(dy, x, t.zeros(1, 512, 512, device="cuda"), [0, n], need_x=False)[1]
    else:
        n = 4_000_000
        rows, cols = {"wide": (10, 300), "narrow": (10, 40), "few": (300, 8)}[case]
        got = grouped.product(t.ones(rows, n, device="cuda"), t.full((1, n, cols), third, device="cuda"), [0, rows])
    off = float((got.double() / (third * n) - 1).abs().max())
    assert off <= (CHAIN + n / (CHAIN * SHARED) + 16) * UNIT
