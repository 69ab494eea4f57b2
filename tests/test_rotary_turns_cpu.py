"""Turns that cannot be made are refused as such, before a device is looked for."""
from decimal import Decimal

import pytest

from tests.test_kv_cpu import fv  # noqa: F401


@pytest.mark.parametrize("change", [dict(base=5e-324), dict(factor=5e-324), dict(factor=1e-310, base=1e-3), dict(factor=5e-324, original=10)])
def test_frequencies_beyond_floats(fv, change):  # noqa: F811
    with pytest.raises(fv.FerrovecError, match="frequencies"):
        fv.Rotary(128, **change)


@pytest.mark.parametrize("change", [dict(base=1e308), dict(factor=1e308), dict(base=1e-300), dict(frequencies=[1e308 / (i + 1) for i in range(64)]), dict(original=10**15, factor=3.0), dict(frequencies=[0.0] * 64)])
def test_frequencies_far_out_are_turns_all_the_same(fv, change):  # noqa: F811
    """A device is what is missing."""
    with pytest.raises(fv.FerrovecError, match="CPU"):
        fv.Rotary(128, device="cpu", **change)
    from ferrolm_b200.rotary import _frequencies, _turns

    made = dict(base=10000.0, factor=1.0, original=None, fast=32.0, slow=1.0) | change
    w = [Decimal(x) for x in made["frequencies"]] if "frequencies" in made else _frequencies(made["base"], 128, made["factor"], made["original"], 32.0, 1.0)
    assert len(w) == 64 and all(0 <= x < 2**64 for x in _turns(w))
