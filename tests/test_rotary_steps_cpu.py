"""Steps of the rotary phases for frequencies of more than one turn a position."""

import math

import pytest
import torch

from cxlsparse_b200.rotary import Rotary, frequencies

SCALINGS = [dict(type="linear", factor=f) for f in (0.3, 0.08, 0.075, 0.05, 0.011, 1e-4)] + [
    dict(type="ntk", factor=1e-4), dict(type="yarn", factor=0.01, original=4096)]


@pytest.mark.parametrize("scaling", SCALINGS, ids=str)
def test_steps_hold_any_frequency(scaling):
    """The phase of a position against the frequency's own, in fp64: off by the
    rounding of the frequency (2^-53 of its turns) and of the product."""
    f, _ = frequencies(64, scaling=scaling)
    steps = Rotary(64, scaling=scaling, device="cpu").steps
    for position in (1, 2, 977, 65536):
        turns = f / (2 * math.pi) * position
        off = (steps * position).double() * 2.0 ** -64 - turns
        assert ((off - off.round()).abs() <= 2.0 ** -50 * (turns.abs() + position)).all()


@pytest.mark.parametrize("scaling", [dict(type="yarn", factor=math.inf, original=4096),
                                     dict(type="yarn", factor=2.0, original=4096,
                                          magnitude=math.nan),
                                     dict(type="linear", factor=1e-320),
                                     dict(type="ntk", factor=5e-324)], ids=str)
def test_frequencies_that_are_not_finite_are_refused(scaling):
    with pytest.raises(ValueError):
        Rotary(64, scaling=scaling, device="cpu")
