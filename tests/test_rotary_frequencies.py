"""rotary_frequencies: what it refuses, and what it passes over evenly in."""
import math

import pytest

import curoaring as cr


@pytest.mark.parametrize("bad", [dict(fast=4.0, slow=4.0), dict(fast=1.0, slow=32.0), dict(original=0), dict(original=-1),
                                 dict(fast=float("nan")), dict(slow=float("nan"))])
def test_parts_without_a_way_between(bad):
    """Pairs that turn as often as both limits say would be divided by zero."""
    with pytest.raises(cr.CrError) as e:
        cr.rotary_frequencies(64, scaling="parts", factor=4.0, device="cpu", **bad)
    assert e.value.code == cr.CR_ERR_INVALID


def test_parts_pass_over_in_turns():
    plain, _ = cr.rotary_frequencies(64, device="cpu")
    parts, _ = cr.rotary_frequencies(64, scaling="parts", factor=4.0, original=4096, fast=32.0, slow=1.0, device="cpu")
    between = 0
    for f, g in zip(plain.tolist(), parts.tolist()):
        turns = 4096 * f / (2 * math.pi)
        stays = min(1.0, max(0.0, (turns - 1.0) / 31.0))
        between += 0 < stays < 1
        assert abs(g - f * (stays + (1 - stays) / 4)) < 1e-15
    assert between > 3
    # other scalings take no notice of the limits
    assert cr.rotary_frequencies(64, scaling="linear", factor=2.0, fast=1.0, slow=1.0, device="cpu")[0].isfinite().all()
