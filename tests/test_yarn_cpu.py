"""YaRN frequencies at every trained length, the ramp's end past the last pair
among them, against the published formula pair by pair in plain Python."""

import math

import pytest

import flashlite_amd as fl


def published(rot, base, factor, trained, fast, slow):
    def dim_of(turns):
        return rot * math.log(trained / (turns * 2 * math.pi)) / (2 * math.log(base))

    low, high = max(math.floor(dim_of(fast)), 0), min(math.ceil(dim_of(slow)), rot - 1)
    out = []
    for j in range(rot // 2):
        kept = 1.0 / base ** (2 * j / rot)
        ramp = min(max((j - low) / (high - low if high != low else 1e-3), 0.0), 1.0)
        out.append(kept / factor * ramp + kept * (1.0 - ramp))
    return out


@pytest.mark.parametrize("rot", [20, 64, 128])
@pytest.mark.parametrize("trained", [512, 4096, 32768, 65536, 131072, 1 << 20])
@pytest.mark.parametrize("factor,base", [(4.0, 1e4), (8.0, 1e4), (40.0, 5e5)])
def test_published_formula(rot, trained, factor, base):
    got, scale = fl.rotary_frequencies(rot, base=base, method="yarn", factor=factor,
                                       trained=trained)
    # a power, whose exponent's rounding counts up to ln(base) 2^-53, and a few
    # products and sums of positive terms, 2^-53 each: below 20 * 2^-53
    assert got.tolist() == pytest.approx(published(rot, base, factor, trained, 32.0, 1.0),
                                         rel=1e-14)
    assert scale == pytest.approx(0.1 * math.log(factor) + 1.0, rel=1e-15)


@pytest.mark.parametrize("rot,trained,factor", [(128, 131072, 8.0), (128, 65536, 4.0),
                                                (64, 65536, 4.0), (20, 32768, 4.0)])
def test_pairs_between_are_not_divided_in_full(rot, trained, factor):
    kept, _ = fl.rotary_frequencies(rot)
    got, _ = fl.rotary_frequencies(rot, method="yarn", factor=factor, trained=trained)
    turns = kept * trained / (2 * math.pi)
    assert float(turns[-1]) > 1.0  # every pair turns more than `slow` times
    assert bool((got > 1.01 * kept / factor).all())
