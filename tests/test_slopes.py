"""Slopes of head counts that are not powers of two: the published table."""
import pytest

from molot_amd import attn


def powers(exponents):
    return [2.0 ** e for e in exponents]


@pytest.mark.parametrize("nq,exponents", [
    (1, [-8]), (2, [-4, -8]), (3, [-4, -8, -2]), (5, [-2, -4, -6, -8, -1]),
    (6, [-2, -4, -6, -8, -1, -3]), (7, [-2, -4, -6, -8, -1, -3, -5]),
    (8, range(-1, -9, -1)),
    (12, [*range(-1, -9, -1), -0.5, -1.5, -2.5, -3.5]),
    (71, [-(h + 1) / 8 for h in range(64)] + [-(2 * k + 1) / 16 for k in range(7)])])
def test_interleaved(nq, exponents):
    """nq heads: those of the power of two below, then every other one of twice as many.
    (The fp32 values round 2^e once: half a step.)"""
    got = attn.alibi_slopes(nq, interleaved=True)
    assert got.tolist() == pytest.approx(powers(exponents), rel=2.0 ** -24)


@pytest.mark.parametrize("nq", [1, 2, 4, 32, 128])
def test_powers_of_two_have_one_table(nq):
    assert attn.alibi_slopes(nq, interleaved=True).equal(attn.alibi_slopes(nq))
