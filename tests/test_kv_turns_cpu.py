"""How near the table of angles is to the frequencies that it is made from, by whole numbers."""
from fractions import Fraction

import pytest

import b4gemv

TWO_PI = Fraction(62831853071795864769252867665590057683943387987502, 10 ** 49)


@pytest.mark.parametrize("inv", [[1e6 ** (-i / 64) for i in range(64)], [1e4 ** (-i / 64) * 0.73 for i in range(64)],
                                 [(-1) ** i * 1.7 ** (i - 8) for i in range(64)]])
def test_turns_against_two_pi(inv):
    """2 pi in fp64 is off by 2^-54.5 of itself, the quotient by 2^-53: below 2^-52 together; then half of the last of 64 bits."""
    rotary = b4gemv.Rotary(128, inv_freq=inv, device="cpu")
    for f, t in zip(inv, rotary.turns.tolist()):
        want = Fraction(f) / TWO_PI
        off = (Fraction(t, 1 << 64) - want) % 1
        assert min(off, 1 - off) <= abs(want) / 2 ** 52 + Fraction(1, 1 << 65)
