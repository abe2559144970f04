"""CPU check of the token choice's exponential: the constants as the kernel's
source has them, against 2^f in 60 digits.

The kernel forms p(f) for the fraction f of a power, |f| <= 1/2, in 64 bits and
by fused steps, and states 2^-51 of it, roundings included. The interpolant at
the 11 Chebyshev nodes is off by ln(2)^11 / 11! 2^x 2^-21 = 2^(x - 52.07) at most,
with x between the nodes and f (near f / 12): relative to 2^f that is largest at
f = -1/2, 2^-51.6. The last step rounds by 2^-53.5 of it there, and what the step
before it and the linear coefficient were rounded by adds 2^-54.5 twice: 0.93 of
2^-51 in all."""

import os
import re
from decimal import Decimal, getcontext
from fractions import Fraction

import conftest  # noqa: F401  (paths)

SOURCE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "delta-attention_amd", "csrc",
                      "sample.hip")


def coefficients():
    with open(SOURCE) as f:
        text = f.read()
    m = re.search(r"double p = ([^;]+);\s*constexpr double c\[\] = \{([^}]*)\};", text)
    assert m, "the polynomial is not where it was"
    return [float(m.group(1))] + [float(x) for x in m.group(2).split(",")]


def fused(p, f, k):
    """fma: one rounding (Fraction to float rounds to the nearest)."""
    return float(Fraction(p) * Fraction(f) + Fraction(k))


def test_the_polynomial_is_the_power():
    getcontext().prec = 60
    co = coefficients()
    assert len(co) == 11 and co[-1] == 1.0
    ln2, worst = Decimal(2).ln(), Decimal(0)
    n = 4000
    for i in range(-n, n + 1):
        f = float(Fraction(i, 2 * n))
        p = co[0]
        for k in co[1:]:
            p = fused(p, f, k)
        power = (Decimal(f) * ln2).exp()
        worst = max(worst, abs(Decimal(p) / power - 1))
    assert worst <= Decimal(2) ** -51, float(worst)
