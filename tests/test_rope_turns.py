"""The frequencies that kc_rope makes (kestrel_b200/csrc/rope_turns.h), on the CPU,
against its formulas with 70 digits.

A phase is position * turn modulo 2^64, exact, so its error at position 2^31 is 2^31
times that of the turn. A turn is w / 2 pi; with u = 2^-64 the roundings of w are the
power's (2 u of it, and none of its exponent), the divisor's (u), the scaling's (5 u
at most) and 2 pi's and its division's (2 u): 10 u w / 2 pi, and u / 2 for the whole
number: 2.1 u where w is 1 at most, 6.9 u at 4. So angles are good to 2^-31 of a turn
at every int32 position, and to 2^-30 where the frequency is above 1."""
import os
import random
import shutil
import subprocess
from decimal import ROUND_CEILING, ROUND_FLOOR, Decimal as D, getcontext

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PI = D("3.14159265358979323846264338327950288419716939937510582097494459230781640628620899")
NONE, LINEAR, YARN, BANDS = range(4)
getcontext().prec = 70


@pytest.fixture(scope="module")
def driver(tmp_path_factory):
    cxx = shutil.which("g++")
    if not cxx:
        pytest.skip("g++ not found")
    exe = str(tmp_path_factory.mktemp("rope") / "rope_turns_driver")
    subprocess.run([cxx, "-std=c++17", "-O1", "-Wall", "-Werror", "-I", os.path.join(ROOT, "kestrel_b200", "csrc"),
                    os.path.join(ROOT, "tests", "rope_turns_driver.cpp"), "-o", exe], check=True)
    return exe


def f32(x):
    return float(np.float32(x))


def made(exe, cases):
    lines = [" ".join(repr(v) if isinstance(v, float) else str(v) for v in (*c[:8], *(c[8] or []))) for c in cases]
    out = subprocess.run([exe], input="\n".join(lines) + "\n", capture_output=True, text=True, check=True).stdout.splitlines()
    assert len(out) == len(cases)
    return [None if o == "refused" else (float(o.split()[0]), [int(t) for t in o.split()[1:]]) for o in out]


def frequencies(dim, base, scaling, factor, original, low, high, ff):
    base, s, low, high, size = D(base), D(factor), D(low), D(high), D(original)
    lb, out = base.ln(), []
    if scaling == YARN:
        c = lambda x: dim * (size / (2 * PI * x)).ln() / (2 * lb)
        a = max(D(0), c(high).to_integral_value(ROUND_FLOOR))
        b = min(D(dim - 1), c(low).to_integral_value(ROUND_CEILING))
    for i in range(dim // 2):
        w = (lb * -2 * i / dim).exp() / (D(ff[i]) if ff else 1)
        if scaling == LINEAR:
            w /= s
        elif scaling == YARN:
            r = min(D(1), max(D(0), (i - a) / max(D("0.001"), b - a)))
            w *= r / s + 1 - r
        elif scaling == BANDS:
            z = min(D(1), max(D(0), (size * w / (2 * PI) - low) / (high - low)))
            w *= z + (1 - z) / s
        out.append(w)
    return out


def case(rng):
    dim = 2 * rng.choice([1, 2, 10, 16, 32, 40, 64, rng.randint(1, 128), 128])
    base = f32(rng.choice([1e4, 5e5, 1e6, 53646.0, rng.uniform(1.5, 100.0), 10 ** rng.uniform(1, 12)]))
    scaling = rng.choice([NONE, NONE, LINEAR, YARN, BANDS])
    ff = [f32(rng.uniform(0.3, 40.0)) for _ in range(dim // 2)] if rng.random() < 0.3 else None
    if scaling in (NONE, LINEAR) and rng.random() < 0.3:
        base = f32(rng.uniform(0.3, 1.0))
    factor = f32(rng.choice([2.0, 8.0, 4.0, rng.uniform(1.0, 64.0)]))
    low, high = {YARN: (1.0, 32.0), BANDS: (1.0, 4.0)}.get(scaling, (0.0, 0.0))
    return dim, base, scaling, factor, rng.choice([512, 4096, 8192, 32768, 131072]), low, high, 0.0, ff


# Bases and sizes whose far phases were off by more than 2^-33 of a turn.
KNOWN = [(80, f32(53646.0), NONE, 1.0, 0, 0.0, 0.0, 0.0, None), (128, f32(0.4486), NONE, 1.0, 0, 0.0, 0.0, 0.0, None)]


def bridged(dim, base, want):
    """A base whose powers the divisors bring back to frequencies near `want`."""
    ff = [f32(D(base) ** (D(-2 * i) / dim) / D(want)) for i in range(dim // 2)]
    return dim, base, NONE, 1.0, 0, 0.0, 0.0, 0.0, ff


def test_turns(driver):
    rng = random.Random(5)
    cases = KNOWN + [case(rng) for _ in range(400)]
    cases += [bridged(dim, f32(base), want) for dim in (6, 96, 128) for base in (1e36, 1e-36, 2e20) for want in (0.9, 3.9)]
    taken = 0
    for c, got in zip(cases, made(driver, cases)):
        dim, base, scaling, factor, original, low, high, _, ff = c
        w = frequencies(dim, base, scaling, factor, original, low, high, ff)
        if max(w) > D(4):
            assert got is None
            continue
        taken += 1
        for x, turn in zip(w, got[1]):
            off = abs((x / (2 * PI) - D(turn) / 2 ** 64 + D("0.5")) % 1 - D("0.5"))
            u = D(2) ** -64
            assert off <= 10 * u * x / (2 * PI) + u / 2, (c, x, off / u)
            assert off * 2 ** 31 <= D(2) ** (-31 if x <= 1 else -30)
    assert taken > 300


def test_frequencies_past_the_limit(driver):
    at = lambda base, ff=None: (4, base, NONE, 1.0, 0, 0.0, 0.0, 0.0, ff)
    assert [g is None for g in made(driver, [at(1e4), at(f32(0.0625)), at(f32(0.0624)), at(1e4, [0.25, 1.0]), at(1e4, [f32(0.249), 1.0])])] == \
        [False, False, True, False, True]
