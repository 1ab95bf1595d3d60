"""The fixed-point frequencies of Rotary against long arithmetic of another kind
(no GPU needed)."""
import math
from decimal import Decimal, localcontext
from fractions import Fraction

import numpy as np
import pytest
import torch

from amass_kv_b200.rotary import Rotary, rotary_frequencies

LLAMA = dict(type="llama3", factor=8.0, low_freq_factor=1.0,
             high_freq_factor=4.0, original_max_position=8192)
YARN = dict(type="yarn", factor=16.0, original_max_position=4096)


def pi():
    """16 atan(1/5) - 4 atan(1/239) in integers of 2^-300."""
    one = 1 << 300

    def atan(n):
        s, x, k = 0, one // n, 0
        while x:
            s += (-x if k & 1 else x) // (2 * k + 1)
            x //= n * n
            k += 1
        return s
    return Fraction(16 * atan(5) - 4 * atan(239), one)


def exact(r, base, sc):
    """The frequencies as fractions, right to 70 digits."""
    kind = (sc or {}).get("type")
    s = Fraction(sc["factor"]) if sc else Fraction(1)
    with localcontext() as ctx:
        ctx.prec = 80
        lb = Decimal(base).ln()
        if kind == "ntk":
            lb += Decimal(sc["factor"]).ln() * r / (r - 2)
        f = [Fraction((-lb * 2 * i / r).exp()) for i in range(r // 2)]
        if kind == "yarn":                   # dimensions by their logarithms
            tau = Decimal(pi().numerator) * 2 / Decimal(pi().denominator)
            dims = [r * (Decimal(4096) / (t * tau)).ln() / (2 * lb)
                    for t in (32, 1)]
    if kind == "linear":
        return [x / s for x in f]
    if kind == "llama3":
        keep = [(8192 * x / (2 * pi()) - 1) / 3 for x in f]
    elif kind == "yarn":
        lo = max(math.floor(dims[0]), 0)
        hi = min(math.ceil(dims[1]), r - 1)
        keep = [1 - Fraction(i - lo, hi - lo) for i in range(r // 2)]
    else:
        return f
    keep = [min(max(k, Fraction(0)), Fraction(1)) for k in keep]
    return [x / s * (1 - k) + x * k for x, k in zip(f, keep)]


@pytest.mark.parametrize("sc", [None, dict(type="linear", factor=2.5),
                                dict(type="ntk", factor=8.0), LLAMA, YARN],
                         ids=lambda s: s["type"] if s else "plain")
@pytest.mark.parametrize("r,base", [(128, 500000.0), (64, 10000.0),
                                    (20, 10000.0), (256, 1234.5)])
def test_turns(r, base, sc):
    """Every frequency is the nearest 64-bit fraction of a turn: half a unit,
    and as much again at position 2^40 as 2^40 halves of one."""
    rot = Rotary("cpu", rotary_dim=r, base=base, scaling=sc)
    f = exact(r, base, sc)
    tau = 2 * pi()
    for got, x in zip(rot.freq.tolist(), f):
        assert abs(got - x / tau * 2 ** 64) <= Fraction(1, 2) + Fraction(
            1, 10 ** 30)
        far = Fraction(got * (2 ** 40 - 1) % 2 ** 64, 2 ** 64)
        off = abs(far - x / tau * (2 ** 40 - 1) % 1)
        assert min(off, 1 - off) <= Fraction(2 ** 40, 2 ** 65)
    # fp64 to the nearest
    g, _ = rotary_frequencies(r, base, sc)
    assert g.dtype == torch.float64
    assert g.tolist() == [float(x) for x in f]


def test_numbers_of_other_types():
    want = Rotary("cpu", rotary_dim=64, base=500000.0,
                  scaling=dict(type="ntk", factor=4.0))
    for r, base, s in ((np.int64(64), np.float32(500000), np.int32(4)),
                       (64, 500000, 4), (64, torch.tensor(5e5), 4.0)):
        rot = Rotary("cpu", rotary_dim=r, base=base,
                     scaling=dict(type="ntk", factor=s))
        assert torch.equal(rot.freq, want.freq)
