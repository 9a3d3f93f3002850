"""rotary_frequencies between its plain and its divided pairs, against its definition in decimals of 50 places."""
import decimal
import itertools

import pytest

D = decimal.Decimal


def _yarn(rot, base, factor, window):
    """Pair by pair: its turns in the window decide, and between the whole indexes around 32 turns and one the index itself."""
    with decimal.localcontext(decimal.Context(prec=50)):
        pi = D("3.14159265358979323846264338327950288419716939937511")
        base, factor, window = D(base), D(factor), D(window)
        plain = [(base.ln() * (D(-2 * i) / rot)).exp() for i in range(rot // 2)]

        def index(turns):  # real i with window base^(-2 i / rot) = 2 pi turns
            return (window / (2 * pi * turns)).ln() * rot / (2 * base.ln())
        lo = index(32).to_integral_value(decimal.ROUND_FLOOR)
        hi = index(1).to_integral_value(decimal.ROUND_CEILING)
        out = []
        for i, f in enumerate(plain):
            turns = window * f / (2 * pi)
            keep = D(1) if turns >= 32 else D(0) if turns <= 1 else 1 - (i - lo) / (hi - lo)
            out.append(f * (keep + (1 - keep) / factor))
        return [float(x) for x in out], float(1 + factor.ln() / 10)


@pytest.mark.parametrize("rot,base", [(128, 10000), (64, 500), (256, 1000000), (2, 10000), (6, 10000), (128, 12), (64, 1.5)])
def test_yarn(rot, base):
    import h3mi
    for factor, window in itertools.product((1.5, 16, 64), (1, 6.2, 7, 100, 201, 202, 600, 4096, 8192, 131072)):
        f, amplitude = h3mi.rotary_frequencies(rot, base=base, scaling="yarn", factor=factor, window=window, device="cpu")
        want, amp = _yarn(rot, base, factor, window)
        # base^e: e's rounding counts by e ln base, below 14, and a few roundings more.  What is kept is a number of 0 to 1, off by
        # three roundings of half that grain at most, and so is the factor that it makes, which is 1 / factor at least.
        assert all(abs(a - b) <= (20 + 2 * factor) * 2.0 ** -53 * b for a, b in zip(f.tolist(), want)), (factor, window)
        assert abs(amplitude - amp) <= 4 * 2.0 ** -53 * amp


def test_yarn_at_128_elements():
    """The numbers of 16 times 8192 tokens, base 10000: pairs 26 to 49 are between."""
    import h3mi
    f = h3mi.rotary_frequencies(128, scaling="yarn", factor=16.0, device="cpu")[0]
    plain = h3mi.rotary_frequencies(128, device="cpu")[0]
    part = (f / plain - 1 / 16) / (1 - 1 / 16)
    want = [1.0] * 26 + [(50 - i) / 25 for i in range(26, 50)] + [0.0] * 14
    assert all(abs(a - b) < 1e-12 for a, b in zip(part.tolist(), want))


@pytest.mark.parametrize("kw", [dict(window=float("inf")), dict(window=float("nan")), dict(window=-1), dict(factor=float("nan")), dict(base=float("inf"))])
def test_refusals(kw):
    import h3mi
    with pytest.raises(ValueError):
        h3mi.rotary_frequencies(128, **{"scaling": "yarn", "factor": 4.0, "device": "cpu", **kw})
