"""fp32 queries over an fp16 cache, cut so that a result shows every bit of them.

A row sees two keys, e_0 of value 1 and e_1 of value -1 (all others score -1000: no weight), with scores ``base`` and
base - x, x a multiple of ``step`` up to 2^-3: 512 and 2^-14, or 0.75 and 2^-24, so that a query has 24 bits. The output is

    (w0 - w1) / (w0 + w1) = (1 - 2^-x) / (1 + 2^-x),     w0 = 1, w1 = 2^-x in units of the largest

The scores are products with 1, so exact as long as the query is, and so is the exponential's argument, -x, in fp32 (not so
that of a weight that is made larger by its exponent: 14 - x has steps of 2^-20). In fp32, w1 is off by an ulp of the
exponential, 2^-24 below 1; the numerator's terms are exact, multiples of 2^-24; the sum and the quotient are rounded once
each. d out / d w1 is -2 / (1 + w1)^2, so the output is off by 2^-24 (2 / (1 + w1)^2 + 2 out) at most.

A weight received is 2^(score - lse), lse = base + log2(1 + w1) rounded to 24 bits: its exponent is off by half a step of
that (2^-15, or 2^-24), the logarithm's 2^-22 and the exponential's ulp.

The kernels split such values into three fp16 planes of 11 bits; a lost one shows: the third of the query is 2^-14 of a
score of 512, 4e-5 of a weight, where x is an odd multiple, the third of a weight up to 3 times 2^-24."""
import math

import torch

SCALE = math.log(2.0)                  # a score is the query's value in powers of 2 ...
assert torch.tensor(1.4426950408889634 * SCALE).item() == 1.0      # ... without a rounding


BASES = {512.0: 2.0 ** -14, 0.75: 2.0 ** -24}                       # a base and its step


def gaps(n, seed, base):
    """n odd multiples of the base's step up to 2^-3."""
    gen = torch.Generator().manual_seed(seed)
    most = int(2.0 ** -3 / BASES[base])
    return (2 * torch.randint(0, most // 2, (n,), generator=gen).double() + 1) * BASES[base]


def answer(x, base):
    """The output, its bound; the weights received by e_0 and e_1, their relative bound (of one row)."""
    w = torch.exp2(-x)
    out = -torch.expm1(-x * math.log(2.0)) / (1 + w)
    lse = 2.0 ** -15 if base == 512.0 else 2.0 ** -24
    return out, 2.0 ** -24 * (2 / (1 + w) ** 2 + 2 * out), 1 / (1 + w), w / (1 + w), \
        (lse + 2.0 ** -22) * math.log(2.0) + 2.0 ** -23


def cut(v, keep):
    """The value that the first ``keep`` of the planes of fp32 values hold."""
    out, rest = torch.zeros_like(v), v
    for _ in range(keep):
        m, e = torch.frexp(rest)
        part = torch.ldexp(torch.trunc(m * 2048.0) / 2048.0, e)
        out, rest = out + part, rest - part
    return out


def emulate(x, base, query_planes, weight_planes, bias=0):
    """The output as the kernels make it, of so many planes, weights by 2^bias larger by their exponents."""
    top, low = (cut(torch.full_like(x, base), query_planes), cut(base - x, query_planes))
    w0, w1 = (torch.exp2((s - (base - bias)).float().double()).float().double() for s in (top, low))
    return ((cut(w0, weight_planes) - cut(w1, weight_planes)) / (w0 + w1).float().double()).float().double()
