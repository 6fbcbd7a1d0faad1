"""fp32 queries over an fp16 cache, cut so that a result shows every bit of them.

A row sees two keys, e_0 of value 1 and e_1 of value -1 (all other keys are 0, their weights 2^-512 of the largest), with
scores 512 and 512 - x, x a multiple of 2^-14 up to 2^-3: 24 bits of the query. The output is

    (w0 - w1) / (w0 + w1) = (1 - 2^-x) / (1 + 2^-x),     w0 = 1, w1 = 2^-x in units of the largest

The scores are products with 1, so exact as long as the query is, and so is the exponential's argument. In fp32, w1 is off
by an ulp of the exponential, 2^-24 below 1; the numerator's terms are exact, multiples of 2^-24; the sum and the quotient
are rounded once each. d out / d w1 is -2 / (1 + w1)^2, so the output is off by 2^-24 (2 / (1 + w1)^2 + 2 out) at most.

A weight received is 2^(score - lse), lse = 512 + log2(1 + w1) rounded to 24 bits: its exponent is off by 2^-15, the
logarithm's 2^-22 and the exponential's ulp.

The kernels split such values into three fp16 planes of 11 bits; a lost one shows: the third of the query is 2^-14 of the
score, 4e-5 of a weight, where x is an odd multiple, the third of a weight up to 3 times 2^-24."""
import math

import torch

SCALE = math.log(2.0)                  # a score is the query's value in powers of 2 ...
assert torch.tensor(1.4426950408889634 * SCALE).item() == 1.0      # ... without a rounding


def gaps(n, seed):
    """n odd multiples of 2^-14 up to 2^-3."""
    gen = torch.Generator().manual_seed(seed)
    return (2 * torch.randint(0, 1024, (n,), generator=gen).double() + 1) * 2.0 ** -14


def answer(x):
    """The output, its bound; the weights received by e_0 and e_1, their relative bound (of one row)."""
    w = torch.exp2(-x)
    out = -torch.expm1(-x * math.log(2.0)) / (1 + w)
    return out, 2.0 ** -24 * (2 / (1 + w) ** 2 + 2 * out), 1 / (1 + w), w / (1 + w), \
        (2.0 ** -15 + 2.0 ** -22) * math.log(2.0) + 2.0 ** -23


def cut(v, keep):
    """The value that the first ``keep`` of the planes of fp32 values hold."""
    out, rest = torch.zeros_like(v), v
    for _ in range(keep):
        m, e = torch.frexp(rest)
        part = torch.ldexp(torch.trunc(m * 2048.0) / 2048.0, e)
        out, rest = out + part, rest - part
    return out


def emulate(x, query_planes, weight_planes):
    """The output as the kernels make it, of so many planes."""
    gap = 512.0 - cut((512.0 - x) / 1024.0, query_planes) * 1024.0
    w = torch.exp2(-gap).float().double()
    return ((1.0 - cut(w, weight_planes)) / (1.0 + w).float().double()).float().double()
