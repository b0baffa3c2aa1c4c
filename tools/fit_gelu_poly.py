#!/usr/bin/env python
"""Coefficients of the polynomial GELU used by the GEMM epilogues (vitpose_amd/csrc/common.h).

gelu(x)  = (x + |x|) / 2 - h(|x|),          h(a) = a erfc(a / sqrt 2) / 2
gelu'(x) = 1/2 + copysign(1/2 - d(|x|), x), d(a) = h'(a) = erfc(a / sqrt 2) / 2 - a phi(a)
h and d are smooth and decay like a Gaussian; on [0, A] each is fitted by a degree-DEG polynomial in
s = 2 a / A - 1 (Chebyshev least squares on a dense grid, converted to the monomial basis, whose
coefficients stay below 2 in magnitude on [-1, 1]), and a is clamped to A beyond.  The script prints the
coefficients and the maximum absolute error of the float32 Horner evaluation against scipy's erfc.

Then the form of vitpose_amd/csrc/fp8.hip, whose error goes by the result: h(a) = exp(-a^2 / 2) s P(s), s = a / (a + 4.25), P of
degree 7 fitted to the least largest RELATIVE error on [0, 14.5] (least squares, weights multiplied by the error each round)."""
import numpy as np
from numpy.polynomial import Polynomial, chebyshev as C
from scipy.special import erfc, erfcx, ndtr

A, DEG = 4.5, 11


def h(a):
    return a * erfc(a / np.sqrt(2)) / 2


def d(a):
    return erfc(a / np.sqrt(2)) / 2 - a * np.exp(-a * a / 2) / np.sqrt(2 * np.pi)


def horner32(mono, s):
    acc = np.full_like(s, np.float32(mono[-1]))
    for k in mono[-2::-1]:
        acc = acc * s + np.float32(k)
    return acc


def relative(c=4.25, far=14.5, degree=7, rounds=200):
    top = far / (far + c)
    s = top * (0.5 - 0.5 * np.cos(np.pi * (np.arange(6000) + 0.5) / 6000))
    a = c * s / (1 - s)
    g = a * erfcx(a / np.sqrt(2)) / 2 / s
    v, weight, best = C.chebvander(2 * s / top - 1, degree), np.ones_like(s), (np.inf, None)
    for _ in range(rounds):
        root = np.sqrt(weight)
        co = np.linalg.lstsq(v / g[:, None] * root[:, None], root, rcond=None)[0]
        e = np.abs(v @ co / g - 1)
        best = min(best, (e.max(), co), key=lambda b: b[0])
        weight = weight * e / (weight * e).sum()
    mono = Polynomial(C.cheb2poly(best[1]))(Polynomial([-1, 2 / top])).coef
    print(f'// P: degree {degree} in s = a / (a + {c}), highest power first; max relative error of the fit {best[0]:.2e}')
    print('{' + ', '.join(f'{k:.9e}f' for k in mono[::-1]) + '}')
    x = np.concatenate([np.linspace(-11, 6, 400001), -np.logspace(-25, 0, 50000)]).astype(np.float32)
    t = np.minimum(np.abs(x), np.float32(far))
    sx = t * (np.float32(1) / (t + np.float32(c)))
    p = horner32(mono, sx) * sx * np.exp2(t * t * np.float32(-0.5 / np.log(2)))
    got = (np.float32(0.5) * np.abs(x) + np.float32(0.5) * x - p).astype(np.float64)
    ref = x.astype(np.float64) * ndtr(x.astype(np.float64))
    for lo, hi in ((0, 3), (3, 6), (6, 11)):
        at = (np.abs(x) >= lo) & (np.abs(x) <= hi) & (x != 0)
        print(f'// max relative error, {lo} <= |x| <= {hi}: {np.abs(got / np.where(ref == 0, 1, ref) - 1)[at].max():.2e}')


def main():
    a = np.linspace(0, A, 20001)
    s = 2 * a / A - 1
    x = np.linspace(-9, 9, 400001).astype(np.float32)
    ax = np.minimum(np.abs(x), np.float32(A))
    sx = ax * np.float32(2 / A) - np.float32(1)
    for name, f in (('H', h), ('D', d)):
        mono = C.cheb2poly(C.chebfit(s, f(a), DEG))
        print(f'// {name}: degree {DEG} in s = 2 a / {A} - 1, highest power first')
        print('{' + ', '.join(f'{c:.9e}f' for c in mono[::-1]) + '}')
        p = horner32(mono, sx).astype(np.float64)
        xd = x.astype(np.float64)
        if name == 'H':
            got = 0.5 * (xd + np.abs(xd)) - p
            ref = xd * (1 - erfc(xd / np.sqrt(2)) / 2)
        else:
            got = 0.5 + np.copysign(0.5 - p, xd)
            ref = (1 - erfc(xd / np.sqrt(2)) / 2) + xd * np.exp(-xd * xd / 2) / np.sqrt(2 * np.pi)
        print(f'// max |error| on [-9, 9]: {np.abs(got - ref).max():.2e}')


if __name__ == '__main__':
    main()
    relative()
