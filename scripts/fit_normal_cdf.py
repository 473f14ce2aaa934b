#!/usr/bin/env python3
"""Coefficients of the normal distribution in rebel_amd/csrc/layer_norm_kernel.h: Phi(-x) = exp(-x^2 / 2) P(x), P(x) = u poly(u),
u = 1 / (1 + a x), fitted to the least relative error of P on [0, 14] (reweighted least squares).  Prints, for each degree, the best a,
the error in exact arithmetic and with every step rounded to f32, and the coefficients from u^1 up."""
import numpy as np
from scipy.special import erfcx


def fit(a, degree, end=14.0):
    k = np.arange(6000)
    x = np.concatenate([end * (1 - np.cos(np.pi * (k + 0.5) / 6000)) / 2, np.linspace(0, 4, 6000)])
    want = erfcx(x / np.sqrt(2)) / 2
    u = 1 / (1 + a * x)
    basis = np.stack([u ** (j + 1) for j in range(degree)], 1) / want[:, None]
    weight = np.ones_like(x)
    for _ in range(200):
        c = np.linalg.lstsq(basis * weight[:, None], weight, rcond=None)[0]
        off = np.abs(basis @ c - 1)
        weight *= (off / off.max() + 1e-3) ** 0.25
        weight /= weight.max()
    return c, off.max()


for degree in (6, 7, 8, 9):
    a = min(np.linspace(0.15, 0.6, 19), key=lambda v: fit(v, degree)[1])
    c, off = fit(a, degree)
    f = np.float32
    x = np.linspace(0, 14, 200001).astype(f)
    u = f(1) / (f(1) + f(a) * x)
    p = np.full_like(x, f(c[-1]))
    for v in c[-2::-1]:
        p = (p.astype(np.float64) * u + f(v)).astype(f)
    p = p * u
    want = erfcx(x.astype(np.float64) / np.sqrt(2)) / 2
    print(degree, "a %.3f" % a, "relative error %.2e, in f32 %.2e" % (off, np.abs(p / want - 1).max()), ", ".join("%.9e" % v for v in c))
