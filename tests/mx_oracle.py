"""The microscaled 4-bit format and its experts in numpy, in 64 bits: the
definition that the kernels are tested against."""

from __future__ import annotations

import numpy as np

E2M1 = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6], np.float64)
VALUES = np.concatenate([E2M1, -E2M1])


def quantize(w):
    """float64 [R, C] (C a multiple of 32) -> (codes uint8 [R, C], scales
    uint8 [R, C/32]), by search over the eight magnitudes."""
    w = np.asarray(w, np.float64)
    g = w.reshape(w.shape[0], -1, 32)
    finite = np.isfinite(g).all(-1)
    top = np.where(finite, np.abs(np.where(np.isfinite(g), g, 0)).max(-1), 0)
    _, e = np.frexp(top)
    s = np.where(top > 0, np.clip(e - 1 - 2, -127, 127), -127)
    a = np.abs(np.where(finite[..., None], g, 0)) / np.exp2(s.astype(np.float64))[..., None]
    dist = np.abs(a[..., None] - E2M1)
    # nearest; of two equally near the one with an even mantissa bit (even index)
    order = dist * 4 + (np.arange(8) % 2) * 1e-9
    code = order.argmin(-1).astype(np.uint8) | (np.signbit(g).astype(np.uint8) << 3)
    code[~finite] = 0
    scales = np.where(finite, s + 127, 255).astype(np.uint8)
    return code.reshape(w.shape), scales


def pack(codes):
    c = codes.astype(np.uint32).reshape(codes.shape[0], -1, 8)
    return (c << (4 * np.arange(8, dtype=np.uint32))).sum(-1, dtype=np.uint64).astype(np.uint32)


def unpack(words):
    c = (words[..., None] >> (4 * np.arange(8, dtype=np.uint32))) & 15
    return c.reshape(words.shape[0], -1).astype(np.uint8)


def dequant(codes, scales):
    """float64 values of codes [R, C] and scales [R, C/32]."""
    unit = np.exp2(scales.astype(np.float64) - 127)
    unit = np.where(scales == 255, np.nan, unit)
    v = VALUES[codes].reshape(codes.shape[0], -1, 32) * unit[..., None]
    return v.reshape(codes.shape)


def group_max(v):
    """The largest magnitude of each value's group of 32."""
    g = np.abs(v.reshape(*v.shape[:-1], -1, 32)).max(-1, keepdims=True)
    return np.broadcast_to(g, (*g.shape[:-1], 32)).reshape(v.shape)


def ffn(x, gate, up, down):
    """(y, bound): the expert on rows x [m, hidden] in 64 bits, and how far
    the kernel's fp32 value may be off before it is rounded to bf16.

    An activation is held to 2^-10 of its group's largest: it is bf16, and exact
    in two pieces where it is an eighth of the largest and more.  An intermediate
    is held to 2^-8 of its group's largest M: with 2^e the group's unit and M in
    [3.875, 7.75) 2^e, the second piece (unit 2^(e-5), steps of 1/8, 1/4, 1/2 up
    to 7.5) leaves 2^-10, 2^-9 and 2^-8 2^e of rests of up to 1/16, 1/8 and 15/64
    2^e, and 1/4 - 15/64 = 2^-6 2^e of a rest of 1/4 2^e, which only a value of
    4 2^e and more leaves, so that M is 4 2^e too.  The sums are fp32, off by at most one rounding
    for each of the reduction's 128-wide steps and pieces and the waves' sums
    (under 2^-16 of the sum of magnitudes); silu's derivative is below 1.1, its
    fp32 value is off by under 2^-20."""
    g, u = x @ gate.T, x @ up.T
    dx = 2.0 ** -10 * group_max(x)
    ax = np.abs(x) * 2.0 ** -16 + dx
    dg, du = ax @ np.abs(gate).T, ax @ np.abs(up).T
    with np.errstate(over="ignore"):
        sg = g / (1 + np.exp(-g))
    h = sg * u
    dh = 1.1 * dg * (np.abs(u) + du) + np.abs(sg) * du + 2.0 ** -20 * np.abs(h)
    ah = dh + 2.0 ** -8 * group_max(np.abs(h) + dh) + 2.0 ** -16 * np.abs(h)
    return h @ down.T, ah @ np.abs(down).T
