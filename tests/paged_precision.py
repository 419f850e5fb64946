"""Inputs of the paged cache whose results show single bits of the arithmetic
and single rows, and what each is allowed to be off by; used on the CPU (where
mistakes are planted in a model of the arithmetic) and on the GPU."""
from __future__ import annotations

import math

import numpy as np

AMP = 25.0                     # |k| of the two-key inputs, exact in bf16 and tf32


def bf16(x):
    """Round to nearest even bf16."""
    u = np.asarray(x, np.float32).view(np.uint32)
    return ((u + 0x7fff + ((u >> 16) & 1)) & np.uint32(0xffff0000)).view(np.float32)


def terms(x, n):
    """x as the sum of its first n bf16 terms, each rounded from what those
    before it leave."""
    x = np.asarray(x, np.float32)
    rest, total = x.copy(), np.zeros(x.shape, np.float64)
    for _ in range(n):
        t = bf16(rest)
        total += t
        rest = (rest - t).astype(np.float32)
    return total


def scale_log2(hd):
    return np.float32(1.4426950408889634 / np.float32(math.sqrt(hd)))


def coherent_queries(rng, heads, hd):
    """[heads, hd] queries in [1, 1.05) for which two bf16 terms leave a
    remainder of one sign in the even dimensions and of the other in the odd
    ones, of q itself and of q * log2(e) / sqrt(hd) (kernels split either)."""
    found = {1: [], -1: []}
    need = heads * hd // 2
    while min(len(v) for v in found.values()) < need:
        x = (1 + 0.05 * rng.random(1 << 18)).astype(np.float32)
        y = (x * scale_log2(hd)).astype(np.float32)
        rx, ry = (a.astype(np.float64) - terms(a, 2) for a in (x, y))
        for sign in found:
            ok = (sign * rx > 0.6 * 2.0 ** -17) & (sign * ry / y > 0.25 * 2.0 ** -17)
            found[sign].extend(x[ok].tolist())
    q = np.zeros((heads, hd), np.float32)
    q[:, 0::2] = np.reshape(found[1][:need], (heads, hd // 2))
    q[:, 1::2] = np.reshape(found[-1][:need], (heads, hd // 2))
    return q


def key(hd):
    """The first of the two keys; the other is its negative."""
    k = np.full(hd, AMP, np.float32)
    k[1::2] = -AMP
    return k


def two_key_result(q, plus, minus):
    """Attention over `plus` rows of key() with value 1 and `minus` rows of
    -key() with value -1, in 64 bits: one number per head."""
    s = np.asarray(q, np.float64) @ key(q.shape[-1]).astype(np.float64) / math.sqrt(q.shape[-1])
    a, b = plus * np.exp(s), minus * np.exp(-s)
    return (a - b) / (a + b)


def two_key_tolerance(hd, dtype):
    """Off by at most this.  The difference D of the two scores moves the
    result by |dD| / 2 at most.  A, the sum of |q k| / sqrt(hd), is below
    1.05 * 25 * sqrt(hd); products and partial sums of a score stay below
    4 A / hd (checked on the CPU).  A tensor-core step (hd / 16 for each of
    three parts of q, and one to join them) cuts each of its 17 addends at
    2^-24 of the largest: less than 2^-20 * 4 A / hd, for two scores.  fp32
    rows: q as two tf32 leaves less than 1.5 * 2^-22 of it, and a step has 8
    dimensions of four products.  ex2, the weights (two bf16 of a shared
    prefix: 2^-17), sums and the division: 2^-16 with room."""
    a = 1.05 * AMP * math.sqrt(hd)
    steps = 3 * hd / 16 + 1 if dtype == "bf16" else 4 * hd / 8 + 1
    left = 0.0 if dtype == "bf16" else 1.5 * 2.0 ** -22
    return 0.5 * 2 * a * (steps * 2.0 ** -20 * 4 / hd + left) + 2.0 ** -16


def chain_tolerance(chunks, steps=0):
    """sum p / sum p of a stream whose warps add `chunks` chunks one after the
    other, in binary32 to nearest in both sums: 2 * chunks roundings of at most
    2^-24 that have no common sign, eight standard deviations of them; a
    chunk's own products (6 steps) and parts of the weights 2^-20; `steps`
    tensor-core steps of a shared prefix that one accumulator gathers, each cut
    at 2^-23 of it."""
    return 8 * math.sqrt(2 * chunks) * 2.0 ** -24 + 2.0 ** -20 + steps * 2.0 ** -23
