"""The inputs and tolerances of test_paged_precision_gpu.py on the CPU: what
they are said to be holds, and a mistake planted in a model of the arithmetic
is seen."""
from __future__ import annotations

import numpy as np
import pytest

import paged_precision as pp


@pytest.mark.parametrize("hd", [32, 64, 128])
def test_a_lost_part_of_q_is_seen(hd):
    """Three bf16 terms are all of q; with the third one lost, of q or of the
    scaled q, the result is off by more than the tolerance."""
    rng = np.random.default_rng(hd)
    q = pp.coherent_queries(rng, 16, hd)
    assert np.array_equal(pp.terms(q, 3), q.astype(np.float64))
    part = np.cumsum(q.astype(np.float64) * pp.key(hd), -1)
    assert np.abs(part).max() <= (np.abs(q) * pp.AMP).sum(-1).min() * 4 / hd
    right = pp.two_key_result(q, 500, 500)
    assert np.abs(right).max() < 0.95                    # the result moves with the scores
    tol = pp.two_key_tolerance(hd, "bf16")
    lost = pp.two_key_result(pp.terms(q, 2), 500, 500)
    sl2 = pp.scale_log2(hd)
    scaled = pp.two_key_result(pp.terms((q * sl2).astype(np.float32), 2) / np.float64(sl2), 500, 500)
    assert np.median(np.abs(lost - right)) > 1.5 * tol
    assert np.median(np.abs(scaled - right)) > 1.5 * tol
    kept = pp.two_key_result(pp.terms((q * sl2).astype(np.float32), 3) / np.float64(sl2), 500, 500)
    assert np.abs(kept - right).max() < tol / 4


def test_a_truncating_accumulator_is_seen():
    """sum p v with v = 1, gathered over all chunks by an accumulator that
    truncates, is off by more than the tolerance; each chunk added in binary32
    to nearest is not."""
    rng = np.random.default_rng(0)
    chunks = 1024
    p = np.exp2(-4 * rng.random((chunks, 6))).astype(np.float32) * 16   # a chunk's six products
    trunc, near, l = np.float64(0), np.float32(0), np.float32(0)
    for c in range(chunks):
        for x in p[c]:
            s = trunc + np.float64(x)
            ulp = 2.0 ** (np.floor(np.log2(s)) - 23)
            trunc = np.floor(s / ulp) * ulp
        near = np.float32(near + np.float32(p[c].sum()))
        l = np.float32(l + np.float32(p[c].sum()))
    exact = p.astype(np.float64).sum()
    tol = pp.chain_tolerance(chunks)
    assert abs(trunc / exact - 1) > 4 * tol
    assert abs(np.float64(near) / l - 1) <= tol and abs(near / exact - 1) <= tol


def test_a_lost_or_doubled_row_is_seen():
    """Counts of random bits: a row, a chunk or a page left out or taken twice
    moves some dimension by far more than the rounding of a quotient."""
    rng = np.random.default_rng(1)
    n, hd = 100_003, 64
    v = rng.integers(0, 2, (n, hd)).astype(np.float64)
    right, tol = v.mean(0), 2.0 ** -22
    for at, rows in ((0, 1), (5000, 1), (n - 1, 1), (32 * 77, 32), (16 * 100, 16), (0, 2048)):
        out = np.delete(v, np.s_[at:at + rows], 0).mean(0)
        twice = np.concatenate([v, v[at:at + rows]]).mean(0)
        assert (np.abs(out / right - 1) > 8 * tol).any(), rows
        assert (np.abs(twice / right - 1) > 8 * tol).any(), rows
