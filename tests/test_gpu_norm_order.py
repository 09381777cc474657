"""The mean of a norm is added in one order whatever the number of rows, so that no code hangs on the batch.

r = fp32(1 / sqrt(mean + eps)) changes by a whole step where the 64-bit value lies next to the border between two
fp32 numbers and two orders of addition fall on its two sides.  Such rows are made here: random ones whose last
elements bring the exact sum of squares to that of a border, kept where two orders that a launch might take give two r.
"""
from fractions import Fraction

import numpy as np
import pytest

import mx
import tier_amd
from mx import MxRows
from rows import Rows, f32
from tier_amd import hip

F32 = tier_amd.F32
EPS = np.float32(1e-5)


def r_of(s, K):
    return np.float32(1.0 / np.sqrt(s / K + np.float64(EPS)))


def sum_by(x, threads, units):
    """The squares of a row added by `threads` lanes, each `units` groups of four in turn, lanes by halves, waves in turn."""
    q = np.zeros(threads * units * 4)
    q[:len(x)] = x.astype(np.float64) ** 2
    q = q.reshape(units, threads, 4)
    s = np.zeros(threads)
    for u in range(units):
        for i in range(4):
            s = s + q[u, :, i]
    s = s.reshape(-1, 64)
    while s.shape[1] > 1:
        h = s.shape[1] // 2
        s = s[:, :h] + s[:, h:]
    total = s[0, 0]
    for w in s[1:, 0]:
        total = total + w
    return total


def border_row(K, seed):
    """A row whose exact sum of squares is that of a border between two r, but for some 2^-60 of it."""
    rng = np.random.default_rng(seed)
    x = rng.standard_normal(K).astype(np.float32)
    at = rng.choice(K, 5, replace=False)
    x[at] = 0
    exact = sum(Fraction(float(v)) ** 2 for v in x)
    r = r_of(float(exact) * 1.003, K)
    border = (Fraction(float(r)) + Fraction(float(np.nextafter(r, np.float32(0))))) / 2
    left = (1 / border ** 2 - Fraction(float(EPS))) * K - exact
    for i in at:
        v = np.float32(np.sqrt(float(left)))
        if Fraction(float(v)) ** 2 > left:
            v = np.nextafter(v, np.float32(0))
        x[i] = v
        left -= Fraction(float(v)) ** 2
    return x


def border_rows(K, n):
    """n rows on which one unit a thread and two a thread disagree."""
    units, rows, seed = -(-K // 4), [], 0
    one, two = -(-units // 64) * 64, -(-units // 128) * 64
    while len(rows) < n:
        x, seed = border_row(K, seed), seed + 1
        assert seed < 60 * n
        if r_of(sum_by(x, one, 1), K) != r_of(sum_by(x, two, 2), K):
            rows.append(x)
    return np.array(rows)


def test_border_rows():
    """Such rows exist, and both r are next to each other."""
    for x in border_rows(1100, 3):
        a, b = r_of(sum_by(x, 320, 1), 1100), r_of(sum_by(x, 192, 2), 1100)
        assert a != b and np.nextafter(a, b) == b


@pytest.mark.gpu
@pytest.mark.parametrize("K", [1100, 4000])
def test_r_and_codes_do_not_depend_on_the_number_of_rows(gpu, K):
    """Twelve such rows alone, among some and among many: r, y, int8 and microscaled codes bit for bit."""
    x = border_rows(K, 12)
    g = f32(1 + 0.2 * np.random.default_rng(1).standard_normal(K))
    rb = tier_amd.i8_row_bytes(K)

    def outputs(M):
        X, Y = Rows(F32, M, K, np.resize(x, (M, K))), Rows(F32, M, K)
        Q, S, R, C = hip.DeviceBuffer(M * rb), f32(np.zeros(M)), f32(np.zeros(M)), MxRows(mx.E4M3, M, K)
        tier_amd.rms_norm(X.ptr, F32, K, None, 0, g.ptr, EPS, None, 0, Y.ptr, K, Q.ptr, rb, S.ptr, R.ptr, M, K)
        R2 = f32(np.zeros(M))
        tier_amd.rms_norm_mx(X.ptr, F32, K, None, 0, g.ptr, EPS, None, 0, None, 0, mx.E4M3, C.q.ptr, C.rb, C.s.ptr, C.sb,
                             R2.ptr, M, K)
        R3 = f32(np.zeros(M))
        tier_amd.rms_norm(X.ptr, F32, K, None, 0, g.ptr, EPS, None, 0, None, 0, None, 0, None, R3.ptr, M, K)
        hip.synchronize()
        c, s = C.get()
        assert np.array_equal(R.download(np.float32), R2.download(np.float32))
        assert np.array_equal(R.download(np.float32), R3.download(np.float32))
        return R.download(np.float32), Y.bits(), Q.download(np.int8).reshape(M, rb), S.download(np.float32), c, s

    few = outputs(12)
    exact = np.array([r_of(sum_by(v, -(-K // 256) * 64, 1), K) for v in x])
    assert (np.abs(few[0].view(np.int32) - exact.view(np.int32)) <= 1).all()
    for M in (516, 600):
        for a, b in zip(few, outputs(M)):
            assert np.array_equal(b, np.resize(a, (M,) + a.shape[1:]))
    one = outputs(1)
    for a, b in zip(few, one):
        assert np.array_equal(a[:1], b)
