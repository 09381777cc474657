"""Microscaled products keep the bits of every product of two elements, whatever the output's type.

A product of E4M3 and E2M1 elements has 6 significant bits, and the fp32 sum of a block's products loses nothing
but what its additions round: at most 8 of them for each block of 32 (as in test_gpu_mx.py), each by 2^-23 of what the
sum's magnitudes add up to.  The bias adds one rounding and the output its own.  In particular no result may
depend on how far apart neighbouring elements lie.
"""
import numpy as np
import pytest

import mx
import tier_amd
from mx import E2M1, E4M3, MxRows
from rows import TINY, UNIT, Rows, f32, to_bits
from test_gpu_mx_tiles import SIZES, some_rows
from tier_amd import hip

pytestmark = pytest.mark.gpu
F32, F16, BF16 = tier_amd.F32, tier_amd.F16, tier_amd.BF16


def check_kept(got, t, x, w, bias=None):
    """got against x w^T + bias within the bound of the header comment."""
    want, mag = x @ w.T, np.abs(x) @ np.abs(w).T
    b = np.zeros(w.shape[0]) if bias is None else bias.astype(np.float64)
    err = 8 * -(-x.shape[1] // 32) * 2.0 ** -23 * mag + 2.0 ** -24 * (mag + np.abs(b))
    want = want + b
    dead = np.isnan(want)
    assert np.isnan(got[dead]).all() and np.isfinite(got[~dead]).all()
    ok = np.abs(got - want) <= err + UNIT[t] * (np.abs(want) + err) + TINY[t]
    assert ok[~dead].all(), (np.argwhere(~ok & ~dead)[:5], np.nanmax(np.abs(got - want) / np.maximum(mag, 1e-300)))


def cancelling_block(M, seed):
    """E4M3 codes of one block a row: the largest number and its negative, small ones and some between.  With weights
    of one magnitude every sum is a whole number of 2^-10 below 2^13, which fp32 holds."""
    rng = np.random.default_rng(seed)
    c = np.zeros((M, 32), np.int64)
    for r in range(M):
        p = rng.permutation(32)
        c[r, p[:2]] = 0x7e, 0xfe
        c[r, p[2:8]] = rng.integers(1, 0x30, 6)
        c[r, p[8:14]] = rng.integers(0x30, 0x58, 6) & 0xf8
    return c


@pytest.mark.parametrize("t", (F32, F16, BF16))
@pytest.mark.parametrize("M,N", [(1, 150), (2, 150), (1, 5300), (2, 5300), (30, 150), (140, 150), (600, 3000)])
def test_a_block_is_exact(gpu, t, M, N):
    """Through mx_gemm and, from numbers that the codes stand for, through mx_linear: the exact sum, rounded once."""
    c, K = cancelling_block(M, M), 32
    wc = np.zeros((N, K), np.int64)
    wc[:] = np.random.default_rng(N).integers(1, 8, (N, 1))
    x, w = mx.numbers(E4M3, c), mx.numbers(E2M1, wc)
    assert ((np.abs(x) @ w.T) < 2.0 ** 13).all()
    X, W = MxRows(E4M3, M, K, c, np.full((M, 1), 127)), MxRows(E2M1, N, K, wc, np.full((N, 1), 127))
    want = to_bits(t, (x @ w.T).astype(np.float32))
    Y = Rows(t, M, N)
    tier_amd.mx_gemm(X.q.ptr, E4M3, X.rb, X.s.ptr, X.sb, W.q.ptr, W.rb, W.s.ptr, W.sb, None, Y.ptr, t, N, M, N, K)
    hip.synchronize()
    assert np.array_equal(Y.bits(), want)
    V, Y = Rows(F32, M, K, x), Rows(t, M, N)
    tier_amd.mx_linear(V.ptr, F32, K, E4M3, W.q.ptr, W.rb, W.s.ptr, W.sb, None, Y.ptr, t, N, M, N, K)
    hip.synchronize()
    assert np.array_equal(Y.bits(), want)


def random_codes(fmt, rows, K, seed, lo, hi):
    rng = np.random.default_rng(seed)
    c = rng.integers(0, 1 << fmt, (rows, K), dtype=np.uint8)
    if fmt == E4M3:
        c = np.where(c & 127 == 127, np.uint8(5), c)
    return c, rng.integers(lo, hi, (rows, -(-K // 32)))


@pytest.mark.parametrize("K", [100, 1100])
@pytest.mark.parametrize("M,N", SIZES + [(3, 70), (40, 10001), (33, 5000)])
def test_16_bit_outputs_of_every_tile(gpu, M, N, K):
    """E4M3 elements of every size side by side."""
    wc, ws = random_codes(E2M1, N, K, N + K, 114, 122)
    c, s = random_codes(E4M3, M, K, M + K, 114, 122)
    W, w = MxRows(E2M1, N, K, wc, ws), mx.values(E2M1, wc, ws)
    X, pick = MxRows(E4M3, M, K, c, s), some_rows(M, N)
    x = mx.values(E4M3, c[pick], s[pick])
    bias = np.random.default_rng(1).standard_normal(N).astype(np.float32)
    for t in (F16, BF16):
        Y = Rows(t, M, N, pad=1, skip=1)
        tier_amd.mx_gemm(X.q.ptr, E4M3, X.rb, X.s.ptr, X.sb, W.q.ptr, W.rb, W.s.ptr, W.sb, f32(bias).ptr, Y.ptr, t, Y.ld, M, N, K)
        hip.synchronize()
        check_kept(Y.values()[pick], t, x, w, bias)
        assert Y.outside_kept()
