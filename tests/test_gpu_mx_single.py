"""A microscaled linear of one or two tokens: every form of its own kernel, which quantizes x by itself.

Rows of more pieces of 2048 elements than are in flight at once (K past 6144), both kinds of workgroup (5120 columns
and fewer), every output type, odd strides, a bias, and blocks of x that are NaN, infinite or zero.  Bounds as in
test_gpu_mx_bits.py.
"""
import functools

import numpy as np
import pytest

import mx
import tier_amd
from mx import E2M1, FORMATS, MxRows
from rows import TYPES, Rows, f32
from test_gpu_mx_bits import check_kept, random_codes
from tier_amd import hip

pytestmark = pytest.mark.gpu
F32, F16, BF16 = tier_amd.F32, tier_amd.F16, tier_amd.BF16


@functools.lru_cache(maxsize=1)
def weight(N, K):
    c, s = random_codes(E2M1, N, K, N + K, 115, 120)
    return MxRows(E2M1, N, K, c, s, pad=N % 2), mx.values(E2M1, c, s)


def linear(X, fmt, W, t, bias=None):
    """mx_linear of X; the values of Y, whose rows are three elements longer than they need be."""
    M, N, K = X.rows, W.rows, X.cols
    Y = Rows(t, M, N, pad=3, skip=1)
    tier_amd.mx_linear(X.ptr, X.t, X.ld, fmt, W.q.ptr, W.rb, W.s.ptr, W.sb, None if bias is None else f32(bias).ptr,
                       Y.ptr, t, Y.ld, M, N, K)
    hip.synchronize()
    assert Y.outside_kept()
    return Y.values()


@pytest.mark.parametrize("N,K", [(33, 6200), (33, 14336), (5119, 2100), (5120, 2100), (5300, 6200), (5300, 12401)])
@pytest.mark.parametrize("M", [1, 2])
@pytest.mark.parametrize("fmt", FORMATS)
def test_every_form(gpu, fmt, M, N, K):
    W, w = weight(N, K)
    rng = np.random.default_rng(M + K)
    x, bias = rng.standard_normal((M, K)).astype(np.float32), rng.standard_normal(N).astype(np.float32)
    x[:, 5::53] *= 9
    for i, t in enumerate(TYPES):
        for b in (None, bias):
            X = Rows(TYPES[(i + (b is None)) % 3], M, K, x, pad=1, skip=1)
            c, s = mx.quantize(fmt, X.values())
            check_kept(linear(X, fmt, W, t, b), t, mx.values(fmt, c, s), w, b)


@pytest.mark.parametrize("N", [40, 5300])
@pytest.mark.parametrize("M", [1, 2])
@pytest.mark.parametrize("fmt", FORMATS)
def test_every_code(gpu, fmt, M, N):
    """Numbers of the format, each block with one of its largest binade, which fixes the block's scale: x quantizes to
    itself, every element of it next to every other."""
    K = 2100
    W, w = weight(N, K)
    c, s = random_codes(fmt, M, K, N, 115, 120)
    c[:, ::32] = 6 + c[:, ::32] % 2 if fmt == E2M1 else 0x78 + c[:, ::32] % 7
    x = mx.values(fmt, c.astype(np.int64), s)
    got, scales = mx.quantize(fmt, x.astype(np.float32))
    assert np.array_equal(scales, s) and np.array_equal(mx.numbers(fmt, got), mx.numbers(fmt, c.astype(np.int64)))
    for t in (F32, BF16):
        check_kept(linear(Rows(F32, M, K, x.astype(np.float32)), fmt, W, t), t, x, w)


@pytest.mark.parametrize("N", [40, 5300])
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("fmt", FORMATS)
def test_special_blocks(gpu, fmt, t, N):
    """A token that holds a NaN or an infinity is NaN and the other is not; zero blocks, a zero token and tiny ones are
    numbers; a NaN scale of W makes its column NaN."""
    K = 2100
    wc, ws = random_codes(E2M1, N, K, 3, 115, 120)
    ws[N // 2, -1] = 255
    W, w = MxRows(E2M1, N, K, wc, ws), mx.values(E2M1, wc, ws)
    rng = np.random.default_rng(4)
    plain = rng.standard_normal(K).astype(np.float32)
    holes = plain.copy()
    holes[32:64], holes[K - 40:] = 0, 0
    tiny = plain.copy()
    tiny[64:96] *= np.float32(2.0 ** -20)
    bad = [plain.copy() for _ in range(3)]
    bad[0][70], bad[1][K - 1], bad[2][0] = np.nan, np.inf, -np.inf
    for rows in ([holes], [np.zeros(K)], [bad[0]], [bad[1]], [bad[0], holes], [tiny, bad[1]], [bad[2], np.zeros(K)]):
        x = np.array(rows, np.float32)
        X = Rows(t, len(rows), K, x)
        c, s = mx.quantize(fmt, X.values())
        with np.errstate(invalid="ignore"):
            xv = mx.values(fmt, c, s)
            for yt in (F32, BF16):
                got = linear(X, fmt, W, yt)
                check_kept(got, yt, xv, w)
                assert np.isnan(got[:, N // 2]).all()
                for r, row in enumerate(rows):
                    assert np.isnan(got[r]).all() == (not np.isfinite(row).all())
