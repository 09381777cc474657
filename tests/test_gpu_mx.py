"""Microscaled rows and products against the formats' definition in 64 bits.

Codes and scales are exact by definition: a power of two and one rounding.  Every product of two elements is
exact, and so is the sum of a block's (their lowest bits and largest sums fit 24 bits after E4M3 x
is split, which fp32 outputs do).  A result is then off by the additions in fp32, at most 8 of them for each
block of 32 (its four groups of 8, the split, the step and the parts of K), each by 2^-23 of what the sum's
magnitudes add up to, and by the bias and the output's rounding.  16-bit outputs take E4M3 without the split:
a product then loses what lies 13 bits below the largest of its eight, 2^-13 of it at most.
"""
import numpy as np
import pytest

import mx
import tier_amd
from mx import E2M1, E4M3, FORMATS, MxRows
from rows import TINY, TYPES, UNIT, Rows, f32
from tier_amd import hip

pytestmark = pytest.mark.gpu
F32, F16, BF16 = tier_amd.F32, tier_amd.F16, tier_amd.BF16


def _x(M, K, seed):
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((M, K)).astype(np.float32)
    x[:, 5::53] *= 9
    return x


def weight(N, K, seed, pad=0):
    """An E2M1 weight on the device and its values."""
    rng = np.random.default_rng(seed)
    c, s = mx.quantize(E2M1, (rng.standard_normal((N, K)) * 0.02).astype(np.float32))
    return MxRows(E2M1, N, K, c, s, pad), mx.values(E2M1, c, s)


def check(got, t, fmt, x, w, bias=None):
    """got against x w^T + bias within the bound of the header comment."""
    want, mag = x @ w.T, np.abs(x) @ np.abs(w).T
    b = np.zeros(w.shape[0]) if bias is None else bias.astype(np.float64)
    blocks = -(-x.shape[1] // 32)
    err = 8 * blocks * 2.0 ** -23 * mag + 2.0 ** -24 * (mag + np.abs(b))
    if fmt == E4M3 and t != F32:  # of eight products the largest counts for seven others
        xb = np.zeros((x.shape[0], blocks * 4, 8))
        xb.reshape(x.shape[0], -1)[:, :x.shape[1]] = np.abs(x)
        wb = np.zeros((w.shape[0], blocks * 4, 8))
        wb.reshape(w.shape[0], -1)[:, :w.shape[1]] = np.abs(w)
        err = err + 7 * 2.0 ** -13 * (xb.max(-1) @ wb.max(-1).T)
    want = want + b
    dead = np.isnan(want)
    assert np.isnan(got[dead]).all() and np.isfinite(got[~dead]).all()
    ok = np.abs(got - want) <= err + UNIT[t] * (np.abs(want) + err) + TINY[t]
    assert ok[~dead].all(), (np.argwhere(~ok & ~dead)[:5], np.nanmax(np.abs(got - want) / np.maximum(mag, 1e-300)))


# ------------------------------------------------------------------- quantizer
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("M,K,pad,skip", [(1, 1, 0, 0), (3, 31, 0, 1), (2, 32, 1, 0), (5, 1408, 0, 0), (2, 5121, 2, 3),
                                          (1, 257, 0, 0), (3, 512, 1, 8), (70, 300, 1, 1), (2, 20000, 0, 0),
                                          (600, 1, 0, 0), (600, 1408, 1, 1), (513, 5121, 0, 0), (515, 17000, 1, 3)])
def test_quant(gpu, fmt, t, M, K, pad, skip):
    X = Rows(t, M, K, _x(M, K, K + M), pad, skip)
    Q = MxRows(fmt, M, K, pad=pad)
    tier_amd.mx_quant(X.ptr, t, X.ld, fmt, Q.q.ptr, Q.rb, Q.s.ptr, Q.sb, M, K)
    hip.synchronize()
    c, s = Q.get()
    want, scales = mx.quantize(fmt, X.values())
    assert np.array_equal(s, scales) and np.array_equal(c, want)


@pytest.mark.parametrize("fmt", FORMATS)
def test_quant_special_blocks(gpu, fmt):
    """Every number of the format and the ties between them, saturation, zeros, tiny and subnormal blocks, the
    largest numbers, NaN and infinities: one block each."""
    lv, rows = mx.LEVELS[fmt], []
    v = np.concatenate([lv, (lv[1:] + lv[:-1]) / 2, np.nextafter(lv[1:], 0), np.nextafter(lv[:-1], 1e9)])
    v = np.concatenate([v, -v])
    for i in range(0, len(v), 31):  # 31 and one that fixes the scale at 1
        b = np.zeros(32)
        b[1:1 + len(v[i:i + 31])] = v[i:i + 31]
        b[0] = 2.0 ** mx.EMAX[fmt]
        rows.append(b)
    for first in (lv[-1] * 1.01, 2.0 ** (mx.EMAX[fmt] + 1) * 0.999, 1e-45, 2.0 ** -126, 2.0 ** -127, 2.0 ** -120, 3.4e38,
                  np.nan, np.inf, -np.inf, -0.0, 0.0):
        b = np.zeros(32)
        b[3:6] = [first, first / 3, -first / 1000]
        rows.append(b)
    x = np.array(rows, np.float32).reshape(1, -1)
    K = x.shape[1]
    X, Q = Rows(F32, 1, K, x), MxRows(fmt, 1, K)
    tier_amd.mx_quant(X.ptr, F32, K, fmt, Q.q.ptr, Q.rb, Q.s.ptr, Q.sb, 1, K)
    hip.synchronize()
    c, s = Q.get()
    want, scales = mx.quantize(fmt, x)
    assert np.array_equal(s, scales)
    assert np.array_equal(c, want)


# ------------------------------------------------------------------ MXFP4 rows
@pytest.mark.parametrize("N,K,pad", [(1, 32, 0), (5, 96, 1), (3, 512, 0), (7, 2880, 2)])
def test_from_mxfp4(gpu, N, K, pad):
    rng = np.random.default_rng(N + K)
    rb = tier_amd.q_row_bytes(tier_amd.MXFP4, K)
    blocks = rng.integers(0, 256, (N, K // 32, 17), dtype=np.uint8)
    blocks[..., 0] = rng.integers(0, 255, (N, K // 32))  # (255 is NaN in the one and 2^128 in the other)
    host = np.full((N, rb + 3 * pad), 0x77, np.uint8)
    host[:, :rb] = blocks.reshape(N, rb)
    W, Q = hip.to_device(host), MxRows(E2M1, N, K, pad=pad)
    tier_amd.mx_from_mxfp4(W.ptr, rb + 3 * pad, Q.q.ptr, Q.rb, Q.s.ptr, Q.sb, N, K)
    hip.synchronize()
    c, s = Q.get()
    want = tier_amd.dequant_host(np.ascontiguousarray(host[:, :rb]), tier_amd.MXFP4, K)
    assert np.array_equal(mx.values(E2M1, c, s).astype(np.float32), want)
    assert np.array_equal(s, blocks[..., 0])


# -------------------------------------------------------------------- products
SHAPES = [(1, 1, 1), (1, 7, 31), (1, 1024, 5120), (2, 129, 1408), (3, 16, 512), (5, 333, 257), (8, 1024, 2048),
          (16, 64, 4096), (17, 130, 1000), (33, 257, 640), (37, 512, 5120), (64, 96, 768), (130, 200, 1024),
          (257, 321, 513), (300, 640, 1536), (1, 5300, 640), (2, 5300, 1030)]


@pytest.mark.parametrize("xfmt", FORMATS)
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_gemm(gpu, xfmt, M, N, K):
    """Every output type, with and without a bias, odd strides."""
    c, s = mx.quantize(xfmt, _x(M, K, M + K))
    X, x = MxRows(xfmt, M, K, c, s, pad=M % 3), mx.values(xfmt, c, s)
    W, w = weight(N, K, N + K, pad=N % 2)
    rng = np.random.default_rng(9)
    for t, with_bias in ((F32, True), (F16, False), (BF16, True), (F32, False)):
        bias = rng.standard_normal(N).astype(np.float32) if with_bias else None
        Y = Rows(t, M, N, pad=3 if with_bias else 0, skip=1 if with_bias else 0)
        tier_amd.mx_gemm(X.q.ptr, xfmt, X.rb, X.s.ptr, X.sb, W.q.ptr, W.rb, W.s.ptr, W.sb,
                         f32(bias).ptr if with_bias else None, Y.ptr, t, Y.ld, M, N, K)
        hip.synchronize()
        check(Y.values(), t, xfmt, x, w, bias)
        assert Y.outside_kept()


@pytest.mark.parametrize("xfmt", FORMATS)
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("M,N,K", [(1, 1024, 5120), (1, 33, 100), (2, 5300, 1030), (3, 65, 2000), (40, 300, 1408)])
def test_linear_is_quant_and_gemm(gpu, xfmt, t, M, N, K):
    X = Rows(t, M, K, _x(M, K, M), 1, 1)
    W, w = weight(N, K, N)
    Y, ws = Rows(F32, M, N), tier_amd.mx_linear_ws_bytes(xfmt, M, N, K)
    tier_amd.mx_linear(X.ptr, t, X.ld, xfmt, W.q.ptr, W.rb, W.s.ptr, W.sb, None, Y.ptr, F32, N, M, N, K)
    hip.synchronize()
    c, s = mx.quantize(xfmt, X.values())
    check(Y.values(), F32, xfmt, mx.values(xfmt, c, s), w)
    S, Y2 = hip.DeviceBuffer(ws + 16), Rows(F32, M, N)
    S.fill_bytes(0x55)
    tier_amd.mx_linear(X.ptr, t, X.ld, xfmt, W.q.ptr, W.rb, W.s.ptr, W.sb, None, Y2.ptr, F32, N, M, N, K, S.ptr, ws)
    hip.synchronize()
    assert np.array_equal(Y.bits(), Y2.bits()) and (S.download(np.uint8)[ws:] == 0x55).all()


@pytest.mark.parametrize("xfmt", FORMATS)
@pytest.mark.parametrize("M,N,K", [(1, 40, 2048), (2, 40, 1024), (20, 70, 1024), (150, 140, 768)])
def test_gemm_every_code(gpu, xfmt, M, N, K):
    """Random codes and scales: every element of either format next to every other."""
    rng = np.random.default_rng(M)
    c = rng.integers(0, 1 << xfmt, (M, K))
    if xfmt == E4M3:
        c = np.where(c & 127 == 127, 3, c)
    s = rng.integers(110, 140, (M, K // 32))
    wc, wsc = rng.integers(0, 16, (N, K)), rng.integers(110, 140, (N, K // 32))
    X, W = MxRows(xfmt, M, K, c, s), MxRows(E2M1, N, K, wc, wsc)
    for t in (F32, BF16):
        Y = Rows(t, M, N)
        tier_amd.mx_gemm(X.q.ptr, xfmt, X.rb, X.s.ptr, X.sb, W.q.ptr, W.rb, W.s.ptr, W.sb, None, Y.ptr, t, N, M, N, K)
        hip.synchronize()
        check(Y.values(), t, xfmt, mx.values(xfmt, c, s), mx.values(E2M1, wc, wsc))


@pytest.mark.parametrize("M", [1, 2, 30, 140])
def test_gemm_keeps_every_bit_of_a_block(gpu, M):
    """One block of E4M3 x, fp32 out, sums that fit 24 bits: exact, whatever lies next to what."""
    rng = np.random.default_rng(M)
    K, N = 32, 150
    c = np.zeros((M, K), np.int64)
    for r in range(M):  # the largest, cancelled, next to the smallest there are beside a step of 2^-9
        p = rng.permutation(K)
        c[r, p[:2]] = 0x7e, 0xfe
        c[r, p[2:8]] = rng.integers(1, 0x30, 6)
        c[r, p[8:14]] = rng.integers(0x30, 0x7e, 6) & 0xf8
    wc = np.zeros((N, K), np.int64)
    wc[:] = rng.integers(1, 8, (N, 1))
    X, W = MxRows(E4M3, M, K, c, np.full((M, 1), 127)), MxRows(E2M1, N, K, wc, np.full((N, 1), 127))
    Y = Rows(F32, M, N)
    tier_amd.mx_gemm(X.q.ptr, E4M3, X.rb, X.s.ptr, X.sb, W.q.ptr, W.rb, W.s.ptr, W.sb, None, Y.ptr, F32, N, M, N, K)
    hip.synchronize()
    x, w = mx.numbers(E4M3, c), mx.numbers(E2M1, wc)
    want, mag = x @ w.T, np.abs(x) @ w.T
    # two parts and four groups of eight each: their fp32 additions alone
    assert (np.abs(Y.values() - want) <= 8 * 2.0 ** -23 * mag).all()
    small = mag < 2.0 ** 13  # whole sums of 2^-10 under 24 bits
    assert np.array_equal(Y.values()[small], want[small])


@pytest.mark.parametrize("xfmt", FORMATS)
@pytest.mark.parametrize("M,N,K", [(1, 70, 700), (2, 70, 700), (9, 70, 700), (70, 300, 1300)])
def test_nan_scales_and_far_scales(gpu, xfmt, M, N, K):
    """A NaN block makes its row (its column) NaN and no other; scales far apart meet without harm."""
    rng = np.random.default_rng(3)
    c, s = mx.quantize(xfmt, _x(M, K, 5))
    wc, ws = mx.quantize(E2M1, rng.standard_normal((N, K)).astype(np.float32))
    s[0, 2], ws[N // 2, -1] = 255, 255
    c[0, 64:96] = 0
    s[-1, 1] += 60 if M > 1 else 0
    ws[N - 1, 1] -= 60
    X, W = MxRows(xfmt, M, K, c, s), MxRows(E2M1, N, K, wc, ws)
    Y = Rows(F32, M, N)
    tier_amd.mx_gemm(X.q.ptr, xfmt, X.rb, X.s.ptr, X.sb, W.q.ptr, W.rb, W.s.ptr, W.sb, None, Y.ptr, F32, N, M, N, K)
    hip.synchronize()
    x, w = mx.values(xfmt, c, s), mx.values(E2M1, wc, ws)
    with np.errstate(invalid="ignore"):
        check(Y.values(), F32, xfmt, x, w)
    assert np.isnan(Y.values()[0]).all() and np.isnan(Y.values()[:, N // 2]).all()


def test_mxfp4_base_through_the_product(gpu):
    """Rows of a base's MXFP4 blocks, laid out once, give what the dequantized rows give."""
    N, K, M = 96, 2880, 4
    rng = np.random.default_rng(1)
    blocks = rng.integers(0, 256, (N, K // 32, 17), dtype=np.uint8)
    blocks[..., 0] = rng.integers(118, 126, (N, K // 32))
    W = MxRows(E2M1, N, K)
    raw = hip.to_device(blocks)
    tier_amd.mx_from_mxfp4(raw.ptr, K // 32 * 17, W.q.ptr, W.rb, W.s.ptr, W.sb, N, K)
    x = _x(M, K, 2)
    X, Y = Rows(F32, M, K, x), Rows(F32, M, N)
    tier_amd.mx_linear(X.ptr, F32, K, E4M3, W.q.ptr, W.rb, W.s.ptr, W.sb, None, Y.ptr, F32, N, M, N, K)
    hip.synchronize()
    c, s = mx.quantize(E4M3, x)
    w = tier_amd.dequant_host(blocks.reshape(N, -1), tier_amd.MXFP4, K).astype(np.float64)
    check(Y.values(), F32, E4M3, mx.values(E4M3, c, s), w)


def test_captured_on_a_stream(gpu):
    """The linear in a graph: replays see new x in place and match the eager call each time."""
    M, N, K, st = 3, 200, 1024, hip.Stream()
    W, w = weight(N, K, 4)
    xs = [Rows(F32, M, K, _x(M, K, i)) for i in range(3)]
    X, Y, Ye = Rows(F32, M, K), Rows(F32, M, N), Rows(F32, M, N)
    n = tier_amd.mx_linear_ws_bytes(E4M3, M, N, K)
    ws, ws2 = hip.DeviceBuffer(n), hip.DeviceBuffer(n)

    def call(y, w_s, stream):
        tier_amd.mx_linear(X.ptr, F32, K, E4M3, W.q.ptr, W.rb, W.s.ptr, W.sb, None, y.ptr, F32, N, M, N, K, w_s.ptr, n,
                           stream)

    call(Ye, ws2, st)
    st.synchronize()
    g = hip.Graph(st, lambda s: call(Y, ws, s))
    try:
        for x in xs:
            hip.copy_d2d(X.ptr, x.ptr, M * K * 4)
            hip.synchronize()
            g.launch(st)
            st.synchronize()
            call(Ye, ws2, st)
            st.synchronize()
            assert np.array_equal(Y.bits(), Ye.bits())
            c, s = mx.quantize(E4M3, x.values())
            check(Y.values(), F32, E4M3, mx.values(E4M3, c, s), w)
    finally:
        g.destroy()
        st.destroy()
